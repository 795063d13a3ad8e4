// Root-mean-square norm of rows, with the residual's addition and, where asked
// for, rows in 8 bits:
//   h = x + r;  y = h / sqrt(mean(h^2) + eps) * gamma
//   s = max |y| / 127;  q = rint(y / s)
//
// One pass: a group of threads holds its row in registers as f32 (h is rounded
// only where it is stored), so x, r and gamma are read once and nothing is read
// back.  The sum of squares and the largest |h gamma| are found together, since
// max |y| = max |h gamma| / sqrt(...): one exchange over the group serves both.
//
// HBM bounds it for many rows (8192 of 4096 bf16 values with a residual to int8: 235 MB
// in 41.2 us by the tracer, 5.7 TB/s; 46.3 to 47.5 a launch of a graph), one group's latency
// for one row (2.6 us by the tracer).  A row takes
// 64 threads (rows to 1024 values, no barrier), 256 (to 8192) or 1024; longer
// rows, and those of fewer than eight values, are read again for the second half
// (rms_norm_long_kernel).
#include <vector>

#include "common.h"
#include "launch.h"

namespace xtk {
namespace {

enum { kF32 = 0, kF16 = 1, kBF16 = 2, kI8 = 3 };

struct NormArgs {
  const void* x;
  const void* r;
  const void* gamma;
  void* sum;
  void* y;
  float* scale;
  TileOff tx, tr, tg, tsum, ty, tscale;
  long long ldx, ldr, ldsum, ldy, ldscale;
  BlockDecode blocks;
  Div31 per;  // rows of a Block
  int block_rows, rows, cols;
  int gamma_elem, y_elem;
  float eps;
};

// Eight values at element alignment; the first n of them where fewer are left.
template <int ELEM>
__device__ __forceinline__ void load8(const void* base, long long at, int n, float (&v)[8]) {
  if constexpr (ELEM == kF32) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    const float* q = static_cast<const float*>(base) + at;
    if (n >= 8) {
      const f4 a = *reinterpret_cast<const f4*>(q), b = *reinterpret_cast<const f4*>(q + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? q[i] : 0.0f;
    }
  } else if constexpr (ELEM == kF16) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8), aligned(2)));
    const _Float16* q = static_cast<const _Float16*>(base) + at;
    if (n >= 8) {
      const h8 a = *reinterpret_cast<const h8*>(q);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)q[i] : 0.0f;
    }
  } else {
    typedef unsigned short s8 __attribute__((ext_vector_type(8), aligned(2)));
    const unsigned short* q = static_cast<const unsigned short*>(base) + at;
    if (n >= 8) {
      const s8 a = *reinterpret_cast<const s8*>(q);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, (unsigned)a[i] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? __builtin_bit_cast(float, (unsigned)q[i] << 16) : 0.0f;
    }
  }
}

// Rounded once, to nearest even, to the stored type.
template <int ELEM>
__device__ __forceinline__ void store8(void* base, long long at, int n, const float (&v)[8]) {
  if constexpr (ELEM == kF32) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    float* q = static_cast<float*>(base) + at;
    if (n >= 8) {
      *reinterpret_cast<f4*>(q) = f4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f4*>(q + 4) = f4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = v[i];
    }
  } else if constexpr (ELEM == kF16) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8), aligned(2)));
    _Float16* q = static_cast<_Float16*>(base) + at;
    if (n >= 8) {
      h8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = (_Float16)v[i];
      *reinterpret_cast<h8*>(q) = a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (_Float16)v[i];
    }
  } else {
    typedef __bf16 b8 __attribute__((ext_vector_type(8), aligned(2)));
    __bf16* q = static_cast<__bf16*>(base) + at;
    if (n >= 8) {
      b8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = (__bf16)v[i];
      *reinterpret_cast<b8*>(q) = a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (__bf16)v[i];
    }
  }
}

__device__ __forceinline__ void load8_of(int elem, const void* base, long long at, int n, float (&v)[8]) {
  if (elem == kF32) load8<kF32>(base, at, n, v);
  else if (elem == kF16) load8<kF16>(base, at, n, v);
  else load8<kBF16>(base, at, n, v);
}

// y / s to int8, half to even.
__device__ __forceinline__ int to_i8(float y, float s) {
  const float v = s != 0.0f ? y / s : 0.0f;
  int i;  // saturates, NaN to 0; assembly because a C++ cast of such values is undefined
  asm("v_cvt_i32_f32 %0, %1" : "=v"(i) : "v"(__builtin_rintf(v)));
  return min(max(i, -127), 127);
}

// Four of them by inv = 1 / s: y inv, and what it leaves of y once more, is the quotient as
// division rounds it, so that halves fall where they should.  |y| is at most 127 s but for a
// few roundings, so none of them passes 127, and 1.5 2^23 more has the integer in its low byte.
__device__ __forceinline__ unsigned to_i8x4(const float* y, float s, float inv) {
  unsigned u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = y[i] * inv;
    u[i] = __builtin_bit_cast(unsigned, fmaf(fmaf(-q, s, y[i]), inv, q) + 12582912.0f);
  }
  return __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u) | __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
}

// What to_i8x4 takes of a row's scale: 0 for scales that are not finite, or too small for the
// remainders to be normal numbers, or from a product `top` of too few bits for its values to
// be at most 127 of them.  Such rows divide.
__device__ __forceinline__ float inverse_scale(float s, unsigned top) {
  return s >= 1.0e-30f && s < __builtin_inff() && __builtin_bit_cast(float, top) >= 1.0e-30f ? 1.0f / s : 0.0f;
}

__device__ __forceinline__ void store_y8(const NormArgs& p, long long at, int n, const float (&y)[8], float s, float inv) {
  if (p.y_elem == kF32) {
    store8<kF32>(p.y, at, n, y);
  } else if (p.y_elem == kF16) {
    store8<kF16>(p.y, at, n, y);
  } else if (p.y_elem == kBF16) {
    store8<kBF16>(p.y, at, n, y);
  } else {
    signed char* q = static_cast<signed char*>(p.y) + at;
    unsigned w[2] = {0, 0};
    if (__builtin_amdgcn_readfirstlane(inv != 0.0f)) {  // of the row, which every lane has
#pragma unroll
      for (int i = 0; i < 2; ++i) w[i] = to_i8x4(y + 4 * i, s, inv);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i >> 2] |= ((unsigned)to_i8(y[i], s) & 255u) << (8 * (i & 3));
    }
    if (n >= 8) {
      typedef unsigned u2 __attribute__((ext_vector_type(2), aligned(1)));
      *reinterpret_cast<u2*>(q) = u2{w[0], w[1]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[i] = (signed char)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
}

// The larger of two magnitudes as their bits: NaN is above infinity, so it stays.
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
  return v;
}

// The sum and the largest magnitude over the T threads of a row (every lane active).
template <int T>
__device__ __forceinline__ void row_reduce(float& ss, unsigned& top, bool want_top) {
  ss = wave_reduce<false>(ss);
  if (want_top) top = wave_umax(top);
  if constexpr (T > 64) {
    __shared__ float part[T / 64];
    __shared__ unsigned tops[T / 64];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      part[wave] = ss;
      tops[wave] = top;
    }
    __syncthreads();
    ss = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
      ss += part[w];
      top = max(top, tops[w]);
    }
  }
}

struct RowAt {
  long long x, r, g, sum, y, scale;
};

__device__ __forceinline__ RowAt row_at(const NormArgs& p, int row) {
  const int b = (int)p.per((unsigned)row);
  const int i = row - b * p.block_rows;
  int bx, by, bz;
  p.blocks(b, bx, by, bz);
  return RowAt{p.tx.at(bx, by, bz) + i * p.ldx,     p.tr.at(bx, by, bz) + i * p.ldr,
               p.tg.at(bx, by, bz),                 p.tsum.at(bx, by, bz) + i * p.ldsum,
               p.ty.at(bx, by, bz) + i * p.ldy,     p.tscale.at(bx, by, bz) + i * p.ldscale};
}

__device__ __forceinline__ float inverse_root(const NormArgs& p, float ss) {
  return 1.0f / sqrtf(ss / (float)p.cols + p.eps);
}

// Eight values as they lie in memory.
template <bool WIDE>
struct Raw8 {
  typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(2)));
  u4 v[WIDE ? 2 : 1];

  __device__ __forceinline__ void load(const void* base, long long at) {
    const unsigned char* const q = static_cast<const unsigned char*>(base) + at * (WIDE ? 4 : 2);
    v[0] = *reinterpret_cast<const u4*>(q);
    if constexpr (WIDE) v[1] = *reinterpret_cast<const u4*>(q + 16);
  }
  // 16 bits: f16 or bf16, told apart lane by lane where the compiler does not know
  __device__ __forceinline__ float value(int i, bool f16) const {
    if constexpr (WIDE) {
      const unsigned u = v[i >> 2][i & 3];
      return __builtin_bit_cast(float, u);
    } else {
      const unsigned u = v[0][i >> 1], half = i & 1 ? u >> 16 : u & 0xffffu;
      const float h = (float)__builtin_bit_cast(_Float16, (unsigned short)half), b = __builtin_bit_cast(float, half << 16);
      return f16 ? h : b;
    }
  }
};

// T threads a row, NV vectors of eight values each; GWIDE: gamma has 32 bits.  Every
// load is on its way before the first value is looked at: none is conditional, and none
// is converted where it is loaded (launches in a graph: one row of 4096 bf16 values 3.0 us,
// with the loads one behind the other 3.6; 8192 rows to int8 47.5 us, and 61).  A vector that
// would pass the row's end starts eight values before it: its first ones are also its
// neighbour's, count once and are stored twice.
template <int ELEM, int T, int NV, bool GWIDE>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rms_norm_kernel(NormArgs p) {
  constexpr int R = T < 256 ? 256 / T : 1;  // rows of a workgroup
  const int row = R == 1 ? (int)blockIdx.x : __builtin_amdgcn_readfirstlane(blockIdx.x * R + threadIdx.x / T);
  if (R > 1 && row >= p.rows) return;  // whole waves, and no barrier below for them
  const RowAt at = row_at(p, row);
  const int t = R == 1 ? threadIdx.x : threadIdx.x % T;
  const bool quantize = p.y_elem == kI8;
  constexpr bool WIDE = ELEM == kF32;
  Raw8<WIDE> x[NV], r[NV];
  Raw8<GWIDE> gr[NV];
  auto begin = [&](int i) { return min((i * T + t) * 8, p.cols - 8); };
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i].load(p.x, at.x + begin(i));
#pragma unroll
  for (int i = 0; i < NV; ++i) gr[i].load(p.gamma, at.g + begin(i));
  if (p.r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) r[i].load(p.r, at.r + begin(i));
  }
  int g16 = p.gamma_elem == kF16;
  asm volatile("" : "+v"(g16));
  float h[NV][8], g[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[i][e] = x[i].value(e, ELEM == kF16);
      g[i][e] = gr[i].value(e, g16 != 0);
    }
  if (p.r) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] += r[i].value(e, ELEM == kF16);
  }
  float ss = 0.0f;
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int twice = (i * T + t) * 8 - begin(i);  // values that a neighbour counts
    float s8 = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = e >= twice ? h[i][e] : 0.0f;
      s8 = fmaf(v, v, s8);
    }
    ss += s8;
  }
  if (quantize) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        top = max(top, __builtin_bit_cast(unsigned, h[i][e] * g[i][e]) & 0x7fffffffu);
  }
  row_reduce<T>(ss, top, quantize);
  const float inv = inverse_root(p, ss);
  float s = 0.0f, is = 0.0f;
  if (quantize) {
    s = __builtin_bit_cast(float, top) * inv / 127.0f;
    is = inverse_scale(s, top);
    if (t == 0) p.scale[at.scale] = s;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * T + t) * 8 >= p.cols) continue;
    const int c = begin(i);
    if (p.sum) store8<ELEM>(p.sum, at.sum + c, 8, h[i]);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = h[i][e] * inv * g[i][e];
    store_y8(p, at.y + c, 8, y, s, is);
  }
}

// Rows that the registers of a workgroup do not hold, and rows of fewer than eight
// values (T = 64, a row a workgroup): x and r are read twice,
// the second time from L2.  Nothing is stored before the second pass, and then by
// the thread that has just read those values again, since it may lie over x or r.
template <int ELEM, int T>
__global__ __launch_bounds__(T) void rms_norm_long_kernel(NormArgs p) {
  const RowAt at = row_at(p, blockIdx.x);
  const int t = threadIdx.x;
  const bool quantize = p.y_elem == kI8;
  float ss = 0.0f;
  unsigned top = 0;
  auto row8 = [&](int c, float (&h)[8], float (&g)[8]) {
    float r[8];
    load8<ELEM>(p.x, at.x + c, p.cols - c, h);
    if (p.r) {
      load8<ELEM>(p.r, at.r + c, p.cols - c, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] += r[e];
    }
    load8_of(p.gamma_elem, p.gamma, at.g + c, p.cols - c, g);
  };
  for (int c = t * 8; c < p.cols; c += T * 8) {
    float h[8], g[8], s8 = 0.0f;
    row8(c, h, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s8 = fmaf(h[e], h[e], s8);
      top = max(top, __builtin_bit_cast(unsigned, h[e] * g[e]) & 0x7fffffffu);
    }
    ss += s8;
  }
  row_reduce<T>(ss, top, quantize);
  const float inv = inverse_root(p, ss);
  float s = 0.0f, is = 0.0f;
  if (quantize) {
    s = __builtin_bit_cast(float, top) * inv / 127.0f;
    is = inverse_scale(s, top);
  }
  for (int c = t * 8; c < p.cols; c += T * 8) {
    float h[8], g[8], y[8];
    row8(c, h, g);
    if (p.sum) store8<ELEM>(p.sum, at.sum + c, p.cols - c, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = h[e] * inv * g[e];
    store_y8(p, at.y + c, p.cols - c, y, s, is);
  }
  // behind the second pass: the scales of rows of one value may lie over x or r
  if (quantize && t == 0) p.scale[at.scale] = s;
}

// What a launch takes: threads a row, workgroups and their threads, and whether the
// rows are read twice.
struct NormGrid {
  int row;
  long long wgs;
  int threads;
  bool twice;
  NormGrid(int cols, long long rows)
      : row(cols <= 1024 ? 64 : cols <= 8192 ? 256 : 1024), twice(cols < 8 || cols > 32768) {
    threads = twice ? row : row < 256 ? 256 : row;
    wgs = (rows + threads / row - 1) / (threads / row);
  }
};

template <int ELEM, int T, bool GWIDE>
void run(const NormArgs& a, const NormGrid& g, hipStream_t s) {
  const unsigned wgs = static_cast<unsigned>(g.wgs);
  const int nv = ((a.cols + 7) / 8 + T - 1) / T;  // vectors a thread
  if (nv <= 1) rms_norm_kernel<ELEM, T, 1, GWIDE><<<wgs, g.threads, 0, s>>>(a);
  else if (nv <= 2) rms_norm_kernel<ELEM, T, 2, GWIDE><<<wgs, g.threads, 0, s>>>(a);
  else rms_norm_kernel<ELEM, T, 4, GWIDE><<<wgs, g.threads, 0, s>>>(a);
}

template <int ELEM, bool GWIDE>
void run_elem(const NormArgs& a, const NormGrid& g, hipStream_t s) {
  const unsigned wgs = static_cast<unsigned>(g.wgs);
  if (g.twice && g.row == 64) rms_norm_long_kernel<ELEM, 64><<<wgs, 64, 0, s>>>(a);
  else if (g.twice) rms_norm_long_kernel<ELEM, 1024><<<wgs, 1024, 0, s>>>(a);
  else if (g.row == 64) run<ELEM, 64, GWIDE>(a, g, s);
  else if (g.row == 256) run<ELEM, 256, GWIDE>(a, g, s);
  else run<ELEM, 1024, GWIDE>(a, g, s);
}

int elem_of(xt::Elem e) {
  return e == xt::Elem::F32 ? kF32 : e == xt::Elem::F16 ? kF16 : e == xt::Elem::BF16 ? kBF16 : kI8;
}

}  // namespace

hipError_t launch_rms_norm(const xt::Plan& p, void* const* bufs, hipStream_t s, std::string& why) {
  const xt::NormPlan& n = p.norm;
  // a result may lie over x or r: every thread stores over what it has read, and
  // nothing that another reads
  std::vector<const xt::Access2D*> ins = {&n.x, &n.gamma}, outs = {&n.y};
  if (n.residual) ins.push_back(&n.r);
  if (n.keep_sum) outs.push_back(&n.sum);
  if (n.quantize) outs.push_back(&n.scale);
  for (size_t i = 0; i < outs.size(); ++i) {
    for (const xt::Access2D* in : ins)
      if (!result_apart(p, bufs, *outs[i], *in, in != &n.gamma, why)) return hipErrorInvalidValue;
    for (size_t j = 0; j < i; ++j)
      if (buffers_meet(p, bufs, outs[i]->arg, outs[j]->arg)) {
        why = "buffers " + std::to_string(outs[j]->arg) + " and " + std::to_string(outs[i]->arg) +
              " are both stored and meet";
        return hipErrorInvalidValue;
      }
  }
  auto off = [](const xt::Access2D& a) { return TileOff{a.addr.c0, a.addr.sx, a.addr.sy, a.addr.sz}; };
  NormArgs a{};
  a.x = bufs[n.x.arg];
  a.r = n.residual ? bufs[n.r.arg] : nullptr;
  a.gamma = bufs[n.gamma.arg];
  a.sum = n.keep_sum ? bufs[n.sum.arg] : nullptr;
  a.y = bufs[n.y.arg];
  a.scale = n.quantize ? static_cast<float*>(bufs[n.scale.arg]) : nullptr;
  a.tx = off(n.x);
  a.tr = off(n.r);
  a.tg = off(n.gamma);
  a.tsum = off(n.sum);
  a.ty = off(n.y);
  a.tscale = off(n.scale);
  a.ldx = n.x.ld;
  a.ldr = n.r.ld;
  a.ldsum = n.sum.ld;
  a.ldy = n.y.ld;
  a.ldscale = n.scale.ld;
  a.blocks = block_decode(p.grid[0], p.grid[1], false);
  a.per = div31(static_cast<unsigned>(n.x.rows));
  a.block_rows = static_cast<int>(n.x.rows);
  const long long rows = grid_blocks(p) * n.x.rows;
  a.rows = static_cast<int>(rows);
  a.cols = static_cast<int>(n.x.cols);
  a.gamma_elem = elem_of(n.gamma.elem);
  a.y_elem = elem_of(n.y.elem);
  a.eps = n.eps;
  const NormGrid g(a.cols, rows);
  if (!grid_fits(g.wgs, g.threads)) {
    why = "rms_norm: " + std::to_string(rows) + " rows exceed one launch";
    return hipErrorInvalidValue;
  }
  const bool wide = a.gamma_elem == kF32;
  if (n.x.elem == xt::Elem::F32) wide ? run_elem<kF32, true>(a, g, s) : run_elem<kF32, false>(a, g, s);
  else if (n.x.elem == xt::Elem::F16) wide ? run_elem<kF16, true>(a, g, s) : run_elem<kF16, false>(a, g, s);
  else wide ? run_elem<kBF16, true>(a, g, s) : run_elem<kBF16, false>(a, g, s);
  return hipGetLastError();
}

}  // namespace xtk
