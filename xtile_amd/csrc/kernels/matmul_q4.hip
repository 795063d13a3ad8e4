// Products with 4-bit weights:
//   y[m, n] = rs[m] sum_g s[n, g] sum_{k in group g} x[m, k] w[n, k]
//
// The weights are read once, 16 bytes a lane straight into registers, and bound
// the kernel: x, of few rows, comes from L2.  A workgroup takes 16 NT rows of
// weights and 16 MT rows of x; its waves split K in chunks of 128 and meet once,
// in LDS, in a fixed order.
//
// A chunk: lane (n = lane % 16, q = lane / 16) loads the 32 weights of row n at
// k = 32 q.  A 4 x 4 transpose over the quarters of the wave (four swaps of lane
// halves and rows) turns that into one word for each step of 32 K values: in step
// t lane (n, q) has the eight weights at k = 32 t + 8 q, so a step lies within one
// group of 32 whatever the group's size.  x goes as the MFMA's rows, the weights
// as its columns, so a lane's results are all of one weight row and take one scale.
//
// Unpacking: the bytes hold weight + 8 (0..15).  Nibbles i and i + 4 of a word are
// neighbours along K; shifted to the top four bits of the mantissa of 16.0 (both
// types) they read as 16 + (weight + 8), exactly, two a shift and an and-or.  The
// 24 comes off after the product as 24 sum(x), one MFMA of x by a constant a step:
// the f32 sums are of values at most 31 x where the weights' own reach 8 x.  For
// int8 rows the nibbles are the MFMA's bytes as they are, less 8 sum(x), in
// integers; x's bytes are put in the nibbles' order by two v_perm a word pair.
#include "launch.h"

#include <type_traits>

#include "common.h"

namespace xtk {
namespace {

enum { kF32 = 0, kF16 = 1, kBF16 = 2, kI8 = 3 };

typedef int int4v __attribute__((ext_vector_type(4)));

struct Q4Args {
  const unsigned char* x;
  const unsigned char* w;
  const void* s;
  const float* rs;
  void* y;
  TileOff tx, tw, ts, trs, ty;
  long long ldx, ldw, lds, ldrs, ldy;  // elements (weights: bytes)
  BlockDecode blocks;
  Div31 d_tiles, d_nt;  // tiles of a Block, n tiles
  int tiles, ntiles;
  int M, N, K, chunks, group;
  Div31 d_group;  // units of 32 FL weights in a group
  int s_elem, y_elem;
};

typedef unsigned u4a __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned u2a __attribute__((ext_vector_type(2), aligned(1)));

// Register t of quarter q <-> register q of quarter t.
__device__ __forceinline__ void transpose_quarters(unsigned (&d)[4]) {
  auto swap32 = [](unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  auto swap16 = [](unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  swap32(d[0], d[2]);
  swap32(d[1], d[3]);
  swap16(d[0], d[1]);
  swap16(d[2], d[3]);
}

__device__ __forceinline__ float scale_at(const void* s, int elem, long long i) {
  if (elem == kF32) return static_cast<const float*>(s)[i];
  if (elem == kF16) return (float)static_cast<const _Float16*>(s)[i];
  return __builtin_bit_cast(float, (unsigned)static_cast<const unsigned short*>(s)[i] << 16);
}

// FL: steps of 32 between two additions to the result (1, 2 or 4): at most the group.
template <int ELEM, int MT, int NT, int W, int FL>
__global__ __launch_bounds__(64 * W) void matmul_q4_kernel(Q4Args p) {
  constexpr bool I8 = ELEM == kI8;
  constexpr int ES = I8 ? 1 : 2;
  typedef typename std::conditional<I8, int4v, float4v>::type acc_t;
  __shared__ float part[W][NT * MT][4][64];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, q = lane >> 4;
  const int b = (int)p.d_tiles(blockIdx.x);
  const int tile = blockIdx.x - b * p.tiles;
  const int tm = (int)p.d_nt(tile), tn = tile - tm * p.ntiles;
  int bx, by, bz;
  p.blocks(b, bx, by, bz);
  const int m0 = tm * 16 * MT, n0 = tn * 16 * NT;

  const unsigned char* w[NT];
  long long sc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {  // rows past the end read the last one; their results are not stored
    const int n = min(n0 + 16 * j + col, p.N - 1);
    w[j] = p.w + p.tw.at(bx, by, bz) + n * p.ldw;
    sc[j] = p.ts.at(bx, by, bz) + n * p.lds;
  }
  const unsigned char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = p.x + (p.tx.at(bx, by, bz) + min(m0 + 16 * i + col, p.M - 1) * p.ldx + q * 8) * ES;

  float4v y[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) y[i][j] = float4v{0, 0, 0, 0};

  struct Chunk {
    unsigned w[NT][4];
    uint4v x[MT][4];
    float s[NT][4 / FL];
  };
  // steps: of 32 K values in this chunk (fewer than four in a last one)
  auto fetch = [&](int c, int steps, Chunk& k) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const u4a v = *reinterpret_cast<const u4a*>(w[j] + (long long)c * 64 + (q < steps ? q : 0) * 16);
#pragma unroll
      for (int t = 0; t < 4; ++t) k.w[j][t] = v[t];
#pragma unroll
      for (int f = 0; f < 4 / FL; ++f) {
        const int g = (int)p.d_group((unsigned)(c * (4 / FL) + (f * FL < steps ? f : 0)));
        k.s[j][f] = scale_at(p.s, p.s_elem, sc[j] + g);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const unsigned char* at = x[i] + ((long long)c * 128 + (t < steps ? t : 0) * 32) * ES;
        if constexpr (I8) {
          const u2a v = *reinterpret_cast<const u2a*>(at);
          k.x[i][t] = uint4v{v[0], v[1], 0, 0};
        } else {
          k.x[i][t] = (uint4v)(*reinterpret_cast<const u4a*>(at));
        }
      }
  };
  auto compute = [&](int steps, Chunk& k) {
#pragma unroll
    for (int j = 0; j < NT; ++j) transpose_quarters(k.w[j]);
#pragma unroll
    for (int f = 0; f < 4 / FL; ++f) {
      if (f * FL >= steps) break;
      acc_t acc[MT][NT], off[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        off[i] = acc_t{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = acc_t{0, 0, 0, 0};
      }
#pragma unroll
      for (int u = 0; u < FL; ++u) {
        const int t = f * FL + u;
        if (t >= steps) break;
        if constexpr (I8) {
          const long eights = 0x0808080808080808L;
          long xi[MT];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const unsigned lo = __builtin_amdgcn_perm(k.x[i][t][1], k.x[i][t][0], 0x05010400u);
            const unsigned hi = __builtin_amdgcn_perm(k.x[i][t][1], k.x[i][t][0], 0x07030602u);
            xi[i] = (long)(((unsigned long)hi << 32) | lo);
            off[i] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xi[i], eights, off[i], 0, 0, 0);
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const unsigned d = k.w[j][t];
            const long wj = (long)(((unsigned long)((d >> 4) & 0x0f0f0f0fu) << 32) | (d & 0x0f0f0f0fu));
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xi[i], wj, acc[i][j], 0, 0, 0);
          }
        } else {
          // 16 + u: f16 0x4c00 | u << 6, bf16 0x4180 | u << 3
          constexpr unsigned one = ELEM == kF16 ? 0x4c004c00u : 0x41804180u, mask = ELEM == kF16 ? 0x03c003c0u : 0x00780078u;
          constexpr unsigned c24 = ELEM == kF16 ? 0x4e004e00u : 0x41c041c0u;
          constexpr int up = ELEM == kF16 ? 6 : 3;
          auto mma = [](uint4v a, uint4v bb, float4v c) {
            if constexpr (ELEM == kF16)
              return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, bb), c, 0, 0, 0);
            else
              return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, bb), c, 0, 0, 0);
          };
#pragma unroll
          for (int i = 0; i < MT; ++i) off[i] = mma(k.x[i][t], uint4v{c24, c24, c24, c24}, off[i]);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const unsigned d = k.w[j][t];
            uint4v v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = ((up >= 4 * e ? d << (up - 4 * e) : d >> (4 * e - up)) & mask) | one;
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][j] = mma(k.x[i][t], v, acc[i][j]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[i][j][r] = fmaf((float)(acc[i][j][r] - off[i][r]), k.s[j][f], y[i][j][r]);
    }
  };

  auto steps_of = [&](int c) { return min(4, (p.K >> 5) - 4 * c); };
  Chunk k0, k1;
  int c = wave;
  if (c < p.chunks) {
    fetch(c, steps_of(c), k0);
    while (true) {
      const int c1 = c + W;
      if (c1 < p.chunks) fetch(c1, steps_of(c1), k1);
      compute(steps_of(c), k0);
      if (c1 >= p.chunks) break;
      const int c2 = c1 + W;
      if (c2 < p.chunks) fetch(c2, steps_of(c2), k0);
      compute(steps_of(c1), k1);
      if (c2 >= p.chunks) break;
      c = c2;
    }
  }

  // the waves' parts, summed in the order of the waves
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[wave][i * NT + j][r][lane] = y[i][j][r];
  __syncthreads();
  const long long y0 = p.ty.at(bx, by, bz), r0 = p.trs.at(bx, by, bz);
  for (int e = threadIdx.x; e < NT * MT * 256; e += 64 * W) {
    const int ij = e >> 8, r = (e >> 6) & 3, l = e & 63;
    float v = 0.0f;
#pragma unroll
    for (int u = 0; u < W; ++u) v += part[u][ij][r][l];
    const int m = m0 + 16 * (ij / NT) + 4 * (l >> 4) + r, n = n0 + 16 * (ij % NT) + (l & 15);
    if (m >= p.M || n >= p.N) continue;
    if (p.rs) v *= p.rs[r0 + m * p.ldrs];
    const long long at = y0 + m * p.ldy + n;
    if (p.y_elem == kF32) static_cast<float*>(p.y)[at] = v;
    else if (p.y_elem == kF16) static_cast<_Float16*>(p.y)[at] = (_Float16)v;
    else static_cast<__bf16*>(p.y)[at] = (__bf16)v;
  }
}

template <int ELEM, int MT, int NT, int W>
void run_fl(Q4Args& a, int wgs, hipStream_t s) {
  a.d_group = div31(a.group / (a.group % 128 == 0 ? 128 : a.group % 64 == 0 ? 64 : 32));
  if (a.group % 128 == 0) matmul_q4_kernel<ELEM, MT, NT, W, 4><<<wgs, 64 * W, 0, s>>>(a);
  else if (a.group % 64 == 0) matmul_q4_kernel<ELEM, MT, NT, W, 2><<<wgs, 64 * W, 0, s>>>(a);
  else matmul_q4_kernel<ELEM, MT, NT, W, 1><<<wgs, 64 * W, 0, s>>>(a);
}

template <int ELEM>
bool run(Q4Args& a, long long blocks, hipStream_t s) {
  const int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4, nt = 1, w = 8;
  a.ntiles = (a.N + 16 * nt - 1) / (16 * nt);
  const long long tiles = (long long)a.ntiles * ((a.M + 16 * mt - 1) / (16 * mt));
  if (tiles > 0x7fffffffLL || !grid_fits(tiles * blocks, 64 * w)) return false;
  a.tiles = (int)tiles;
  a.d_tiles = div31(a.tiles);
  a.d_nt = div31(a.ntiles);
  const int wgs = (int)(tiles * blocks);
  if (mt == 1) run_fl<ELEM, 1, 1, 8>(a, wgs, s);
  else if (mt == 2) run_fl<ELEM, 2, 1, 8>(a, wgs, s);
  else run_fl<ELEM, 4, 1, 8>(a, wgs, s);
  return true;
}

int elem_of(xt::Elem e) {
  return e == xt::Elem::F32 ? kF32 : e == xt::Elem::F16 ? kF16 : e == xt::Elem::BF16 ? kBF16 : kI8;
}

}  // namespace

hipError_t launch_matmul_q4(const xt::Plan& p, void* const* bufs, hipStream_t s, std::string& why) {
  const xt::Q4Plan& q = p.q4;
  for (const xt::Access2D* in : {&q.x, &q.w, &q.scales, q.row_scale ? &q.rows : &q.x})
    if (!result_apart(p, bufs, q.y, *in, false, why)) return hipErrorInvalidValue;
  auto off = [](const xt::Access2D& a) { return TileOff{a.addr.c0, a.addr.sx, a.addr.sy, a.addr.sz}; };
  Q4Args a{};
  a.x = static_cast<const unsigned char*>(bufs[q.x.arg]);
  a.w = static_cast<const unsigned char*>(bufs[q.w.arg]);
  a.s = bufs[q.scales.arg];
  a.rs = q.row_scale ? static_cast<const float*>(bufs[q.rows.arg]) : nullptr;
  a.y = bufs[q.y.arg];
  a.tx = off(q.x);
  a.tw = off(q.w);
  a.ts = off(q.scales);
  a.trs = off(q.rows);
  a.ty = off(q.y);
  a.ldx = q.x.ld;
  a.ldw = q.w.ld;
  a.lds = q.scales.ld;
  a.ldrs = q.rows.ld;
  a.ldy = q.y.ld;
  a.blocks = block_decode(p.grid[0], p.grid[1], false);
  a.M = static_cast<int>(q.y.rows);
  a.N = static_cast<int>(q.y.cols);
  a.K = static_cast<int>(q.K);
  a.chunks = (a.K + 127) / 128;
  a.group = static_cast<int>(q.group);
  a.s_elem = elem_of(q.scales.elem);
  a.y_elem = elem_of(q.y.elem);
  bool ok;
  if (q.x.elem == xt::Elem::I8) ok = run<kI8>(a, grid_blocks(p), s);
  else if (q.x.elem == xt::Elem::F16) ok = run<kF16>(a, grid_blocks(p), s);
  else ok = run<kBF16>(a, grid_blocks(p), s);
  if (!ok) {
    why = "matmul_q4: " + std::to_string(a.M) + " x " + std::to_string(a.N) + " tiles exceed one launch";
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace xtk
