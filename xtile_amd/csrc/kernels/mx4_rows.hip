// Rows in microscaled 4-bit floating point, and their values:
//   e = max(floor(log2 max |x|) - 2, -127) of a block of 32;  q = round(x / 2^e)
//   y = q 2^e
// q is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, halfway to the even code,
// magnitudes above 6 held at 6; the byte e + 127 is a block's scale, 255 where it has
// an infinity or NaN (its q are 0, its y NaN).  The largest magnitude's exponent is
// that of its bits as an integer, which is also how infinities and NaN are found.
//
// HBM bounds it.  A thread has eight neighbours of a row, a quad of lanes a block, whose
// largest magnitude meets by two DPP steps; the conversions are the hardware's, two values
// at a time with the scale applied.
//
// Results are stored past the caches, which otherwise drop for them what is still to be read.
// In a graph over 3 sets of buffers, whose inputs the Infinity Cache then keeps, and over 24,
// whose inputs come from HBM: 8192 rows of 4096 in bf16 with their values 24.3 us (6.2 TB/s) and
// 28.0 (5.4), stored through the caches 31.6 and 31.3; 11008 such rows back to fp16 18 to 19 us
// and 23.0 (4.9 TB/s), through them 25 and 24.3.  Where no values are stored the rows are read
// past them too: the 8192 rows 17.7 us and 19.0 (4.5 TB/s), read through them 17.3 and 19.8; with
// values that costs 3 us of the 24.3 and saves 0.7 of the 28.0.
#include "common.h"
#include "launch.h"

namespace xtk {
namespace {

enum { kF32 = 0, kF16 = 1, kBF16 = 2 };

typedef float float2v __attribute__((ext_vector_type(2)));

struct Mx4RowsArgs {
  const void* x;
  unsigned char* q;  // null: not wanted
  unsigned char* s;
  void* y;
  TileOff tx, tq, ts, ty;
  long long ldx, ldq, lds, ldy;  // elements
  BlockDecode blocks;
  Div31 per_row, per_block;  // units of eight values of a row, rows of a Block
  int units_row, rows;
  unsigned units;  // of the grid, below 2^31
};

// Where a unit lies.
struct UnitAt {
  int x, y, z;
  long long row;
  int c;
  __device__ __forceinline__ long long in(const TileOff& t, long long ld, int per) const {
    return t.at(x, y, z) + row * ld + (long long)c * per;
  }
};

__device__ __forceinline__ UnitAt unit_at(const Mx4RowsArgs& p, unsigned u) {
  UnitAt a;
  const unsigned row = p.per_row(u);
  a.c = (int)(u - row * (unsigned)p.units_row);
  const int b = (int)p.per_block(row);
  a.row = (long long)(row - (unsigned)b * (unsigned)p.rows);
  p.blocks(b, a.x, a.y, a.z);
  return a;
}

// Eight neighbours at element alignment, as they are stored.
template <int ELEM>
struct Eight {
  typedef unsigned u4a __attribute__((ext_vector_type(4), aligned(2)));
  uint4v w[ELEM == kF32 ? 2 : 1];
  template <bool PAST>
  __device__ __forceinline__ void load(const void* base, long long at) {
    const unsigned char* const from = static_cast<const unsigned char*>(base) + at * (ELEM == kF32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < (ELEM == kF32 ? 2 : 1); ++i) {
      const u4a* const v = reinterpret_cast<const u4a*>(from + 16 * i);
      if constexpr (PAST) w[i] = (uint4v)__builtin_nontemporal_load(v);
      else w[i] = (uint4v)(*v);
    }
  }
  __device__ __forceinline__ void store(void* base, long long at) const {
    unsigned char* const to = static_cast<unsigned char*>(base) + at * (ELEM == kF32 ? 4 : 2);
#pragma unroll
    for (int i = 0; i < (ELEM == kF32 ? 2 : 1); ++i) __builtin_nontemporal_store((u4a)w[i], reinterpret_cast<u4a*>(to + 16 * i));
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (ELEM == kF32) {
        const unsigned u = w[i / 4][i % 4];  // a bit cast of the element itself would read element 0
        v[i] = __builtin_bit_cast(float, u);
      } else {
        const unsigned short h = (unsigned short)(w[0][i / 2] >> (16 * (i % 2)));
        v[i] = ELEM == kF16 ? (float)__builtin_bit_cast(_Float16, h) : __builtin_bit_cast(float, (unsigned)h << 16);
      }
    }
  }
  // Rounded to nearest even, where the type does not hold them.
  __device__ __forceinline__ void set(const float (&v)[8]) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < (ELEM == kF32 ? 8 : 4); ++i) {
      if constexpr (ELEM == kF32) w[i / 4][i % 4] = __builtin_bit_cast(unsigned, v[i]);
      else if constexpr (ELEM == kF16) w[0][i] = __builtin_bit_cast(unsigned, h2{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
      else w[0][i] = __builtin_bit_cast(unsigned, b2{(__bf16)v[2 * i], (__bf16)v[2 * i + 1]});
    }
  }
};

// The values of eight codes times 2^(byte - 127): an exact product of a normal number and
// a power that may be below them; NaN for a byte of 255.
__device__ __forceinline__ void values_of(unsigned codes, unsigned byte, float (&v)[8]) {
  const float2v a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1),
                c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3);
  const float m = __builtin_bit_cast(float, byte == 255 ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
  v[0] = a[0] * m;
  v[1] = a[1] * m;
  v[2] = b[0] * m;
  v[3] = b[1] * m;
  v[4] = c[0] * m;
  v[5] = c[1] * m;
  v[6] = d[0] * m;
  v[7] = d[1] * m;
}

// U units a thread, 256 apart, all loaded before the first is looked at.
template <int ELEM, int U, bool VALUES>
__global__ __launch_bounds__(256) void quantize_mx4_kernel(Mx4RowsArgs p) {
  typedef unsigned u1a __attribute__((aligned(1)));
  const unsigned u0 = blockIdx.x * (256u * U) + threadIdx.x;
  Eight<ELEM> e[U];
  UnitAt at[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    // a quad of lanes has a whole block: none is past the end but with its block
    at[i] = unit_at(p, min(u0 + 256u * i, p.units - 1));
    e[i].template load<!VALUES>(p.x, at[i].in(p.tx, p.ldx, 8));
  }
  issue_fence();
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float v[8];
    e[i].values(v);
    unsigned most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = max(most, __builtin_bit_cast(unsigned, v[k]) & 0x7fffffffu);
    most = max(most, (unsigned)__builtin_amdgcn_update_dpp(0, (int)most, 0xb1, 0xf, 0xf, false));  // its neighbour's
    most = max(most, (unsigned)__builtin_amdgcn_update_dpp(0, (int)most, 0x4e, 0xf, 0xf, false));  // the other two's
    const unsigned field = most >> 23;
    const bool odd = field == 255;
    const unsigned byte = odd ? 255u : field > 2 ? field - 2 : 0u;
    // x 2^(127 - byte), whose exponent's field is 254 - byte: a normal number
    const float up = __builtin_bit_cast(float, (254u - (odd ? 127u : byte)) << 23);
    unsigned codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0] * up, v[1] * up, 1.0f, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2] * up, v[3] * up, 1.0f, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4] * up, v[5] * up, 1.0f, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6] * up, v[7] * up, 1.0f, 3);
    if (odd) codes = 0;
    if (u0 + 256u * i >= p.units) continue;
    if (p.q) __builtin_nontemporal_store(codes, reinterpret_cast<u1a*>(p.q + at[i].in(p.tq, p.ldq, 4)));
    if (p.s && (threadIdx.x & 3) == 0) p.s[at[i].in(p.ts, p.lds, 0) + (at[i].c >> 2)] = (unsigned char)byte;
    if constexpr (VALUES) {
      values_of(codes, byte, v);
      Eight<ELEM> y;
      y.set(v);
      y.store(p.y, at[i].in(p.ty, p.ldy, 8));
    }
  }
}

template <int ELEM, int U>
__global__ __launch_bounds__(256) void dequantize_mx4_kernel(Mx4RowsArgs p) {
  typedef unsigned u1a __attribute__((aligned(1)));
  const unsigned u0 = blockIdx.x * (256u * U) + threadIdx.x;
  unsigned codes[U], byte[U];
  UnitAt at[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    at[i] = unit_at(p, min(u0 + 256u * i, p.units - 1));
    codes[i] = *reinterpret_cast<const u1a*>(p.q + at[i].in(p.tq, p.ldq, 4));
    byte[i] = p.s[at[i].in(p.ts, p.lds, 0) + (at[i].c >> 2)];
  }
  issue_fence();
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (u0 + 256u * i >= p.units) continue;
    float v[8];
    values_of(codes[i], byte[i], v);
    Eight<ELEM> y;
    y.set(v);
    y.store(p.y, at[i].in(p.ty, p.ldy, 8));
  }
}

template <int ELEM, int U>
void run_of(const Mx4RowsArgs& a, bool back, hipStream_t s) {
  const unsigned wgs = (a.units + 256 * U - 1) / (256 * U);
  if (back) dequantize_mx4_kernel<ELEM, U><<<wgs, 256, 0, s>>>(a);
  else if (a.y) quantize_mx4_kernel<ELEM, U, true><<<wgs, 256, 0, s>>>(a);
  else quantize_mx4_kernel<ELEM, U, false><<<wgs, 256, 0, s>>>(a);
}

// One unit a thread for few of them: 64 rows of 4096 with values in 2.5 us against 2.8 with two,
// 1024 in f32 8.5 against 8.9.  The large ones above over 3 sets of buffers: with one 26 us
// against 24.3, without values 20 against 17.7, back to fp16 21.3 against 18 to 19; with four 24.4, 18.3
// and 18.9.
template <int ELEM>
void run(const Mx4RowsArgs& a, bool back, hipStream_t s) {
  if (a.units <= 1u << 19) run_of<ELEM, 1>(a, back, s);
  else run_of<ELEM, 2>(a, back, s);
}

}  // namespace

hipError_t launch_mx4_rows(const xt::Plan& p, void* const* bufs, hipStream_t s, std::string& why) {
  const xt::Mx4RowsPlan& m = p.mx4_rows;
  // Every result apart from every other and from what is read; values may lie over x:
  // a thread has read what it stores there.
  const xt::Access2D* outs[3] = {m.back ? nullptr : &m.q, m.back ? nullptr : &m.s, &m.y};
  const xt::Access2D* ins[3] = {&m.x, m.back ? &m.q : nullptr, m.back ? &m.s : nullptr};
  for (const xt::Access2D* o : outs) {
    if (!o || o->arg < 0) continue;
    for (const xt::Access2D* in : ins)
      if (in && in->arg >= 0 && !result_apart(p, bufs, *o, *in, !m.back && o == &m.y, why)) return hipErrorInvalidValue;
    for (const xt::Access2D* other : outs)
      if (other && other != o && other->arg >= 0 && buffers_meet(p, bufs, o->arg, other->arg)) {
        why = "buffers " + std::to_string(o->arg) + " and " + std::to_string(other->arg) + " are both stored and meet";
        return hipErrorInvalidValue;
      }
  }
  auto off = [](const xt::Access2D& a) { return TileOff{a.addr.c0, a.addr.sx, a.addr.sy, a.addr.sz}; };
  auto at = [&](const xt::Access2D& a) { return a.arg < 0 ? nullptr : bufs[a.arg]; };
  Mx4RowsArgs a{};
  a.x = at(m.x);
  a.q = static_cast<unsigned char*>(at(m.q));
  a.s = static_cast<unsigned char*>(at(m.s));
  a.y = at(m.y);
  a.tx = off(m.x);
  a.tq = off(m.q);
  a.ts = off(m.s);
  a.ty = off(m.y);
  a.ldx = m.x.ld;
  a.ldq = m.q.ld;
  a.lds = m.s.ld;
  a.ldy = m.y.ld;
  a.blocks = block_decode(p.grid[0], p.grid[1], false);
  a.rows = static_cast<int>(m.back ? m.q.rows : m.x.rows);
  a.units_row = static_cast<int>(m.cols / 8);
  a.per_row = div31(a.units_row);
  a.per_block = div31(a.rows);
  const long long units = grid_blocks(p) * a.rows * a.units_row;  // below 2^31, as planned
  a.units = static_cast<unsigned>(units);
  switch (m.back ? m.y.elem : m.x.elem) {
    case xt::Elem::F32: run<kF32>(a, m.back, s); break;
    case xt::Elem::F16: run<kF16>(a, m.back, s); break;
    default: run<kBF16>(a, m.back, s); break;
  }
  return hipGetLastError();
}

}  // namespace xtk
