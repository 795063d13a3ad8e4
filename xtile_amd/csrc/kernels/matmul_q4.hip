// Products with 4-bit weights:
//   y[m, n] = rs[m] sum_g s[n, g] sum_{k in group g} x[m, k] w[n, k]
//
// The weights are read once and bound the kernel: x, of few rows, comes from L2.  A
// workgroup takes 16 NT rows of weights and 16 MT rows of x; its waves split K in chunks
// of 128 and meet once, in LDS, in a fixed order.
//
// A wave brings a chunk's weights, rows of x and scales into a ring of its own in LDS
// by DMA, so that nothing but its own loads makes it wait and neighbouring lanes read
// neighbouring bytes.  Loaded straight into the fragments' registers, where neighbours
// are of different rows, every load takes its 64 lookups in the cache apart: 16 rows of
// int8 by 4096 x 11008 weights took 16.8 us so and take 9.7 us.  Two chunks in a ring
// leave several workgroups on a CU; three and four are slower (11008 x 4096, groups of
// 32: 11.8, 13.1 and 13.4 us), as are four waves and sixteen in place of eight (13.9,
// 16.1).  One token by 4096 x 4096 takes 5.8 us, by 11008 x 4096 10.7 (2.6 TB/s): with
// 16 KB to 88 KB of weights for a CU, the way there and back is most of it.
//
// Of the fragments, x goes as the MFMA's rows and the weights as its columns, so a
// lane's results are all of one weight row and take one scale; lane (n, q) has the
// eight weights at k = 32 t + 8 q in step t, one word.
//
// Unpacking: the bytes hold weight + 8 (0..15).  Nibbles i and i + 4 of a word are
// neighbours along K; shifted to the top four bits of the mantissa of 16.0 (both
// types) they read as 16 + (weight + 8), exactly, two a shift and an and-or.  The
// 24 comes off after the product as 24 sum(x), one MFMA of x by a constant a step:
// the f32 sums are of values at most 31 x where the weights' own reach 8 x.  For
// int8 rows the nibbles are the MFMA's bytes as they are, less 8 sum(x), in
// integers; x's bytes are put in the nibbles' order by two v_perm a word pair.
#include "launch.h"

#include <algorithm>
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
  int M, N, K, group;
  int dma;
  Div31 d_group;  // steps of 32 FL weights in a group
  int s_elem, y_elem;
};

typedef unsigned u4a __attribute__((ext_vector_type(4), aligned(1)));

// Four bytes a lane into LDS by DMA; as dma16.
__device__ __forceinline__ void dma4(i32x4 rsrc, unsigned lds, unsigned voff) {
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" : : "v"(voff), "s"(rsrc), "{m0}"(lds) : "memory");
}

constexpr unsigned kNone = 1u << 31;  // an offset behind every row: such lanes read zeros

// What a workgroup of W waves holds.  ROWS: rows of x, of which the MFMA takes 16 at a
// time (fewer are read again and again, for results that are not stored).
template <bool I8, int ROWS, int NT, int W, int NS>
struct Q4Shape {
  static constexpr int MT = ROWS <= 16 ? 1 : ROWS / 16;
  static constexpr int ES = I8 ? 1 : 2, PIECES = 8 * ES;  // pieces of 16 bytes in a row's 128 values
  // a stage: the weights, x, the scales; instructions that bring x, and all three
  static constexpr int X0 = 1024 * NT, S0 = X0 + ROWS * PIECES * 16, STAGE = S0 + 256 * NT;
  static constexpr int XI = ROWS * PIECES / 64, PER = XI + 2 * NT;
  static constexpr int LDS = W * NS * STAGE;
  static_assert(XI * 64 == ROWS * PIECES && LDS <= 160 * 1024 && NS >= 2 && NS <= 4 && (NS - 1) * PER < 64, "");
  static_assert(W * MT * NT * 1024 <= LDS, "the waves' parts take the rings' place");
};

// FL: steps of 32 between two additions to the result (1, 2 or 4): at most the group.
// S32: scales of 32 bits.  NS: chunks in a wave's ring.
template <int ELEM, int ROWS, int NT, int W, int NS, int FL, bool S32>
__global__ __launch_bounds__(64 * W) void matmul_q4_kernel(Q4Args p) {
  constexpr bool I8 = ELEM == kI8;
  typedef Q4Shape<I8, ROWS, NT, W, NS> S;
  constexpr int ES = S::ES, MT = S::MT, XI = S::XI, PIECES = S::PIECES, NF = 4 / FL;
  typedef typename std::conditional<I8, int4v, float4v>::type acc_t;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[S::LDS];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, q = lane >> 4;
  const int b = (int)p.d_tiles(blockIdx.x);
  const int tile = blockIdx.x - b * p.tiles;
  const int tm = (int)p.d_nt(tile), tn = tile - tm * p.ntiles;
  int bx, by, bz;
  p.blocks(b, bx, by, bz);
  const int m0 = tm * 16 * MT, n0 = tn * 16 * NT;
  const unsigned char* const w = p.w + p.tw.at(bx, by, bz) + n0 * p.ldw;
  const unsigned char* const x = p.x + (p.tx.at(bx, by, bz) + m0 * p.ldx) * ES;

  // A lane's pieces: the weights' row lane / 4, piece (lane % 4) ^ row / 2 % 4; x's row
  // lane / PIECES of each instruction's, piece (lane % PIECES) ^ row % 8.  Neighbours
  // read neighbours in memory, and fragments, of one piece of 16 rows, lie over all banks.
  const int wn = lane >> 2, wt = (lane & 3) ^ ((lane >> 3) & 3);
  unsigned wat[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) wat[n] = wn + 16 * n < p.N - n0 ? (unsigned)(wn + 16 * n) * (unsigned)p.ldw + wt * 16 : kNone;
  constexpr int XR = 64 / PIECES;  // rows of an instruction: 4 or 8
  unsigned xat[XI];
  const int xr = lane / PIECES;
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int row = i * XR + xr, c = (lane % PIECES) ^ (row & 7);
    xat[i] = row < p.M - m0 ? (unsigned)row * (unsigned)p.ldx * ES + c * 16 : kNone;
  }
  // Its scale: row lane / 4, the group of step FL (lane % 4) of a chunk.  DMA takes four
  // bytes, of which a scale of 16 bits is either half, so the address is rounded down to
  // them; they lie within the memory that holds the scale.
  const int sf0 = lane & 3;
  const unsigned char* const st = static_cast<const unsigned char*>(p.s) + ((p.ts.at(bx, by, bz) + n0 * p.lds) << (S32 ? 2 : 1));
  const unsigned odd = (unsigned)reinterpret_cast<uintptr_t>(st) & 3;  // 16 bits: 0 or 2
  const unsigned char* const s0 = st - odd;
  unsigned char* const ring = lds + wave * NS * S::STAGE;
  auto issue = [&](int c, int slot) {
    unsigned char* const at = ring + slot * S::STAGE;
    const unsigned char* const wc = w + (long long)c * 64;
    const unsigned char* const xc = x + (long long)c * 128 * ES;
    const int left = p.K - c * 128;  // pieces past it are zeros
    const bool whole = left >= 128;
    const unsigned group = p.d_group((unsigned)(c * NF + sf0));
    unsigned wo[NT], so[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      wo[n] = whole || wt * 32 < left ? wat[n] : kNone;
      const unsigned s = (((unsigned)(wn + 16 * n) * (unsigned)p.lds + group) << (S32 ? 2 : 1)) + odd;
      so[n] = wn + 16 * n < p.N - n0 && sf0 < NF && sf0 * FL * 32 < left ? s & ~3u : kNone;
    }
    if (p.dma) {
      // the low half of its generic address (a cast between address spaces compares with null first)
      const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<uintptr_t>(at));
#pragma unroll
      for (int n = 0; n < NT; ++n) dma16(raw_rsrc(wc, kNone), to + 1024 * n, wo[n], 0);
      const i32x4 rs = raw_rsrc(xc, kNone);
#pragma unroll
      for (int i = 0; i < XI; ++i) {
        const int k = ((lane % PIECES) ^ ((i * XR + xr) & 7)) * (16 / ES);
        dma16(rs, to + S::X0 + 1024 * i, whole || k < left ? xat[i] : kNone, 0);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) dma4(raw_rsrc(s0, kNone), to + S::S0 + 256 * n, so[n]);
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint4v v = {0, 0, 0, 0};
        if (wo[n] < kNone) v = (uint4v)(*reinterpret_cast<const u4a*>(wc + wo[n]));
        *reinterpret_cast<uint4v*>(at + 1024 * n + lane * 16) = v;
        unsigned e = 0;
        if (so[n] < kNone) e = *reinterpret_cast<const unsigned*>(s0 + so[n]);
        *reinterpret_cast<unsigned*>(at + S::S0 + 256 * n + lane * 4) = e;
      }
#pragma unroll
      for (int i = 0; i < XI; ++i) {
        const int k = ((lane % PIECES) ^ ((i * XR + xr) & 7)) * (16 / ES);
        uint4v u = {0, 0, 0, 0};
        if (xat[i] < kNone && k < left) u = (uint4v)(*reinterpret_cast<const u4a*>(xc + xat[i]));
        *reinterpret_cast<uint4v*>(at + S::X0 + 1024 * i + lane * 16) = u;
      }
    }
  };

  float4v y[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) y[i][n] = float4v{0, 0, 0, 0};

  // where this lane's fragments lie in a stage: a word of weights, and of x the piece of
  // a row's step, in which int8 rows have two quarters' eight bytes
  const int wfrag = col * 64 + q * 4, wsw = (col >> 1) & 3;
  const int xrow = ROWS < 16 ? col % ROWS : col, xsw = xrow & 7;
  const int xfrag = S::X0 + xrow * PIECES * 16 + (I8 ? (q & 1) * 8 : 0), xpiece = I8 ? q >> 1 : q;
  int f16 = p.s_elem == kF16;
  asm volatile("" : "+v"(f16));  // told apart lane by lane: a branch would part the products
  const bool f16_scales = f16 != 0;
  const unsigned srow_col = (unsigned)col * (unsigned)p.lds + (odd >> 1);

  auto compute = [&](const unsigned (&d)[NT][4], const uint4v (&xf)[MT][4], const unsigned (&sc)[NT][NF], int c) {
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      // one step: its correction is where its products begin; more: two sums side by side
      constexpr bool CHAIN = FL == 1;
      acc_t acc[MT][NT], off[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        off[i] = acc_t{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[i][n] = acc_t{0, 0, 0, 0};
      }
#pragma unroll
      for (int u = 0; u < FL; ++u) {
        const int t = f * FL + u;
        if constexpr (I8) {
          const long eights = CHAIN ? (long)0xf8f8f8f8f8f8f8f8UL : 0x0808080808080808L;
          long xi[MT];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const unsigned lo = __builtin_amdgcn_perm(xf[i][t][1], xf[i][t][0], 0x05010400u);
            const unsigned hi = __builtin_amdgcn_perm(xf[i][t][1], xf[i][t][0], 0x07030602u);
            xi[i] = (long)(((unsigned long)hi << 32) | lo);
            off[i] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xi[i], eights, off[i], 0, 0, 0);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const long wj = (long)(((unsigned long)((d[n][t] >> 4) & 0x0f0f0f0fu) << 32) | (d[n][t] & 0x0f0f0f0fu));
#pragma unroll
            for (int i = 0; i < MT; ++i)
              acc[i][n] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xi[i], wj, CHAIN ? off[i] : acc[i][n], 0, 0, 0);
          }
        } else {
          // 16 + u: f16 0x4c00 | u << 6, bf16 0x4180 | u << 3
          constexpr unsigned one = ELEM == kF16 ? 0x4c004c00u : 0x41804180u, mask = ELEM == kF16 ? 0x03c003c0u : 0x00780078u;
          constexpr unsigned c24 = (ELEM == kF16 ? 0x4e004e00u : 0x41c041c0u) | (CHAIN ? 0x80008000u : 0);
          constexpr int up = ELEM == kF16 ? 6 : 3;
          auto mma = [](uint4v a, uint4v bb, float4v c) {
            if constexpr (ELEM == kF16)
              return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, bb), c, 0, 0, 0);
            else
              return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, bb), c, 0, 0, 0);
          };
#pragma unroll
          for (int i = 0; i < MT; ++i) off[i] = mma(xf[i][t], uint4v{c24, c24, c24, c24}, off[i]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint4v v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = ((up >= 4 * e ? d[n][t] << (up - 4 * e) : d[n][t] >> (4 * e - up)) & mask) | one;
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][n] = mma(xf[i][t], v, CHAIN ? off[i] : acc[i][n]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float sf;
        if constexpr (S32) {
          sf = __builtin_bit_cast(float, sc[n][f]);
        } else {
          // rows 16 apart begin in the same half of their four bytes
          const unsigned half = sc[n][f] >> (((srow_col + p.d_group((unsigned)(c * NF + f))) & 1) * 16);
          const float h = (float)__builtin_bit_cast(_Float16, (unsigned short)half), b = __builtin_bit_cast(float, half << 16);
          sf = f16_scales ? h : b;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            y[i][n][r] = fmaf((float)(CHAIN ? acc[i][n][r] : acc[i][n][r] - off[i][r]), sf, y[i][n][r]);
      }
    }
  };

  const int chunks = (p.K + 127) >> 7, mine = max(0, (chunks - wave + W - 1) / W);
#pragma unroll
  for (int j = 0; j < NS; ++j)
    if (j < mine) issue(wave + j * W, j);
  int slot = 0;
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    const int ahead = p.dma ? min(mine - 1 - j, NS - 1) : 0;
    switch (ahead) {
      case 0: XTK_WAIT_VM(0); break;
      case 1: XTK_WAIT_VM(S::PER); break;
      case 2: XTK_WAIT_VM(NS > 2 ? 2 * S::PER : 0); break;
      default: XTK_WAIT_VM(NS > 3 ? 3 * S::PER : 0); break;
    }
    asm volatile("" ::: "memory");
    const unsigned char* const at = ring + slot * S::STAGE;
    unsigned d[NT][4], sc[NT][NF];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int f = 0; f < NF; ++f) sc[n][f] = *reinterpret_cast<const unsigned*>(at + S::S0 + 256 * n + col * 16 + f * 4);
    uint4v xf[MT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int n = 0; n < NT; ++n) d[n][t] = *reinterpret_cast<const unsigned*>(at + 1024 * n + wfrag + ((t ^ wsw) << 4));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const unsigned char* const xp = at + xfrag + i * 256 * PIECES;
        if constexpr (I8) {
          const uint2v e = *reinterpret_cast<const uint2v*>(xp + (((2 * t + xpiece) ^ xsw) << 4));
          xf[i][t] = uint4v{e[0], e[1], 0, 0};
        } else {
          xf[i][t] = *reinterpret_cast<const uint4v*>(xp + (((4 * t + xpiece) ^ xsw) << 4));
        }
      }
    }
    // every fragment is in registers before the slot is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (j + NS < mine) issue(wave + (j + NS) * W, slot);
    slot = slot + 1 == NS ? 0 : slot + 1;
    compute(d, xf, sc, wave + j * W);
  }
  __syncthreads();  // every ring is done with

  // the waves' parts, summed in the order of the waves
  float* const part = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) part[(((wave * MT + i) * NT + n) * 4 + r) * 64 + lane] = y[i][n][r];
  __syncthreads();
  const long long y0 = p.ty.at(bx, by, bz), r0 = p.trs.at(bx, by, bz);
  for (int e = threadIdx.x; e < MT * NT * 256; e += 64 * W) {
    const int i = e / (256 * NT), j = (e >> 8) % NT, r = (e >> 6) & 3, l = e & 63;
    const int m = m0 + 16 * i + 4 * (l >> 4) + r, n = n0 + 16 * j + (l & 15);
    if (m >= p.M || n >= p.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int u = 0; u < W; ++u) v += part[u * MT * NT * 256 + e];
    if (p.rs) v *= p.rs[r0 + m * p.ldrs];
    const long long at = y0 + m * p.ldy + n;
    if (p.y_elem == kF32) static_cast<float*>(p.y)[at] = v;
    else if (p.y_elem == kF16) static_cast<_Float16*>(p.y)[at] = (_Float16)v;
    else static_cast<__bf16*>(p.y)[at] = (__bf16)v;
  }
}

template <int ELEM, bool S32, int ROWS, int NT, int W, int NS>
void run_fl(Q4Args& a, int wgs, hipStream_t s) {
  const int fl = a.group % 128 == 0 ? 4 : a.group % 64 == 0 ? 2 : 1;
  a.d_group = div31(a.group / (32 * fl));
  if (fl == 4) matmul_q4_kernel<ELEM, ROWS, NT, W, NS, 4, S32><<<wgs, 64 * W, 0, s>>>(a);
  else if (fl == 2) matmul_q4_kernel<ELEM, ROWS, NT, W, NS, 2, S32><<<wgs, 64 * W, 0, s>>>(a);
  else matmul_q4_kernel<ELEM, ROWS, NT, W, NS, 1, S32><<<wgs, 64 * W, 0, s>>>(a);
}

// near32: 32 rows of weights, and of their scales, lie within a lane's 31 bits.
template <int ELEM, bool S32>
bool run(Q4Args& a, long long blocks, bool near32, hipStream_t s) {
  constexpr int FEW = ELEM == kI8 ? 8 : 4;  // rows that one instruction brings
  auto tiles_of = [&](int mt, int nt) {
    return (long long)((a.N + 16 * nt - 1) / (16 * nt)) * ((a.M + 16 * mt - 1) / (16 * mt));
  };
  // As many rows of x to a workgroup as leave one for every CU.  64 rows of 16 bits are
  // sixteen times their weights' bytes, from L2: there a workgroup takes 32 rows of
  // weights if three quarters of the CUs still get one (42 rows by 7906 x 8192: 26.6 us,
  // with 16 rows 37; fewer rows of x, or of int8, are better off with twice the
  // workgroups: 24 by 11008 x 4096 18.1 us against 20.8).
  int mt = a.M <= 16 ? 1 : a.M <= 32 ? 2 : 4;
  while (mt > 1 && tiles_of(mt, 1) * blocks < 256) mt >>= 1;
  const int nt = ELEM != kI8 && mt == 4 && near32 && tiles_of(mt, 2) * blocks >= 192 ? 2 : 1;
  const long long tiles = tiles_of(mt, nt);
  if (tiles > 0x7fffffffLL || !grid_fits(tiles * blocks, 512)) return false;
  a.tiles = (int)tiles;
  a.ntiles = (a.N + 16 * nt - 1) / (16 * nt);
  a.d_tiles = div31(a.tiles);
  a.d_nt = div31(a.ntiles);
  const int wgs = (int)(tiles * blocks);
  if (a.M <= FEW) run_fl<ELEM, S32, FEW, 1, 8, 2>(a, wgs, s);
  else if (mt == 1) run_fl<ELEM, S32, 16, 1, 8, 2>(a, wgs, s);
  else if (mt == 2) run_fl<ELEM, S32, 32, 1, 8, ELEM == kI8 ? 3 : 2>(a, wgs, s);
  else if constexpr (ELEM == kI8) run_fl<ELEM, S32, 64, 1, 8, 2>(a, wgs, s);
  else if (nt == 1) run_fl<ELEM, S32, 64, 1, 4, 2>(a, wgs, s);
  else run_fl<ELEM, S32, 64, 2, 4, 2>(a, wgs, s);
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
  a.group = static_cast<int>(q.group);
  // DMA takes rows of whole 16 bytes; others go through registers
  auto pieces = [&](const xt::Access2D& t, int per) {
    const xt::TileAddr& d = t.addr;
    return reinterpret_cast<uintptr_t>(bufs[t.arg]) % 16 == 0 && t.ld % per == 0 && d.c0 % per == 0 && d.sx % per == 0 &&
           d.sy % per == 0 && d.sz % per == 0;
  };
  a.dma = pieces(q.x, q.x.elem == xt::Elem::I8 ? 16 : 8) && pieces(q.w, 16);
  a.s_elem = elem_of(q.scales.elem);
  a.y_elem = elem_of(q.y.elem);
  // what a lane adds to its tile's address has 31 bits
  auto near = [](int rows, long long ld, long long cols, int bytes) { return ((rows - 1) * ld + cols) * bytes < (1LL << 31); };
  const int xs = q.x.elem == xt::Elem::I8 ? 1 : 2, ss = a.s_elem == kF32 ? 4 : 2;
  auto near_weights = [&](int rows) { return near(rows, a.ldw, 64, 1) && near(rows, a.lds, a.K / 32 + 1, ss); };
  if (!near(std::min(a.M, 64), a.ldx, 128, xs) || !near_weights(std::min(a.N, 16))) {
    why = "matmul_q4: rows that a workgroup reads together span 2^31 bytes or more";
    return hipErrorInvalidValue;
  }
  bool ok;
  const bool s32 = a.s_elem == kF32;
  const bool near32 = near_weights(std::min(a.N, 32));
  const long long blocks = grid_blocks(p);
  if (q.x.elem == xt::Elem::I8) ok = s32 ? run<kI8, true>(a, blocks, near32, s) : run<kI8, false>(a, blocks, near32, s);
  else if (q.x.elem == xt::Elem::F16) ok = s32 ? run<kF16, true>(a, blocks, near32, s) : run<kF16, false>(a, blocks, near32, s);
  else ok = s32 ? run<kBF16, true>(a, blocks, near32, s) : run<kBF16, false>(a, blocks, near32, s);
  if (!ok) {
    why = "matmul_q4: " + std::to_string(a.M) + " x " + std::to_string(a.N) + " tiles exceed one launch";
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace xtk
