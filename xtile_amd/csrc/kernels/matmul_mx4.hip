// Products of rows in microscaled 4-bit floating point:
//   y[m, n] = sum_b 2^(xs[m, b] + ws[n, b] - 254) sum_{k in block b} x[m, k] w[n, k]
//
// The MFMA takes 4-bit operands as they lie in memory: of a lane's row, one block of
// 32 neighbours, 16 bytes, and the byte of its scale, which a selector takes out of a
// register's four.  Which blocks meet in one MFMA is free, as long as both operands
// agree, so that lanes have neighbouring scale bytes in one register.
//
// A stage of LDS has 256 of K: rows of 128 bytes, brought by DMA in 16-byte pieces (eight
// neighbouring lanes a row), piece c of row r at c ^ r / 2 % 8, so that 16 rows' pieces
// of one block lie over all banks; and for each row three words that hold its eight
// scale bytes, which begin anywhere within the first.
#include "launch.h"

#include <algorithm>
#include <cmath>

#include "common.h"

namespace xtk {
namespace {

enum { kF32 = 0, kF16 = 1, kBF16 = 2 };

typedef int int4w __attribute__((ext_vector_type(4)));
typedef int int8w __attribute__((ext_vector_type(8)));
typedef unsigned u4a __attribute__((ext_vector_type(4), aligned(1)));

constexpr unsigned kNone = 1u << 31;  // an offset behind every row: such lanes read zeros
constexpr int kStageK = 256, kBlocks = kStageK / 32;

struct Mx4Args {
  const unsigned char *x, *xs, *w, *ws;
  void* y;
  TileOff tx, txs, tw, tws, ty;
  long long ldx, ldxs, ldw, ldws, ldy;  // bytes; y: elements
  BlockDecode blocks;
  Div31 d_tiles, d_nt;  // tiles of a Block, n tiles
  Div31 d_group, d_width, d_last;  // of many rows: a group's tiles, its columns, the last one's
  int tiles, ntiles, mtiles, group, nwg;
  int M, N, blocks_k;  // blocks of 32 of a row
  int dma, whole;  // whole: scales in rows of whole words
  int y_elem;
};

// Four bytes a lane into LDS by DMA; as dma16.
__device__ __forceinline__ void dma4(i32x4 rsrc, unsigned lds, unsigned voff) {
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" : : "v"(voff), "s"(rsrc), "{m0}"(lds) : "memory");
}

// The low half of a generic address (a cast between address spaces compares with null first).
__device__ __forceinline__ unsigned lds_at(const void* p) { return (unsigned)reinterpret_cast<uintptr_t>(p); }

__device__ __forceinline__ int piece_of(int row, int c) { return c ^ ((row >> 1) & 7); }

// Eight rows' pieces of a stage that one instruction of a wave brings: rows first + lane / 8.
struct Pieces {
  unsigned off;  // from the rows' first byte, or kNone
  int block;
  __device__ __forceinline__ void begin(int first, int rows, long long ld) {
    const int lane = threadIdx.x & 63, row = first + (lane >> 3);
    block = piece_of(row, lane & 7);
    off = row < rows ? (unsigned)row * (unsigned)ld + block * 16 : kNone;
  }
  // from: the rows at this stage's first block; left: blocks from there on
  __device__ __forceinline__ void issue(bool dma, const unsigned char* from, int left, unsigned char* to) const {
    const unsigned at = block < left ? off : kNone;
    if (dma) {
      dma16(raw_rsrc(from, kNone), __builtin_amdgcn_readfirstlane(lds_at(to)), at, 0);
    } else {
      uint4v v = {0, 0, 0, 0};
      if (at < kNone) v = (uint4v)(*reinterpret_cast<const u4a*>(from + at));
      *reinterpret_cast<uint4v*>(to + 16 * (threadIdx.x & 63)) = v;
    }
  }
};

// Three words a row of scales, 64 of which one instruction brings: words first on, of rows
// below `count`.  Rows begin at any byte: a word that holds none of the eight bytes, or none
// of a row's, is not read.
struct Scales {
  unsigned off;  // of the word, less the bytes before it
  int before;    // bytes of the word before the row's first
  __device__ __forceinline__ void begin(const unsigned char* base, int first, int count, int rows, long long ld) {
    const int word = first + (threadIdx.x & 63), row = word / 3, i = word - 3 * row;
    const unsigned at = (unsigned)row * (unsigned)ld, odd = ((unsigned)reinterpret_cast<uintptr_t>(base) + at) & 3;
    before = (int)odd - 4 * i;
    off = row < min(count, rows) && before > -kBlocks ? at - (unsigned)before : kNone;
  }
  // from: the scales at this stage's first block.  The descriptor begins three bytes
  // earlier, for words that begin before their row.
  __device__ __forceinline__ void issue(const unsigned char* from, int left, unsigned char* to) const {
    const unsigned at = off != kNone && -before < left ? off + 3u : kNone;
    const unsigned odd = (unsigned)reinterpret_cast<uintptr_t>(from - 3) & 3;
    // a descriptor's base is a multiple of four
    dma4(raw_rsrc(from - 3 - odd, kNone), __builtin_amdgcn_readfirstlane(lds_at(to)), at == kNone ? kNone : at + odd);
  }
};

// Of a row's three words, bytes 4 h .. 4 h + 3 behind the first `odd`, those of blocks past
// the row's end as 0 (a scale of 255 would make NaN of the zeros there).
__device__ __forceinline__ int scale_word(const unsigned char* three, int h, int odd, int left) {
  const unsigned lo = reinterpret_cast<const unsigned*>(three)[h], hi = reinterpret_cast<const unsigned*>(three)[h + 1];
  const unsigned v = __builtin_amdgcn_alignbyte(hi, lo, odd);
  const int n = left - 4 * h;
  return (int)(n >= 4 ? v : n <= 0 ? 0u : v & ((1u << (8 * n)) - 1));
}

__device__ __forceinline__ int odd_of(const unsigned char* base, int row, long long ld) {
  return (int)(((unsigned)reinterpret_cast<uintptr_t>(base) + (unsigned)row * (unsigned)ld) & 3);
}

__device__ __forceinline__ int8w wide(uint4v a) { return int8w{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}; }

__device__ __forceinline__ void put(void* y, int elem, long long at, float v) {
  if (elem == kF32) static_cast<float*>(y)[at] = v;
  else if (elem == kF16) static_cast<_Float16*>(y)[at] = (_Float16)v;
  else static_cast<__bf16*>(y)[at] = (__bf16)v;
}

// Four neighbours of a row, at element alignment.
__device__ __forceinline__ void put4(void* y, int elem, long long at, float4v v) {
  if (elem == kF32) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    *reinterpret_cast<f4*>(static_cast<float*>(y) + at) = (f4)v;
  } else if (elem == kF16) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4), aligned(2)));
    *reinterpret_cast<h4*>(static_cast<_Float16*>(y) + at) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  } else {
    typedef __bf16 b4 __attribute__((ext_vector_type(4), aligned(2)));
    *reinterpret_cast<b4*>(static_cast<__bf16*>(y) + at) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
  }
}

// Few rows of x: a workgroup has 16 rows of weights and 16 of x, its W waves split K in
// stages, each in a ring of two of its own, and meet once, in LDS, in a fixed order.
// XR: rows of x in LDS (8, of which the MFMA's 16 are the same ones twice, or 16).
template <int XR, int W>
struct FewShape {
  static constexpr int X0 = 2048, S0 = X0 + XR * 128, STAGE = S0 + 512;
  static constexpr int XI = XR / 8, PER = 2 + XI + 2;  // instructions of a stage
  static constexpr int LDS = W * 2 * STAGE;
  static_assert(LDS <= 160 * 1024 && W * 1024 <= LDS, "");
};

template <int XR, int W>
__global__ __launch_bounds__(64 * W) void matmul_mx4_few_kernel(Mx4Args p) {
  typedef FewShape<XR, W> S;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[S::LDS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int b = (int)p.d_tiles(blockIdx.x);
  const int tile = blockIdx.x - b * p.tiles;
  const int tm = (int)p.d_nt(tile), tn = tile - tm * p.ntiles;
  int bx, by, bz;
  p.blocks(b, bx, by, bz);
  const int m0 = tm * 16, n0 = tn * 16, mrows = p.M - m0, nrows = p.N - n0;
  const unsigned char* const w = p.w + p.tw.at(bx, by, bz) + n0 * p.ldw;
  const unsigned char* const ws = p.ws + p.tws.at(bx, by, bz) + n0 * p.ldws;
  const unsigned char* const x = p.x + p.tx.at(bx, by, bz) + m0 * p.ldx;
  const unsigned char* const xs = p.xs + p.txs.at(bx, by, bz) + m0 * p.ldxs;

  Pieces pw[2], px[S::XI];
  Scales sw, sx;
#pragma unroll
  for (int i = 0; i < 2; ++i) pw[i].begin(8 * i, nrows, p.ldw);
#pragma unroll
  for (int i = 0; i < S::XI; ++i) px[i].begin(8 * i, mrows, p.ldx);
  sw.begin(ws, 0, 16, nrows, p.ldws);
  sx.begin(xs, 0, XR, mrows, p.ldxs);
  unsigned char* const ring = lds + wave * 2 * S::STAGE;
  auto issue = [&](int c, int slot) {
    unsigned char* const at = ring + slot * S::STAGE;
    const int left = p.blocks_k - c * kBlocks;
    const long long d = (long long)c * 128;
#pragma unroll
    for (int i = 0; i < 2; ++i) pw[i].issue(p.dma, w + d, left, at + 1024 * i);
#pragma unroll
    for (int i = 0; i < S::XI; ++i) px[i].issue(p.dma, x + d, left, at + S::X0 + 1024 * i);
    sw.issue(ws + c * kBlocks, left, at + S::S0);
    sx.issue(xs + c * kBlocks, left, at + S::S0 + 256);
  };

  float4v y = {0, 0, 0, 0};
  const int stages = (p.blocks_k + kBlocks - 1) / kBlocks, mine = max(0, (stages - wave + W - 1) / W);
  if (mine > 0) issue(wave, 0);
  if (mine > 1) issue(wave + W, 1);
  // this lane's row of x, and where the scales of its two rows begin
  const int xrow = col % XR, wodd = odd_of(ws, col, p.ldws), xodd = odd_of(xs, xrow, p.ldxs);
  int slot = 0;
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    if (p.dma && j + 1 < mine) XTK_WAIT_VM(S::PER);
    else XTK_WAIT_VM(0);
    asm volatile("" ::: "memory");
    const int left = p.blocks_k - (wave + j * W) * kBlocks;
    const unsigned char* const at = ring + slot * S::STAGE;
    // MFMA i has blocks 2 g + i; a lane's two scale bytes are moved to the low half
    uint4v wf[2], xf[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      wf[i] = *reinterpret_cast<const uint4v*>(at + col * 128 + piece_of(col, 2 * g + i) * 16);
      xf[i] = *reinterpret_cast<const uint4v*>(at + S::X0 + xrow * 128 + piece_of(xrow, 2 * g + i) * 16);
    }
    const int sa = scale_word(at + S::S0 + 256 + xrow * 12, g >> 1, xodd, left) >> (16 * (g & 1));
    const int sb = scale_word(at + S::S0 + col * 12, g >> 1, wodd, left) >> (16 * (g & 1));
    // every fragment is in registers before the slot is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (j + 2 < mine) issue(wave + (j + 2) * W, slot);
    slot ^= 1;
    y = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(xf[0]), wide(wf[0]), y, 4, 4, 0, sa, 0, sb);
    y = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(xf[1]), wide(wf[1]), y, 4, 4, 1, sa, 1, sb);
  }
  __syncthreads();  // every ring is done with

  // the waves' parts, summed in the order of the waves
  float* const part = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int r = 0; r < 4; ++r) part[(wave * 4 + r) * 64 + lane] = y[r];
  __syncthreads();
  const int e = threadIdx.x, r = e >> 6, l = e & 63;
  const int m = m0 + 4 * (l >> 4) + r, n = n0 + (l & 15);
  if (e >= 256 || m >= p.M || n >= p.N) return;
  float v = 0.0f;
#pragma unroll
  for (int u = 0; u < W; ++u) v += part[u * 256 + e];
  put(p.y, p.y_elem, p.ty.at(bx, by, bz) + m * p.ldy + n, v);
}

template <int XR, int W>
bool run_few(Mx4Args& a, long long blocks, hipStream_t s) {
  const long long nt = (a.N + 15) / 16, tiles = nt * ((a.M + 15) / 16);
  if (tiles > 0x7fffffffLL || !grid_fits(tiles * blocks, 64 * W)) return false;
  a.tiles = static_cast<int>(tiles);
  a.ntiles = static_cast<int>(nt);
  a.d_tiles = div31(a.tiles);
  a.d_nt = div31(a.ntiles);
  matmul_mx4_few_kernel<XR, W><<<static_cast<unsigned>(tiles * blocks), 64 * W, 0, s>>>(a);
  return true;
}

// Tiles of 32 MT x 32 NT of the result, between the two: the waves split K as above, on
// 32 x 32 x 64 MFMAs; a lane's half has blocks 4 h + i of a stage in step i.
template <int MT, int NT, int W>
struct MidShape {
  static constexpr int X0 = NT * 4096, S0 = X0 + MT * 4096;
  static constexpr int WI = (NT * 96 + 63) / 64, XI = (MT * 96 + 63) / 64;  // instructions for scales
  static constexpr int STAGE = S0 + 256 * (WI + XI), PER = 4 * (MT + NT) + WI + XI;
  static constexpr int PARTS = W * MT * NT * 4096;
  static constexpr int LDS = W * 2 * STAGE > PARTS ? W * 2 * STAGE : PARTS;
  static_assert(LDS <= 160 * 1024 && PER < 64, "");
};

template <int MT, int NT, int W>
__global__ __launch_bounds__(64 * W) void matmul_mx4_mid_kernel(Mx4Args p) {
  typedef MidShape<MT, NT, W> S;
  typedef float float16v __attribute__((ext_vector_type(16)));
  __shared__ __attribute__((aligned(1024))) unsigned char lds[S::LDS];
  const int lane = threadIdx.x & 63, lrow = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = (int)p.d_tiles(blockIdx.x);
  const int tile = blockIdx.x - b * p.tiles;
  const int tm = (int)p.d_nt(tile), tn = tile - tm * p.ntiles;
  int bx, by, bz;
  p.blocks(b, bx, by, bz);
  const int m0 = tm * 32 * MT, n0 = tn * 32 * NT, mrows = p.M - m0, nrows = p.N - n0;
  const unsigned char* const w = p.w + p.tw.at(bx, by, bz) + n0 * p.ldw;
  const unsigned char* const ws = p.ws + p.tws.at(bx, by, bz) + n0 * p.ldws;
  const unsigned char* const x = p.x + p.tx.at(bx, by, bz) + m0 * p.ldx;
  const unsigned char* const xs = p.xs + p.txs.at(bx, by, bz) + m0 * p.ldxs;

  Pieces pw[4 * NT], px[4 * MT];
  Scales sw[S::WI], sx[S::XI];
#pragma unroll
  for (int i = 0; i < 4 * NT; ++i) pw[i].begin(8 * i, nrows, p.ldw);
#pragma unroll
  for (int i = 0; i < 4 * MT; ++i) px[i].begin(8 * i, mrows, p.ldx);
#pragma unroll
  for (int i = 0; i < S::WI; ++i) sw[i].begin(ws, 64 * i, 32 * NT, nrows, p.ldws);
#pragma unroll
  for (int i = 0; i < S::XI; ++i) sx[i].begin(xs, 64 * i, 32 * MT, mrows, p.ldxs);
  unsigned char* const ring = lds + wave * 2 * S::STAGE;
  auto issue = [&](int c, int slot) {
    unsigned char* const at = ring + slot * S::STAGE;
    const int left = p.blocks_k - c * kBlocks;
    const long long d = (long long)c * 128;
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) pw[i].issue(p.dma, w + d, left, at + 1024 * i);
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i) px[i].issue(p.dma, x + d, left, at + S::X0 + 1024 * i);
#pragma unroll
    for (int i = 0; i < S::WI; ++i) sw[i].issue(ws + c * kBlocks, left, at + S::S0 + 256 * i);
#pragma unroll
    for (int i = 0; i < S::XI; ++i) sx[i].issue(xs + c * kBlocks, left, at + S::S0 + 256 * (S::WI + i));
  };

  float16v acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
  const int stages = (p.blocks_k + kBlocks - 1) / kBlocks, mine = max(0, (stages - wave + W - 1) / W);
  if (mine > 0) issue(wave, 0);
  if (mine > 1) issue(wave + W, 1);
  const int wodd = odd_of(ws, lrow, p.ldws), xodd = odd_of(xs, lrow, p.ldxs);  // of rows 32 apart alike
  const int row = lrow * 128, piece = piece_of(lrow, 4 * hi) * 16;  // block 4 hi + ks: its last bits changed by ks
  int slot = 0;
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    if (p.dma && j + 1 < mine) XTK_WAIT_VM(S::PER);
    else XTK_WAIT_VM(0);
    asm volatile("" ::: "memory");
    const int left = p.blocks_k - (wave + j * W) * kBlocks;
    const unsigned char* const at = ring + slot * S::STAGE;
    uint4v wf[4][NT], xf[4][MT];
    int ss[NT + MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) ss[i] = scale_word(at + S::S0 + (32 * i + lrow) * 12, hi, wodd, left);
#pragma unroll
    for (int i = 0; i < MT; ++i) ss[NT + i] = scale_word(at + S::S0 + 256 * S::WI + (32 * i + lrow) * 12, hi, xodd, left);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int i = 0; i < NT; ++i) wf[ks][i] = *reinterpret_cast<const uint4v*>(at + 4096 * i + row + (piece ^ (16 * ks)));
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[ks][i] = *reinterpret_cast<const uint4v*>(at + S::X0 + 4096 * i + row + (piece ^ (16 * ks)));
    }
    // every fragment is in registers before the slot is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (j + 2 < mine) issue(wave + (j + 2) * W, slot);
    slot ^= 1;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float16v& d = acc[i][n];
        const int sa = ss[NT + i], sb = ss[n];
        d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(xf[0][i]), wide(wf[0][n]), d, 4, 4, 0, sa, 0, sb);
        d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(xf[1][i]), wide(wf[1][n]), d, 4, 4, 1, sa, 1, sb);
        d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(xf[2][i]), wide(wf[2][n]), d, 4, 4, 2, sa, 2, sb);
        d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(xf[3][i]), wide(wf[3][n]), d, 4, 4, 3, sa, 3, sb);
      }
  }
  __syncthreads();  // every ring is done with

  // the waves' parts, summed in the order of the waves; four neighbours of a row a thread
  float* const part = reinterpret_cast<float*>(lds);
  constexpr int COLS = 32 * NT, ALL = 1024 * MT * NT;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        part[wave * ALL + (32 * i + 8 * (v >> 2) + 4 * hi + (v & 3)) * COLS + 32 * n + lrow] = acc[i][n][v];
  __syncthreads();
  const long long y0 = p.ty.at(bx, by, bz);
  for (int e = 4 * threadIdx.x; e < ALL; e += 256 * W) {
    const int m = m0 + e / COLS, n = n0 + e % COLS;
    if (m >= p.M || n >= p.N) continue;
    float4v v = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < W; ++u) v += *reinterpret_cast<const float4v*>(part + u * ALL + e);
    const long long to = y0 + m * p.ldy + n;
    if (n + 4 <= p.N) put4(p.y, p.y_elem, to, v);
    else
      for (int k = 0; k < p.N - n; ++k) put(p.y, p.y_elem, to + k, k == 0 ? v[0] : k == 1 ? v[1] : v[2]);
  }
}

template <int MT, int NT, int W>
bool run_mid(Mx4Args& a, long long blocks, hipStream_t s) {
  const long long nt = (a.N + 32 * NT - 1) / (32 * NT), tiles = nt * ((a.M + 32 * MT - 1) / (32 * MT));
  if (tiles > 0x7fffffffLL || !grid_fits(tiles * blocks, 64 * W)) return false;
  a.tiles = static_cast<int>(tiles);
  a.ntiles = static_cast<int>(nt);
  a.d_tiles = div31(a.tiles);
  a.d_nt = div31(a.ntiles);
  matmul_mx4_mid_kernel<MT, NT, W><<<static_cast<unsigned>(tiles * blocks), 64 * W, 0, s>>>(a);
  return true;
}

// Many rows of x: BM x BN of the result a workgroup, NW waves of WM x WN on 32 x 32 x 64
// MFMAs.  A stage has 256 of K, rows of 128 bytes (whole cache lines: rows of 64 bytes ask
// L2 twice as often, which bounded the kernel), in one of NB buffers, and four steps of
// products; a lane's half has blocks 4 h + i of it in step i.  A stage's last fragments are
// read before its last step.  The barrier there says that every wave is done with the
// stage's buffer and that the next stage has landed: behind it the last step runs, the next
// stage's first fragments are read, and the DMA into that buffer begins, which has until the
// NB - 1st such barrier to land.  So no barrier is followed by an LDS round trip (a bare
// s_barrier: __syncthreads would wait for LDS reads too).
//
// The result is computed transposed (the weights are the MFMA's rows), so that a lane has
// four neighbours of a row, and leaves through LDS in 16-byte pieces.
//
// A row's scales are a few bytes of a line that L2 is asked for each time: WHOLE, rows of them
// that begin at whole words, takes those of four stages at once (SG), 32 bytes by two
// neighbouring lanes, and others two stages' five words, or, with more than two buffers, where a
// wait that leaves DMA in flight has to count it, one stage's three: 1024 x 4096 x 4096 in 128 x
// 128 17.9 us against 20.8, 1024 x 11008 x 4096 in 256 x 256 36.1 against 39.3 (without any
// scales they take 17.4 and 34.4).
template <int P>
struct Phase {
  static constexpr int value = P;
};
template <int BM, int BN, int NW, int NB, bool WHOLE>
struct ManyShape {
  static constexpr int WC = NW / 2, WM = BM / 2, WN = BN / WC, MI = WM / 32, NI = WN / 32;
  static constexpr int SG = WHOLE ? 4 : NB == 2 ? 2 : 1, WORDS = WHOLE ? 8 : 2 * SG + 1;
  static constexpr int AB = BM * 128, SCALES = (BM + BN) * WORDS * 4, STAGE = (BM + BN) * 128 + (SG == 1 ? SCALES : 0);
  static constexpr int LDS = NB * STAGE + (SG == 1 ? 0 : 2 * SCALES);
  static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW, PD = PA + PB;  // data instructions of a wave and stage
  static constexpr int ONE = WHOLE ? 1024 : 256;                          // bytes of an instruction for scales
  static constexpr int PS = SCALES / ONE / NW;                            // of them, of SG stages
  static constexpr int PER = PD + (WHOLE ? 0 : PS);                       // that a wait counts a stage
  static constexpr int PRODUCTS = MI * NI, HALF = PD / 2, EVERY = PRODUCTS / HALF;  // of a step; data instructions
  static_assert(PS * ONE * NW == SCALES && BM * WORDS * 4 / ONE % PS == 0, "a wave has scales of one operand");
  static_assert(PRODUCTS % HALF == 0 && PA % 2 == 0 && MI >= NI && (MI == 4 || MI == 2) && (PS + SG - 1) / SG <= PRODUCTS && (!WHOLE || PS <= SG), "the steps' schedule");
  static_assert(LDS <= 160 * 1024 && (NB - 1) * (PD + PS) < 64, "");
};

template <int BM, int BN, int NW, int NB, bool WHOLE>
__global__ __launch_bounds__(64 * NW, BM * BN > 128 * 128 || NB > 2 ? 1 : 2)
void matmul_mx4_many_kernel(Mx4Args p) {
  typedef ManyShape<BM, BN, NW, NB, WHOLE> S;
  typedef float float16v __attribute__((ext_vector_type(16)));
  constexpr int MI = S::MI, NI = S::NI, PA = S::PA, PB = S::PB, PS = S::PS, SG = S::SG, WORDS = S::WORDS;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[S::LDS];

  const int lane = threadIdx.x & 63, lrow = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WC, wn = wave % S::WC;
  const int id = xcd_contiguous(blockIdx.x, p.nwg);
  const int b = (int)p.d_tiles(id);
  int tile = id - b * p.tiles;
  // tiles in groups of p.group tile columns, row by row, so that neighbours share panels in L2
  const int gi = (int)p.d_group(tile), first = gi * p.group;
  tile -= gi * p.group * p.mtiles;
  const int width = min(p.group, p.ntiles - first);
  const int tm = width == p.group ? (int)p.d_width(tile) : (int)p.d_last(tile), tn = first + tile - tm * width;
  int bx, by, bz;
  p.blocks(b, bx, by, bz);
  const int m0 = tm * BM, n0 = tn * BN, mrows = min(BM, p.M - m0), nrows = min(BN, p.N - n0);
  const unsigned char* const x = p.x + p.tx.at(bx, by, bz) + m0 * p.ldx;
  const unsigned char* const xs = p.xs + p.txs.at(bx, by, bz) + m0 * p.ldxs;
  const unsigned char* const w = p.w + p.tw.at(bx, by, bz) + n0 * p.ldw;
  const unsigned char* const ws = p.ws + p.tws.at(bx, by, bz) + n0 * p.ldws;
  const int nk = (p.blocks_k + kBlocks - 1) / kBlocks;  // stages

  // What this lane brings: of rows 8 i + lane / 8 of its wave's instructions the piece that
  // lies at lane % 8; it is another, 4 apart, in every second instruction.  Rows past the
  // last lie behind the descriptors' ends and read as zeros, and so does all that comes
  // behind the last stage: its place in LDS is filled without a branch, which would part the
  // products from what goes between them.
  const int piece = piece_of(lane >> 3, lane & 7);
  const unsigned va = (8u * wave * PA + (lane >> 3)) * (unsigned)p.ldx, vb = (8u * wave * PB + (lane >> 3)) * (unsigned)p.ldw;
  const unsigned aend = (unsigned)mrows * (unsigned)p.ldx, bend = (unsigned)nrows * (unsigned)p.ldw;
  auto dma_one = [&](int s, unsigned char* to, int q) {
    const int left = p.blocks_k - kBlocks * s, c = piece ^ (4 * (q & 1));
    const bool of_a = q < PA;
    const unsigned skip = (unsigned)s * 128, end = s < nk ? (of_a ? aend : bend) - skip : 0u;
    const unsigned row8 = 8u * (unsigned)(of_a ? q : q - PA) * (unsigned)(of_a ? p.ldx : p.ldw);
    const unsigned at = (of_a ? va : vb) + row8 + c * 16;
    const unsigned lds_to = lds_at(to + (of_a ? wave * PA + q : BM / 8 + wave * PB + q - PA) * 1024);
    dma16(raw_rsrc((of_a ? x : w) + skip, end), __builtin_amdgcn_readfirstlane(lds_to), c < left ? at : kNone, 0);
  };
  // Scales, eight bytes a row and stage, in a word more where rows begin at any byte; this
  // wave's are of x's rows or of the weights'.  The descriptor ends with the last row's last scale, in
  // whole words, of which each is held against it.
  const bool of_x = wave * PS < BM * WORDS * 4 / S::ONE;
  const unsigned char* const sbase = of_x ? xs : ws;
  const unsigned sodd = (unsigned)reinterpret_cast<uintptr_t>(sbase) & 3;
  const unsigned sld = (unsigned)(of_x ? p.ldxs : p.ldws);
  unsigned vs[PS];
#pragma unroll
  for (int q = 0; q < PS; ++q) {
    constexpr unsigned PIECES = WORDS * 256 / S::ONE;  // lanes of a row
    const unsigned at = (unsigned)((wave * PS + q) * 64 + lane) - (of_x ? 0 : BM * PIECES), row = at / PIECES;
    // WHOLE: every second eight rows have their two pieces the other way round, or four rows'
    // words would lie in one bank
    vs[q] = ((sodd + row * sld) & ~3u) + S::ONE / 64 * (WHOLE ? (at ^ row >> 3) & 1 : at - PIECES * row);
  }
  const unsigned send = (sodd + (unsigned)((of_x ? mrows : nrows) - 1) * sld + (unsigned)p.blocks_k + 3) & ~3u;
  // where the scales of stage s lie, whose buffer is `at`
  auto scales_at = [&](int s, unsigned char* at) {
    return SG == 1 ? at + (BM + BN) * 128 : lds + NB * S::STAGE + (s / SG & 1) * S::SCALES;
  };
  auto dma_scales = [&](int s, unsigned char* at, int q) {
    const unsigned skip = 8u * (unsigned)s;
    const i32x4 rs = raw_rsrc(sbase - sodd + skip, s < nk ? send - skip : 0u);
    const unsigned to = __builtin_amdgcn_readfirstlane(lds_at(scales_at(s, at) + (wave * PS + q) * S::ONE));
    if constexpr (WHOLE) dma16(rs, to, vs[q], 0);
    else dma4(rs, to, vs[q]);
  };

  const int xodd = odd_of(xs, lrow, p.ldxs), wodd = odd_of(ws, lrow, p.ldws);  // of rows 32 apart alike
  // a row's block 4 hi + ks lies at the place of its block 4 hi, less or more: its last bits
  // changed by ks; rows 32 apart have theirs at the same places
  const int arow = (wm * S::WM + lrow) * 128 + piece_of(lrow, 4 * hi) * 16;
  const int brow = S::AB + (wn * S::WN + lrow) * 128 + piece_of(lrow, 4 * hi) * 16;
  const int turned = WHOLE ? (lrow >> 3 & 1) * 16 : 0;
  const int xword = ((wm * S::WM + lrow) * WORDS * 4 + 4 * hi) ^ turned, wword = ((BM + wn * S::WN + lrow) * WORDS * 4 + 4 * hi) ^ turned;

  float16v acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;
  uint4v af[2][MI], bf[2][NI];
  unsigned raw[MI + NI][2];  // the next stage's scale words as they lie
  int sx[MI], sw[NI];        // this stage's, a byte a step
  auto read_a = [&](const unsigned char* at, int ks, int i) {
    af[ks & 1][i] = *reinterpret_cast<const uint4v*>(at + (ks * 16 ^ arow) + i * 4096);
  };
  auto read_b = [&](const unsigned char* at, int ks, int j) {
    bf[ks & 1][j] = *reinterpret_cast<const uint4v*>(at + (ks * 16 ^ brow) + j * 4096);
  };
  auto read_scale = [&](const unsigned char* at, int phase, int i) {  // of a stage whose group lies at `at`
    const int word = i < MI ? xword + i * 128 * WORDS : wword + (i - MI) * 128 * WORDS;
    const unsigned* const from = reinterpret_cast<const unsigned*>(at + (WHOLE ? word ^ 8 * phase : word + 8 * phase));
    raw[i][0] = from[0];
    raw[i][1] = WHOLE ? 0u : from[1];
  };
  auto take_scales = [&](int s) {
    // those past the row's end as 0: 255 would make NaN of the zeros there
    const int n = p.blocks_k - kBlocks * s - 4 * hi;
    const unsigned mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
#pragma unroll
    for (int i = 0; i < MI + NI; ++i) {
      const unsigned v = __builtin_amdgcn_alignbyte(raw[i][1], raw[i][0], i < MI ? xodd : wodd) & mask;
      if (i < MI) sx[i < MI ? i : 0] = (int)v;
      else sw[i < MI ? 0 : i - MI] = (int)v;
    }
  };
  auto mma = [&](int ks, int i, int j) {
    const int8w a = wide(bf[ks & 1][j]), c = wide(af[ks & 1][i]);
    float16v& d = acc[i][j];
    if (ks == 0) d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, c, d, 4, 4, 0, sw[j], 0, sx[i]);
    else if (ks == 1) d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, c, d, 4, 4, 1, sw[j], 1, sx[i]);
    else if (ks == 2) d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, c, d, 4, 4, 2, sw[j], 2, sx[i]);
    else d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, c, d, 4, 4, 3, sw[j], 3, sx[i]);
  };
  // Step ks: its MI NI products; behind product n issue(n), a DMA instruction or nothing,
  // and what the next step needs, the fragments that its first products take first.
  constexpr int PRODUCTS = S::PRODUCTS, EVERY = S::EVERY, HALF = S::HALF;
  auto step = [&](int ks, const unsigned char* at, int next, auto issue) {
#pragma unroll
    for (int n = 0; n < PRODUCTS; ++n) {
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MI == NI) {  // shells of the larger index
        const int k = n < 1 ? 0 : n < 4 ? 1 : n < 9 ? 2 : 3, r = n - k * k;
        mma(ks, r < k ? r : k, r < k ? k : r - k);
      } else {
        mma(ks, 2 * (n >> 2) + (n & 1), (n >> 1) & 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      issue(n);
      __builtin_amdgcn_sched_barrier(0);
      if (n < MI) read_a(at, next, n);
      if (n < NI) read_b(at, next, n);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto none = [](int) {};

  // prologue: as much as the buffers hold, of the last one half the data; WHOLE: before it the
  // scales of the first four stages and the first ones of the next
  if constexpr (WHOLE) {
#pragma unroll
    for (int q = 0; q < PS; ++q) dma_scales(0, lds, q);
    dma_scales(SG, lds, 0);
  }
#pragma unroll
  for (int s = 0; s < NB; ++s) {
#pragma unroll
    for (int q = 0; q < (s < NB - 1 ? S::PD : HALF); ++q) dma_one(s, lds + s * S::STAGE, q);
    if (!WHOLE && s < NB - 1) {
#pragma unroll
      for (int q = 0; q < PS; ++q) dma_scales(s, lds + s * S::STAGE, q);
    }
  }
  static_assert(WHOLE || SG == 1 || NB == 2, "the first wait leaves the second stage's data");
  XTK_WAIT_VM((NB - 2) * S::PER + HALF);
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int i = 0; i < MI; ++i) read_a(lds, 0, i);
#pragma unroll
  for (int j = 0; j < NI; ++j) read_b(lds, 0, j);
#pragma unroll
  for (int i = 0; i < MI + NI; ++i) read_scale(scales_at(0, lds), 0, i);
  take_scales(0);

  // stage s, of phase s % SG, in `at`, with `last` the buffer before it and `next` the one
  // behind it.  WHOLE: in the last step, behind whose barrier no wave reads the scales of the
  // group before this one, and before its data, so that a wait which leaves those leaves
  // none of them, part of the group behind the next stage's.
  auto stage = [&](int s, unsigned char* at, unsigned char* last, unsigned char* next, auto phase) {
    constexpr int PHASE = decltype(phase)::value, AFTER = (PHASE + 1) % SG;
    step(0, at, 1, [&](int n) {
      if (n % EVERY == 0) dma_one(s + NB - 1, last, HALF + n / EVERY);
    });
    step(1, at, 2, [&](int n) {
      if constexpr (SG == 1) {
        if (n < PS) dma_scales(s + NB - 1, last, n);
      } else if constexpr (SG == 2) {  // of the two stages from the next even one on, in two halves
        constexpr int FIRST = (PS + 1) / 2;
        if (PHASE == 0 && n < FIRST) dma_scales(s + 2, at, n);
        if (PHASE == 1 && n < PS - FIRST) dma_scales(s + 1, at, FIRST + n);
      }
    });
    step(2, at, 3, none);
    XTK_WAIT_VM((NB - 2) * S::PER);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const unsigned char* const scales = scales_at(s + 1, next);
    step(3, next, 0, [&](int n) {
      if constexpr (WHOLE && AFTER < PS)
        if (n == 0) dma_scales(s + 1 - AFTER + SG, at, AFTER);
      if (n % EVERY == 0) dma_one(s + NB, at, n / EVERY);
      if (n >= PRODUCTS - MI) {
        read_scale(scales, AFTER, n - (PRODUCTS - MI));
        if (n - (PRODUCTS - MI) < NI) read_scale(scales, AFTER, MI + n - (PRODUCTS - MI));
      }
    });
    take_scales(s + 1);
  };
  unsigned char *at = lds, *last = lds + (NB - 1) * S::STAGE;
  auto turn = [&](int s, auto phase) {
    unsigned char* const next = at == lds + (NB - 1) * S::STAGE ? lds : at + S::STAGE;
    stage(s, at, last, next, phase);
    last = at;
    at = next;
  };
#pragma unroll 1
  for (int s = 0; s < nk; s += SG) {
    turn(s, Phase<0>{});
    if constexpr (SG >= 2) {
      if (s + 1 < nk) turn(s + 1, Phase<1 % SG>{});
    }
    if constexpr (SG == 4) {
      if (s + 2 < nk) turn(s + 2, Phase<2>{});
      if (s + 3 < nk) turn(s + 3, Phase<3>{});
    }
  }
  XTK_WAIT_VM(0);

  // each wave's 32 rows at a time through a part of LDS of its own
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __syncthreads();
  static_assert(S::LDS >= NW * 32 * (S::WN * 4 + 16), "the waves' parts");
  unsigned char* const own = lds + wave * 32 * (S::WN * 4 + 16);
  const long long y0 = p.ty.at(bx, by, bz);
  auto leave = [&](auto zero) {
    typedef decltype(zero) T;
    constexpr int ES = sizeof(T), PER16 = 16 / ES, PITCH = S::WN * ES + 16, PIECES = S::WN / PER16;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          typedef T t4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<t4*>(own + lrow * PITCH + (32 * j + 8 * g + 4 * hi) * ES) =
              t4{(T)acc[i][j][4 * g], (T)acc[i][j][4 * g + 1], (T)acc[i][j][4 * g + 2], (T)acc[i][j][4 * g + 3]};
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own writes
#pragma unroll
      for (int e = lane; e < 32 * PIECES; e += 64) {
        const int r = e / PIECES, c = e % PIECES;
        const int m = m0 + wm * S::WM + 32 * i + r, n = n0 + wn * S::WN + c * PER16;
        if (m >= p.M || n >= p.N) continue;
        const T* const from = reinterpret_cast<const T*>(own + r * PITCH + c * 16);
        T* const to = static_cast<T*>(p.y) + y0 + m * p.ldy + n;
        if (n + PER16 <= p.N) {
          typedef unsigned u4e __attribute__((ext_vector_type(4), aligned(2)));
          *reinterpret_cast<u4e*>(to) = (u4e)(*reinterpret_cast<const uint4v*>(from));
        } else {
          for (int k = 0; k < p.N - n; ++k) to[k] = from[k];
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  };
  if (p.y_elem == kF32) leave(0.0f);
  else if (p.y_elem == kF16) leave((_Float16)0);
  else leave((__bf16)0.0f);
}

template <int BM, int BN, int NW, int NB>
bool run_many(Mx4Args& a, long long blocks, hipStream_t s) {
  const long long mt = (a.M + BM - 1) / BM, nt = (a.N + BN - 1) / BN, tiles = mt * nt;
  if (tiles > 0x7fffffffLL || !grid_fits(tiles * blocks, 64 * NW)) return false;
  a.tiles = static_cast<int>(tiles);
  a.mtiles = static_cast<int>(mt);
  a.ntiles = static_cast<int>(nt);
  a.nwg = static_cast<int>(tiles * blocks);
  a.group = static_cast<int>(std::min(nt, 8LL));
  a.d_tiles = div31(a.tiles);
  a.d_group = div31(a.group * a.mtiles);
  a.d_width = div31(a.group);
  a.d_last = div31(a.ntiles % a.group ? a.ntiles % a.group : a.group);
  if (a.whole) matmul_mx4_many_kernel<BM, BN, NW, NB, true><<<a.nwg, 64 * NW, 0, s>>>(a);
  else matmul_mx4_many_kernel<BM, BN, NW, NB, false><<<a.nwg, 64 * NW, 0, s>>>(a);
  return true;
}

// The kernel by estimated time, in us, fitted to graph replays of 34 products from 1 x 840 x
// 1696 to 4096 x 11008 x 4096: a round of tiles costs its start and end and its stages; a
// wave of few and mid tiles has a W-th of them.  (Measured: 64 x 4096 x 4096 in tiles of 16 x
// 16 8.5 us, 32 x 32 6.6, 64 x 64 10.2; 256 x 4096 x 4096 in 32 x 64 14.8, 64 x 64 11.9, 128
// x 128 15.4; 512 x 11008 x 4096 in 128 x 128 with three buffers 29.4, with two and twice
// the workgroups on a CU 24.8, in 256 x 256 34.1; 1024 x 11008 x 4096 in 128 x 128 41.7, in
// 256 x 256 36.1.)
bool run(Mx4Args& a, long long blocks, hipStream_t s) {
  const int stages = (a.blocks_k + kBlocks - 1) / kBlocks;
  auto tiles = [&](int bm, int bn) { return double(blocks) * double((a.M + bm - 1) / bm) * double((a.N + bn - 1) / bn); };
  auto share = [&](int waves) { return double((stages + waves - 1) / waves); };
  auto rounds = [](double t, int at_once) { return std::ceil(t / at_once); };
  // more workgroups than two a CU: four waves each, of which four fit on one
  const double small = tiles(16, 16);
  const bool eight = small <= 512;
  const double by_16 = 2.2 + (eight ? std::max(1.0 + 0.9 * share(8), small / 256 * (0.5 + 0.78 * share(8)))
                                    : std::max(1.0 + 0.55 * share(4), small / 256 * (0.37 + 0.3 * share(4))));
  double us[7] = {by_16,
                  2.4 + rounds(tiles(32, 32), 256) * (2.0 + 0.95 * share(8)),
                  2.3 + rounds(tiles(32, 64), 256) * (2.3 + 0.95 * share(4)),
                  2.5 + rounds(tiles(64, 64), 256) * (3.9 + 1.35 * share(4)),
                  2.0 + rounds(tiles(128, 128), 256) * (2.5 + (a.whole ? 0.82 : 1.0) * stages),
                  2.0 + rounds(tiles(128, 128), 512) * (2.2 + (a.whole ? 1.28 : 1.35) * stages),
                  2.0 + rounds(tiles(256, 256), 256) * (4.0 + (a.whole ? 1.95 : 2.2) * stages)};
  // large tiles take their rows by DMA only
  const int kernels = a.dma ? 7 : 4;
  auto launch = [&](int kernel) {
    switch (kernel) {
      case 0:
        if (a.M <= 8) return eight ? run_few<8, 8>(a, blocks, s) : run_few<8, 4>(a, blocks, s);
        return eight ? run_few<16, 8>(a, blocks, s) : run_few<16, 4>(a, blocks, s);
      case 1: return run_mid<1, 1, 8>(a, blocks, s);
      case 2: return run_mid<1, 2, 4>(a, blocks, s);
      case 3: return run_mid<2, 2, 4>(a, blocks, s);
      case 4: return run_many<128, 128, 4, 3>(a, blocks, s);
      case 5: return run_many<128, 128, 4, 2>(a, blocks, s);
      default: return run_many<256, 256, 8, 2>(a, blocks, s);
    }
  };
  // the next where one's tiles exceed a launch
  for (int i = 0; i < kernels; ++i) {
    double* const least = std::min_element(us, us + kernels);
    if (launch(static_cast<int>(least - us))) return true;
    *least = HUGE_VAL;
  }
  return false;
}

}  // namespace

hipError_t launch_matmul_mx4(const xt::Plan& p, void* const* bufs, hipStream_t s, std::string& why) {
  const xt::Mx4Plan& m = p.mx4;
  for (const xt::Access2D* in : {&m.x, &m.xs, &m.w, &m.ws})
    if (!result_apart(p, bufs, m.y, *in, false, why)) return hipErrorInvalidValue;
  auto off = [](const xt::Access2D& a) { return TileOff{a.addr.c0, a.addr.sx, a.addr.sy, a.addr.sz}; };
  auto at = [&](const xt::Access2D& a) { return static_cast<const unsigned char*>(bufs[a.arg]); };
  Mx4Args a{};
  a.x = at(m.x);
  a.xs = at(m.xs);
  a.w = at(m.w);
  a.ws = at(m.ws);
  a.y = bufs[m.y.arg];
  a.tx = off(m.x);
  a.txs = off(m.xs);
  a.tw = off(m.w);
  a.tws = off(m.ws);
  a.ty = off(m.y);
  a.ldx = m.x.ld;
  a.ldxs = m.xs.ld;
  a.ldw = m.w.ld;
  a.ldws = m.ws.ld;
  a.ldy = m.y.ld;
  a.blocks = block_decode(p.grid[0], p.grid[1], false);
  a.M = static_cast<int>(m.y.rows);
  a.N = static_cast<int>(m.y.cols);
  a.blocks_k = static_cast<int>(m.K / 32);
  a.y_elem = m.y.elem == xt::Elem::F32 ? kF32 : m.y.elem == xt::Elem::F16 ? kF16 : kBF16;
  // DMA takes rows of whole 16 bytes; others go through registers
  auto pieces = [&](const xt::Access2D& t, int of) {
    const xt::TileAddr& d = t.addr;
    return reinterpret_cast<uintptr_t>(bufs[t.arg]) % of == 0 && t.ld % of == 0 && d.c0 % of == 0 && d.sx % of == 0 &&
           d.sy % of == 0 && d.sz % of == 0;
  };
  a.dma = pieces(m.x, 16) && pieces(m.w, 16);
  a.whole = pieces(m.xs, 4) && pieces(m.ws, 4);
  // what a lane adds to its tile's address has 31 bits
  auto near = [](long long rows, long long ld) { return rows * ld + 256 < (1LL << 31); };
  const int mr = std::min(a.M, 256), nr = std::min(a.N, 256);
  if (!near(mr, a.ldx) || !near(mr, a.ldxs) || !near(nr, a.ldw) || !near(nr, a.ldws)) {
    why = "matmul_mx4: rows that a workgroup reads together span 2^31 bytes or more";
    return hipErrorInvalidValue;
  }
  const long long blocks = grid_blocks(p);
  const bool ok = run(a, blocks, s);
  if (!ok) {
    why = "matmul_mx4: " + std::to_string(a.M) + " x " + std::to_string(a.N) + " tiles exceed one launch";
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace xtk
