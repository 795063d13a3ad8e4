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
  int tiles, ntiles;
  int M, N, blocks_k;  // blocks of 32 of a row
  int dma;
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

// Three words of 21 rows' scales that one instruction brings (lane 3 r + i: word i of row
// first + r), at most `count` of them.  Rows begin at any byte: a word that holds none of
// the eight bytes, or none of a row's, is not read.
struct Scales {
  unsigned off;  // of the word, less the bytes before it
  int before;    // bytes of the word before the row's first
  __device__ __forceinline__ void begin(const unsigned char* base, int first, int count, int rows, long long ld) {
    const int lane = threadIdx.x & 63, r = lane / 3, i = lane - 3 * r, row = first + r;
    const unsigned at = (unsigned)row * (unsigned)ld, odd = ((unsigned)reinterpret_cast<uintptr_t>(base) + at) & 3;
    before = (int)odd - 4 * i;
    off = r < count && row < rows && before > -kBlocks ? at - (unsigned)before : kNone;
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

// Few rows of x: a workgroup has 16 rows of weights and 16 MT of x, its W waves split K in
// stages, each in a ring of its own, and meet once, in LDS, in a fixed order.
// XR: rows of x in LDS (8, of which the MFMA's 16 are the same ones twice, or 16 MT).
template <int MT, int XR, int W, int NS>
struct FewShape {
  static constexpr int X0 = 2048, S0 = X0 + XR * 128, STAGE = S0 + 256 * (1 + MT);
  static constexpr int XI = XR / 8, PER = 2 + XI + 1 + MT;  // instructions of a stage
  static constexpr int LDS = W * NS * STAGE;
  static_assert(LDS <= 160 * 1024 && (NS - 1) * PER < 64 && W * MT * 1024 <= LDS, "");
};

template <int MT, int XR, int W, int NS>
__global__ __launch_bounds__(64 * W) void matmul_mx4_few_kernel(Mx4Args p) {
  typedef FewShape<MT, XR, W, NS> S;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[S::LDS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int b = (int)p.d_tiles(blockIdx.x);
  const int tile = blockIdx.x - b * p.tiles;
  const int tm = (int)p.d_nt(tile), tn = tile - tm * p.ntiles;
  int bx, by, bz;
  p.blocks(b, bx, by, bz);
  const int m0 = tm * 16 * MT, n0 = tn * 16, mrows = p.M - m0, nrows = p.N - n0;
  const unsigned char* const w = p.w + p.tw.at(bx, by, bz) + n0 * p.ldw;
  const unsigned char* const ws = p.ws + p.tws.at(bx, by, bz) + n0 * p.ldws;
  const unsigned char* const x = p.x + p.tx.at(bx, by, bz) + m0 * p.ldx;
  const unsigned char* const xs = p.xs + p.txs.at(bx, by, bz) + m0 * p.ldxs;

  Pieces pw[2], px[S::XI];
  Scales sw, sx[MT];
#pragma unroll
  for (int i = 0; i < 2; ++i) pw[i].begin(8 * i, nrows, p.ldw);
#pragma unroll
  for (int i = 0; i < S::XI; ++i) px[i].begin(8 * i, mrows, p.ldx);
  sw.begin(ws, 0, 16, nrows, p.ldws);
#pragma unroll
  for (int i = 0; i < MT; ++i) sx[i].begin(xs, 16 * i, 16, mrows, p.ldxs);
  unsigned char* const ring = lds + wave * NS * S::STAGE;
  auto issue = [&](int c, int slot) {
    unsigned char* const at = ring + slot * S::STAGE;
    const int left = p.blocks_k - c * kBlocks;
    const long long d = (long long)c * 128;
#pragma unroll
    for (int i = 0; i < 2; ++i) pw[i].issue(p.dma, w + d, left, at + 1024 * i);
#pragma unroll
    for (int i = 0; i < S::XI; ++i) px[i].issue(p.dma, x + d, left, at + S::X0 + 1024 * i);
    sw.issue(ws + c * kBlocks, left, at + S::S0);
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i].issue(xs + c * kBlocks, left, at + S::S0 + 256 * (1 + i));
  };

  float4v y[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) y[i] = float4v{0, 0, 0, 0};
  const int stages = (p.blocks_k + kBlocks - 1) / kBlocks, mine = max(0, (stages - wave + W - 1) / W);
#pragma unroll
  for (int j = 0; j < NS; ++j)
    if (j < mine) issue(wave + j * W, j);
  // this lane's row of each operand: where it lies, and its scales' first byte
  const int xrow = XR < 16 ? col % XR : col;
  const int wodd = odd_of(ws, col, p.ldws);
  int xodd[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xodd[i] = odd_of(xs, 16 * i + xrow, p.ldxs);
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
    const int left = p.blocks_k - (wave + j * W) * kBlocks;
    const unsigned char* const at = ring + slot * S::STAGE;
    // MFMA i has blocks 2 g + i; a lane's two scale bytes are moved to the low half
    uint4v wf[2], xf[MT][2];
    int sc[1 + MT];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      wf[i] = *reinterpret_cast<const uint4v*>(at + col * 128 + piece_of(col, 2 * g + i) * 16);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int row = XR < 16 ? xrow : 16 * t + col;
        xf[t][i] = *reinterpret_cast<const uint4v*>(at + S::X0 + row * 128 + piece_of(row, 2 * g + i) * 16);
      }
    }
    sc[0] = scale_word(at + S::S0 + col * 12, g >> 1, wodd, left) >> (16 * (g & 1));
#pragma unroll
    for (int t = 0; t < MT; ++t)
      sc[1 + t] = scale_word(at + S::S0 + 256 * (1 + t) + xrow * 12, g >> 1, xodd[t], left) >> (16 * (g & 1));
    // every fragment is in registers before the slot is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (j + NS < mine) issue(wave + (j + NS) * W, slot);
    slot = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      y[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(xf[t][0]), wide(wf[0]), y[t], 4, 4, 0, sc[1 + t], 0, sc[0]);
      y[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(xf[t][1]), wide(wf[1]), y[t], 4, 4, 1, sc[1 + t], 1, sc[0]);
    }
  }
  __syncthreads();  // every ring is done with

  // the waves' parts, summed in the order of the waves
  float* const part = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[((wave * MT + i) * 4 + r) * 64 + lane] = y[i][r];
  __syncthreads();
  const long long y0 = p.ty.at(bx, by, bz);
  for (int e = threadIdx.x; e < MT * 256; e += 64 * W) {
    const int i = e >> 8, r = (e >> 6) & 3, l = e & 63;
    const int m = m0 + 16 * i + 4 * (l >> 4) + r, n = n0 + (l & 15);
    if (m >= p.M || n >= p.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int u = 0; u < W; ++u) v += part[u * MT * 256 + e];
    put(p.y, p.y_elem, y0 + m * p.ldy + n, v);
  }
}

template <int MT, int XR, int W, int NS>
bool run_few(Mx4Args& a, long long blocks, hipStream_t s) {
  const long long nt = (a.N + 15) / 16, tiles = nt * ((a.M + 16 * MT - 1) / (16 * MT));
  if (tiles > 0x7fffffffLL || !grid_fits(tiles * blocks, 64 * W)) return false;
  a.tiles = static_cast<int>(tiles);
  a.ntiles = static_cast<int>(nt);
  a.d_tiles = div31(a.tiles);
  a.d_nt = div31(a.ntiles);
  matmul_mx4_few_kernel<MT, XR, W, NS><<<static_cast<unsigned>(tiles * blocks), 64 * W, 0, s>>>(a);
  return true;
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
  auto pieces = [&](const xt::Access2D& t) {
    const xt::TileAddr& d = t.addr;
    return reinterpret_cast<uintptr_t>(bufs[t.arg]) % 16 == 0 && t.ld % 16 == 0 && d.c0 % 16 == 0 && d.sx % 16 == 0 &&
           d.sy % 16 == 0 && d.sz % 16 == 0;
  };
  a.dma = pieces(m.x) && pieces(m.w);
  // what a lane adds to its tile's address has 31 bits
  auto near = [](long long rows, long long ld) { return rows * ld + 256 < (1LL << 31); };
  const int mr = std::min(a.M, 64), nr = std::min(a.N, 16);
  if (!near(mr, a.ldx) || !near(mr, a.ldxs) || !near(nr, a.ldw) || !near(nr, a.ldws)) {
    why = "matmul_mx4: rows that a workgroup reads together span 2^31 bytes or more";
    return hipErrorInvalidValue;
  }
  const long long blocks = grid_blocks(p);
  const bool ok = a.M <= 8    ? run_few<1, 8, 8, 2>(a, blocks, s)
                  : a.M <= 16 ? run_few<1, 16, 8, 2>(a, blocks, s)
                  : a.M <= 32 ? run_few<2, 32, 8, 2>(a, blocks, s)
                              : run_few<4, 64, 4, 2>(a, blocks, s);
  if (!ok) {
    why = "matmul_mx4: " + std::to_string(a.M) + " x " + std::to_string(a.N) + " tiles exceed one launch";
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace xtk
