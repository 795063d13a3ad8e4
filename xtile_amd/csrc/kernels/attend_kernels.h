// The attention kernels: see attend.hip for the mathematics and the choices.
#pragma once

#include "common.h"

namespace xtk {

// Element offset of a Block's tile from the argument's first one: the pointers start
// at that, and every step is at least 0.
struct Walk {
  unsigned long long sx, sy, sz;
  __device__ __forceinline__ unsigned long long at(unsigned x, unsigned y, unsigned z) const {
    return x * sx + y * sy + z * sz;
  }
};

struct AttendArgs {
  const unsigned char* q;
  const unsigned char* k;
  const unsigned char* v;
  unsigned char* o;
  const float* slopes;
  const int *start, *length, *prefix, *qdocs, *kdocs;
  Walk tq, tk, tv, to, tslopes, tstart, tlength, tprefix, tqdocs, tkdocs;
  long long q_head, q_row, o_head, o_row, ldk, ldv, slope_step, qdoc_step;   // strides in elements
  BlockDecode blocks;
  Div31 d_heads, d_work, d_splits;  // d_work: row tiles x splits of a Block
  int heads, rows, keys;            // rows: query rows of a Block, heads x tokens
  int tiles, splits, nwg;
  float scale_log2;  // scale * log2 e, what the products are multiplied by without a cap
  float cap_in, cap_log2;  // 2 scale log2 e / cap and cap * log2 e; cap_log2 0: no cap
  // Products of at most cap_near take cap_poly (attend.hip); a tile of none above it does,
  // and one of others takes the exponential, or, by FINE kernels, what each score asks for.
  float cap_near, cap_poly[4];
  int causal, window, dma;
  float* work;
};

// For kernels that choose for each score: the polynomial is in (mul s)^2.  An argument of
// its own, behind the others: in their midst it moves the scalar registers of every kernel
// (causal, 64 columns: 49 us -> 52).
struct FineCap {
  float mul;
};

// attend_*.hip, one instantiation each for d of 32, 64, ... 256; fine: null for none.
template <int D>
hipError_t run_attend(bool bf16, bool few, const AttendArgs& a, const FineCap* fine, hipStream_t s);

}  // namespace xtk

#ifdef XTK_ATTEND_KERNELS

#include "launch.h"

namespace xtk {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) unsigned char lds_t;
typedef unsigned u4a __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u2a __attribute__((ext_vector_type(2), aligned(2)));

constexpr int kFar = 1 << 30;  // positions are held within this
// Weights may reach 2^kSlack times that of the largest score that the sums are relative to.
// In half precision they are held 2^kRaise times larger: at most 2^15, and what is lost
// begins at 2^-32 of the largest instead of 2^-25, of which a long row may have enough to matter.
constexpr float kSlack = 8.0f, kRaise = 7.0f;

// The LDS address of a pointer into LDS: the low half of its generic address (a cast
// between address spaces compares with null first).
__device__ __forceinline__ unsigned lds_at(const void* p) { return (unsigned)reinterpret_cast<uintptr_t>(p); }

// Four bytes a lane into LDS by DMA; as dma16.
__device__ __forceinline__ void dma4(i32x4 rsrc, unsigned lds, unsigned voff) {
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" : : "v"(voff), "s"(rsrc), "{m0}"(lds) : "memory");
}

__device__ __forceinline__ float both_halves(float v, bool is_max) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const float a = __builtin_bit_cast(float, (unsigned)r[0]), b = __builtin_bit_cast(float, (unsigned)r[1]);
  return is_max ? fmaxf(a, b) : a + b;
}

template <bool BF16>
__device__ __forceinline__ float16v mma(uint4v a, uint4v b, float16v c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// l + the sum of a packed pair.
template <bool BF16>
__device__ __forceinline__ float add_pair(unsigned w, float l) {
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), __builtin_bit_cast(b2, 0x3f803f80u), l, false);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), __builtin_bit_cast(h2, 0x3c003c00u), l, false);
  }
}

// The capped score, in units of log2, of a product s within cap_near (w: its square,
// times mul^2), of a larger one, and of any.
__device__ __forceinline__ float capped_near(const AttendArgs& p, float s, float w) {
  return s * fmaf(w, fmaf(w, fmaf(w, p.cap_poly[3], p.cap_poly[2]), p.cap_poly[1]), p.cap_poly[0]);
}
__device__ __forceinline__ float capped_far(const AttendArgs& p, float s) {
  return fmaf(-2.0f * p.cap_log2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * p.cap_in) + 1.0f), p.cap_log2);
}
__device__ __forceinline__ float capped(const AttendArgs& p, const FineCap& c, float s) {
  const float z = s * c.mul;
  return fabsf(s) <= p.cap_near ? capped_near(p, s, z * z) : capped_far(p, s);
}

template <bool BF16>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, b2{(__bf16)a, (__bf16)b});
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, h2{(_Float16)a, (_Float16)b});
  }
}

// The last key that a window hides from a row at pos: -1 for none, or without windows.
__device__ __forceinline__ int before(const AttendArgs& p, int window, int pos) {
  return !p.window || pos < window ? -1 : pos - window;
}

// What one wave's 32 query rows see, and its running softmax.  Lane (c = lane % 32,
// h = lane / 32) holds row c; of a tile of 32 keys it holds the scores of keys
// 8 (r / 4) + 4 h + r % 4 in register r, and of the result columns
// 32 n + 8 (r / 4) + 4 h + r % 4 in register r of acc[n].
// FINE: the cap looks at each score.
template <int D, bool BF16, bool FINE = false>
struct Rows {
  static constexpr int N = D / 32, KK = D / 16;
  static constexpr int PITCH = 2 * D;  // bytes of a key row in LDS
  static constexpr int VAHEAD = D < 128 ? 2 : 1;  // steps of 16 keys whose values are read ahead

  // Where a key row's 16-byte chunks lie in LDS: chunk c at c ^ ksw (keys), c ^ vsw
  // (values), so that the 16 rows of a fragment read, and the four rows of a
  // transposing read, fall into distinct banks for every D.
  static __device__ __forceinline__ int ksw(int row) {
    return D % 128 == 0 ? row & 15 : D % 64 == 0 ? (row >> 1) & 7 : (row >> 2) & 3;
  }
  static __device__ __forceinline__ int vsw(int row) {
    return D % 128 == 0 ? 4 * (row & 3) : D % 64 == 0 ? 4 * ((row >> 1) & 1) : 0;
  }

  int lane, col, hi;
  int row, token;        // this lane's row of the Block (the last one past the end) and its token
  int pos, above, below; // sees key j when below < j <= above (or j < prefix)
  int p0, p1;            // positions of the wave's first and last row
  int w0, w1;            // the last keys before their windows
  float slope;           // times log2 e
  int doc;               // this lane's document
  uint4v q[KK];
  float16v acc[N];
  float m, l;
  // LDS offsets of this lane's part of a key and of a value fragment, for each step;
  // the widest heads, short of registers, keep one of a key row and work out the rest
  static constexpr bool LEAN = D == 256;
  int koff[LEAN ? 1 : KK], voff[N];

  __device__ __forceinline__ void begin(const AttendArgs& p, int first, int bx, int by, int bz, int start, int window) {
    lane = threadIdx.x & 63;
    col = lane & 31;
    hi = lane >> 5;
    row = min(first + col, p.rows - 1);
    token = (int)p.d_heads((unsigned)row);
    const int head = row - token * p.heads;
    pos = start + token;
    p0 = start + (int)p.d_heads((unsigned)min(first, p.rows - 1));
    p1 = start + (int)p.d_heads((unsigned)min(first + 31, p.rows - 1));
    above = p.causal ? min(pos, kFar) : kFar;
    below = before(p, window, pos);
    w0 = before(p, window, p0);
    w1 = before(p, window, p1);
    slope = p.slopes ? p.slopes[p.tslopes.at(bx, by, bz) + head * p.slope_step] * 1.44269504088896340736f : 0.0f;
    doc = p.qdocs ? p.qdocs[p.tqdocs.at(bx, by, bz) + token * p.qdoc_step] : 0;
    const unsigned char* at = p.q + (p.tq.at(bx, by, bz) + head * p.q_head + token * p.q_row + 8 * hi) * 2;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) q[kk] = (uint4v)(*reinterpret_cast<const u4a*>(at + kk * 32));
    reset();
    const int g = lane >> 4, li = lane & 15;
    const int key = 4 * hi + (li >> 2), chunk = 2 * (g & 1) + ((li & 3) >> 1);
#pragma unroll
    for (int n = 0; n < N; ++n) voff[n] = key * PITCH + ((((chunk ^ vsw(key)) << 4) + 8 * (li & 1)) ^ (n << 6));
#pragma unroll
    for (int kk = 0; kk < (LEAN ? 1 : KK); ++kk) koff[kk] = col * PITCH + (((2 * kk + hi) ^ ksw(col)) << 4);
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][r] = 0.0f;
    m = -__builtin_inff();
    l = 0.0f;
  }

  // Behind a loop: the sums as they are, or the loop would copy them to the registers
  // that what follows wants them in, once a tile.
  __device__ __forceinline__ void hold() {
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("" : "+v"(acc[n]));
  }

  __device__ __forceinline__ uint4v key_fragment(const unsigned char* K, int kt, int kk) const {
    if constexpr (LEAN) {
      int at = koff[0];
      asm volatile("" : "+v"(at));
      return *reinterpret_cast<const uint4v*>(K + (at ^ (kk << 5)) + kt * 32 * PITCH);
    }
    return *reinterpret_cast<const uint4v*>(K + koff[LEAN ? 0 : kk] + kt * 32 * PITCH);
  }

  // Values of keys 32 kt + 16 u + {4 h + 0..3, 8 + 4 h + 0..3}, column 32 n + c.
  __device__ __forceinline__ uint4v value_fragment(const unsigned char* V, int kt, int u, int n) const {
    lds_t* const f = (lds_t*)lds_at(V + voff[n] + (kt * 32 + u * 16) * PITCH);
    const uint2v lo = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                     reinterpret_cast<short4v __attribute__((address_space(3)))*>(f)));
    const uint2v up = __builtin_bit_cast(
        uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    reinterpret_cast<short4v __attribute__((address_space(3)))*>(f + 8 * PITCH)));
    return uint4v{lo[0], lo[1], up[0], up[1]};
  }

  // Whether the wave's rows see all of keys [key0, key0 + n), documents aside, or none.
  __device__ __forceinline__ bool sees_all(const AttendArgs& p, int key0, int n, int len, int pre) const {
    return key0 + n <= len && (key0 + n <= pre || ((!p.causal || key0 + n - 1 <= p0) && key0 > w1));
  }
  __device__ __forceinline__ bool sees_none(const AttendArgs& p, int key0, int n, int pre) const {
    return key0 >= pre && ((p.causal && key0 > p1) || key0 + n - 1 <= w0);
  }

  // Of a lane's 16 registers of a tile of 32 keys, as bits, those whose key is at most
  // x past the lane's first: register r holds key 8 (r / 4) + r % 4.
  static __device__ __forceinline__ unsigned up_to(int x) {
    const int y = min(max(x, -1), 31);
    return (1u << (4 * (y >> 3) + min((y & 7) + 1, 4))) - 1u;  // -1: 4 (-1) + 4
  }

  __device__ __forceinline__ int doc_of(const int* docs, const int* kdocs, int t, int i, int base, int len) const {
    if (docs) return docs[t * 32 + 4 * hi + i];
    return base + i < len ? kdocs[base + i] : 0;
  }

  // T tiles of 32 keys from key0 on.  docs: their documents in LDS, or null, then from
  // kdocs.
  template <int T>
  __device__ __forceinline__ void tile(const AttendArgs& p, const FineCap& c, const unsigned char* K, const unsigned char* V,
                                       const int* docs, const int* kdocs, int key0, int len, int pre) {
    bool part = !sees_all(p, key0, 32 * T, len, pre);
    bool by_doc = false, by_key = false;  // rows, or keys, of several documents
    int tile_doc = 0;
    if (kdocs) {
      const int i = key0 + (lane & (32 * T - 1));
      const int d = docs ? docs[lane & (32 * T - 1)] : i < len ? kdocs[i] : 0;
      tile_doc = __builtin_amdgcn_readfirstlane(d);
      by_key = __builtin_amdgcn_ballot_w64(i < len && d != tile_doc) != 0;
      if (!by_key) {
        const unsigned long long same = __builtin_amdgcn_ballot_w64(doc == tile_doc);
        if (same == 0) return;
        by_doc = ~same != 0;
      }
      part |= by_doc || by_key;
    }

    float16v s[T];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = 0.0f;
    // fragments AHEAD steps before their products: one LDS read takes longer than a
    // step's products, and the scheduler would read each just before its use
    constexpr int AHEAD = KK < 4 ? KK : 4;
    uint4v kf[AHEAD][T];
#pragma unroll
    for (int kk = 0; kk < AHEAD; ++kk)
#pragma unroll
      for (int t = 0; t < T; ++t) kf[kk][t] = key_fragment(K, t, kk);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
      for (int t = 0; t < T; ++t) s[t] = mma<BF16>(kf[kk % AHEAD][t], q[kk], s[t]);
      if (kk + AHEAD < KK) {
#pragma unroll
        for (int t = 0; t < T; ++t) kf[kk % AHEAD][t] = key_fragment(K, t, kk + AHEAD);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // the values of the first products, read behind the scores' arithmetic
    uint4v vf[VAHEAD][N];
#pragma unroll
    for (int x = 0; x < VAHEAD; ++x)
#pragma unroll
      for (int n = 0; n < N; ++n) vf[x][n] = value_fragment(V, 0, x, n);
    __builtin_amdgcn_sched_barrier(0);

    float mul = p.scale_log2;
    if (FINE || p.cap_log2 > 0.0f) {
      float big[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) big[r & 3] = fmaxf(big[r & 3], fabsf(s[t][r]));
      const float most = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
      mul = 1.0f;
      if (__builtin_amdgcn_ballot_w64(most > p.cap_near) == 0) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float z = FINE ? s[t][r] * c.mul : s[t][r];
            s[t][r] = capped_near(p, s[t][r], z * z);
          }
      } else {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = FINE ? capped(p, c, s[t][r]) : capped_far(p, s[t][r]);
      }
    }
    if (p.slopes) {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const float away = (float)(pos - (key0 + t * 32 + 4 * hi));
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[t][r] = fmaf(-slope, fabsf(away - (float)(8 * (r >> 2) + (r & 3))), s[t][r] * mul);
      }
      mul = 1.0f;
    }
    if (part) {
      unsigned seen[T];  // bit r for register r
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const int base = key0 + t * 32 + 4 * hi;
        unsigned bits = ((up_to(above - base) & ~up_to(below - base)) | up_to(pre - 1 - base)) & up_to(len - 1 - base);
        if (by_doc && doc != tile_doc) bits = 0;
        if (by_key) {
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              bits &= ~((doc_of(docs, kdocs, t, 8 * w + e, base, len) != doc ? 1u : 0u) << (4 * w + e));
        }
        seen[t] = bits;
      }
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {  // -inf where the bit is clear
          const unsigned keep = (unsigned)((int)(seen[t] << (31 - r)) >> 31);
          const float x = s[t][r];  // a bit cast of the element itself would read element 0
          s[t][r] = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, x) & keep) | (~keep & 0xff800000u));
        }
    }

    // the running maximum, in units of log2; four chains, since each step waits for the last
    float most[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) most[r & 3] = fmaxf(most[r & 3], s[t][r]);
    float top = both_halves(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), true) * mul;
    if constexpr (!BF16) top -= kRaise;  // and so m is, wherever it goes with l and the sums
    // weights may reach 2^kSlack: the sums are rescaled only where a row's maximum
    // has grown by more (most tiles of a long row raise some row's by a little)
    if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0) {
      const float now = fmaxf(m, top);
      const float alpha = __builtin_amdgcn_exp2f(m - (now == -__builtin_inff() ? 0.0f : now));
      m = now;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[n][r] *= alpha;
    }
    add_values<T>(V, s, vf, mul);
  }

  // Whether a value may have spoilt a row's sums: a weight of 0, of a key that the row does
  // not see or by rounding, times an infinity or NaN is NaN, and stays; and a weight above
  // one, between rescalings, may take a value near the largest past it.  (Infinities that
  // belong in the result look alike; odd_rows, which does such rows again, tells them apart.
  // Where the total is not finite either, the row's own scores are not.)
  __device__ __forceinline__ bool spoilt() const {
    float t = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) t = fmaf(acc[n][r], 0.0f, t);
    return __builtin_amdgcn_ballot_w64(t != 0.0f && l - l == 0.0f) != 0;
  }

  // Weights e^(score - m), rounded to the values' type (off by half a step each, as
  // the result is), and their products with the values; l takes the rounded weights,
  // so that a row's weights sum to one.  vf: the values of the first VAHEAD steps.
  template <int T>
  __device__ __forceinline__ void add_values(const unsigned char* V, float16v (&s)[T], uint4v (&vf)[VAHEAD][N], float mul) {
    const float use = m == -__builtin_inff() ? 0.0f : m;
    uint4v w[T][2];
    auto weigh = [&](int t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], mul, -use));
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[t][u][e] = pack2<BF16>(s[t][8 * u + 2 * e], s[t][8 * u + 2 * e + 1]);
          l = add_pair<BF16>(w[t][u][e], l);
        }
    };
    weigh(0);
    // ahead of the other wave of the SIMD: its arithmetic fills the matrix unit's time
    // (causal, 4096 tokens, 32 heads of 128, capped: 210 -> 188 us)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      // the next tile's weights between this one's products
      if (t + 1 < T) weigh(t + 1);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int x = 2 * t + u;
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] = mma<BF16>(vf[x % VAHEAD][n], w[t][u], acc[n]);
        if (x + VAHEAD < 2 * T) {
#pragma unroll
          for (int n = 0; n < N; ++n) vf[x % VAHEAD][n] = value_fragment(V, (x + VAHEAD) / 2, (x + VAHEAD) % 2, n);
        }
      }
      if (t + 1 < T) {
#pragma unroll
        for (int x = 0; x < 2 * N; ++x) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                // a product,
          __builtin_amdgcn_sched_group_barrier(0x402, 48 / (2 * N) + 1, 0);  // its share of the arithmetic
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);                // and of the reads
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
};

// The tiles of BN keys that a workgroup's rows may see: tiles [a0, a0 + na) of the
// prefix, then [b0, b0 + nb).
struct Tiles {
  int a0, na, b0, n;
  __device__ __forceinline__ int at(int i) const { return i < na ? a0 + i : b0 + (i - na); }
};

// p0, p1: the workgroup's first and last position; [d0, d1): the keys whose
// documents may be its rows'.
__device__ __forceinline__ Tiles tiles_of(const AttendArgs& p, int bn, int p0, int p1, int window, int len, int pre, int d0,
                                          int d1) {
  const int b0 = max(before(p, window, p0) + 1, d0);
  const int b1 = min(p.causal ? min(len, max(p1, -1) + 1) : len, d1);
  const int a1 = min(pre, d1);
  Tiles t;
  t.a0 = d0 / bn;
  t.na = a1 > d0 ? (a1 + bn - 1) / bn - t.a0 : 0;
  t.b0 = max(b0 / bn, t.na ? t.a0 + t.na : 0);
  t.n = t.na + (b1 > b0 ? max(0, (b1 + bn - 1) / bn - t.b0) : 0);
  return t;
}

// The smallest (or largest) over a wave, in every lane: wave_reduce for integers.
template <bool IS_MAX>
__device__ __forceinline__ int wave_extreme(int v) {
  constexpr int id = IS_MAX ? -0x7fffffff - 1 : 0x7fffffff;
  auto op = [](int a, int b) { return IS_MAX ? max(a, b) : min(a, b); };
  int a = v;
  a = op(a, __builtin_amdgcn_update_dpp(id, v, 0x111, 0xf, 0xf, false));
  a = op(a, __builtin_amdgcn_update_dpp(id, v, 0x112, 0xf, 0xf, false));
  a = op(a, __builtin_amdgcn_update_dpp(id, v, 0x113, 0xf, 0xf, false));
  a = op(a, __builtin_amdgcn_update_dpp(id, a, 0x114, 0xf, 0xe, false));
  a = op(a, __builtin_amdgcn_update_dpp(id, a, 0x118, 0xf, 0xc, false));
  a = op(a, __builtin_amdgcn_update_dpp(id, a, 0x142, 0xa, 0xf, false));
  a = op(a, __builtin_amdgcn_update_dpp(id, a, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(a, 63);
}

// Keys [d0, d1), of the first `keys`, outside of which no key's document lies between
// those of tokens t0 to t1: all that packed documents need not read.  mem: two ints a
// wave.
template <int W>
__device__ __forceinline__ void document_keys(const AttendArgs& p, const int* qdocs, const int* kdocs, int t0, int t1,
                                              int keys, int* mem, int& d0, int& d1) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int lo = 0x7fffffff, hi = -0x7fffffff - 1;
#pragma unroll 2
  for (int t = t0 + lane; t <= t1; t += 64) {  // every wave by itself
    const int d = qdocs[t * p.qdoc_step];
    lo = min(lo, d);
    hi = max(hi, d);
  }
  lo = wave_extreme<false>(lo);
  hi = wave_extreme<true>(hi);
  int first = keys, last = -1;
  typedef int i4a __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int STEP = 256 * W;  // keys a round
  const int mine = 4 * (int)threadIdx.x;
  int j = 0;
  for (; j + 4 * STEP <= keys; j += 4 * STEP) {
    i4a d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) d[u] = *reinterpret_cast<const i4a*>(kdocs + j + u * STEP + mine);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d[u][e] >= lo && d[u][e] <= hi) {
          const int at = j + u * STEP + mine + e;
          first = min(first, at);
          last = max(last, at);
        }
  }
#pragma unroll 4
  for (j += threadIdx.x; j < keys; j += 64 * W) {
    const int d = kdocs[j];
    if (d >= lo && d <= hi) {
      first = min(first, j);
      last = max(last, j);
    }
  }
  first = wave_extreme<false>(first);
  last = wave_extreme<true>(last);
  if (lane == 0) {
    mem[2 * wave] = first;
    mem[2 * wave + 1] = last;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) {
    first = min(first, mem[2 * w]);
    last = max(last, mem[2 * w + 1]);
  }
  d0 = __builtin_amdgcn_readfirstlane(first);
  d1 = __builtin_amdgcn_readfirstlane(last) + 1;
  __syncthreads();
}

struct BlockAt {
  int x, y, z, tile, split, start, window, len, pre;
  long long block;
};

// A first position, held within +-kFar; so far past every key its window is shorter by what
// that takes off, which leaves the keys that the rows see, and scores but for one constant.
__device__ __forceinline__ void hold_start(const AttendArgs& p, int start, BlockAt& b) {
  b.start = min(max(start, -kFar), kFar - 1);
  if (start > kFar - 1) b.window = max(p.window - (start - (kFar - 1)), 0);
}

template <bool FEW>
__device__ __forceinline__ BlockAt block_at(const AttendArgs& p) {
  BlockAt b;
  const int id = xcd_contiguous(blockIdx.x, p.nwg);
  const int blk = (int)p.d_work((unsigned)id);
  const int rest = id - blk * p.tiles * p.splits;
  const int tile = (int)p.d_splits((unsigned)rest);
  b.split = rest - tile * p.splits;
  b.tile = p.tiles - 1 - tile;  // a causal Block's last rows see the most keys: they go first
  b.block = blk;
  p.blocks(blk, b.x, b.y, b.z);
  if constexpr (FEW) {
    b.start = 0;
    b.window = p.window;
    b.len = p.keys;
    b.pre = 0;
    if (p.start || p.length || p.prefix) {
      // all on their way at once, what is absent reads one that is there: a twentieth of
      // a short cache's time (878 keys 11.1 -> 10.6 us; more rows lose a fiftieth by it)
      const int* const any = p.start ? p.start : p.length ? p.length : p.prefix;
      const int start = *(p.start ? p.start + p.tstart.at(b.x, b.y, b.z) : any);
      const int len = *(p.length ? p.length + p.tlength.at(b.x, b.y, b.z) : any);
      const int pre = *(p.prefix ? p.prefix + p.tprefix.at(b.x, b.y, b.z) : any);
      if (p.start) hold_start(p, start, b);
      if (p.length) b.len = min(max(len, 0), p.keys);
      if (p.prefix) b.pre = min(max(pre, 0), b.len);
    }
  } else {
    b.start = 0;
    b.window = p.window;
    if (p.start) hold_start(p, p.start[p.tstart.at(b.x, b.y, b.z)], b);
    b.len = p.length ? min(max(p.length[p.tlength.at(b.x, b.y, b.z)], 0), p.keys) : p.keys;
    b.pre = p.prefix ? min(max(p.prefix[p.tprefix.at(b.x, b.y, b.z)], 0), b.len) : 0;
  }
  b.start = __builtin_amdgcn_readfirstlane(b.start);
  b.window = __builtin_amdgcn_readfirstlane(b.window);
  b.len = __builtin_amdgcn_readfirstlane(b.len);
  b.pre = __builtin_amdgcn_readfirstlane(b.pre);
  return b;
}

// No row up to token t1 sees this key or a later one, documents aside.
__device__ __forceinline__ int last_key(const AttendArgs& p, const BlockAt& b, int t1) {
  return p.causal ? min(b.len, max(max(b.start + t1, -1) + 1, b.pre)) : b.len;
}

// BN keys of D values each from an array to LDS, by STEP waves: instruction i of a
// wave fills 1 KB, lane L at byte 16 L, with the chunk that belongs there.  Rows past
// `left` become zeros.
template <int D, int BN, bool VALUES, int STEP>
struct Fill {
  typedef Rows<D, false> R;
  static constexpr int IN = BN * D * 2 / 1024 / STEP;
  static_assert(IN * 1024 * STEP == BN * D * 2, "whole instructions");
  // Where an instruction takes whole rows, the swizzle of its first row and that of
  // the lane's row among them are apart (the rows' bits are): two registers, the row's
  // offset and the chunk's, serve all instructions.  That fits three workgroups on a CU
  // at 64 columns (documents of 8192 tokens: 57 -> 51 us) and leaves nothing in scratch
  // at 256.  Otherwise each has its own: at 128 the arithmetic costs more than the
  // registers (a batch of decoded tokens: 175 us against 179).
  static constexpr bool WHOLE = 1024 % (2 * D) == 0 && D != 128;
  static constexpr int RPI = 512 / D;
  const unsigned char* base;
  unsigned pitch;
  unsigned off[WHOLE ? 2 : IN];
  int lane, first;

  static __device__ __forceinline__ int swizzle(int row) { return VALUES ? R::vsw(row) : R::ksw(row); }

  __device__ __forceinline__ void begin(const unsigned char* b, long long ld, int wave) {
    base = b;
    pitch = (unsigned)(ld * 2);
    lane = threadIdx.x & 63;
    first = wave;
    if constexpr (WHOLE) {
      const int row = lane / (D / 8), c = lane % (D / 8);
      off[0] = (unsigned)row * pitch;
      off[1] = (unsigned)(c ^ swizzle(row)) << 4;
    } else {
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        const int pos = (i * STEP + first) * 1024 + lane * 16, row = pos / (2 * D), c = (pos % (2 * D)) >> 4;
        off[i] = (unsigned)row * pitch + ((c ^ swizzle(row)) << 4);
      }
    }
  }

  // Byte offset of the chunk that instruction i of this wave brings; chunk: off[1].
  __device__ __forceinline__ unsigned at(int i, unsigned chunk) const {
    if constexpr (WHOLE) {
      const int row = (i * STEP + first) * RPI;
      return (unsigned)row * pitch + off[0] + (chunk ^ ((unsigned)swizzle(row) << 4));
    } else {
      return off[i];
    }
  }

  __device__ __forceinline__ void issue(bool dma, int key0, int left, unsigned char* to) const {
    const unsigned char* from = base + (long long)key0 * pitch;
    unsigned chunk = off[WHOLE ? 1 : 0];
    if constexpr (WHOLE) asm volatile("" : "+v"(chunk));  // or the offsets would be kept, a register each
    if (dma) {
      const i32x4 rs = raw_rsrc(from, (unsigned)(min(left, BN) - 1) * pitch + 2 * D);
      const unsigned lds = __builtin_amdgcn_readfirstlane(lds_at(to) + first * 1024);
#pragma unroll
      for (int i = 0; i < IN; ++i) dma16(rs, lds + i * STEP * 1024, at(i, chunk), 0);
    } else {
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        const int pos = (i * STEP + first) * 1024 + lane * 16;
        uint4v v = {0, 0, 0, 0};
        if (pos / (2 * D) < left) v = (uint4v)(*reinterpret_cast<const u4a*>(from + at(i, chunk)));
        *reinterpret_cast<uint4v*>(to + pos) = v;
      }
    }
  }
};

// Every LDS access of this wave is done, then the barrier: a bare s_barrier, since
// __syncthreads would also wait for the DMA in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Four neighbouring result columns of a row, rounded once.
template <bool BF16>
__device__ __forceinline__ void store4(const AttendArgs& p, const BlockAt& b, int row, int d, float x, float y, float z,
                                       float w) {
  const int token = (int)p.d_heads((unsigned)row), head = row - token * p.heads;
  unsigned char* const at = p.o + (p.to.at(b.x, b.y, b.z) + head * p.o_head + token * p.o_row + d) * 2;
  *reinterpret_cast<u2a*>(at) = u2a{pack2<BF16>(x, y), pack2<BF16>(z, w)};
}

// The workspace: D sums of each (row, split), then a maximum and a total each.
__device__ __forceinline__ float* sums_of(const AttendArgs& p, int D, long long row, int split) {
  return p.work + (row * p.splits + split) * D;
}
__device__ __forceinline__ float* total_of(const AttendArgs& p, int D, long long rows, long long row, int split) {
  return p.work + rows * p.splits * D + 2 * (row * p.splits + split);
}

// The kernel's arguments (AttendArgs comes first), loaded where they are used: what only the
// way of odd rows reads would take scalar registers in every launch's loop (2048 tokens, 16
// heads of 32 columns, causal: 30.5 us if kept in registers, 26.6 if loaded here).
__device__ __forceinline__ const AttendArgs& args_here() {
  auto at = (const __attribute__((address_space(4))) AttendArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const AttendArgs*)at;
}

// Rows first, first + step, ... below last over the keys of tiles [i0, i1) of bn, a
// wave each and in vector arithmetic: the way for keys among which values are not finite
// or near the largest, of which only what a row sees is ever multiplied, by weights of 32
// bits and at most one.  Lane j of 64 keys has
// the score of key j; then the lanes have the columns.
template <int D, bool BF16, bool FINE>
__device__ __forceinline__ void odd_rows(const AttendArgs& p, const FineCap& c, const BlockAt& b, const Tiles& tiles,
                                         int bn, int i0, int i1, const int* kdocs, int first, int last, int step,
                                         long long all_rows) {
  const int lane = threadIdx.x & 63;
  auto value = [](unsigned short x) {
    return BF16 ? __builtin_bit_cast(float, (unsigned)x << 16) : (float)__builtin_bit_cast(_Float16, x);
  };
  const unsigned short* const keys = reinterpret_cast<const unsigned short*>(p.k) + p.tk.at(b.x, b.y, b.z);
  const unsigned short* const values = reinterpret_cast<const unsigned short*>(p.v) + p.tv.at(b.x, b.y, b.z);
#pragma unroll 1
  for (int row = first; row < last; row += step) {
    const int token = (int)p.d_heads((unsigned)row), head = row - token * p.heads, pos = b.start + token;
    const unsigned short* const q = reinterpret_cast<const unsigned short*>(p.q) + p.tq.at(b.x, b.y, b.z) +
                                    head * p.q_head + token * p.q_row;
    const float slope = p.slopes ? p.slopes[p.tslopes.at(b.x, b.y, b.z) + head * p.slope_step] * 1.44269504088896340736f : 0.0f;
    const int doc = p.qdocs ? p.qdocs[p.tqdocs.at(b.x, b.y, b.z) + token * p.qdoc_step] : 0;
    auto sees = [&](int j, int end) {
      return j < end && j < b.len && (j < b.pre || ((!p.causal || j <= pos) && j > before(p, b.window, pos))) &&
             (!kdocs || kdocs[j] == doc);
    };
    auto score = [&](int j) {
      const unsigned short* const k = keys + (long long)j * p.ldk;
      float s = 0.0f;
#pragma unroll 1
      for (int d = 0; d < D; ++d) s = fmaf(value(q[d]), value(k[d]), s);
      s = FINE ? capped(p, c, s) : p.cap_log2 > 0.0f ? capped_far(p, s) : s * p.scale_log2;
      return p.slopes ? fmaf(-slope, fabsf((float)(pos - j)), s) : s;
    };
    // the maximum, minus infinity where the row sees nothing (as in tile), and what the
    // scores are taken relative to
    float m = -__builtin_inff(), use = 0.0f, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
      for (int i = i0; i < i1; ++i) {
        const int key0 = tiles.at(i) * bn, j = key0 + lane;
        const bool in = sees(j, key0 + bn);
        const float s = in ? score(j) : -__builtin_inff();
        if (pass == 0) {
          m = fmaxf(m, s);
          continue;
        }
        const float w = in ? __builtin_amdgcn_exp2f(s - use) : 0.0f;
        l += w;
        unsigned long long left = __builtin_amdgcn_ballot_w64(in);
#pragma unroll 1
        while (left) {
          const int e = __builtin_ctzll(left);
          left &= left - 1;
          const float we = __shfl(w, e, 64);
#pragma unroll
          for (int c = 0; c < (D + 63) / 64; ++c)
            if (c * 64 + lane < D) o[c] = fmaf(we, value(values[(long long)(key0 + e) * p.ldv + c * 64 + lane]), o[c]);
        }
      }
      if (pass == 0) {
        m = wave_reduce<true>(m);
        use = m == -__builtin_inff() ? 0.0f : m;
      }
    }
    l = wave_reduce<false>(l);
    const long long at = b.block * p.rows + row;
    float* const t = p.splits > 1 ? total_of(p, D, all_rows, at, b.split) : nullptr;
    if (t && lane == 0) {
      t[0] = m;
      t[1] = l;
    }
#pragma unroll
    for (int c = 0; c < (D + 63) / 64; ++c) {
      if (c * 64 + lane >= D) continue;
      if (t) {
        sums_of(p, D, at, b.split)[c * 64 + lane] = o[c];
      } else {
        const unsigned both = pack2<BF16>(l == 0.0f ? 0.0f : o[c] / l, 0.0f);
        reinterpret_cast<unsigned short*>(p.o)[p.to.at(b.x, b.y, b.z) + head * p.o_head + token * p.o_row + c * 64 + lane] =
            (unsigned short)both;
      }
    }
  }
}

// Whether any wave of the workgroup says so; no LDS access is left out standing.
template <int W>
__device__ __forceinline__ bool any_wave(bool x, unsigned char* lds) {
  int* const at = reinterpret_cast<int*>(lds);
  if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = x;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) any |= at[w];
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(any) != 0;
}

// More than 32 rows: 128 of them, 32 a wave, the keys in tiles of 64 that four waves
// share, two of them in LDS.  G groups of four waves have the same rows and take tiles
// in turn, and the second's results join the first's: where workgroups are so few that
// a SIMD would have one wave, whose products and arithmetic wait for each other.
template <int D, bool BF16, int G, bool FINE>
__global__ __launch_bounds__(256 * G, G == 2 ? 2 : D <= 64 ? 3 : D <= 128 ? 2 : 1)
void attend_rows_kernel(AttendArgs p, long long all_rows, FineCap c) {
  constexpr int BN = 64, KB = BN * D * 2, STAGE = 2 * KB + 256;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * G * STAGE];
  const bool dma = p.dma;
  const int every = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = every & 3, group = G == 1 ? 0 : every >> 2;
  const BlockAt b = block_at<false>(p);
  const int first = b.tile * 128, last = min(first + 127, p.rows - 1);
  const int t0 = (int)p.d_heads((unsigned)first), t1 = (int)p.d_heads((unsigned)last);
  const int* const kdocs = p.kdocs ? p.kdocs + p.tkdocs.at(b.x, b.y, b.z) : nullptr;
  int d0 = 0, d1 = b.len;
  if (kdocs)
    document_keys<4 * G>(p, p.qdocs + p.tqdocs.at(b.x, b.y, b.z), kdocs, t0, t1, last_key(p, b, t1), reinterpret_cast<int*>(lds),
                     d0, d1);
  const Tiles tiles = tiles_of(p, BN, b.start + t0, b.start + t1, b.window, b.len, b.pre, d0, d1);
  const int share = (int)p.d_splits((unsigned)(tiles.n + p.splits - 1));  // tiles of a split
  const int i0 = min(b.split * share, tiles.n), i1 = min(i0 + share, tiles.n);

  Fill<D, BN, false, 4> fk;
  Fill<D, BN, true, 4> fv;
  fk.begin(p.k + p.tk.at(b.x, b.y, b.z) * 2, p.ldk, wave);
  fv.begin(p.v + p.tv.at(b.x, b.y, b.z) * 2, p.ldv, wave);
  auto issue = [&](int i, unsigned char* at) {
    const int key0 = tiles.at(i) * BN, left = b.len - key0;
    fk.issue(dma, key0, left, at);
    fv.issue(dma, key0, left, at + KB);
    if (kdocs) dma4(raw_rsrc(kdocs + key0, (unsigned)min(left, BN) * 4), lds_at(at + 2 * KB), (threadIdx.x & 63) * 4);
  };
  unsigned char* const stages = lds + group * 2 * STAGE;
  if (i0 + group < i1) issue(i0 + group, stages);
  Rows<D, BF16, FINE> rows;
  rows.begin(p, first + 32 * wave, b.x, b.y, b.z, b.start, b.window);
#pragma unroll 1
  for (int i = i0 + group, n = 0; i - group < i1; i += G, n ^= 1) {
    // one barrier a tile: behind it this tile has landed, and every wave is done with
    // the one before, whose place the next one takes while this one is worked on
    unsigned char* const at = stages + n * STAGE;
    XTK_WAIT_VM(0);
    lds_barrier();
    if (i + G < i1) issue(i + G, stages + (n ^ 1) * STAGE);
    if (G > 1 && i >= i1) continue;
    const int key0 = tiles.at(i) * BN;
    if (!rows.sees_none(p, key0, BN, b.pre))
      rows.template tile<2>(p, c, at, at + KB, reinterpret_cast<const int*>(at + 2 * KB), kdocs, key0, b.len, b.pre);
  }
  rows.hold();
  lds_barrier();
  if (any_wave<4 * G>(rows.spoilt(), lds)) {
    odd_rows<D, BF16, FINE>(args_here(), c, b, tiles, BN, i0, i1, kdocs, first + every, last + 1, 4 * G, all_rows);
    return;
  }
  if constexpr (G == 2) {
    // behind what the rows leave through below
    float* const theirs = reinterpret_cast<float*>(lds + 4 * 32 * (2 * D + 16)) + wave * (32 * D + 128);
    static_assert(4 * 32 * (2 * D + 16) + 4 * (32 * D + 128) * 4 <= 2 * G * STAGE, "the second group's results");
    if (group == 1) {
#pragma unroll
      for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *reinterpret_cast<float4v*>(theirs + (4 * n + w) * 256 + rows.lane * 4) =
              float4v{rows.acc[n][4 * w], rows.acc[n][4 * w + 1], rows.acc[n][4 * w + 2], rows.acc[n][4 * w + 3]};
      theirs[32 * D + rows.lane] = rows.m;
      theirs[32 * D + 64 + rows.lane] = rows.l;
    }
    __syncthreads();
    if (group == 1) return;
    const float m1 = theirs[32 * D + rows.lane], l1 = theirs[32 * D + 64 + rows.lane];
    const float m = fmaxf(rows.m, m1), use = m == -__builtin_inff() ? 0.0f : m;
    const float a0 = __builtin_amdgcn_exp2f(rows.m - use), a1 = __builtin_amdgcn_exp2f(m1 - use);
    rows.m = m;
    rows.l = rows.l * a0 + l1 * a1;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4v o = *reinterpret_cast<const float4v*>(theirs + (4 * n + w) * 256 + rows.lane * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) rows.acc[n][4 * w + e] = rows.acc[n][4 * w + e] * a0 + o[e] * a1;
      }
  }

  const float l = both_halves(rows.l, false);
  if (p.splits == 1) {
    // through LDS, so that a row leaves in 16-byte pieces side by side: a lane has
    // four columns of eight here and there.  Each wave has its own part; rows 16 bytes
    // apart from a multiple of the banks.
    constexpr int PITCH = 2 * D + 16;
    unsigned char* const own = lds + wave * 32 * PITCH;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = l == 0.0f ? 0.0f : rows.acc[n][4 * w + e] * inv;
        *reinterpret_cast<uint2v*>(own + rows.col * PITCH + (32 * n + 8 * w + 4 * rows.hi) * 2) =
            uint2v{pack2<BF16>(o[0], o[1]), pack2<BF16>(o[2], o[3])};
      }
    unsigned char* const out = p.o + p.to.at(b.x, b.y, b.z) * 2;
    constexpr int C = D / 8;  // pieces of a row
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
      const int e = i * 64 + rows.lane, r = e / C, c = e % C, row = first + 32 * wave + r;
      if (row >= p.rows) continue;
      const int token = (int)p.d_heads((unsigned)row), head = row - token * p.heads;
      *reinterpret_cast<u4a*>(out + (head * p.o_head + token * p.o_row + c * 8) * 2) =
          (u4a)(*reinterpret_cast<const uint4v*>(own + r * PITCH + c * 16));
    }
    return;
  }
  if (first + 32 * wave + rows.col >= p.rows) return;
  const long long row = b.block * p.rows + rows.row;
  float* const sums = sums_of(p, D, row, b.split);
#pragma unroll
  for (int n = 0; n < D / 32; ++n)
#pragma unroll
    for (int w = 0; w < 4; ++w)
      *reinterpret_cast<float4v*>(sums + 32 * n + 8 * w + 4 * rows.hi) =
          float4v{rows.acc[n][4 * w], rows.acc[n][4 * w + 1], rows.acc[n][4 * w + 2], rows.acc[n][4 * w + 3]};
  if (rows.hi == 0) {
    float* const t = total_of(p, D, all_rows, row, b.split);
    t[0] = rows.m;
    t[1] = l;
  }
}

// Waves of a workgroup of few rows, and tiles of 32 keys in a wave's ring: what
// fills 160 KB of LDS, twice over where that leaves enough in flight.
template <int D>
struct Few {
  static constexpr int W = D <= 160 ? 4 : 2, TILE = 32 * D * 4;
  static constexpr int NS = D == 32 ? 4 : D == 64 ? 2 : D == 96 || D == 192 ? 3 : 2;
  static constexpr int LDS = W * NS * TILE;
  static_assert(LDS <= 160 * 1024 && W * 256 + W * 32 * (D + 4) * 4 <= LDS, "rings, then the waves' results");
  static_assert((NS - 1) * (D / 8) < 64, "vmcnt is six bits");
};

// Up to 32 rows: every wave has them all and takes tiles of 32 keys in turn, each in
// a ring of its own, so that nothing but its own loads makes a wave wait.
template <int D, bool BF16, bool FINE>
__global__ __launch_bounds__(64 * Few<D>::W) void attend_few_kernel(AttendArgs p, long long all_rows, FineCap c) {
  typedef Few<D> F;
  constexpr int W = F::W, NS = F::NS, KB = 32 * D * 2, PER = D / 8;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[F::LDS];
  const bool dma = p.dma;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const BlockAt b = block_at<true>(p);
  const int t1 = (int)p.d_heads((unsigned)(p.rows - 1));
  const int* const kdocs = p.kdocs ? p.kdocs + p.tkdocs.at(b.x, b.y, b.z) : nullptr;
  int d0 = 0, d1 = b.len;
  if (kdocs)
    document_keys<W>(p, p.qdocs + p.tqdocs.at(b.x, b.y, b.z), kdocs, 0, t1, last_key(p, b, t1), reinterpret_cast<int*>(lds),
                     d0, d1);
  const Tiles tiles = tiles_of(p, 32, b.start, b.start + t1, b.window, b.len, b.pre, d0, d1);
  const int share = (int)p.d_splits((unsigned)(tiles.n + p.splits - 1));  // tiles of a split
  const int i0 = min(b.split * share, tiles.n), i1 = min(i0 + share, tiles.n);
  const int mine = max(0, (i1 - i0 - wave + W - 1) / W);

  Fill<D, 32, false, 1> fk;
  Fill<D, 32, true, 1> fv;
  fk.begin(p.k + p.tk.at(b.x, b.y, b.z) * 2, p.ldk, 0);
  fv.begin(p.v + p.tv.at(b.x, b.y, b.z) * 2, p.ldv, 0);
  unsigned char* const ring = lds + wave * NS * F::TILE;
  auto key_of = [&](int j) { return tiles.at(i0 + wave + j * W) * 32; };
  auto issue = [&](int j, int slot) {
    unsigned char* const at = ring + slot * F::TILE;
    const int key0 = key_of(j);
    fk.issue(dma, key0, b.len - key0, at);
    fv.issue(dma, key0, b.len - key0, at + KB);
  };
#pragma unroll
  for (int j = 0; j < NS; ++j)
    if (j < mine) issue(j, j);
  Rows<D, BF16, FINE> rows;
  rows.begin(p, 0, b.x, b.y, b.z, b.start, b.window);
  int slot = 0;
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    const int ahead = dma ? min(mine - 1 - j, NS - 1) : 0;
    switch (ahead) {
      case 0: XTK_WAIT_VM(0); break;
      case 1: XTK_WAIT_VM(PER); break;
      case 2: XTK_WAIT_VM(NS > 2 ? 2 * PER : 0); break;
      default: XTK_WAIT_VM(NS > 3 ? 3 * PER : 0); break;
    }
    asm volatile("" ::: "memory");
    unsigned char* const at = ring + slot * F::TILE;
    rows.template tile<1>(p, c, at, at + KB, nullptr, kdocs, key_of(j), b.len, b.pre);
    // every fragment is in registers before the slot is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (j + NS < mine) issue(j + NS, slot);
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  // At 256 columns the accumulators would otherwise meet themselves in other registers,
  // and scratch; narrower heads lose a few of 120 us by it.
  if constexpr (D == 256) rows.hold();
  __syncthreads();  // every ring is done with
  if (any_wave<W>(rows.spoilt(), lds)) {
    odd_rows<D, BF16, FINE>(args_here(), c, b, tiles, 32, i0, i1, kdocs, wave, p.rows, W, all_rows);
    return;
  }

  // the waves' results meet in the rings
  float* const total = reinterpret_cast<float*>(lds);
  float* const part = total + W * 64;
  const float own = both_halves(rows.l, false);
  __syncthreads();
  if (rows.hi == 0) {
    total[(wave * 32 + rows.col) * 2] = rows.m;
    total[(wave * 32 + rows.col) * 2 + 1] = own;
  }
  __syncthreads();
  auto joined = [&](int c, float& m, float& l) {
    m = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, total[(w * 32 + c) * 2]);
    const float use = m == -__builtin_inff() ? 0.0f : m;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) l += total[(w * 32 + c) * 2 + 1] * __builtin_amdgcn_exp2f(total[(w * 32 + c) * 2] - use);
    return use;
  };
  float m, l;
  const float f = __builtin_amdgcn_exp2f(rows.m - joined(rows.col, m, l));
  if (rows.col < p.rows) {
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        *reinterpret_cast<float4v*>(part + (wave * 32 + rows.col) * (D + 4) + 32 * n + 8 * w + 4 * rows.hi) =
            float4v{rows.acc[n][4 * w] * f, rows.acc[n][4 * w + 1] * f, rows.acc[n][4 * w + 2] * f,
                    rows.acc[n][4 * w + 3] * f};
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.rows * (D / 4); e += 64 * W) {
    const int c = e / (D / 4), d = 4 * (e % (D / 4));
    float4v o = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w) o += *reinterpret_cast<const float4v*>(part + (w * 32 + c) * (D + 4) + d);
    joined(c, m, l);
    if (p.splits == 1) {
      const float inv = 1.0f / l;
      if (l == 0.0f) o = float4v{0, 0, 0, 0};
      else o *= inv;
      store4<BF16>(p, b, c, d, o[0], o[1], o[2], o[3]);
    } else {
      const long long row = b.block * p.rows + c;
      *reinterpret_cast<float4v*>(sums_of(p, D, row, b.split) + d) = o;
      if (d == 0) {
        float* const t = total_of(p, D, all_rows, row, b.split);
        t[0] = m;
        t[1] = l;
      }
    }
  }
}

// The splits of rows joined, in a fixed order: D / 4 threads (a column quad each) take
// every G-th split of a row.  G = 1: 256 / (D / 4) rows a workgroup, for few splits;
// else one row with as many groups as fit, and up to 256 splits.
template <int D, bool BF16, bool FEW>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs p, long long all_rows) {
  constexpr int Q = D / 4, G = 256 / Q;
  const int tid = threadIdx.x, g = tid / Q, d = 4 * (tid % Q);
  const long long row = FEW ? (long long)blockIdx.x * G + g : blockIdx.x;
  if (FEW && (g >= G || row >= all_rows)) return;
  BlockAt b;
  const int blk = (int)p.d_work((unsigned)row);
  const int r = (int)(row - (long long)blk * p.rows);
  p.blocks(blk, b.x, b.y, b.z);
  float4v o = {0, 0, 0, 0};
  float total = 0.0f;
  if constexpr (FEW) {
    float m = -__builtin_inff();
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, *total_of(p, D, all_rows, row, s));
    if (m == -__builtin_inff()) m = 0.0f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
      const float2 t = *reinterpret_cast<const float2*>(total_of(p, D, all_rows, row, s));
      const float f = __builtin_amdgcn_exp2f(t.x - m);
      total += t.y * f;
      o += f * *reinterpret_cast<const float4v*>(sums_of(p, D, row, s) + d);
    }
  } else {
    __shared__ float f[256];
    __shared__ float red[8];
    __shared__ __attribute__((aligned(16))) float part[G][D];
    const int lane = tid & 63, wave = tid >> 6;
    const float2 t = tid < p.splits ? *reinterpret_cast<const float2*>(total_of(p, D, all_rows, row, tid))
                                    : float2{-__builtin_inff(), 0.0f};
    // the first sums are on their way before the maximum is known
    float4v v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      v[u] = g < G && g + u * G < p.splits ? *reinterpret_cast<const float4v*>(sums_of(p, D, row, g + u * G) + d)
                                           : float4v{0, 0, 0, 0};
    float m = wave_reduce<true>(t.x);
    if (lane == 0) red[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    if (m == -__builtin_inff()) m = 0.0f;
    const float own = __builtin_amdgcn_exp2f(t.x - m);
    f[tid] = own;
    const float l = wave_reduce<false>(t.y * own);
    if (lane == 0) red[4 + wave] = l;
    __syncthreads();
    if (g < G) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (g + u * G < p.splits) o += f[g + u * G] * v[u];
#pragma unroll 8
      for (int s = g + 4 * G; s < p.splits; s += G)
        o += f[s] * *reinterpret_cast<const float4v*>(sums_of(p, D, row, s) + d);
      *reinterpret_cast<float4v*>(&part[g][d]) = o;
    }
    __syncthreads();
    if (tid >= Q) return;
    o = float4v{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < G; ++w) o += *reinterpret_cast<const float4v*>(&part[w][d]);
    total = (red[4] + red[5]) + (red[6] + red[7]);
  }
  if (total == 0.0f) o = float4v{0, 0, 0, 0};
  else o *= 1.0f / total;
  store4<BF16>(p, b, r, d, o[0], o[1], o[2], o[3]);
}

// Whether two groups of waves share the rows' keys: where there is no second workgroup
// for a CU, nor a split that would fill it, and each group gets two tiles at least (577
// keys, 160 workgroups of 96 columns: 17.6 -> 16.6 us; 332 keys of 32: 15.5 -> 11.5; of
// 135 keys 9.6 -> 10.6; a split of 1520 keys in five 19.8 -> 21.1).
inline bool pairs_of(const AttendArgs& a, int d) { return d <= 128 && a.nwg <= 256 && a.splits == 1 && a.keys > 192; }

template <int D, bool BF16, bool FINE>
void run_attend_rows(bool few, const AttendArgs& a, long long all_rows, const FineCap& c, hipStream_t s) {
  if (few) {
    attend_few_kernel<D, BF16, FINE><<<a.nwg, 64 * Few<D>::W, 0, s>>>(a, all_rows, c);
    return;
  }
  if constexpr (D <= 128)
    if (pairs_of(a, D)) {
      attend_rows_kernel<D, BF16, 2, FINE><<<a.nwg, 512, 0, s>>>(a, all_rows, c);
      return;
    }
  attend_rows_kernel<D, BF16, 1, FINE><<<a.nwg, 256, 0, s>>>(a, all_rows, c);
}

template <int D, bool BF16>
hipError_t run_attend_elem(bool few, const AttendArgs& a, const FineCap* fine, hipStream_t s) {
  const long long blocks = a.nwg / ((long long)a.tiles * a.splits), all_rows = blocks * a.rows;
  if (fine) run_attend_rows<D, BF16, true>(few, a, all_rows, *fine, s);
  else run_attend_rows<D, BF16, false>(few, a, all_rows, FineCap{}, s);
  if (a.splits > 1) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    AttendArgs j = a;
    j.d_work = div31(static_cast<unsigned>(a.rows));
    constexpr int rows = 256 / (D / 4);
    if (a.splits <= 16)
      attend_join_kernel<D, BF16, true><<<static_cast<unsigned>((all_rows + rows - 1) / rows), 256, 0, s>>>(j, all_rows);
    else
      attend_join_kernel<D, BF16, false><<<static_cast<unsigned>(all_rows), 256, 0, s>>>(j, all_rows);
  }
  return hipGetLastError();
}

}  // namespace

template <int D>
hipError_t run_attend(bool bf16, bool few, const AttendArgs& a, const FineCap* fine, hipStream_t s) {
  return bf16 ? run_attend_elem<D, true>(few, a, fine, s) : run_attend_elem<D, false>(few, a, fine, s);
}

}  // namespace xtk

#endif
