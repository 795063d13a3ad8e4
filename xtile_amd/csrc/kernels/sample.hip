// A token of each row of logits (xtile_amd.dsl.sample states which).
//
// Weights are 64-bit integers, rint(2^S e^((x - max) / t)): their sums are exact, so
// neither the order of additions nor the number of workgroups changes a result.  S leaves
// room for the sum of a row (S + log2 V < 62, and at most 50 for the conversion).
//
// What top-k, top-p and min-p leave is in each case a beginning of the tokens' order
// (largest logit first, equal ones by index), so what they leave together is the
// shortest of the three, and it is enough to know its weight.  The drawn token is then
// found as the cut of top-p is: the first at which the running sum reaches a value.
//
// The order is not made.  One pass takes the largest logit, a second counts and sums the
// tokens in kBins bins of their distance from it, the next gathers the few tokens of the
// bin in which the sum reaches the value (or of all bins up to there, if they are few,
// which then serve every further question), and only those are sorted.  A bin with too
// many is parted by 11 bits of the order's key (the logit's bits, then the index) as often
// as it takes, at most five times.
#include "launch.h"

#include <algorithm>

#include "common.h"

namespace xtk {
namespace {

enum { kF32 = 0, kF16 = 1, kBF16 = 2 };

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048, kList = 2048;
constexpr int kIndexBits = 22;  // xt::kSampleVocab
static_assert(xt::kSampleVocab == 1LL << kIndexBits && kBins == 2 * kThreads && kList == 2 * kThreads, "");

struct SampleArgs {
  const unsigned char* x;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  int* y;
  TileOff tx, tu, tt, tk, tp, tm, ty;
  long long ldx, ldu, ldt, ldk, ldp, ldm, ldy;  // elements
  BlockDecode blocks;
  Div31 per_block;  // rows of a Block
  int rows, vocab;
  int shift;  // S
};

struct RowAt {
  int x, y, z;
  long long r;
  template <class T>
  __device__ __forceinline__ T in(const T* base, const TileOff& t, long long ld, T absent) const {
    return base ? base[t.at(x, y, z) + r * ld] : absent;
  }
};

__device__ __forceinline__ RowAt row_at(const SampleArgs& p, int row) {
  RowAt a;
  const int b = (int)p.per_block((unsigned)row);
  a.r = row - b * p.rows;
  p.blocks(b, a.x, a.y, a.z);
  return a;
}

// NaN as minus infinity, minus zero as zero.
__device__ __forceinline__ float clean(float x) { return x != x ? -__builtin_inff() : x + 0.0f; }

// f(logit, index) of logits first to last - 1 of a row, by `threads` threads.
template <int ELEM, class F>
__device__ __forceinline__ void each(const unsigned char* row, int first, int last, int threads, F f) {
  constexpr int N = ELEM == kF32 ? 4 : 8, ES = ELEM == kF32 ? 4 : 2, U = 4;
  typedef unsigned u4a __attribute__((ext_vector_type(4), aligned(2)));
  auto value = [](uint4v w, int i) {
    if constexpr (ELEM == kF32) {
      const unsigned u = w[i];  // a bit cast of the element itself would read element 0
      return __builtin_bit_cast(float, u);
    } else {
      const unsigned short h = (unsigned short)(w[i / 2] >> (16 * (i % 2)));
      return ELEM == kF16 ? (float)__builtin_bit_cast(_Float16, h) : __builtin_bit_cast(float, (unsigned)h << 16);
    }
  };
  int i = first + (int)threadIdx.x * N;
  for (; i + (U - 1) * threads * N + N <= last; i += U * threads * N) {
    uint4v w[U];
#pragma unroll
    for (int k = 0; k < U; ++k) w[k] = (uint4v)(*reinterpret_cast<const u4a*>(row + (long long)(i + k * threads * N) * ES));
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) f(clean(value(w[k], e)), i + k * threads * N + e);
  }
#pragma unroll 1
  for (; i < last; i += threads * N) {
    uint4v w = {0, 0, 0, 0};
    const int n = min(N, last - i);
    if (n == N) {
      w = (uint4v)(*reinterpret_cast<const u4a*>(row + (long long)i * ES));
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < n) {
          if constexpr (ELEM == kF32) w[e] = *reinterpret_cast<const unsigned*>(row + (long long)(i + e) * ES);
          else w[e / 2] |= (unsigned)*reinterpret_cast<const unsigned short*>(row + (long long)(i + e) * ES) << (16 * (e % 2));
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < n) f(clean(value(w, e)), i + e);
  }
}

// A row's weights and bins.
struct Weights {
  float top;      // the largest logit
  float per_bin;  // bins a unit of distance
  double c;       // log2 e / t
  bool only_top;  // no other logit has a weight
  int shift;

  __device__ __forceinline__ void begin(float largest, float t, int s) {
    top = largest;
    shift = s;
    only_top = !(t > 0.0f) || largest == __builtin_inff();
    c = only_top ? 0.0 : 1.4426950408889634 / (double)t;
    // weights end at 2^-(S + 1)
    per_bin = (float)(c * ((kBins - 1) / (double)(s + 2)));
  }

  // Never more for a larger logit: each step here is monotonic.
  __device__ __forceinline__ int bin(float x) const {
    if (x == top) return 0;
    if (only_top) return kBins - 1;
    return (int)fminf((top - x) * per_bin, (float)(kBins - 1));
  }

  // rint(2^S 2^z): 2^z as 2^k e^r, |r| <= ln 2 / 2, by eleven terms of the exponential's
  // series (off by 7e-15), and a sum with 2^52, whose low bits are the integer.
  __device__ __forceinline__ u64 weight(float x) const {
    if (x == top) return 1ull << shift;
    const double z = ((double)x - (double)top) * c;
    if (only_top || x == -__builtin_inff() || !(z > -(double)(shift + 1))) return 0;
    const double k = __builtin_rint(z), r = (z - k) * 0.6931471805599453;
    double e = 1.0 / 39916800;
    e = __builtin_fma(e, r, 1.0 / 3628800);
    e = __builtin_fma(e, r, 1.0 / 362880);
    e = __builtin_fma(e, r, 1.0 / 40320);
    e = __builtin_fma(e, r, 1.0 / 5040);
    e = __builtin_fma(e, r, 1.0 / 720);
    e = __builtin_fma(e, r, 1.0 / 120);
    e = __builtin_fma(e, r, 1.0 / 24);
    e = __builtin_fma(e, r, 1.0 / 6);
    e = __builtin_fma(e, r, 0.5);
    e = __builtin_fma(e, r, 1.0);
    e = __builtin_fma(e, r, 1.0);
    const double v = __builtin_ldexp(e, (int)k + shift) + 4503599627370496.0;
    return __builtin_bit_cast(u64, v) & ((1ull << 52) - 1);
  }

  // The smallest weight that min-p keeps.
  __device__ __forceinline__ u64 least(float min_p) const {
    const double m = min_p > 1.0f ? 1.0 : min_p > 0.0f ? (double)min_p : 0.0;  // NaN: 0
    return (u64)__builtin_ceil(__builtin_ldexp(m, shift));
  }
};

// Ascending in the tokens' order.
__device__ __forceinline__ u64 order_of(float x, int index) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const unsigned rising = u & 0x80000000u ? ~u : u | 0x80000000u;
  return ((u64)~rising << kIndexBits) | (unsigned)index;
}

struct Shared {
  u64 sum[kBins];  // running sums once scanned
  u64 fine[kBins];
  u64 order[kList], weight[kList];
  unsigned count[kBins], fine_count[kBins];
  u64 wave_sum[kWaves];
  unsigned wave_count[kWaves];
  float wave_top[kWaves];
  u64 kept;
  // what the search found
  u64 at_sum;       // running sum up to and with it
  u64 base_sum;     // of what comes before a bin
  unsigned base_count, in_bin;
  int bin, index, listed;
};

template <class T>
__device__ __forceinline__ T shfl_up(T v, int by) {
  if constexpr (sizeof(T) == 8) {
    const unsigned lo = __shfl_up((unsigned)v, by, 64), hi = __shfl_up((unsigned)(v >> 32), by, 64);
    return ((u64)hi << 32) | lo;
  } else {
    return __shfl_up(v, by, 64);
  }
}

// a[2 t], a[2 t + 1] of each thread t become running sums over all 2 kThreads.
template <class T>
__device__ __forceinline__ void scan(T* a, T* waves) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const T a0 = a[2 * t], a1 = a[2 * t + 1];
  T s = a0 + a1;
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    const T o = shfl_up(s, by);
    if (lane >= by) s += o;
  }
  if (lane == 63) waves[wave] = s;
  __syncthreads();
  T before = 0;
  for (int w = 0; w < wave; ++w) before += waves[w];
  a[2 * t] = before + s - a1;
  a[2 * t + 1] = before + s;
  __syncthreads();
}

// The bin in which a scanned row of sums reaches `value`, which it does.
template <class T>
__device__ __forceinline__ void find_bin(Shared& s, const T* running, T value, const u64* sum, const unsigned* count) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 2 * threadIdx.x + i;
    const T before = b ? running[b - 1] : T(0);
    if (before < value && value <= running[b]) {
      s.bin = b;
      s.base_sum = b ? sum[b - 1] : 0;
      s.base_count = b ? count[b - 1] : 0;
      s.in_bin = count[b] - s.base_count;
    }
  }
  __syncthreads();
}

// The listed tokens in order.
__device__ __forceinline__ void sort_list(Shared& s, int n) {
  int size = 64;
  while (size < n) size *= 2;
  for (int i = threadIdx.x; i < size; i += kThreads)
    if (i >= n) {
      s.order[i] = ~0ull;
      s.weight[i] = 0;
    }
  __syncthreads();
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      const int t = threadIdx.x;
      if (t < size / 2) {
        const int a = 2 * j * (t / j) + t % j, b = a + j;
        const u64 x = s.order[a], y = s.order[b];
        if ((x > y) == ((a & k) == 0)) {
          s.order[a] = y;
          s.order[b] = x;
          const u64 wx = s.weight[a];
          s.weight[a] = s.weight[b];
          s.weight[b] = wx;
        }
      }
      __syncthreads();
    }
  for (int i = size + threadIdx.x; i < kList; i += kThreads) s.weight[i] = 0;
  __syncthreads();
}

// What the search remembers between its questions: bins lo to hi, of n tokens, listed in
// order, with base_sum and base_count before them (hi < 0: none).
struct Listed {
  int lo = 0, hi = -1, n = 0;
  u64 base_sum = 0;
  unsigned base_count = 0;
};

// The token at which the row's running sum (of weights, or BY_COUNT the number of tokens)
// reaches `value`, at least 1 and at most the whole: s.index, s.at_sum.
template <int ELEM, bool BY_COUNT>
__device__ __forceinline__ void search(Shared& s, const unsigned char* row, int vocab, const Weights& w, Listed& l, u64 value) {
  if constexpr (BY_COUNT) find_bin<unsigned>(s, s.count, (unsigned)value, s.sum, s.count);
  else find_bin<u64>(s, s.sum, value, s.sum, s.count);
  const int bin = s.bin;
  const u64 upto = s.sum[bin];
  const unsigned with = s.base_count + s.in_bin, in_bin = s.in_bin;
  u64 base_sum = s.base_sum;
  unsigned base_count = s.base_count;
  if (BY_COUNT && with == (unsigned)value) {  // it ends with the bin: whose token is last is not asked
    __syncthreads();
    if (threadIdx.x == 0) s.at_sum = upto;
    __syncthreads();
    return;
  }
  __syncthreads();
  if (bin < l.lo || bin > l.hi) {
    int shift = kIndexBits + 32;  // bits of the order not yet looked at
    u64 prefix = 0;
    unsigned n = in_bin;
    l.lo = l.hi = bin;
    if (with <= kList) {
      l.lo = 0;
      n = with;
      base_sum = 0;
      base_count = 0;
    }
    while (n > kList && shift > 0) {  // part the bin by the next bits
      const int next = max(shift - 11, 0);
      for (int i = threadIdx.x; i < kBins; i += kThreads) {
        s.fine[i] = 0;
        s.fine_count[i] = 0;
      }
      __syncthreads();
      each<ELEM>(row, 0, vocab, kThreads, [&](float x, int i) {
        if (w.bin(x) != bin) return;
        const u64 o = order_of(x, i);
        if ((o >> shift) != prefix) return;
        const int d = (int)(o >> next) & ((1 << (shift - next)) - 1);
        atomicAdd(&s.fine[d], w.weight(x));
        atomicAdd(&s.fine_count[d], 1u);
      });
      __syncthreads();
      scan(s.fine, s.wave_sum);
      scan(s.fine_count, s.wave_count);
      if constexpr (BY_COUNT) find_bin<unsigned>(s, s.fine_count, (unsigned)value - base_count, s.fine, s.fine_count);
      else find_bin<u64>(s, s.fine, value - base_sum, s.fine, s.fine_count);
      prefix = (prefix << (shift - next)) | (unsigned)s.bin;
      shift = next;
      base_sum += s.base_sum;
      base_count += s.base_count;
      n = s.in_bin;
      l.hi = -1;  // part of a bin serves no other question
      __syncthreads();
    }
    const int lo = l.lo;
    const bool whole = shift == kIndexBits + 32;
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    each<ELEM>(row, 0, vocab, kThreads, [&](float x, int i) {
      const int b = w.bin(x);
      if (b < lo || b > bin) return;
      const u64 o = order_of(x, i);
      if (!whole && (o >> shift) != prefix) return;
      const int at = atomicAdd(&s.listed, 1);
      if (at >= kList) return;  // as counted, there are no more
      s.order[at] = o;
      s.weight[at] = w.weight(x);
    });
    __syncthreads();
    l.n = (int)n;
    l.base_sum = base_sum;
    l.base_count = base_count;
    sort_list(s, l.n);
    scan(s.weight, s.wave_sum);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 2 * threadIdx.x + i;
    const u64 before = l.base_sum + (e ? s.weight[e - 1] : 0), with_it = l.base_sum + s.weight[e];
    const bool here = BY_COUNT ? l.base_count + e + 1 == (unsigned)value : before < value && value <= with_it;
    if (e < l.n && here) {
      s.index = (int)(s.order[e] & ((1u << kIndexBits) - 1));
      s.at_sum = with_it;
    }
  }
  __syncthreads();
}

// From a row's bins, in s.sum and s.count, and s.kept, the weight of what min-p keeps,
// the drawn token; every thread of the workgroup has it.
template <int ELEM>
__device__ __forceinline__ int pick(Shared& s, const unsigned char* row, int vocab, const Weights& w, int top_k, float top_p,
                                    float u) {
  scan(s.sum, s.wave_sum);
  scan(s.count, s.wave_count);
  Listed l;
  u64 kept = s.sum[kBins - 1];
  if (top_k > 0 && top_k < vocab) {
    search<ELEM, true>(s, row, vocab, w, l, (u64)top_k);
    kept = s.at_sum;
  }
  if (top_p < 1.0f) {  // NaN: all
    // the running sum before a kept token is below p of the total
    const u64 reach = top_p > 0.0f ? (u64)__builtin_ceil((double)top_p * (double)kept) : 1;
    search<ELEM, false>(s, row, vocab, w, l, min(max(reach, 1ull), kept));
    kept = min(kept, s.at_sum);
  }
  kept = min(kept, s.kept);
  const double share = u > 0.0f ? (double)u : 0.0;  // NaN: 0
  const u64 reach = share < 1.0 ? (u64)(share * (double)kept) + 1 : kept;
  search<ELEM, false>(s, row, vocab, w, l, min(reach, kept));
  return s.index;
}

template <int ELEM>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs p) {
  __shared__ Shared s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const RowAt at = row_at(p, blockIdx.x);
  const unsigned char* const row = p.x + (p.tx.at(at.x, at.y, at.z) + at.r * p.ldx) * (ELEM == kF32 ? 4 : 2);
  int* const out = p.y + p.ty.at(at.x, at.y, at.z) + at.r * p.ldy;
  for (int i = t; i < kBins; i += kThreads) {
    s.sum[i] = 0;
    s.count[i] = 0;
  }
  if (t == 0) s.kept = 0;
  float top = -__builtin_inff();
  each<ELEM>(row, 0, p.vocab, kThreads, [&](float x, int) { top = fmaxf(top, x); });
  top = wave_reduce<true>(top);
  if (lane == 0) s.wave_top[wave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) top = fmaxf(top, s.wave_top[i]);
  if (top == -__builtin_inff()) {
    if (t == 0) *out = -1;
    return;
  }
  Weights w;
  w.begin(top, at.in(p.temperature, p.tt, p.ldt, 1.0f), p.shift);
  const u64 least = w.least(at.in(p.min_p, p.tm, p.ldm, 0.0f));
  u64 kept = 0;
  each<ELEM>(row, 0, p.vocab, kThreads, [&](float x, int) {
    const u64 e = w.weight(x);
    const int b = w.bin(x);
    atomicAdd(&s.sum[b], e);
    atomicAdd(&s.count[b], 1u);
    if (e >= least) kept += e;
  });
  atomicAdd(&s.kept, kept);
  __syncthreads();
  const int token = pick<ELEM>(s, row, p.vocab, w, at.in(p.top_k, p.tk, p.ldk, 0), at.in(p.top_p, p.tp, p.ldp, 1.0f),
                               at.in(p.u, p.tu, p.ldu, 0.0f));
  if (t == 0) *out = token;
}

}  // namespace

hipError_t launch_sample(const xt::Plan& p, void* const* bufs, void* work, hipStream_t s, std::string& why) {
  (void)work;
  const xt::SamplePlan& t = p.sample;
  for (const xt::Access2D* in : {&t.x, &t.u, &t.extra[0], &t.extra[1], &t.extra[2], &t.extra[3]})
    if (in->arg >= 0 && !result_apart(p, bufs, t.y, *in, false, why)) return hipErrorInvalidValue;
  auto off = [](const xt::Access2D& a) { return TileOff{a.addr.c0, a.addr.sx, a.addr.sy, a.addr.sz}; };
  auto at = [&](const xt::Access2D& a) { return a.arg < 0 ? nullptr : bufs[a.arg]; };
  SampleArgs a{};
  a.x = static_cast<const unsigned char*>(at(t.x));
  a.u = static_cast<const float*>(at(t.u));
  a.temperature = static_cast<const float*>(at(t.extra[0]));
  a.top_k = static_cast<const int*>(at(t.extra[1]));
  a.top_p = static_cast<const float*>(at(t.extra[2]));
  a.min_p = static_cast<const float*>(at(t.extra[3]));
  a.y = static_cast<int*>(at(t.y));
  a.tx = off(t.x);
  a.tu = off(t.u);
  a.tt = off(t.extra[0]);
  a.tk = off(t.extra[1]);
  a.tp = off(t.extra[2]);
  a.tm = off(t.extra[3]);
  a.ty = off(t.y);
  a.ldx = t.x.ld;
  a.ldu = t.u.ld;
  a.ldt = t.extra[0].ld;
  a.ldk = t.extra[1].ld;
  a.ldp = t.extra[2].ld;
  a.ldm = t.extra[3].ld;
  a.ldy = t.y.ld;
  a.blocks = block_decode(p.grid[0], p.grid[1], false);
  a.rows = static_cast<int>(t.x.rows);
  a.per_block = div31(a.rows);
  a.vocab = static_cast<int>(t.x.cols);
  int bits = 0;
  while ((1LL << bits) < t.x.cols) ++bits;
  a.shift = std::min(50, 61 - bits);
  const long long rows = grid_blocks(p) * a.rows;  // below 2^22, as planned
  const unsigned wgs = static_cast<unsigned>(rows);
  switch (t.x.elem) {
    case xt::Elem::F32: sample_kernel<kF32><<<wgs, kThreads, 0, s>>>(a); break;
    case xt::Elem::F16: sample_kernel<kF16><<<wgs, kThreads, 0, s>>>(a); break;
    default: sample_kernel<kBF16><<<wgs, kThreads, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

}  // namespace xtk
