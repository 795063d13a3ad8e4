// A token of each row of logits (xtile_amd.dsl.sample states which).
//
// Weights are 64-bit integers, rint(2^S e^((x - max) / t)), the exponential's series off by
// 2.2e-13 of it (250 units at S = 50, none below 2^41): their sums are exact, so
// neither the order of additions nor the number of workgroups changes a result.  S leaves
// room for the sum of a row (S + log2 V < 62, and at most 50 for the conversion).  What rounds
// to no unit is left out: V 2^-(S + 1) of the largest weight at most, 2^-24 at 2^19 logits and
// 2^-18 at 2^22.
//
// What top-k, top-p and min-p leave is in each case a beginning of the tokens' order
// (largest logit first, equal ones by index), so what they leave together is the
// shortest of the three, and it is enough to know its weight.  The drawn token is then
// found as the cut of top-p is: the first at which the running sum reaches a value.
//
// The order is not made.  One pass takes the largest logit, a second counts and sums the
// tokens in kBins bins of their distance from it (for few top-k tokens it only counts), the
// next lists the few tokens of the bin in which the sum reaches the value (or of all bins up
// to there, if they are at most kHead, which then serve every question), and only those are
// sorted.
// A bin with too many is parted by 11 bits of the order's key (the logit's bits, then the
// index) as often as it takes, at most five times.
//
// What bounds it is the arithmetic of a row on one CU: a weight is some twenty 64-bit
// operations, so 32768 weights and their bins take 10 us there, against 3 for their loads; a
// scan of the bins takes 1, a list with its search 5.  Rows of few top-k tokens make no weights
// but those of a list of at most kList.  Few long rows are dealt to many workgroups in slices,
// a kernel for each pass (xt::sample_slices has the rule).  Replayed in a graph: 1 row of 32768
// logits, top-k 50 and top-p, 17 us, without cuts 23; 1 row of 131072, top-p, 31 to 38, top-k
// 50, 23; 256 rows of 32768 44; 64 rows of 131072, top-p and min-p, 59 to 63, of which the
// largest logit takes 8 (34 MB at 4 TB/s), the bins 18, the lists 18, and what is left of a row
// 17.  Where few tokens have a weight most logits are added to one bin, one after the other: of
// 1 row of 131072 23 to 27, of 64 of them 86 to 96, and with top-k, a workgroup a row, 130 to 262.
#include "launch.h"

#include <algorithm>

#include "common.h"

namespace xtk {
namespace {

enum { kF32 = 0, kF16 = 1, kBF16 = 2 };

typedef unsigned long long u64;

constexpr int kBins = 2048, kList = 2048;
constexpr int kIndexBits = 22;  // xt::kSampleVocab
constexpr u64 kAll = 1ull << 62;  // more than any sum: what is kept where nothing is dropped
static_assert(xt::kSampleVocab == 1LL << kIndexBits && kBins == kList, "");

struct RowWork;

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
  int slices;
  Div31 d_slices;
  RowWork* work;
};

struct RowAt {
  int x, y, z;
  long long r;
  template <class T>
  __device__ __forceinline__ const T* in(const T* base, const TileOff& t, long long ld) const {
    return base + t.at(x, y, z) + r * ld;
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

typedef unsigned u4a __attribute__((ext_vector_type(4), aligned(2)));

// Sixteen bytes' logits, n of them, at index i: four at a time to f4(values, index, n).
template <int ELEM, class F>
__device__ __forceinline__ void by_four(uint4v w, int i, int n, F f4) {
#pragma unroll
  for (int q = 0; q < (ELEM == kF32 ? 1 : 2); ++q) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (ELEM == kF32) {
        const unsigned u = w[e];  // a bit cast of the element itself would read element 0
        v[e] = __builtin_bit_cast(float, u);
      } else {
        const unsigned short h = (unsigned short)(w[2 * q + e / 2] >> (16 * (e % 2)));
        v[e] = ELEM == kF16 ? (float)__builtin_bit_cast(_Float16, h) : __builtin_bit_cast(float, (unsigned)h << 16);
      }
    }
    if (n > 4 * q) f4(v, i + 4 * q, min(n - 4 * q, 4));
  }
}

// The first n logits of sixteen bytes that the row may not have whole.
template <int ELEM>
__device__ __forceinline__ uint4v load_some(const unsigned char* row, int i, int n) {
  constexpr int N = ELEM == kF32 ? 4 : 8, ES = ELEM == kF32 ? 4 : 2;
  uint4v w = {0, 0, 0, 0};
  if (n >= N) return (uint4v)(*reinterpret_cast<const u4a*>(row + (long long)i * ES));
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < n) {
      if constexpr (ELEM == kF32) w[e] = *reinterpret_cast<const unsigned*>(row + (long long)(i + e) * ES);
      else w[e / 2] |= (unsigned)*reinterpret_cast<const unsigned short*>(row + (long long)(i + e) * ES) << (16 * (e % 2));
    }
  return w;
}

// Logits first to last - 1 of a row, dealt to `threads` threads, read at every pass.
template <int ELEM>
struct Read {
  static constexpr int kWide = ELEM == kF32 ? 8 : 4;  // loads that leave registers for a list
  const unsigned char* row;
  int first, last, threads;
  // f4(values, index, n) of four neighbours at a time, of which n are some; U loads on their
  // way at once.
  template <int U, class F>
  __device__ __forceinline__ void each4(F f4) const {
    constexpr int N = ELEM == kF32 ? 4 : 8, ES = ELEM == kF32 ? 4 : 2;
    int i = first + (int)threadIdx.x * N;
    for (; i + (U - 1) * threads * N + N <= last; i += U * threads * N) {
      uint4v w[U];
#pragma unroll
      for (int k = 0; k < U; ++k) w[k] = (uint4v)(*reinterpret_cast<const u4a*>(row + (long long)(i + k * threads * N) * ES));
      issue_fence();
#pragma unroll
      for (int k = 0; k < U; ++k) by_four<ELEM>(w[k], i + k * threads * N, N, f4);
    }
#pragma unroll 1
    for (; i < last; i += threads * N) {
      const int n = min(N, last - i);
      by_four<ELEM>(load_some<ELEM>(row, i, n), i, n, f4);
    }
  }
};

constexpr int kThreads = 1024;
constexpr int kHeld = 32768;  // logits of 16 bits that a row's workgroup keeps in registers, 32 a thread

// A row of at most kHeld of them, read once.
template <int ELEM>
struct Held {
  static constexpr int N = 8, PER = kHeld / (kThreads * N), kWide = 1;
  uint4v w[PER];
  int last;
  __device__ __forceinline__ void begin(const unsigned char* row, int vocab) {
    last = vocab;
#pragma unroll
    for (int k = 0; k < PER; ++k) w[k] = load_some<ELEM>(row, index(k), vocab - index(k));
  }
  static __device__ __forceinline__ int index(int k) { return (k * kThreads + (int)threadIdx.x) * N; }
  template <int U, class F>
  __device__ __forceinline__ void each4(F f4) const {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      // one piece's arithmetic at a time, and none kept for the next pass: so it has registers
      uint4v x = w[k];
      int i = index(k);
      asm volatile("" : "+v"(x), "+v"(i));
      if (i < last) by_four<ELEM>(x, i, min(N, last - i), f4);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// The largest of logits, over a workgroup of `threads`; minus infinity for none.  waves: a
// float a wave.
template <class X>
__device__ __forceinline__ float largest(const X& x, int threads, float* waves) {
  float top = -__builtin_inff();
  x.template each4<8>([&](const float (&v)[4], int, int n) {
    if (n == 4) {  // NaN is passed over
      top = fmaxf(fmaxf(top, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) top = fmaxf(top, v[e]);
    }
  });
  top = wave_reduce<true>(top);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = top;
  __syncthreads();
  for (int i = 0; i < threads / 64; ++i) top = fmaxf(top, waves[i]);
  return top + 0.0f;
}

// Tokens of the first bins that are listed together, and that top-k takes without the sums of
// all the others: a list of 256 is sorted in 2 us, of 512 in 4, of 2048 in 25.
constexpr int kHead = 256;

// Parameters of a row.
struct Asked {
  float temperature, top_p, u, min_p;
  int top_k;
  u64 least;  // of min-p: the smallest weight that it keeps
  __device__ __forceinline__ bool some(int vocab) const { return top_k > 0 && top_k < vocab; }
  __device__ __forceinline__ bool few(int vocab) const { return some(vocab) && top_k <= kHead; }
  // NaN: all
  __device__ __forceinline__ bool cuts() const { return top_p < 1.0f; }
  // the smallest running sum that ends what top-p keeps of `total`: before a kept token it is
  // below p of that
  __device__ __forceinline__ u64 cut(u64 total) const {
    const u64 reach = top_p > 0.0f ? (u64)__builtin_ceil((double)top_p * (double)total) : 1;
    return min(max(reach, (u64)1), total);
  }
  // the running sum that the drawn token of `kept` reaches
  __device__ __forceinline__ u64 drawn(u64 kept) const {
    const double share = u > 0.0f ? (double)u : 0.0;  // NaN: 0
    return min(share < 1.0 ? (u64)(share * (double)kept) + 1 : kept, kept);
  }
};

// All of them on their way at once: what is absent reads what is there.
__device__ __forceinline__ Asked asked_of(const SampleArgs& p, const RowAt& at) {
  const float* const u = at.in(p.u, p.tu, p.ldu);
  const int* const none = reinterpret_cast<const int*>(u);
  const float *const t = p.temperature ? at.in(p.temperature, p.tt, p.ldt) : u, *const top_p = p.top_p ? at.in(p.top_p, p.tp, p.ldp) : u,
              *const min_p = p.min_p ? at.in(p.min_p, p.tm, p.ldm) : u;
  const int* const k = p.top_k ? at.in(p.top_k, p.tk, p.ldk) : none;
  Asked a{*t, *top_p, *u, *min_p, *k, 0};
  if (!p.temperature) a.temperature = 1.0f;
  if (!p.top_p) a.top_p = 1.0f;
  if (!p.min_p) a.min_p = 0.0f;
  if (!p.top_k) a.top_k = 0;
  const double m = a.min_p > 1.0f ? 1.0 : a.min_p > 0.0f ? (double)a.min_p : 0.0;  // NaN: 0
  a.least = (u64)__builtin_ceil(__builtin_ldexp(m, p.shift));
  return a;
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
    // weights end at 2^-(S + 1); finite, so that no distance of 0 makes a NaN
    per_bin = fminf((float)(c * ((kBins - 1) / (double)(s + 2))), 1e38f);
  }

  // Never more for a larger logit: each step here is monotonic.
  __device__ __forceinline__ int bin(float x) const {
    return only_top ? (x == top ? 0 : kBins - 1) : bin_of_many(x);
  }
  __device__ __forceinline__ int bin_of_many(float x) const { return (int)fminf((top - x) * per_bin, (float)(kBins - 1)); }

  // The first tokens of the order, all that have a weight among them, from running counts: those
  // before the last bin, which begins where weights are a quarter.  At temperatures near float's
  // largest it begins at distances past float's range, and may have any.
  __device__ __forceinline__ int weighted(const unsigned* running, int vocab) const {
    return only_top || per_bin >= 1e-35f ? (int)running[kBins - 2] : vocab;
  }

  // A logit that no logit of bins up to `last` is below.
  __device__ __forceinline__ float least_of(int last) const {
    if (last >= kBins - 1 || !(per_bin > 0.0f)) return -__builtin_inff();
    if (only_top) return top;
    const float far = (float)(last + 1) / per_bin;  // three roundings of 2^-24 in bin and here
    return top - far * 1.000001f - fabsf(top) * 2.4e-7f - 1e-37f;
  }

  // A logit that no logit of bins from `first` on is above.
  __device__ __forceinline__ float most_of(int first) const {
    if (first <= 0) return __builtin_inff();
    if (only_top) return top;
    const float far = (float)first / per_bin;
    return top - far * 0.999999f + fabsf(top) * 2.4e-7f + 1e-37f;
  }

  // rint(2^S 2^z): 2^z as 2^k 2^r, |r| <= 1/2, by eleven terms of its series (off by
  // 2.2e-13), and a sum with 2^52, whose low bits are the integer.
  __device__ __forceinline__ u64 weight(float x) const {
    return only_top ? (x == top ? 1ull << shift : 0) : weight_of_many(x);
  }
  __device__ __forceinline__ u64 weight_of_many(float x) const {
    const double z = ((double)x - (double)top) * c;
    // z to the nearest integer in the low bits of a sum with 3 2^51
    const double sum = z + 6755399441055744.0, r = z - (sum - 6755399441055744.0);
    double e = 7.054911620801121e-09;  // (ln 2)^10 / 10!, and so on
    e = __builtin_fma(e, r, 1.0178086009239696e-07);
    e = __builtin_fma(e, r, 1.3215486790144305e-06);
    e = __builtin_fma(e, r, 1.5252733804059838e-05);
    e = __builtin_fma(e, r, 0.00015403530393381606);
    e = __builtin_fma(e, r, 0.0013333558146428441);
    e = __builtin_fma(e, r, 0.009618129107628477);
    e = __builtin_fma(e, r, 0.055504108664821576);
    e = __builtin_fma(e, r, 0.2402265069591007);
    e = __builtin_fma(e, r, 0.6931471805599453);
    e = __builtin_fma(e, r, 1.0);
    const u64 bits = __builtin_bit_cast(u64, e) + ((u64)(__builtin_bit_cast(unsigned, (int)__builtin_bit_cast(u64, sum)) + shift) << 52);
    const double v = __builtin_bit_cast(double, bits) + 4503599627370496.0;
    const u64 w = __builtin_bit_cast(u64, v) & ((1ull << 52) - 1);
    return z > -(double)(shift + 1) ? w : 0;  // minus infinity, and NaN of it: 0
  }
};

// Ascending in the tokens' order.
__device__ __forceinline__ u64 order_of(float x, int index) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const unsigned rising = u & 0x80000000u ? ~u : u | 0x80000000u;
  return ((u64)~rising << kIndexBits) | (unsigned)index;
}

template <class T>
__device__ __forceinline__ T shfl_up(T v, int by) {
  if constexpr (sizeof(T) == 8) {
    const unsigned lo = __shfl_up((unsigned)v, by, 64), hi = __shfl_up((unsigned)(v >> 32), by, 64);
    return ((u64)hi << 32) | lo;
  } else {
    return __shfl_up(v, by, 64);
  }
}

// Running sums over a wave: the last lane has the whole.
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    const T o = shfl_up(v, by);
    if ((int)(threadIdx.x & 63) >= by) v += o;
  }
  return v;
}

// The kBins values of `a` and, where there is one, of `b`, of THREADS threads, become running
// sums.  mem: eight bytes and four a wave.
template <int THREADS>
struct ScanMem {
  u64 a[THREADS / 64];
  unsigned b[THREADS / 64];
};
template <int THREADS, bool A, bool B>
__device__ __forceinline__ void scan(u64* a, unsigned* b, ScanMem<THREADS>& mem) {
  constexpr int PER = kBins / THREADS;
  const int t = threadIdx.x, wave = t >> 6;
  u64 v[PER], s = 0;
  unsigned u[PER], c = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if constexpr (A) v[i] = s += a[PER * t + i];
    if constexpr (B) u[i] = c += b[PER * t + i];
  }
  u64 upto = s;
  unsigned upto_c = c;
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    u64 o = 0;
    unsigned oc = 0;
    if constexpr (A) o = shfl_up(upto, by);
    if constexpr (B) oc = shfl_up(upto_c, by);
    if ((t & 63) >= by) {
      upto += o;
      upto_c += oc;
    }
  }
  if ((t & 63) == 63) {
    if constexpr (A) mem.a[wave] = upto;
    if constexpr (B) mem.b[wave] = upto_c;
  }
  __syncthreads();
  u64 before = upto - s;
  unsigned before_c = upto_c - c;
#pragma unroll
  for (int w = 0; w < THREADS / 64 - 1; ++w) {
    if constexpr (A) before += w < wave ? mem.a[w] : 0;
    if constexpr (B) before_c += w < wave ? mem.b[w] : 0;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if constexpr (A) a[PER * t + i] = before + v[i];
    if constexpr (B) b[PER * t + i] = before_c + u[i];
  }
  __syncthreads();
}

// The bin in which running sums reach `value`, which they do, in every thread.  `turn`: each
// question's answer lies apart from the one before, which threads may still read.
struct Found {
  int at[2];
};
template <int THREADS, class T>
__device__ __forceinline__ int bin_with(const T* running, T value, Found& found, int& turn) {
  constexpr int PER = kBins / THREADS;
  int* const at = &found.at[turn ^= 1];
  T before = threadIdx.x ? running[PER * threadIdx.x - 1] : T(0);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const T upto = running[PER * threadIdx.x + i];
    if (before < value && value <= upto) *at = PER * threadIdx.x + i;
    before = upto;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*at);
}

// The same of two values, the first at most the second.
struct FoundBoth {
  int at[2][2];
};
template <int THREADS>
__device__ __forceinline__ void bins_with(const u64* running, u64 low, u64 high, FoundBoth& found, int& turn, int& lo, int& hi) {
  constexpr int PER = kBins / THREADS;
  int* const at = found.at[turn ^= 1];
  u64 before = threadIdx.x ? running[PER * threadIdx.x - 1] : 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const u64 upto = running[PER * threadIdx.x + i];
    if (before < low && low <= upto) at[0] = PER * threadIdx.x + i;
    if (before < high && high <= upto) at[1] = PER * threadIdx.x + i;
    before = upto;
  }
  __syncthreads();
  lo = __builtin_amdgcn_readfirstlane(at[0]);
  hi = __builtin_amdgcn_readfirstlane(at[1]);
}

// Adds logits to the bins, in LDS: counts, and with SUMS weights and, where
// there is a min-p (KEPT), to `kept` those of what it keeps.  MANY: not only the largest have
// weights; these are questions for a whole row, and a branch for each logit would keep the
// arithmetic of one from filling another's waits.
template <bool SUMS, bool KEPT, bool MANY, class X>
__device__ __forceinline__ void add_bins_of(const X& logits, const Weights& w, u64 least, u64* sum, unsigned* count, u64* kept) {
  u64 mine = 0;
  logits.template each4<4>([&](const float (&v)[4], int, int n) {
    int b[4];
    u64 is[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = clean(v[e]);
      b[e] = MANY ? w.bin_of_many(x) : w.bin(x);
      if constexpr (SUMS) is[e] = MANY ? w.weight_of_many(x) : w.weight(x);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= n) break;
      atomicAdd(&count[b[e]], 1u);
      if constexpr (SUMS) {
        atomicAdd(&sum[b[e]], is[e]);
        if constexpr (KEPT) mine += is[e] >= least ? is[e] : 0;
      }
    }
  });
  if constexpr (KEPT) {
    mine = wave_scan(mine);
    if ((threadIdx.x & 63) == 63) atomicAdd(kept, mine);
  }
}

template <class X>
__device__ __forceinline__ void add_bins(const X& logits, const Weights& w, bool sums, u64 least, u64* sum, unsigned* count,
                                         u64* kept) {
  if (w.only_top) {
    add_bins_of<true, true, false>(logits, w, least, sum, count, kept);
  } else if (!sums) {
    add_bins_of<false, false, true>(logits, w, least, sum, count, kept);
  } else if (least) {
    add_bins_of<true, true, true>(logits, w, least, sum, count, kept);
  } else {
    add_bins_of<true, false, true>(logits, w, least, sum, count, kept);
    if (threadIdx.x == 0) *kept = kAll;
  }
}

// Bins lo to hi of a row's logits; none of them where lo > hi.
struct Between {
  int lo, hi;
  float least, most;  // no logit of them is outside; minus infinity stands for NaN too
  __device__ __forceinline__ void begin(const Weights& w, int l, int h) {
    lo = l;
    hi = h;
    least = l > h ? w.top : w.least_of(h);
    most = l > h ? w.top : w.most_of(l);
  }
  __device__ __forceinline__ bool tail() const { return least == -__builtin_inff(); }
};

// give(run, order, logit) of each logit that lies in one of R runs of bins.
template <class X, int R, class F>
__device__ __forceinline__ void each_in(const X& logits, const Weights& w, const Between (&run)[R], F give) {
  bool tail = false;
#pragma unroll
  for (int q = 0; q < R; ++q) tail |= run[q].tail();
  logits.template each4<X::kWide>([&](const float (&v)[4], int i, int n) {
    // of a wave's 256 few are among them: between two is what is the median of the three
    bool in[4] = {tail, tail, tail, tail};
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] |= __builtin_amdgcn_fmed3f(v[e], run[q].least, run[q].most) == v[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!in[e] || e >= n) continue;
      const float x = clean(v[e]);
      const int b = w.bin(x);
#pragma unroll
      for (int q = 0; q < R; ++q)
        if (b >= run[q].lo && b <= run[q].hi) give(q, order_of(x, i + e), x);
    }
  });
}

// A list of tokens with their weights, which become running sums once it is in order.
struct List {
  alignas(16) u64 order[kList + 2];
  u64 weight[kList];
  unsigned rank[1024];
  ScanMem<1024> mem;
  u64 at_sum;  // what a search found: the running sum up to and with it
  int index;
  int n;
};

// The first n tokens in order, by 1024 threads.
__device__ __forceinline__ void sort_list(List& s, int n) {
  constexpr int kThreads = 1024;
  const int t = threadIdx.x;
  if (n <= 1024) {
    // each token's place is the number of those before it, which one to sixteen threads count
    const int size = n <= 64 ? 64 : n <= 256 ? 256 : n <= 512 ? 512 : 1024, parts = kThreads / size, i = t % size, part = t / size;
    const int each = ((n + parts - 1) / parts + 1) & ~1;
    const u64 mine = i < n ? s.order[i] : ~0ull, weight = i < n ? s.weight[i] : 0;
    s.rank[t] = 0;
    if (t == 0 && n % 2) s.order[n] = ~0ull;  // two are read at a time
    __syncthreads();
    // compared as doubles, in half the time: orders are below 2^54, whose doubles rise as they do
    const double key = __builtin_bit_cast(double, mine);
    unsigned before = 0;
#pragma unroll 4
    for (int j = part * each; j < min(n, (part + 1) * each); j += 2) {
      const double2 o = *reinterpret_cast<const double2*>(s.order + j);
      before += (o.x < key) + (o.y < key);
    }
    if (i < n && before) atomicAdd(&s.rank[i], before);
    __syncthreads();
    const int at = i < n ? (int)s.rank[i] : i;
    if (part == 0) {
      s.order[at] = mine;
      s.weight[at] = weight;
    }
    for (int e = size + t; e < kList; e += kThreads) s.weight[e] = 0;
    __syncthreads();
  } else {
    const int size = kList;
    for (int i = t; i < kList; i += kThreads)
      if (i >= n) {
        s.order[i] = ~0ull;
        s.weight[i] = 0;
      }
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
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
  }
  scan<kThreads, true, false>(s.weight, nullptr, s.mem);
}

// The token of a sorted list of n, base_sum before it, at which the running sum reaches `value`.
__device__ __forceinline__ void search_list(List& s, int n, u64 base_sum, u64 value) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 2 * threadIdx.x + i;
    const u64 before = base_sum + (e ? s.weight[e - 1] : 0), with_it = base_sum + s.weight[e];
    if (e < n && before < value && value <= with_it) {
      s.index = (int)(s.order[e] & ((1u << kIndexBits) - 1));
      s.at_sum = with_it;
    }
  }
  __syncthreads();
}

// The drawn token from a sorted list of the first n tokens, which has all that remains: top-k of
// them, or all that have a weight.
__device__ __forceinline__ int pick_few(List& s, int n, const Asked& a) {
  const u64 total = s.weight[min(a.top_k, n) - 1];
  u64 kept = total;
  if (a.least > 0) {  // min-p: the running sum before the first token that it does not keep
    if (threadIdx.x == 0) s.n = n;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int e = 2 * threadIdx.x + i;
      if (e < n && s.weight[e] - (e ? s.weight[e - 1] : 0) < a.least) atomicMin(&s.n, e);
    }
    __syncthreads();
    kept = min(kept, s.weight[s.n - 1]);  // the first one is kept
  }
  if (a.cuts()) {
    search_list(s, n, 0, a.cut(total));
    kept = min(kept, s.at_sum);
    __syncthreads();
  }
  search_list(s, n, 0, a.drawn(kept));
  return s.index;
}

// A workgroup's memory for one row.  Bins are parted in the list's place.
struct Shared {
  u64 sum[kBins];  // running sums once scanned
  unsigned count[kBins];
  union {
    List list;
    struct {
      u64 sum[kBins];
      unsigned count[kBins];
    } fine;
  };
  ScanMem<1024> mem;
  float top[16];
  u64 kept;  // the weight of what min-p keeps
  Found found;
};

// Tokens of bins lo to hi, whose order begins with `prefix` above `shift` bits, n of them, listed
// in order.
template <class X>
__device__ __forceinline__ void make_list(Shared& s, const X& logits, const Weights& w, int lo, int hi, int shift, u64 prefix,
                                          int n) {
  if (threadIdx.x == 0) s.list.n = 0;
  __syncthreads();
  Between run[1];
  run[0].begin(w, lo, hi);
  each_in(logits, w, run, [&](int, u64 o, float x) {
    if ((o >> shift) != prefix) return;
    const int at = atomicAdd(&s.list.n, 1);
    if (at >= kList) return;  // as counted, there are no more
    s.list.order[at] = o;
    s.list.weight[at] = w.weight(x);
  });
  __syncthreads();
  sort_list(s.list, n);
}

// What the search remembers between its questions: bins lo to hi, of n tokens, listed in
// order, with base_sum before them (hi < 0: none).
struct Listed {
  int lo = 0, hi = -1, n = 0;
  u64 base_sum = 0;
  unsigned base_count = 0;
  int turn = 0;
};

// The token at which the row's running sum (of weights, or BY_COUNT the number of tokens)
// reaches `value`, at least 1 and at most the whole: s.list.index, and the running sum up to
// and with it.
template <bool BY_COUNT, class X>
__device__ __forceinline__ u64 search(Shared& s, const X& logits, const Weights& w, Listed& l, u64 value) {
  int bin;
  if constexpr (BY_COUNT) bin = bin_with<kThreads, unsigned>(s.count, (unsigned)value, s.found, l.turn);
  else bin = bin_with<kThreads, u64>(s.sum, value, s.found, l.turn);
  const unsigned with = s.count[bin];
  // whose token is last is not asked, nor which of those that add nothing
  if (BY_COUNT && (with == (unsigned)value || s.sum[bin] == (bin ? s.sum[bin - 1] : 0))) return s.sum[bin];
  if (bin < l.lo || bin > l.hi) {
    int shift = kIndexBits + 32;  // bits of the order not yet looked at
    u64 prefix = 0, base_sum = bin ? s.sum[bin - 1] : 0;
    unsigned base_count = bin ? s.count[bin - 1] : 0, n = with - base_count;
    l.lo = l.hi = bin;
    if (with <= kHead) {
      l.lo = 0;
      n = with;
      base_sum = 0;
      base_count = 0;
    }
    const int lo = l.lo;
    while (n > kList && shift > 0) {  // part the bin by the next bits
      const int next = max(shift - 11, 0);
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += kThreads) {
        s.fine.sum[i] = 0;
        s.fine.count[i] = 0;
      }
      __syncthreads();
      Between run[1];
      run[0].begin(w, bin, bin);
      each_in(logits, w, run, [&](int, u64 o, float x) {
        if ((o >> shift) != prefix) return;
        const int d = (int)(o >> next) & ((1 << (shift - next)) - 1);
        atomicAdd(&s.fine.sum[d], w.weight(x));
        atomicAdd(&s.fine.count[d], 1u);
      });
      __syncthreads();
      scan<kThreads, true, true>(s.fine.sum, s.fine.count, s.mem);
      int d;
      if constexpr (BY_COUNT) d = bin_with<kThreads, unsigned>(s.fine.count, (unsigned)value - base_count, s.found, l.turn);
      else d = bin_with<kThreads, u64>(s.fine.sum, value - base_sum, s.found, l.turn);
      prefix = (prefix << (shift - next)) | (unsigned)d;
      shift = next;
      n = s.fine.count[d] - (d ? s.fine.count[d - 1] : 0);
      base_sum += d ? s.fine.sum[d - 1] : 0;
      base_count += d ? s.fine.count[d - 1] : 0;
      l.hi = -1;  // part of a bin serves no other question
    }
    l.n = (int)n;
    l.base_sum = base_sum;
    l.base_count = base_count;
    __syncthreads();
    make_list(s, logits, w, lo, bin, shift, prefix, l.n);
  }
  if constexpr (BY_COUNT) {
    const int at = (int)((unsigned)value - l.base_count) - 1;
    return l.base_sum + s.list.weight[at];
  } else {
    search_list(s.list, l.n, l.base_sum, value);
    const u64 sum = s.list.at_sum;
    __syncthreads();
    return sum;
  }
}

// From a row's bins, in s.count and, but for few top-k tokens, s.sum, and s.kept, the drawn
// token; every thread of the workgroup has it.
template <class X>
__device__ __forceinline__ int pick(Shared& s, const X& logits, int vocab, const Weights& w, const Asked& a) {
  Listed l;
  if (a.few(vocab)) {
    scan<kThreads, false, true>(nullptr, s.count, s.mem);
    const int k = min(a.top_k, w.weighted(s.count, vocab));
    const int bin = bin_with<kThreads, unsigned>(s.count, (unsigned)k, s.found, l.turn);
    const int with = (int)s.count[bin];
    if (with <= kList) {
      make_list(s, logits, w, 0, bin, kIndexBits + 32, 0, with);
      return pick_few(s.list, with, a);
    }
    // thousands of nearly equal ones: with the weights of all
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.sum[i] = 0;
      s.count[i] = 0;
    }
    if (threadIdx.x == 0) s.kept = 0;
    __syncthreads();
    add_bins(logits, w, true, a.least, s.sum, s.count, &s.kept);
    __syncthreads();
  }
  scan<kThreads, true, true>(s.sum, s.count, s.mem);
  u64 kept = s.sum[kBins - 1];
  if (a.some(vocab)) kept = search<true>(s, logits, w, l, (u64)a.top_k);
  if (a.cuts()) kept = min(kept, search<false>(s, logits, w, l, a.cut(kept)));
  search<false>(s, logits, w, l, a.drawn(min(kept, s.kept)));
  return s.list.index;
}

template <int ELEM>
__device__ __forceinline__ const unsigned char* logits_of(const SampleArgs& p, const RowAt& at) {
  return p.x + (p.tx.at(at.x, at.y, at.z) + at.r * p.ldx) * (ELEM == kF32 ? 4 : 2);
}

__device__ __forceinline__ Weights weights_of(const SampleArgs& p, const Asked& a, float top) {
  Weights w;
  w.begin(top, a.temperature, p.shift);
  return w;
}

__device__ __forceinline__ void put_token(const SampleArgs& p, const RowAt& at, int token) {
  if (threadIdx.x == 0) p.y[p.ty.at(at.x, at.y, at.z) + at.r * p.ldy] = token;
}

// A row's bins by one workgroup, then its token.
template <class X>
__device__ __forceinline__ int sample_row(const SampleArgs& p, const X& logits, const Asked& a, Shared& s, float top) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.sum[i] = 0;
    s.count[i] = 0;
  }
  if (threadIdx.x == 0) s.kept = 0;
  const Weights w = weights_of(p, a, top);
  __syncthreads();
  add_bins(logits, w, !a.few(p.vocab), a.least, s.sum, s.count, &s.kept);
  __syncthreads();
  return pick(s, logits, p.vocab, w, a);
}

// A workgroup a row; HELD: of at most kHeld logits, which it keeps.
template <int ELEM, bool HELD>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs p) {
  __shared__ Shared s;
  const RowAt at = row_at(p, blockIdx.x);
  const Asked a = asked_of(p, at);
  auto token = [&](const auto& logits) {
    const float top = largest(logits, kThreads, s.top);
    put_token(p, at, top == -__builtin_inff() ? -1 : sample_row(p, logits, a, s, top));
  };
  if constexpr (HELD) {
    Held<ELEM> logits;
    logits.begin(logits_of<ELEM>(p, at), p.vocab);
    token(logits);
  } else {
    token(Read<ELEM>{logits_of<ELEM>(p, at), 0, p.vocab, kThreads});
  }
}

// Few rows: a row's slices have workgroups of their own, in three kernels.  The largest logit
// of each; the bins of each, added to the row's; and the tokens of the bins in which the
// ends of top-k's and top-p's beginnings and the drawn token lie: three runs, the second
// and third from the least to the most that the one before can leave, or the first bins as
// one.  Then a workgroup a row sorts those.  Where a run is too long the last kernel has the
// row to itself.
constexpr int kSliceThreads = 512;
constexpr int kNear = 680;  // tokens of a run that a slice keeps in LDS until it hands them on

struct Run {
  int lo, hi, n;       // bins, tokens
  unsigned base_count;  // before them
  u64 base_sum;
};

// A row's part of the workspace.
struct RowWork {
  u64 sum[kBins];
  unsigned count[kBins];
  u64 order[3][kList], weight[3][kList];  // the runs' tokens
  Run run[3];                              // 0 tokens: none
  u64 kept;   // the weight of what min-p keeps
  u64 total;  // and of what top-k does, where that is known without a list
  int listed[3];
  int alone;  // the last kernel has the row to itself
  u64 unused;
  float top[xt::kSampleSlices];
};
static_assert(sizeof(RowWork) == xt::kSampleRowWork && sizeof(RowWork) % 16 == 0, "as planned");

// Logits [first, last) of a slice: whole runs of eight but for the last one's.
__device__ __forceinline__ void slice_of(const SampleArgs& p, int slice, int& first, int& last) {
  const int each = ((int)p.d_slices((unsigned)(p.vocab + p.slices - 1)) + 7) & ~7;
  first = min(slice * each, p.vocab);
  last = min(first + each, p.vocab);
}

template <int ELEM>
__global__ __launch_bounds__(kSliceThreads) void sample_top_kernel(SampleArgs p) {
  __shared__ float waves[kSliceThreads / 64];
  const int r = (int)p.d_slices(blockIdx.x), slice = blockIdx.x - r * p.slices;
  const RowAt at = row_at(p, r);
  RowWork& work = p.work[r];
  for (int i = slice * kSliceThreads + threadIdx.x; i < kBins; i += p.slices * kSliceThreads) {
    work.sum[i] = 0;
    work.count[i] = 0;
  }
  int first, last;
  slice_of(p, slice, first, last);
  const float top = largest(Read<ELEM>{logits_of<ELEM>(p, at), first, last, kSliceThreads}, kSliceThreads, waves);
  if (threadIdx.x == 0) {
    work.top[slice] = top;
    if (slice == 0) {
      work.kept = 0;
      work.listed[0] = work.listed[1] = work.listed[2] = 0;
    }
  }
}

__device__ __forceinline__ float top_of(const SampleArgs& p, const RowWork& work) {
  const int lane = threadIdx.x & 63;
  return wave_reduce<true>(lane < p.slices ? work.top[lane] : -__builtin_inff());
}

template <class T>
__device__ __forceinline__ T add_to(T* at, T v) {
  return __hip_atomic_fetch_add(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int ELEM>
__global__ __launch_bounds__(kSliceThreads) void sample_bins_kernel(SampleArgs p) {
  __shared__ u64 sum[kBins];
  __shared__ unsigned count[kBins];
  __shared__ u64 kept;
  const int r = (int)p.d_slices(blockIdx.x), slice = blockIdx.x - r * p.slices;
  const RowAt at = row_at(p, r);
  RowWork& work = p.work[r];
  const Asked a = asked_of(p, at);
  const float top = top_of(p, work);
  if (top == -__builtin_inff()) return;
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads) {
    sum[i] = 0;
    count[i] = 0;
  }
  if (threadIdx.x == 0) kept = 0;
  __syncthreads();
  const Weights w = weights_of(p, a, top);
  int first, last;
  slice_of(p, slice, first, last);
  const bool few = a.few(p.vocab);
  add_bins(Read<ELEM>{logits_of<ELEM>(p, at), first, last, kSliceThreads}, w, !few, a.least, sum, count, &kept);
  __syncthreads();
  // integers: in whatever order they are added, the sums are the same
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads)
    if (count[i]) {
      add_to(&work.count[i], count[i]);
      if (!few && sum[i]) add_to(&work.sum[i], sum[i]);
    }
  if (!few && threadIdx.x == 0) {
    if (a.least || w.only_top) add_to(&work.kept, kept);
    else if (slice == 0) work.kept = kAll;
  }
}

template <int ELEM>
__global__ __launch_bounds__(kSliceThreads) void sample_list_kernel(SampleArgs p) {
  __shared__ u64 sum[kBins];
  __shared__ unsigned count[kBins];
  __shared__ ScanMem<kSliceThreads> mem;
  __shared__ Found found;
  __shared__ FoundBoth both;
  __shared__ int near[3], far[3];
  const int r = (int)p.d_slices(blockIdx.x), slice = blockIdx.x - r * p.slices;
  const RowAt at = row_at(p, r);
  RowWork& work = p.work[r];
  const Asked a = asked_of(p, at);
  const float top = top_of(p, work);
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads) {
    sum[i] = work.sum[i];
    count[i] = work.count[i];
  }
  if (top == -__builtin_inff()) return;
  const bool few = a.few(p.vocab);
  const Weights w = weights_of(p, a, top);
  int turn = 0;
  if (threadIdx.x < 3) near[threadIdx.x] = 0;
  __syncthreads();
  scan<kSliceThreads, true, true>(sum, count, mem);
  auto run_of = [&](int lo, int hi) {
    const unsigned before = lo ? count[lo - 1] : 0;
    return Run{lo, hi, (int)(count[hi] - before), before, lo ? sum[lo - 1] : 0};
  };
  auto before_bin = [&](int b) { return b ? sum[b - 1] : 0; };
  Run run[3] = {{0, 0, 0, 0, 0}, {0, 0, 0, 0, 0}, {0, 0, 0, 0, 0}};
  u64 total = sum[kBins - 1];
  if (few) {
    const int k = min(a.top_k, w.weighted(count, p.vocab));
    run[0] = run_of(0, bin_with<kSliceThreads, unsigned>(count, (unsigned)k, found, turn));
  } else {
    // the least and the most that top-k, top-p and min-p leave
    u64 low = total, high = total;
    bool head = false;  // a run of the first bins, which has whatever comes
    if (a.some(p.vocab)) {
      const int b = bin_with<kSliceThreads, unsigned>(count, (unsigned)a.top_k, found, turn);
      total = high = sum[b];
      // the whole bin, or one without a weight, of which no token adds to those before it
      if (count[b] == (unsigned)a.top_k || before_bin(b) == high) {
        low = high;
      } else {
        low = before_bin(b) + 1;
        run[0] = run_of(b, b);
      }
    }
    if (a.cuts()) {
      int lo, hi;
      bins_with<kSliceThreads>(sum, a.cut(low), a.cut(high), both, turn, lo, hi);
      head = count[hi] <= kHead;
      run[1] = run_of(head ? 0 : lo, hi);
      low = min(low, before_bin(lo) + 1);
      high = min(high, sum[hi]);
    }
    const u64 by_min = work.kept;
    if (!head) {
      int lo, hi;
      bins_with<kSliceThreads>(sum, a.drawn(min(low, by_min)), a.drawn(min(high, by_min)), both, turn, lo, hi);
      run[2] = run_of(count[hi] <= kHead ? 0 : lo, hi);
    }
  }
  const bool alone = run[0].n > kList || run[1].n > kList || run[2].n > kList;
  if (slice == 0 && threadIdx.x == 0) {
    for (int q = 0; q < 3; ++q) work.run[q] = run[q];
    work.total = total;
    work.alone = alone;
  }
  if (alone) return;
  // the runs' tokens of this slice, in the bins' place, then handed on together; what does not
  // fit goes by itself
  __syncthreads();
  float* const logits = reinterpret_cast<float*>(count);
  static_assert(3 * kNear <= kBins, "the bins' place");
  auto hand_on = [&](int q, int to, u64 o, float x) {
    if (to >= kList) return;  // as counted, there are no more
    work.order[q][to] = o;
    work.weight[q][to] = w.weight(x);
  };
  int first, last;
  slice_of(p, slice, first, last);
  auto take = [&](int q, u64 o, float x) {
    const int to = atomicAdd(&near[q], 1);
    if (to < kNear) {
      sum[q * kNear + to] = o;
      logits[q * kNear + to] = x;
    } else {
      hand_on(q, add_to(&work.listed[q], 1), o, x);
    }
  };
  Between in[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) in[q].begin(w, run[q].lo, run[q].n ? run[q].hi : -1);
  each_in(Read<ELEM>{logits_of<ELEM>(p, at), first, last, kSliceThreads}, w, in, take);
  __syncthreads();
  if (threadIdx.x < 3) {
    const int n = min(near[threadIdx.x], kNear);
    far[threadIdx.x] = n ? add_to(&work.listed[threadIdx.x], n) : 0;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 3; ++q)
    for (int i = threadIdx.x; i < min(near[q], kNear); i += kSliceThreads)
      hand_on(q, far[q] + i, sum[q * kNear + i], logits[q * kNear + i]);
}

template <int ELEM>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs p) {
  __shared__ Shared s;
  const RowAt at = row_at(p, blockIdx.x);
  const RowWork& work = p.work[blockIdx.x];
  const Asked a = asked_of(p, at);
  const float top = top_of(p, work);
  if (top == -__builtin_inff()) {
    put_token(p, at, -1);
    return;
  }
  if (work.alone) {
    put_token(p, at, sample_row(p, Read<ELEM>{logits_of<ELEM>(p, at), 0, p.vocab, kThreads}, a, s, top));
    return;
  }
  // the runs' tokens, on their way together
  constexpr int PER = kList / kThreads;
  u64 order[3][PER], weight[3][PER];
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = threadIdx.x + e * kThreads;
      const bool in = i < work.run[q].n;
      order[q][e] = in ? work.order[q][i] : 0;
      weight[q][e] = in ? work.weight[q][i] : 0;
    }
  auto take = [&](int q) {
    __syncthreads();
    const int n = work.run[q].n;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      s.list.order[threadIdx.x + e * kThreads] = order[q][e];
      s.list.weight[threadIdx.x + e * kThreads] = weight[q][e];
    }
    __syncthreads();
    sort_list(s.list, n);
    return n;
  };
  if (a.few(p.vocab)) {
    const int n = take(0);
    put_token(p, at, pick_few(s.list, n, a));
    return;
  }
  u64 total = work.total;
  if (work.run[0].n) {
    take(0);
    total = work.run[0].base_sum + s.list.weight[a.top_k - (int)work.run[0].base_count - 1];
  }
  u64 kept = min(total, work.kept);
  int q = 2;
  if (work.run[1].n) {
    const int n = take(1);
    search_list(s.list, n, work.run[1].base_sum, a.cut(total));
    kept = min(kept, s.list.at_sum);
    if (!work.run[2].n) q = 1;
    __syncthreads();
  }
  int n = work.run[1].n;
  if (q == 2) n = take(2);
  search_list(s.list, n, work.run[q].base_sum, a.drawn(kept));
  put_token(p, at, s.list.index);
}

template <int ELEM>
hipError_t run(const SampleArgs& a, unsigned rows, hipStream_t s) {
  if (a.slices == 1) {
    // Rows of 16 bits are kept where they fit and are not short: 1 of 32000 without cuts 22.2 us
    // against 25.9 read at every pass, 16 of 30000 with top-k 50 16.8 against 20.6, 256 of 20000
    // with top-p 32.3 against 33.1, 1 of 8192 18.5 against 18.6, of 2000 17.6 against 16.7.  Of
    // 32 bits they take registers that the arithmetic needs: 256 of 32768 47 against 43.
    if constexpr (ELEM != kF32)
      if (a.vocab > 8192 && a.vocab <= kHeld) {
        sample_row_kernel<ELEM, true><<<rows, kThreads, 0, s>>>(a);
        return hipGetLastError();
      }
    sample_row_kernel<ELEM, false><<<rows, kThreads, 0, s>>>(a);
    return hipGetLastError();
  }
  sample_top_kernel<ELEM><<<rows * a.slices, kSliceThreads, 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  sample_bins_kernel<ELEM><<<rows * a.slices, kSliceThreads, 0, s>>>(a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  sample_list_kernel<ELEM><<<rows * a.slices, kSliceThreads, 0, s>>>(a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  sample_pick_kernel<ELEM><<<rows, kThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const xt::Plan& p, void* const* bufs, void* work, hipStream_t s, std::string& why) {
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
  a.slices = work ? t.slices : 1;
  a.d_slices = div31(a.slices);
  a.work = static_cast<RowWork*>(work);
  switch (t.x.elem) {
    case xt::Elem::F32: return run<kF32>(a, wgs, s);
    case xt::Elem::F16: return run<kF16>(a, wgs, s);
    default: return run<kBF16>(a, wgs, s);
  }
}

}  // namespace xtk
