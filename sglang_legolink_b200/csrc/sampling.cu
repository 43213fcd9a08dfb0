// One token per row of logits: temperature, top-k, top-p and min-p, drawn
// with one uniform number per row.
//
//   w_i = exp((x_i - max x) / T);  order: x descending, equal x by index
//   keep the first top_k;  of those, the ones whose predecessors hold less
//   than top_p of the mass;  of those, the ones with w_i >= min_p
//   token = first kept one, in index order, with  sum_{j <= i} w_j > u * S
//
// Every filter keeps a prefix of the order, so what is kept is a threshold:
// all values above `tau` and the first `quota` tokens equal to it.  No row is
// sorted.
//
// Few candidates (top-k to 1024, a nucleus or a min-p set of that size): a
// lower bound on tau picks them out of the row (the ranges' own maxima bound
// the k-th largest; the mass per power of two of the weight bounds the
// nucleus; min-p is a bound), and one CTA sorts them.  Else tau comes from
// radix selection on the values' order-preserving integer keys, with token
// counts (top-k) or weights (top-p) summed per bin; top-p selects within the
// power of two that its cut falls in.
//
// Weights are integers: w in units of 2^-44, computed in double to 1.2e-12 of
// itself and rounded.  Integer sums do not depend on their order, so a row
// gives the same token whatever batch, cluster size or device it is drawn on,
// and the sums over a whole vocabulary (2^19 tokens at most: 2^63) are exact.
// A token below 2^-45 of the largest has weight 0 and is never drawn.
//
// A cluster of CTAs owns a row and holds it in shared memory, so the logits
// are read from memory once; the passes over the row run on shared memory and
// exchange their sums through it (distributed shared memory).  The passes are
// functions of their own, not inlined: two CTAs of 512 threads a SM leave 64
// registers, and what the rest of the kernel keeps alive would spill inside
// their loops, to memory that has no L1 left.
//
// What bounds it: one row, the chain of some ten block and cluster steps of
// 0.5 to 2 us (10.3 us for one row of 152064 tokens with top-k and top-p); a
// batch of flat rows, the double operations of the exact sums (256 rows with
// temperature alone 91 us, of which reading the logits is 12; 64 rows with
// top-p 67 us, with three passes that evaluate every token).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstddef>
#include <utility>

#include "common.cuh"
#include "sampling.h"

namespace cg = cooperative_groups;

namespace ll {

constexpr int SMP_THREADS = 512;
constexpr int SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_MAX_CLUSTER = 8;
constexpr int SMP_BINS = 2048;
constexpr double SMP_ONE = 17592186044416.0;  // 2^44

// Order-preserving keys of the values: larger value, larger key.  -0 and +0
// share a key (they are equal values).  Logits are held as they are, NaN
// replaced by -inf (never drawn).
template <typename Raw>
struct Key;
template <>
struct Key<uint16_t> {  // bf16
  static constexpr uint32_t kNegInf = 0x007Fu, kPosInf = 0xFF80u;
  static constexpr int kPerVec = 8;
  static constexpr uint32_t kFill = 0xFF80FF80u;  // -inf, twice
  __device__ __forceinline__ static uint32_t of(float x) {
    uint32_t b = __float_as_uint(x);
    if (b == 0x80000000u) b = 0;
    return ((uint32_t)((int)b >> 31) ^ (b | 0x80000000u)) >> 16;
  }
  __device__ __forceinline__ static float value(uint32_t k) {
    const uint32_t b = (k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu);
    return __uint_as_float(b << 16);
  }
  // smallest bf16 >= x (finite)
  __device__ __forceinline__ static float up(float x) {
    const uint32_t b = __float_as_uint(x);
    return __uint_as_float(((b & 0x80000000u) ? b : b + 0xFFFFu) & 0xFFFF0000u);
  }
  __device__ __forceinline__ static void unpack(const uint4& q, float (&x)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ static __nv_bfloat162 pair(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  __device__ __forceinline__ static uint32_t no_nan(uint32_t w) {
    const __nv_bfloat162 r = __hmax2(pair(w), pair(kFill));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ __forceinline__ static float largest(const uint4& q) {
    const __nv_bfloat162 m = __hmax2(__hmax2(pair(q.x), pair(q.y)), __hmax2(pair(q.z), pair(q.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <>
struct Key<uint32_t> {  // fp32
  static constexpr uint32_t kNegInf = 0x007FFFFFu, kPosInf = 0xFF800000u;
  static constexpr int kPerVec = 4;
  static constexpr uint32_t kFill = 0xFF800000u;
  __device__ __forceinline__ static uint32_t of(float x) {
    uint32_t b = __float_as_uint(x);
    if (b == 0x80000000u) b = 0;
    return (uint32_t)((int)b >> 31) ^ (b | 0x80000000u);
  }
  __device__ __forceinline__ static float value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
  __device__ __forceinline__ static float up(float x) { return x; }
  __device__ __forceinline__ static void unpack(const uint4& q, float (&x)[4]) {
    x[0] = __uint_as_float(q.x);
    x[1] = __uint_as_float(q.y);
    x[2] = __uint_as_float(q.z);
    x[3] = __uint_as_float(q.w);
  }
  __device__ __forceinline__ static uint32_t no_nan(uint32_t w) {
    return __float_as_uint(fmaxf(__uint_as_float(w), __uint_as_float(kFill)));
  }
  __device__ __forceinline__ static float largest(const uint4& q) {
    return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
  }
};

constexpr int SMP_RANGES = SMP_MAX_CLUSTER * SMP_WARPS;  // warp ranges of a row
constexpr int SMP_OCTAVES = 16;            // bins of the weight, by powers of two (octave_start), the last one open
constexpr int SMP_LIST = 2048;             // candidates, in one segment per CTA
constexpr int SMP_FEW = 2 * SMP_THREADS;   // of them that one CTA sorts
constexpr float SMP_LOWEST = -3.4028234663852886e38f;

// What a row's passes need to know of it.
struct Row {
  double xmax, inv_t, k1;  // t = (x - xmax) k1 is 32 log2 w
  double u, top_p, min_w;
  double shift;            // approximate weights times it are true to their own error
  float fc, fm;            // approximately log2 w = x fc + fm, a little below 0 at the largest
  float top;               // xmax
  float zero;              // smaller logits weigh less than half a unit
  uint32_t kmax;
};

struct SampleShared {
  Row row;
  alignas(16) float wmax[SMP_RANGES];    // largest logit of each warp range
  float wkth[SMP_RANGES];                // the r-th largest of its lanes' largest
  unsigned long long wsum[SMP_RANGES];   // kept weight of each range
  uint32_t wties[SMP_RANGES];            // its tokens equal to tau
  unsigned long long whigh[SMP_RANGES];  // weight of each range above the keys that top-p selects in
  uint32_t octave[2][SMP_MAX_CLUSTER][SMP_OCTAVES];  // each CTA's mass per bin; levels alternate
  uint32_t listed[SMP_MAX_CLUSTER];      // candidates of each CTA
  unsigned long long scan[SMP_WARPS];
  unsigned long long found_above, total, at_target;
  uint32_t found_bin, found_count;
  float bound;
  uint32_t minp_key;
  uint32_t edge[2];
  int redo;
  int at_range;
  uint32_t at_ties;
  uint32_t count_here;
  double exp2_table[32];
  union {
    struct {
      alignas(16) uint32_t count[SMP_BINS];  // read four bins at a time
      alignas(16) unsigned long long weight[SMP_BINS];
    };
    struct {
      alignas(16) unsigned long long list[SMP_LIST];  // key << 32 | ~index
      alignas(16) unsigned long long flat[SMP_FEW];   // of the sort
    };
    uint32_t mine[SMP_OCTAVES][SMP_THREADS];  // each thread's mass per bin
  };
};
static_assert(offsetof(SampleShared, wmax) % 16 == 0 && offsetof(SampleShared, count) % 16 == 0 &&
                  offsetof(SampleShared, weight) % 16 == 0,
              "vector reads");

// w of a logit, in units of 2^-44, with w = 2^(t / 32), t = (x - max) 32 / (T ln 2):
// t = n + f, n whole and |f| <= 1/2;  2^(f / 32) by its Taylor polynomial of
// degree 4 (within 1.2e-12), 2^(n / 32) from a table and the exponent.  Eleven
// double operations; the library's exponential takes about three times that.
// For zero <= x <= max.
__device__ __forceinline__ double real_weight(float x, double xmax, double k1, const double* table) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
  constexpr double c1 = 0.02166084939249829, c2 = 2.3459619820224677e-4, c3 = 1.6938509724371819e-6,
                   c4 = 9.172562701824643e-9;    // (ln 2 / 32)^i / i!
  const double t = ((double)x - xmax) * k1;
  const double m = t + kMagic;
  const int n = __double2loint(m);
  const double f = t - (m - kMagic);
  double p = fma(fma(fma(fma(c4, f, c3), f, c2), f, c1), f, 1.0);
  p *= table[n & 31];
  // * 2^(n >> 5) * 2^44
  return __hiloint2double(__double2hiint(p) + (((n >> 5) + 44) << 20), __double2loint(p));
}
__device__ __forceinline__ unsigned long long to_whole(double w) {
  w += 6755399441055744.0;
  return (((unsigned long long)(uint32_t)__double2hiint(w) << 32) | (uint32_t)__double2loint(w)) - 0x4338000000000000ull;
}
__device__ __forceinline__ unsigned long long exact_weight(float x, double xmax, double k1, const double* table) {
  return to_whole(real_weight(x, xmax, k1, table));
}
// any logit; without a branch, so that several run at once
__device__ __forceinline__ unsigned long long weight_from(float x, float from, double xmax, double k1,
                                                          const double* table) {
  const unsigned long long w = exact_weight(fmaxf(x, from), xmax, k1, table);
  return x >= from ? w : 0ull;
}
__device__ __noinline__ unsigned long long weight_of(const SampleShared& sh, float x) {
  return weight_from(x, sh.row.zero, sh.row.xmax, sh.row.k1, sh.exp2_table);
}

__device__ __forceinline__ unsigned long long warp_add(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ T warp_inclusive(T v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// exclusive prefix over the block of one value per thread (thread order)
__device__ __noinline__ ulonglong2 block_exclusive(unsigned long long v, unsigned long long* scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long inc = warp_inclusive(v, lane);
  __syncthreads();
  if (lane == 31) scan[warp] = inc;
  __syncthreads();
  const unsigned long long w = warp_inclusive(lane < SMP_WARPS ? scan[lane] : 0ull, lane);
  const unsigned long long before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return make_ulonglong2((warp > 0 ? before : 0ull) + inc - v, __shfl_sync(0xffffffffu, w, 31));
}

// Bitonic sort, largest first: thread t holds values 4 t to 4 t + 3.  The
// steps of one round between lanes, then within the thread.
__device__ __forceinline__ void order_pair(unsigned long long& a, unsigned long long& b, bool down) {
  const bool swap = (a < b) == down;
  const unsigned long long x = swap ? b : a, y = swap ? a : b;
  a = x;
  b = y;
}
__device__ __forceinline__ void take(unsigned long long& c, unsigned long long o, bool large) {
  c = large == (o > c) ? o : c;
}
__device__ __forceinline__ void merge_in_warp(unsigned long long (&c)[4], uint32_t lanes, bool down) {
  for (uint32_t j = lanes / 2; j > 0; j /= 2) {
    const bool large = down == ((threadIdx.x & j) == 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) take(c[q], __shfl_xor_sync(0xffffffffu, c[q], j), large);
  }
  order_pair(c[0], c[2], down);
  order_pair(c[1], c[3], down);
  order_pair(c[0], c[1], down);
  order_pair(c[2], c[3], down);
}
// each warp's up to 128 values, in the directions of a longer sort
__device__ __forceinline__ void warp_sort_descending(unsigned long long (&c)[4], uint32_t size) {
  order_pair(c[0], c[1], true);
  order_pair(c[2], c[3], false);
  for (uint32_t k = 4; k <= size && k <= 128; k *= 2) merge_in_warp(c, k / 4, (4 * threadIdx.x & k) == 0);
}
// of n (a power of two, at most 2 SMP_THREADS) values, two a thread of the
// CTA, through `buf`: 8 of its warps sort.  1024 values 2.4 us (two values a
// thread and every step of more than 64 through shared memory: 5.3).
__device__ __noinline__ ulonglong2 sort_descending(ulonglong2 v, unsigned long long* buf, uint32_t n) {
  const uint32_t tid = threadIdx.x, i = 4 * tid;
  ulonglong2* pairs = reinterpret_cast<ulonglong2*>(buf);
  pairs[tid] = v;
  __syncthreads();
  if (i < 2 * SMP_THREADS) {
    auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(SMP_THREADS / 2) : "memory"); };
    const ulonglong2 a = pairs[2 * tid], b = pairs[2 * tid + 1];
    unsigned long long c[4] = {a.x, a.y, b.x, b.y};
    warp_sort_descending(c, n);
    for (uint32_t k = 256; k <= n; k *= 2) {
      const bool down = (i & k) == 0;
      for (uint32_t j = k / 2; j >= 128; j /= 2) {  // between warps
        sync();
        pairs[2 * tid] = make_ulonglong2(c[0], c[1]);
        pairs[2 * tid + 1] = make_ulonglong2(c[2], c[3]);
        sync();
        const bool large = down == ((i & j) == 0);
        const ulonglong2 o = pairs[2 * (tid ^ (j / 4))], p = pairs[2 * (tid ^ (j / 4)) + 1];
        take(c[0], o.x, large);
        take(c[1], o.y, large);
        take(c[2], p.x, large);
        take(c[3], p.y, large);
      }
      merge_in_warp(c, 32, down);
    }
    sync();
    pairs[2 * tid] = make_ulonglong2(c[0], c[1]);
    pairs[2 * tid + 1] = make_ulonglong2(c[2], c[3]);
  }
  __syncthreads();
  return pairs[tid];
}

// ---- passes over a warp's range [a, b) of vectors, results per lane

// Weight of the logits within [from, upto], and (BOTH) of those above upto
// too.  The weights are added up as the bits of 1.5 * 2^52 + w, a masked one
// as those of w = 0.
struct ExactSum {
  unsigned long long s, high;
};
template <typename Raw, bool BOTH>
__device__ __noinline__ ExactSum exact_sum(const uint4* vals, int a, int b, float from, float upto, double xmax,
                                           double k1, const double* table) {
  using K = Key<Raw>;
  unsigned long long s = 0, high = 0;
  uint32_t vectors = 0;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < from) continue;
    ++vectors;
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) {
      const double w = real_weight(x[i], xmax, k1, table);  // anything below from
      const bool in = x[i] >= from && x[i] <= upto;
      const double r = __hiloint2double(in ? __double2hiint(w) : 0, __double2loint(w)) + 6755399441055744.0;
      s += __double_as_longlong(r);
      if (BOTH) {
        const double h = __hiloint2double(x[i] > upto ? __double2hiint(w) : 0, __double2loint(w)) + 6755399441055744.0;
        high += __double_as_longlong(h);
      }
    }
  }
  const unsigned long long zero = (unsigned long long)(vectors * K::kPerVec) * 0x4338000000000000ull;
  return ExactSum{s - zero, high - (BOTH ? zero : 0ull)};
}

// The same where [from, upto] holds few of the tokens: over the set bits of a
// mask, as many rounds as the fullest lane has, not over all of the vector's
// elements (64 flat rows of 152064 tokens: 66.7 us a call, 68.6 without).
template <typename Raw>
__device__ __noinline__ unsigned long long exact_sum_of_few(const uint4* vals, int a, int b, float from, float upto,
                                                            double xmax, double k1, const double* table) {
  using K = Key<Raw>;
  unsigned long long s = 0;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < from) continue;
    float x[K::kPerVec];
    K::unpack(q, x);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) m |= (x[i] >= from && x[i] <= upto ? 1u : 0u) << i;
    for (; m != 0; m &= m - 1) {
      const Raw b = reinterpret_cast<const Raw*>(vals)[v * K::kPerVec + __ffs(m) - 1];
      s += exact_weight(__uint_as_float((uint32_t)b << (32 - 8 * sizeof(Raw))), xmax, k1, table);
    }
  }
  return s;
}

template <typename Raw>
__device__ __noinline__ uint32_t count_equal(const uint4* vals, int a, int b, float tau) {
  using K = Key<Raw>;
  uint32_t n = 0;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    float x[K::kPerVec];
    K::unpack(vals[v], x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) n += x[i] == tau;
  }
  return n;
}

// Bins of a = -log2 w: fifteen of two octaves, the rest (a >= 30) in the last.
// Of a flat row the largest weight is far above most, and top-p's cut falls at
// 15 to 20: with bins of one octave it was in the open one and took a pass
// more (64 such rows 75 us, 67 now; 16 of fp32 65, 47).  Eight bins of one
// octave before wider ones cost more to tell apart than their shorter lists
// of a small nucleus save (68).
__host__ __device__ __forceinline__ constexpr int octave_start(int bin) { return 2 * bin; }
__device__ __forceinline__ float octave_of(float a) {  // + 2^23
  return __fadd_rd(fminf(a * 0.5f, (float)(SMP_OCTAVES - 1)), 8388608.f);
}

// Approximate mass per bin of all logits, to the thread's own sums:
// w 2^(octave_start + 23) <= 2^23, rounded to a whole number.
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename Raw>
__device__ __noinline__ void octave_sums(const uint4* vals, int a, int b, float fc, float fm, uint32_t* mine) {
  using K = Key<Raw>;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    float x[K::kPerVec];
    K::unpack(vals[v], x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) {
      const float arg = fmaf(x[i], fc, fm);  // < 0
      const uint32_t bin = __float_as_uint(octave_of(-arg)) - 0x4B000000u;
      const float m = fmaf(ex2_approx(arg), __uint_as_float((127u + 23u + 2u * bin) << 23),
                           8388608.f);
      mine[bin * SMP_THREADS] += __float_as_uint(m) - 0x4B000000u;
    }
  }
}

// Mass (approximate) of the logits within [flo, fhi] per sixteenth of their
// range of arguments: bins floor((a1 - x) sc).
__device__ __forceinline__ float bin_of(float x, float a1, float sc) {  // + 2^23
  return __fadd_rd(fminf(fmaxf((a1 - x) * sc, 0.f), (float)(SMP_OCTAVES - 1)), 8388608.f);
}
template <typename Raw>
__device__ __noinline__ void refine_sums(const uint4* vals, int a, int b, float a1, float sc, float k, float flo,
                                         float fhi, uint32_t* mine) {
  using K = Key<Raw>;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < flo) continue;
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) {  // outside: no mass, without a branch
      const bool in = x[i] >= flo && x[i] <= fhi;
      const uint32_t bin = __float_as_uint(bin_of(x[i], a1, sc)) - 0x4B000000u;
      // of the heaviest within the keys: at most 2^23
      mine[bin * SMP_THREADS] +=
          __float_as_uint(ex2_approx(in ? fmaf(x[i] - fhi, k, 23.f) : -INFINITY) + 8388608.f) - 0x4B000000u;
    }
  }
}

// Tokens per bin of (key - lo) >> shift, keys in [lo, hi]; given `weight`,
// their weights too.  The key below that of 0 would be -0's and is no value's:
// a range that ends there ends at the one before, since +0 <= -0.
template <typename Raw>
__device__ __noinline__ void histogram(const uint4* vals, int a, int b, uint32_t lo, uint32_t hi, int shift,
                                       uint32_t* count, unsigned long long* weight, double xmax, double k1,
                                       const double* table) {
  using K = Key<Raw>;
  const float flo = K::value(lo), fhi = K::value(hi == K::of(0.f) - 1 ? hi - 1 : hi);
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < flo) continue;
    auto add = [&](float x) {
      const uint32_t bin = (K::of(x) - lo) >> shift;
      atomicAdd(&count[bin], 1u);
      if (weight != nullptr) atomicAdd(&weight[bin], exact_weight(x, xmax, k1, table));
    };
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i)
      if (x[i] >= flo && x[i] <= fhi) add(x[i]);
  }
}

// Candidates within [xlo, xhi] into this CTA's segment of the first CTA's list.
template <typename Raw>
__device__ __noinline__ void collect(const uint4* vals, int a, int b, int token0, float xlo, float xhi,
                                     uint32_t* counter, unsigned long long* to, uint32_t segment) {
  using K = Key<Raw>;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < xlo) continue;
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i)
      if (x[i] >= xlo && x[i] <= xhi) {
        const uint32_t at = atomicAdd(counter, 1u);
        if (at < segment)
          to[at] = (unsigned long long)K::of(x[i]) << 32 | (0xFFFFFFFFu - (uint32_t)(token0 + v * K::kPerVec + i));
      }
  }
}

// Running sums of kept weight over the n <= 128 ranges: weight above tau and
// tokens at tau, of which the first `quota` count `wtau` each.  One warp, four
// entries a lane.  The lane whose entry passes u times
// the total returns entry >= 0, what is left of that target before the entry,
// and of the quota.
struct Found {
  int entry;
  unsigned long long t, total;
  uint32_t quota;
};
__device__ __forceinline__ Found find_entry(const unsigned long long* wsum, const uint32_t* wties, int n,
                                            uint32_t quota, unsigned long long wtau, double u) {
  constexpr int PER = SMP_RANGES / 32;
  const int lane = threadIdx.x & 31;
  unsigned long long s[PER], mine = 0;
  uint32_t left[PER] = {};
#pragma unroll
  for (int j = 0; j < PER; ++j) s[j] = lane * PER + j < n ? wsum[lane * PER + j] : 0ull;
  if (quota > 0) {
    uint32_t k[PER], ties = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      k[j] = lane * PER + j < n ? wties[lane * PER + j] : 0u;
      ties += k[j];
    }
    uint32_t before = warp_inclusive(ties, lane) - ties;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      left[j] = quota > before ? quota - before : 0u;
      before += k[j];
      s[j] += (unsigned long long)min(left[j], k[j]) * wtau;
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) mine += s[j];
  const unsigned long long inc = warp_inclusive(mine, lane);
  Found f{-1, 0, __shfl_sync(0xffffffffu, inc, 31), 0};
  unsigned long long t = u > 0.0 ? (u < 1.0 ? (unsigned long long)(u * (double)f.total) : f.total - 1) : 0ull;
  if (t >= f.total) t = f.total - 1;
  unsigned long long run = inc - mine;
  if (run <= t && t < inc) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (run <= t) {
        f.entry = lane * PER + j;
        f.t = t - run;
        f.quota = left[j];
      }
      run += s[j];
    }
  }
  return f;
}

// The log of a token's share.
__device__ __noinline__ float log_share(const Row& r, float x, double total) {
  return (float)((x == r.top ? 0.0 : ((double)x - r.xmax) * r.inv_t) - log(total));
}

// w >= min_p, in the definition's own terms
__device__ __noinline__ bool heavy(const Row& r, float x) {
  return x == r.top || exp(((double)x - r.xmax) * r.inv_t) >= r.min_w;
}

// Largest key in [lo, hi] at which `above` (the sum over keys larger than hi)
// plus the sum over keys from it to hi reaches a target: tokens, or their
// weights (W).  Tokens: the search may end with the lower end of a bin of keys,
// once no more than `enough` tokens are at or above it.
struct Selected {
  bool ok;  // false: never reached
  uint32_t key, count;       // the key, tokens equal to it
  unsigned long long above;  // sum over larger keys
};
template <typename Raw, bool W>
__device__ __noinline__ Selected select(SampleShared& sh, const uint4* vals, int v0, int v1, uint32_t lo, uint32_t hi,
                                        unsigned long long above, unsigned long long target,
                                        unsigned long long enough = 0) {
  using K = Key<Raw>;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), tid = threadIdx.x;
  Selected r{false, 0, 0, above};
  if (lo > hi) return r;
  while (true) {
    constexpr int PER = SMP_BINS / SMP_THREADS;
    static_assert(PER == 4, "a thread's bins are one 16-byte read");
    const uint32_t span = hi - lo;
    const int shift = span < (uint32_t)SMP_BINS ? 0 : 32 - __clz(span) - 11;
    const int used = ((int)(span >> shift) + PER) & ~(PER - 1);
    const bool weighted = W && shift > 0;
    for (int i = tid; i < used; i += SMP_THREADS) {
      sh.count[i] = 0;
      if (weighted) sh.weight[i] = 0;
    }
    __syncthreads();
    histogram<Raw>(vals, v0, v1, lo, hi, shift, sh.count, weighted ? sh.weight : nullptr, sh.row.xmax, sh.row.k1,
                   sh.exp2_table);
    cluster.sync();
    // thread t merges four bins, thread 0 the largest keys; every CTA's at once
    uint32_t cnt[PER] = {};
    unsigned long long val[PER] = {}, mine = 0;
    const int b0 = used - PER * (tid + 1);
    if (b0 >= 0) {
      uint4 n4[SMP_MAX_CLUSTER];
#pragma unroll
      for (int c = 0; c < SMP_MAX_CLUSTER; ++c)
        n4[c] = c < cs ? *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.count, c) + b0)
                       : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < SMP_MAX_CLUSTER; ++c) {
        cnt[0] += n4[c].w;
        cnt[1] += n4[c].z;
        cnt[2] += n4[c].y;
        cnt[3] += n4[c].x;
      }
      if (weighted)
        for (int c = 0; c < cs; ++c) {
          const ulonglong2* w2 = reinterpret_cast<const ulonglong2*>(cluster.map_shared_rank(sh.weight, c) + b0);
          const ulonglong2 a = w2[0], d = w2[1];
          val[0] += d.y;
          val[1] += d.x;
          val[2] += a.y;
          val[3] += a.x;
        }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (!W) val[j] = cnt[j];
        else if (!weighted && cnt[j] > 0)
          val[j] = cnt[j] * exact_weight(K::value(lo + b0 + PER - 1 - j), sh.row.xmax, sh.row.k1, sh.exp2_table);
        mine += val[j];
      }
    }
    const ulonglong2 ex = block_exclusive(mine, sh.scan);
    if (r.above >= target || r.above + ex.y < target) {  // uniform over the cluster
      cluster.sync();
      return r;
    }
    unsigned long long before = r.above + ex.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (before < target && before + val[j] >= target) {
        sh.found_bin = b0 + PER - 1 - j;
        sh.found_above = before;
        sh.found_count = cnt[j];
      }
      before += val[j];
    }
    cluster.sync();  // the found bin, and every read of the bins
    const uint32_t b = sh.found_bin;
    r.above = sh.found_above;
    if (shift == 0 || (!W && r.above + sh.found_count <= enough)) {
      r.ok = true;
      r.key = lo + (b << shift);
      r.count = sh.found_count;
      return r;
    }
    const uint32_t nlo = lo + (b << shift);
    hi = min(hi, nlo + ((1u << shift) - 1));
    lo = nlo;
  }
}

// Smallest key in [lo, hi] (hi qualifies) from which on `in` holds; one warp.
template <typename In>
__device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, In in) {
  const int lane = threadIdx.x & 31;
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 32 + 1;
    const uint32_t probe =
        (uint32_t)min((unsigned long long)hi, (unsigned long long)lo + (unsigned long long)lane * step);
    const uint32_t ok = __ballot_sync(0xffffffffu, probe == hi || in(probe));
    const int f = __ffs(ok) - 1;  // first probe inside; none: beyond the last one
    const uint32_t from = lo;
    if (f < 0) {
      lo = from + 31 * step + 1;
    } else {
      hi = (uint32_t)min((unsigned long long)hi, (unsigned long long)from + (unsigned long long)f * step);
      if (f > 0) lo = from + (f - 1) * step + 1;
    }
  }
  return lo;
}

// top-p over the whole row: the keys within which its cut falls, from
// approximate masses.  The mass per power or two of the weight (octave_of),
// then, while the bin of the cut holds many tokens for one histogram, the mass
// of its sixteenths.  What is selected
// within the keys is checked against exact sums; the few tokens of a small
// nucleus are enough with the mass below them and its error.
struct Nucleus {
  uint32_t lo, hi;
  double tokens, inside;    // at most so many tokens >= lo of the first level; within [lo, hi]
  double below, err_below;  // mass (units of 1) of the keys < lo of the first level, its error
};
template <typename Raw>
__device__ __noinline__ Nucleus find_nucleus(SampleShared& sh, const uint4* vals, int v0, int v1, int V, float T) {
  using K = Key<Raw>;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float fc = sh.row.fc, fm = sh.row.fm;
  Nucleus r{K::kNegInf + 1, sh.row.kmax, 1e30, 1e30, 0.0, 0.0};
  double goal = 0.0;  // mass still to pass
  for (int level = 0;; ++level) {
#pragma unroll
    for (int b = 0; b < SMP_OCTAVES; ++b) sh.mine[b][tid] = 0;
    const float flo = K::value(r.lo), fhi = K::value(r.hi), sc = (float)SMP_OCTAVES / (fhi - flo);
    if (level == 0) octave_sums<Raw>(vals, v0, v1, fc, fm, &sh.mine[0][tid]);
    else refine_sums<Raw>(vals, v0, v1, fhi, sc, 1.442695f / T, flo, fhi, &sh.mine[0][tid]);
    __syncthreads();
    {  // one warp a bin, in units 512 times coarser: a bin of a CTA fits 32 bits
      static_assert(SMP_WARPS == SMP_OCTAVES && SMP_THREADS == 512, "a warp a bin");
      unsigned long long m = 0;
#pragma unroll
      for (int i = 0; i < SMP_THREADS; i += 32) m += sh.mine[warp][i + lane];
      m = warp_add(m);
      if (lane < cs)
        cluster.map_shared_rank(&sh.octave[level & 1][0][0], lane)[rank * SMP_OCTAVES + warp] = (uint32_t)(m >> 9);
    }
    cluster.sync();
    // every warp, a lane a bin: the bin in which the cut falls
    double mass = 0.0;
    if (lane < SMP_OCTAVES) {
      unsigned long long m = 0;
      for (int c = 0; c < cs; ++c) m += sh.octave[level & 1][c][lane];
      // units: of a bin 2^(9 - 23 - octave_start); of a later level, the weight of hi 2^(9 - 23)
      mass = (double)m * (level == 0 ? __hiloint2double((1023 - 14 - octave_start(lane)) << 20, 0)
                                     : (double)ex2_approx(fmaf(fhi, fc, fm)) * (1.0 / 16384.0));
    }
    const double upto = warp_inclusive(mass, lane), all = __shfl_sync(0xffffffffu, upto, 31);
    if (level == 0) goal = sh.row.top_p * all;
    const uint32_t past = __ballot_sync(0xffffffffu, lane < SMP_OCTAVES - 1 && upto >= goal);
    const int at = past ? __ffs(past) - 1 : SMP_OCTAVES - 1;
    const double in = __shfl_sync(0xffffffffu, mass, at), here = __shfl_sync(0xffffffffu, upto, at);
    goal -= here - in;
    if (level == 0) {
      // tokens: by the bins' smallest weights, and what the coarser units dropped
      const double n = lane < SMP_OCTAVES - 1 ? mass * (double)(1u << octave_start(lane + 1)) * 1.001 + 1.0 : 1e30;
      r.tokens = __shfl_sync(0xffffffffu, warp_inclusive(n, lane), at);
      // error: 2^-22 (ex2) + 2^-22 (rounded to a whole, of 2^21 or more) +
      // 2 * 2^-24 |arg| ln 2 (argument; the open bin: at most 46); its wholes
      // (half of 2^-53 a token), and the coarser units
      double err = lane < SMP_OCTAVES
                       ? mass * ((2.0 + 0.35 * (lane == SMP_OCTAVES - 1 ? 46.0 : octave_start(lane + 1))) *
                                 (1.01 / 4194304.0)) +
                             (lane == SMP_OCTAVES - 1 ? (double)V : 0.0) * __hiloint2double((1023 - 54) << 20, 0) +
                             cs * __hiloint2double((1023 - 14 - octave_start(lane)) << 20, 0)
                       : 0.0;
      err = warp_inclusive(err, lane);
      r.below = all - here;
      r.err_below = __shfl_sync(0xffffffffu, err, 31) - __shfl_sync(0xffffffffu, err, at);
    }
    // the bin's keys
    if (warp < 2) {
      const int b = at + 1 - warp;  // warp 0: first key of bins < at + 1; warp 1: of bins < at
      uint32_t k = warp == 0 ? max(r.lo, K::of(sh.row.zero)) : r.hi + 1;
      if (warp == 0 ? at < SMP_OCTAVES - 1 : at > 0)
        k = first_key(r.lo, r.hi, [&](uint32_t q) {
          const float x = K::value(q);
          return (level == 0 ? octave_of(-fmaf(x, fc, fm)) : bin_of(x, fhi, sc)) < 8388608.f + (float)b;
        });
      if (lane == 0) sh.edge[warp] = k;
    }
    __syncthreads();
    r.lo = sh.edge[0];
    r.hi = sh.edge[1] - 1;
    r.inside = in / (double)ex2_approx(fmaf(K::value(r.lo), fc, fm)) * 1.001 + 1.0;
    // keys that have a bin each are counted, however many tokens they are
    if (r.tokens <= SMP_FEW || r.inside <= SMP_FEW || r.hi - r.lo < SMP_BINS || r.lo >= r.hi || level == 3) break;
    __syncthreads();  // the edges are read
  }
  return r;
}

// Every CTA's candidates within [xlo, xhi] to the first CTA's list; how many,
// or more than SMP_FEW where they do not fit.  All threads of the cluster.
template <typename Raw>
__device__ __noinline__ uint32_t collect_all(SampleShared& sh, const uint4* vals, int a, int b, int token0, float xlo,
                                             float xhi) {
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x;
  const uint32_t segment = SMP_LIST / cs;
  if (tid == 0) sh.count_here = 0;
  __syncthreads();
  collect<Raw>(vals, a, b, token0, xlo, xhi, &sh.count_here, cluster.map_shared_rank(sh.list, 0) + rank * segment,
               segment);
  __syncthreads();
  if (tid < cs) cluster.map_shared_rank(sh.listed, tid)[rank] = sh.count_here;
  cluster.sync();
  uint32_t n = 0;
  for (int c = 0; c < cs; ++c) {
    const uint32_t m = sh.listed[c];
    n = n > SMP_FEW || m > segment ? SMP_FEW + 1 : n + m;
  }
  return n;
}

// The n listed candidates in the order, two a thread, on the first CTA.
__device__ __noinline__ ulonglong2 sorted_list(SampleShared& sh, int cs, uint32_t n) {
  const int tid = threadIdx.x, segment = SMP_LIST / cs;
  ulonglong2 c = make_ulonglong2(0, 0);
  uint32_t base = 0, size = 2;
  for (int r = 0; r < cs; ++r) {
    const uint32_t m = sh.listed[r], i = 2 * tid - base;  // wraps where 2 tid < base
    if (i < m) c.x = sh.list[r * segment + i];
    if (i + 1 < m) c.y = sh.list[r * segment + i + 1];
    base += m;
  }
  while (size < n) size *= 2;
  return sort_descending(c, sh.flat, size);
}

// top-p's cut among the n listed candidates, `above` the weight of all larger
// ones: its key and how many tokens equal to it are kept, to every CTA (0: the
// cut is not among them).
template <typename Raw>
__device__ __noinline__ void cut_in_list(SampleShared& sh, int cs, uint32_t n, unsigned long long above,
                                         unsigned long long goal) {
  using K = Key<Raw>;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  const ulonglong2 c = sorted_list(sh, cs, n);
  const uint32_t k0 = (uint32_t)(c.x >> 32), k1 = (uint32_t)(c.y >> 32);
  const unsigned long long w0 = c.x != 0 ? weight_of(sh, K::value(k0)) : 0ull;
  const unsigned long long w1 = c.y != 0 ? weight_of(sh, K::value(k1)) : 0ull;
  if (tid == 0) sh.found_bin = 0;
  const ulonglong2 ex = block_exclusive(w0 + w1, sh.scan);
  const unsigned long long b0 = above + ex.x, b1 = b0 + w0;
  // the last kept token: what is before it is below the goal, with it no more
  if (b0 < goal && goal <= b0 + w0) sh.found_bin = k0;
  if (b1 < goal && goal <= b1 + w1) sh.found_bin = k1;
  __syncthreads();
  const uint32_t key = sh.found_bin;
  const uint32_t kept = __syncthreads_count(key != 0 && k0 == key && b0 < goal) +
                        __syncthreads_count(key != 0 && k1 == key && b1 < goal);
  if (tid < cs) {
    *cluster.map_shared_rank(&sh.found_bin, tid) = key;
    *cluster.map_shared_rank(&sh.found_count, tid) = kept;
  }
}

// finish_list by one warp, without a barrier: for as many candidates as a
// usual top-k leaves (top-k 50 of 152064 tokens: one row 10.3 us a call, 11.9
// by the whole CTA; 64 rows 13.2 and 17.7).
constexpr int SMP_WARP_FEW = 128;
template <typename Raw>
__device__ __noinline__ bool finish_in_warp(SampleShared& sh, const LLSample& p, int64_t row, int cs, uint32_t n,
                                            uint32_t limit, bool use_p, bool use_m, double below, double err) {
  using K = Key<Raw>;
  const uint32_t lane = threadIdx.x, segment = SMP_LIST / cs;
  unsigned long long c[4] = {0, 0, 0, 0}, w[4];
  uint32_t base = 0, size = 4;
  for (int r = 0; r < cs; ++r) {
    const uint32_t m = sh.listed[r];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t i = 4 * lane + q - base;  // wraps before the segment
      if (i < m) c[q] = sh.list[r * segment + i];
    }
    base += m;
  }
  while (size < n) size *= 2;
  warp_sort_descending(c, size);
  limit = min(limit, n);
  auto weigh = [&](uint32_t count, bool high_half) {  // weights of the first `count`, what is before this lane's, all
    unsigned long long mine = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = K::value((uint32_t)(high_half ? c[q] >> 32 : c[q]));
      w[q] = 4 * lane + q < count ? weight_from(x, sh.row.zero, sh.row.xmax, sh.row.k1, sh.exp2_table) : 0ull;
      mine += w[q];
    }
    const unsigned long long inc = warp_inclusive(mine, (int)lane);
    return make_ulonglong2(inc - mine, __shfl_sync(0xffffffffu, inc, 31));
  };
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (4 * lane + q >= limit) c[q] = 0;
  if (use_p) {
    const ulonglong2 ex = weigh(limit, true);
    const double scale = below >= 0.0 ? sh.row.shift * SMP_ONE : 0.0;
    const double goal = fmax(1.0, ceil(sh.row.top_p * ((double)ex.y + below * scale)));
    const double e = sh.row.top_p * err * scale + 2.0;
    bool near = (double)ex.y < goal + e;
    unsigned long long run = ex.x;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool first = lane == 0 && q == 0;
      near = near || (c[q] != 0 && !first && fabs((double)run - goal) <= e);
      if ((double)run >= goal && !first) c[q] = 0;
      run += w[q];
    }
    if (below >= 0.0 && __any_sync(0xffffffffu, near)) return false;
  }
  if (use_m) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (c[q] != 0 && !heavy(sh.row, K::value((uint32_t)(c[q] >> 32)))) c[q] = 0;
  }
  uint32_t kept = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    kept += c[q] != 0;
    c[q] = c[q] << 32 | c[q] >> 32;
  }
  kept = __reduce_add_sync(0xffffffffu, kept);
  size = 4;
  while (size < kept) size *= 2;
  warp_sort_descending(c, size);
  const ulonglong2 ex = weigh(kept, false);
  const double u = sh.row.u;
  unsigned long long t = u > 0.0 ? (u < 1.0 ? (unsigned long long)(u * (double)ex.y) : ex.y - 1) : 0ull;
  if (t >= ex.y) t = ex.y - 1;
  unsigned long long run = ex.x;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (run <= t && t < run + w[q]) {
      p.out[row] = (int)(0xFFFFFFFFu - (uint32_t)(c[q] >> 32));
      if (p.logprob) p.logprob[row] = log_share(sh.row, K::value((uint32_t)c[q]), (double)ex.y / SMP_ONE);
    }
    run += w[q];
  }
  return true;
}

// The few candidates in sh.list, in segments of one CTA each: filters, draw.
// `below`, `err`: mass (units of 1) of the row's other tokens and its error,
// for a top-p over the whole row; else -1.  False: too near a border.
template <typename Raw>
__device__ __noinline__ bool finish_list(SampleShared& sh, const LLSample& p, int64_t row, int cs, uint32_t n,
                                         uint32_t limit, bool use_p, bool use_m, double below, double err) {
  using K = Key<Raw>;
  const int tid = threadIdx.x;
  if (n <= SMP_WARP_FEW) {
    const bool ok = tid >= 32 || finish_in_warp<Raw>(sh, p, row, cs, n, limit, use_p, use_m, below, err);
    return below < 0.0 || !__syncthreads_or(!ok);
  }
  // two tokens a thread, in the order: weights and what is before them
  ulonglong2 c = sorted_list(sh, cs, n);
  limit = min(limit, n);
  if (2 * tid >= limit) c.x = 0;
  if (2 * tid + 1 >= limit) c.y = 0;
  unsigned long long w0 = c.x != 0 ? weight_of(sh, K::value((uint32_t)(c.x >> 32))) : 0ull;
  unsigned long long w1 = c.y != 0 ? weight_of(sh, K::value((uint32_t)(c.y >> 32))) : 0ull;
  if (use_p) {
    const ulonglong2 ex = block_exclusive(w0 + w1, sh.scan);
    // predecessors' mass below top_p of all; the first token is always kept
    const double scale = below >= 0.0 ? sh.row.shift * SMP_ONE : 0.0;
    const double goal = fmax(1.0, ceil(sh.row.top_p * ((double)ex.y + below * scale)));
    if (below >= 0.0) {
      // the cut for any mass within the error: before the same token, and within the list
      const double e = sh.row.top_p * err * scale + 2.0, b0 = (double)ex.x, b1 = (double)(ex.x + w0);
      const bool near = (c.x != 0 && tid > 0 && fabs(b0 - goal) <= e) || (c.y != 0 && fabs(b1 - goal) <= e) ||
                        (double)ex.y < goal + e;
      if (__syncthreads_or(near)) return false;
    }
    if ((double)ex.x >= goal && tid > 0) c.x = 0;
    if ((double)(ex.x + w0) >= goal) c.y = 0;
  }
  if (use_m) {
    if (c.x != 0 && !heavy(sh.row, K::value((uint32_t)(c.x >> 32)))) c.x = 0;
    if (c.y != 0 && !heavy(sh.row, K::value((uint32_t)(c.y >> 32)))) c.y = 0;
  }
  // the kept ones, which are the first: by index (~index, key), and their running sum
  const uint32_t kept = __syncthreads_count(c.x != 0) + __syncthreads_count(c.y != 0);
  uint32_t size = 2;
  while (size < kept) size *= 2;
  c = sort_descending(make_ulonglong2(c.x << 32 | c.x >> 32, c.y << 32 | c.y >> 32), sh.flat, size);
  w0 = 2 * tid < kept ? weight_of(sh, K::value((uint32_t)c.x)) : 0ull;
  w1 = 2 * tid + 1 < kept ? weight_of(sh, K::value((uint32_t)c.y)) : 0ull;
  const ulonglong2 ex = block_exclusive(w0 + w1, sh.scan);
  const double u = sh.row.u;
  unsigned long long t = u > 0.0 ? (u < 1.0 ? (unsigned long long)(u * (double)ex.y) : ex.y - 1) : 0ull;
  if (t >= ex.y) t = ex.y - 1;
  if (ex.x <= t && t < ex.x + w0 + w1) {
    const unsigned long long d = t < ex.x + w0 ? c.x : c.y;
    p.out[row] = (int)(0xFFFFFFFFu - (uint32_t)(d >> 32));
    if (p.logprob) p.logprob[row] = log_share(sh.row, K::value((uint32_t)d), (double)ex.y / SMP_ONE);
  }
  return true;
}

template <typename Raw>
__global__ void __launch_bounds__(SMP_THREADS, 2) sample_kernel(const __grid_constant__ LLSample p) {
  using K = Key<Raw>;
  constexpr int PV = K::kPerVec;
  constexpr float kNone = -INFINITY;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
  uint4* vals = reinterpret_cast<uint4*>(smem_raw + ((sizeof(SampleShared) + 15) & ~size_t(15)));

  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / cs;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = p.V, ranges = cs * SMP_WARPS;

  // another CTA's shared memory may be written once that CTA has started: every
  // CTA says so here, and the wait is where the load is done
  auto started = cluster.barrier_arrive();
  pdl_trigger();
  if (tid == 0) sh.redo = 0;
  if (tid < 32) sh.exp2_table[tid] = exp2((double)tid / 32.0);
  pdl_wait();
  const float T = p.temperature ? p.temperature[row] : 1.f;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;
  const int k_of = T > 0.f && top_k > 0 && top_k < V ? top_k : 0;
  // few candidates: at least k_of tokens lie at or above the k_of-th largest
  // of the ranges' maxima; with r_want of them wanted from every range, at or
  // above the smallest of the ranges' r_want-th largest lane maxima
  const int r_want = (k_of + ranges - 1) / ranges;

  // ---- load: the row to shared memory, and its largest logit.  Every CTA
  // has a run of 16-byte vectors, every warp of it a range [v0, v1) of them.
  const Raw* src = reinterpret_cast<const Raw*>(p.logits) + row * p.stride;
  const int pad = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(Raw));  // elements before the row in its first vector
  const int nvec = (pad + V + PV - 1) / PV;
  const int per_cta = (nvec + cs - 1) / cs;
  const int cv0 = min(nvec, rank * per_cta), cv_n = min(nvec, cv0 + per_cta) - cv0;
  const int per_warp = (per_cta + SMP_WARPS - 1) / SMP_WARPS;
  const int v0 = min(cv_n, warp * per_warp), v1 = min(cv_n, v0 + per_warp);
  const int token0 = cv0 * PV - pad;  // of vals[0]
  {
    const uint4* vsrc = reinterpret_cast<const uint4*>(src - pad) + cv0;
    float mine = kNone;
    constexpr int DEPTH = 4;  // vectors of a lane in flight
    for (int vb = v0 + lane; vb < v1; vb += 32 * DEPTH) {
      uint4 q[DEPTH];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int v = vb + 32 * d, e0 = token0 + v * PV;  // token of the vector's first element
        if (v < v1 && e0 >= 0 && e0 + PV <= V) q[d] = vsrc[v];
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int v = vb + 32 * d, e0 = token0 + v * PV;
        if (v >= v1) break;
        if (!(e0 >= 0 && e0 + PV <= V)) {  // the row's ends: one element at a time, -inf outside
          uint32_t w[4] = {K::kFill, K::kFill, K::kFill, K::kFill};
#pragma unroll
          for (int i = 0; i < PV; ++i) {
            const int e = e0 + i;
            if (e >= 0 && e < V) {
              const uint32_t b = (uint32_t)src[e];
              if constexpr (PV == 8) w[i / 2] = (i & 1) ? (w[i / 2] & 0xFFFFu) | b << 16 : (w[i / 2] & 0xFFFF0000u) | b;
              else w[i] = b;
            }
          }
          q[d] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        q[d] = make_uint4(K::no_nan(q[d].x), K::no_nan(q[d].y), K::no_nan(q[d].z), K::no_nan(q[d].w));
        mine = fmaxf(mine, K::largest(q[d]));
        vals[v] = q[d];
      }
    }
    float kth = kNone;
    if (r_want > 1 && r_want <= 32) {
      int larger = 0;
      for (int l = 0; l < 32; ++l) {
        const float o = __shfl_sync(0xffffffffu, mine, l);
        larger += o > mine || (o == mine && l < lane);
      }
      const uint32_t at = __ballot_sync(0xffffffffu, larger == r_want - 1);
      kth = __shfl_sync(0xffffffffu, mine, __ffs(at) - 1);
    }
    const float wmax = warp_max(mine);
    cluster.barrier_wait(std::move(started));
    if (lane < cs) {
      cluster.map_shared_rank(sh.wmax, lane)[rank * SMP_WARPS + warp] = wmax;
      cluster.map_shared_rank(sh.wkth, lane)[rank * SMP_WARPS + warp] = kth;
    }
  }
  cluster.sync();
  float xmax = kNone;
  for (int i = lane; i < ranges; i += 32) xmax = fmaxf(xmax, sh.wmax[i]);
  xmax = warp_max(xmax);
  if (xmax == kNone) {  // nothing to draw
    if (rank == 0 && tid == 0) {
      p.out[row] = -1;
      if (p.logprob) p.logprob[row] = kNone;
    }
    return;
  }
  if (!(T > 0.f)) {  // the first of the largest: in the first range that has it
    int at = ranges;
    for (int i = lane; i < ranges; i += 32)
      if (sh.wmax[i] == xmax) at = min(at, i);
    at = __reduce_min_sync(0xffffffffu, at);
    if (at != rank * SMP_WARPS + warp) return;
    for (int vb = v0; vb < v1; vb += 32) {
      const int v = vb + lane;
      int e = INT_MAX;
      if (v < v1) {
        float x[PV];
        K::unpack(vals[v], x);
#pragma unroll
        for (int i = PV - 1; i >= 0; --i)
          if (x[i] == xmax) e = token0 + v * PV + i;
      }
      e = __reduce_min_sync(0xffffffffu, e);
      if (e != INT_MAX) {
        if (lane == 0) {
          p.out[row] = e;
          if (p.logprob) p.logprob[row] = 0.f;
        }
        return;
      }
    }
    return;
  }
  if (xmax == INFINITY) {  // all mass is on the infinities, alike: they become 0, the others -inf
    __syncthreads();       // the ranges' maxima are read
    for (int v = v0 + lane; v < v1; v += 32) {
      float x[PV];
      K::unpack(vals[v], x);
      uint32_t w[4] = {K::kFill, K::kFill, K::kFill, K::kFill};
#pragma unroll
      for (int i = 0; i < PV; ++i)
        if (x[i] == INFINITY) {
          if constexpr (PV == 8) w[i / 2] &= (i & 1) ? 0x0000FFFFu : 0xFFFF0000u;
          else w[i] = 0u;
        }
      vals[v] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (tid < ranges) {
      sh.wmax[tid] = sh.wmax[tid] == INFINITY ? 0.f : kNone;
      sh.wkth[tid] = sh.wkth[tid] == INFINITY ? 0.f : kNone;
    }
    xmax = 0.f;
    __syncthreads();
  }
  if (tid == 0) {
    Row& r = sh.row;
    r.top = xmax;
    r.kmax = K::of(xmax);
    r.xmax = (double)xmax;
    r.inv_t = 1.0 / (double)T;
    r.k1 = 46.16624130844683 * r.inv_t;  // 32 / ln 2
    // rounded up: no logit from it on is outside the polynomial's range
    const float z = fminf(xmax, __double2float_ru(r.xmax - 31.2 * (double)T));
    r.zero = K::up(fmaxf(z, SMP_LOWEST));
    r.fc = (float)(1.4426950408889634 * r.inv_t);
    r.fm = fmaf(-xmax, r.fc, -0.001953125f);  // every argument is below 0
    // 2^-(fm + xmax fc), the exponent within 2^-8: by its series
    const double d = -0.6931471805599453 * ((double)r.fm + r.xmax * (double)r.fc);
    r.shift = 1.0 + d * (1.0 + d * (0.5 + d * (1.0 / 6 + d * (1.0 / 24 + d * (1.0 / 120)))));
    r.u = p.u[row];
    r.top_p = fmax((double)top_p, 0.0);
    r.min_w = fmin((double)min_p, 1.0);
  }
  __syncthreads();

  const bool use_p = top_p < 1.f, use_m = min_p > 0.f;
  // approximate masses: where their arguments neither overflow nor cancel, fm
  // rounded to 2^-12 at most
  const bool nucleus = use_p && k_of == 0 && V > SMP_FEW && T >= 1e-3f && T <= 1e4f && fabsf(xmax) / T * 1.4427f <= 4000.f;
  Nucleus nu{K::kNegInf + 1, sh.row.kmax, 1e30, 1e30, -1.0, 0.0};
  if (nucleus) nu = find_nucleus<Raw>(sh, vals, v0, v1, V, T);

  // What is kept, where it is not few: logits above tau, and the first `quota`
  // equal to it.
  float tau = kNone;
  uint32_t quota = 0;

  // ---- top-k: a lower bound on the k-th largest; with a larger k, itself
  float xlo = INFINITY;
  if (r_want == 1) {
    if (tid < ranges) {
      const float mine = sh.wmax[tid];
      int larger = 0;
#pragma unroll 4
      for (int i = 0; i < ranges; i += 4) {
        const float4 o = *reinterpret_cast<const float4*>(&sh.wmax[i]);
        larger += (o.x > mine || (o.x == mine && i < tid)) + (o.y > mine || (o.y == mine && i + 1 < tid)) +
                  (o.z > mine || (o.z == mine && i + 2 < tid)) + (o.w > mine || (o.w == mine && i + 3 < tid));
      }
      if (larger == k_of - 1) sh.bound = mine;
    }
    __syncthreads();
    xlo = fmaxf(sh.bound, SMP_LOWEST);
  } else if (k_of > 0) {
    float b = r_want <= 32 ? INFINITY : kNone;
    for (int i = lane; i < ranges; i += 32) b = fminf(b, sh.wkth[i]);
    xlo = fmaxf(-warp_max(-b), SMP_LOWEST);
    const Selected r =
        select<Raw, false>(sh, vals, v0, v1, K::of(xlo), sh.row.kmax, 0, (unsigned long long)k_of, SMP_FEW);
    if (r.ok) {
      xlo = K::value(r.key);
      if (r.above + r.count > SMP_FEW) {
        tau = xlo;
        quota = (uint32_t)(k_of - r.above);
      }
    }
  } else if (use_p) {
    if (V <= SMP_FEW) xlo = SMP_LOWEST;  // all of them: sorting beats finding out which
    else if (nu.tokens <= SMP_FEW) xlo = K::value(nu.lo);
  } else if (min_p >= 1e-4f) {
    // a little below max + T log(min_p)
    xlo = __double2float_rd(sh.row.xmax + (double)T * (log(sh.row.min_w) - 1e-6) - 1e-6 * fabs(sh.row.xmax));
    xlo = K::up(fmaxf(xlo, SMP_LOWEST));
    if (!(xlo <= xmax)) xlo = xmax;
  }

  // ---- few candidates: every token at or above `xlo`, finished by one CTA
  if (xlo != INFINITY && tau == kNone) {
    const uint32_t n = collect_all<Raw>(sh, vals, v0, v1, token0, xlo, INFINITY);
    if (n <= SMP_FEW) {
      if (rank == 0 &&
          !finish_list<Raw>(sh, p, row, cs, n, k_of > 0 ? (uint32_t)k_of : n, use_p, use_m, nu.below, nu.err_below) &&
          tid < cs)
        *cluster.map_shared_rank(&sh.redo, tid) = 1;
      if (!nucleus) return;
      cluster.sync();
      if (!sh.redo) return;
    }
  }

  // ---- many: the threshold, selected in the row
  // The smallest logit above x with weight; NaN where there is none.
  auto above_of = [&](float x) {
    if (x >= xmax) return __int_as_float(0x7FFFFFFF);
    return fmaxf(x == kNone ? SMP_LOWEST : K::value(K::of(x) + 1), sh.row.zero);
  };
  // Weight within [from, upto] and tokens at tau per warp range, to every CTA;
  // `both`: and the weight above upto.
  auto sum_pass = [&](float from, float upto, bool both) {
    ExactSum e{0, 0};
    if (both) e = exact_sum<Raw, true>(vals, v0, v1, from, upto, sh.row.xmax, sh.row.k1, sh.exp2_table);
    else if (upto == INFINITY)
      e = exact_sum<Raw, false>(vals, v0, v1, from, upto, sh.row.xmax, sh.row.k1, sh.exp2_table);
    else e.s = exact_sum_of_few<Raw>(vals, v0, v1, from, upto, sh.row.xmax, sh.row.k1, sh.exp2_table);
    const unsigned long long s = warp_add(e.s), high = both ? warp_add(e.high) : 0ull;
    const uint32_t ties = quota > 0 ? __reduce_add_sync(0xffffffffu, count_equal<Raw>(vals, v0, v1, tau)) : 0u;
    if (lane < cs) {
      const int i = rank * SMP_WARPS + warp;
      cluster.map_shared_rank(sh.wsum, lane)[i] = s;
      cluster.map_shared_rank(sh.wties, lane)[i] = ties;
      if (both) cluster.map_shared_rank(sh.whigh, lane)[i] = high;
    }
    cluster.sync();
  };
  float split = INFINITY;  // whigh holds the ranges' weight above it
  if (k_of > 0 && tau == kNone) {  // too many at or above the bound, or fewer tokens than k
    const Selected r =
        select<Raw, false>(sh, vals, v0, v1, K::kNegInf + 1, sh.row.kmax, 0, (unsigned long long)k_of);
    if (r.ok) {
      tau = K::value(r.key);
      quota = (uint32_t)(k_of - r.above);
    }
  }
  if (use_p) {
    // all weights; of a row whose cut is known to lie within keys, apart from those above them
    if (nucleus && nu.lo <= nu.hi) split = K::value(nu.hi);
    sum_pass(above_of(tau), split, true);
    unsigned long long s = 0, above = 0;
    uint32_t ties = 0;
    for (int i = lane; i < ranges; i += 32) {
      s += sh.wsum[i];
      above += sh.whigh[i];
      ties += sh.wties[i];
    }
    above = warp_add(above);
    const unsigned long long total =
        warp_add(s) + above +
        (quota > 0 ? (unsigned long long)min(__reduce_add_sync(0xffffffffu, ties), quota) * weight_of(sh, tau) : 0ull);
    // predecessors' mass below top_p of all; the first token is always kept
    const unsigned long long goal = (unsigned long long)fmax(1.0, ceil(sh.row.top_p * (double)total));
    const uint32_t floor_key = max(K::of(fmaxf(fmaxf(tau, SMP_LOWEST), sh.row.zero)), K::kNegInf + 1);
    Selected r{false, 0, 0, 0};
    bool found = false;
    if (split != INFINITY && nu.inside <= SMP_FEW && nu.hi - nu.lo >= SMP_BINS) {
      const uint32_t n = collect_all<Raw>(sh, vals, v0, v1, token0, K::value(max(floor_key, nu.lo)), split);
      if (n <= SMP_FEW) {
        if (rank == 0) cut_in_list<Raw>(sh, cs, n, above, goal);
        cluster.sync();
        if (sh.found_count > 0) {
          found = true;
          tau = K::value(sh.found_bin);
          quota = sh.found_count;
        }
      }
    } else if (split != INFINITY) {
      r = select<Raw, true>(sh, vals, v0, v1, max(floor_key, nu.lo), nu.hi, above, goal);
    }
    if (!found && !r.ok) {
      split = INFINITY;
      r = select<Raw, true>(sh, vals, v0, v1, floor_key, sh.row.kmax, 0, goal);
    }
    if (r.ok) {  // else everything with weight is kept
      const unsigned long long w = weight_of(sh, K::value(r.key));
      tau = K::value(r.key);
      quota = (uint32_t)min((goal - r.above + w - 1) / w, (unsigned long long)r.count);
    }
  }
  if (use_m) {
    if (warp == 0) {
      // at max + T log(min_p), up to roundings: searched a millionth around it
      uint32_t lo = K::kNegInf + 1, hi = sh.row.kmax;
      const double at = sh.row.xmax + (double)T * log(sh.row.min_w);
      const double margin = 1e-6 * (fabs(at) + fabs(sh.row.xmax) + (double)T);
      if (fabs(at) + margin < 3e38) {
        lo = max(lo, K::of(__double2float_rd(at - margin)));
        hi = min(hi, K::of(__double2float_ru(at + margin)) + 1);
      }
      const uint32_t k = first_key(lo, max(lo, hi), [&](uint32_t q) { return heavy(sh.row, K::value(q)); });
      if (lane == 0) sh.minp_key = k;
    }
    __syncthreads();
    const float below = K::value(sh.minp_key - 1);
    if (below >= tau) {
      tau = below;
      quota = 0;
      if (tau >= split) split = INFINITY;
    }
  }

  // ---- draw: the range in which the running sum passes u * S, then, by its
  // warp, the lane and the token
  const float from = above_of(tau);
  const unsigned long long wtau = quota > 0 ? weight_of(sh, tau) : 0ull;
  sum_pass(from, split, false);
  if (warp == 0) {
    if (split != INFINITY) {
      for (int i = lane; i < ranges; i += 32) sh.wsum[i] += sh.whigh[i];
      __syncwarp();
    }
    const Found f = find_entry(sh.wsum, sh.wties, ranges, quota, wtau, sh.row.u);
    if (f.entry >= 0) {
      sh.at_range = f.entry;
      sh.at_target = f.t;
      sh.at_ties = f.quota;
      sh.total = f.total;
    }
  }
  __syncthreads();
  if (sh.at_range != rank * SMP_WARPS + warp) return;
  unsigned long long t = sh.at_target;
  uint32_t left = sh.at_ties;
  for (int vb = v0; vb < v1; vb += 32) {
    const int v = vb + lane;
    const uint4 q = v < v1 ? vals[v] : make_uint4(K::kFill, K::kFill, K::kFill, K::kFill);
    float x[PV];
    unsigned long long s = 0;
    uint32_t ties = 0, mine = 0;  // ties, and how many of them this lane may keep
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < PV; ++i) s += weight_from(x[i], from, sh.row.xmax, sh.row.k1, sh.exp2_table);
    if (quota > 0) {
#pragma unroll
      for (int i = 0; i < PV; ++i) ties += x[i] == tau;
      const uint32_t tinc = warp_inclusive(ties, lane);
      mine = left > tinc - ties ? left - (tinc - ties) : 0;
      const uint32_t all = __shfl_sync(0xffffffffu, tinc, 31);
      left = left > all ? left - all : 0;
      s += (unsigned long long)min(mine, ties) * wtau;
    }
    const unsigned long long inc = warp_inclusive(s, lane);
    const unsigned long long all = __shfl_sync(0xffffffffu, inc, 31);
    if (t < all) {
      if (inc - s <= t && t < inc) {
        unsigned long long run = inc - s;
        int at = -1;
        float x_at = 0.f;
#pragma unroll
        for (int i = 0; i < PV; ++i) {
          if (at < 0) {
            unsigned long long w = weight_from(x[i], from, sh.row.xmax, sh.row.k1, sh.exp2_table);
            if (mine > 0 && x[i] == tau) {
              w = wtau;
              --mine;
            }
            if (t < run + w) {
              at = i;
              x_at = x[i];
            }
            run += w;
          }
        }
        p.out[row] = token0 + v * PV + at;
        if (p.logprob) p.logprob[row] = log_share(sh.row, x_at, (double)sh.total / SMP_ONE);
      }
      return;
    }
    t -= all;
  }
}

// CTAs per row: enough that two of them, with their share of the row, fit an
// SM (or one, for the longest rows); more while the batch leaves places idle
// and a thread keeps a vector.
template <typename Raw>
static int sample_launch(const LLSample& p, cudaStream_t stream) {
  constexpr int PV = Key<Raw>::kPerVec;
  const int nvec = (p.V + PV - 1) / PV + 1;  // + 1: a row that starts inside a vector
  const size_t fixed = (sizeof(SampleShared) + 15) & ~size_t(15);
  const size_t limit = 227 * 1024;
  auto bytes = [&](int cs) { return fixed + (size_t)((nvec + cs - 1) / cs) * 16; };
  int cs = 1;
  while (cs < SMP_MAX_CLUSTER && bytes(cs) > limit / 2 - 1024) cs *= 2;
  if (bytes(cs) > limit) return -4;
  while (cs < SMP_MAX_CLUSTER && (int64_t)p.B * cs * 2 <= 296 && nvec / (2 * cs) >= SMP_THREADS) cs *= 2;
  auto kern = sample_kernel<Raw>;
  static unsigned long long done = 0;
  if (!smem_on_device(kern, (int)limit, done)) return -7;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * cs));
  cfg.blockDim = dim3(SMP_THREADS);
  cfg.dynamicSmemBytes = bytes(cs);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)cs, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? 0 : -5;
}

}  // namespace ll

extern "C" int ll_sample(const LLSample* p, cudaStream_t stream) {
  if (p->B <= 0) return 0;
  if (p->V <= 0 || p->V > LL_SAMPLE_MAX_VOCAB || p->B > (1 << 27)) return -3;
  return p->fp32 ? ll::sample_launch<uint32_t>(*p, stream) : ll::sample_launch<uint16_t>(*p, stream);
}
