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
// lower bound on tau that one pass finds (the ranges' own maxima bound the
// k-th largest; the mass per power of two of the weight bounds the nucleus;
// min-p is a bound) picks them out of the row, and one CTA sorts them.  Else tau comes from radix selection on the values' order-preserving
// integer keys, with token counts (top-k) or weights (top-p) summed per bin;
// top-p selects within the power of two that its cut falls in.
//
// Exact weights are integers: w in units of 2^-44, computed in double.
// Integer sums do not depend on their order, so a row gives the same token
// whatever batch, cluster size or device it is drawn on, and the sums over a
// whole vocabulary (2^19 tokens at most: 2^63) are exact to 2^-45 of the
// largest weight per token.  A token below 2^-45 of it has weight 0 and is
// never drawn.
//
// An exact weight takes some 25 instructions, and a row of 152064 tokens is
// 150 a thread of a cluster.  Sums over many tokens are therefore first taken
// with the hardware's 2^x (4 instructions a token) together with a bound on
// their error, 2^-22 (1.75 + 0.35 |log2 w|) of each weight:
//   ex2.approx 2^-22; its argument |log2 w| 2^-24 from the product's rounding
//   and as much from the factor's, times ln 2; three rounded additions.
// Where the bound leaves one answer possible, that is the exact one; else (a
// border closer than about 1e-6 of the sum) the row is summed exactly.
//
// A cluster of CTAs owns a row and holds it in shared memory, so the logits
// are read from memory once; the passes over the row run on shared memory and
// exchange their sums through it (distributed shared memory).  The passes are
// functions of their own, not inlined: two CTAs of 512 threads a SM leave 64
// registers, and what the rest of the kernel keeps alive would spill inside
// their loops, to memory that has no L1 left (an exact sum took 110 cycles a
// warp and logit that way, 15 without).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstddef>

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
constexpr int SMP_OCTAVES = 16;            // powers of two of the weight, the last one open
constexpr int SMP_LIST = 2048;             // candidates, in one segment per CTA
constexpr int SMP_FEW = 2 * SMP_THREADS;   // of them that one CTA sorts
constexpr double SMP_FAST_ONE = 1099511627776.0;  // 2^40: unit of the approximate sums
constexpr float SMP_LOWEST = -3.4028234663852886e38f;

// What a row's passes need to know of it.
struct Row {
  double xmax, inv_t, k1;  // t = (x - xmax) k1 is 32 log2 w
  double shift;            // approximate weights times it are true to their own error
  double u, top_p, min_w;
  float top;               // xmax
  float zero;              // smaller logits weigh less than half a unit
  float fc, fm;            // approximately log2 w = x fc + fm, a little below 0 at the largest
  uint32_t kmax;
};

struct SampleShared {
  Row row;
  float wmax[SMP_RANGES];                // largest logit of each warp range
  float wkth[SMP_RANGES];                // the r-th largest of its lanes' largest
  unsigned long long wsum[SMP_RANGES];   // kept weight of each range
  uint32_t wties[SMP_RANGES];            // its tokens equal to tau
  float werr[SMP_RANGES];                // error bound of an approximate sum, in units of 2^-22
  unsigned long long octave[2][SMP_MAX_CLUSTER][SMP_OCTAVES];  // each CTA's mass per bin; levels alternate
  uint32_t listed[SMP_MAX_CLUSTER];      // candidates of each CTA
  unsigned long long scan[SMP_WARPS];
  unsigned long long found_above, total, at_target;
  uint32_t found_bin, found_count;
  float bound;
  uint32_t minp_key;
  uint32_t edge[2];
  int at_range;
  uint32_t at_ties;
  int redo;
  uint32_t count_here;
  double exp2_table[32];
  union {
    struct {
      alignas(16) uint32_t count[SMP_BINS];  // read four bins at a time
      alignas(16) unsigned long long weight[SMP_BINS];
    };
    struct {
      alignas(16) unsigned long long list[SMP_LIST];  // key << 32 | ~index
      alignas(16) unsigned long long flat[SMP_FEW];   // the same without gaps
    };
    uint32_t mine[SMP_OCTAVES][SMP_THREADS];  // each thread's mass per bin
  };
};
static_assert(offsetof(SampleShared, count) % 16 == 0 && offsetof(SampleShared, weight) % 16 == 0, "vector reads");

// w of a logit, in units of 2^-44, with w = 2^(t / 32), t = (x - max) 32 / (T ln 2):
// t = n + f, n whole and |f| <= 1/2;  2^(f / 32) by its Taylor polynomial of
// degree 4 (within 1.2e-12), 2^(n / 32) from a table and the exponent.  Eleven
// double operations; the library's exponential takes about three times that.
// For zero <= x <= max.
__device__ __forceinline__ unsigned long long exact_weight(float x, double xmax, double k1, const double* table) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
  constexpr double c1 = 0.02166084939249829, c2 = 2.3459619820224677e-4, c3 = 1.6938509724371819e-6,
                   c4 = 9.172562701824643e-9;    // (ln 2 / 32)^i / i!
  // float -> double by its bits (the conversion unit is slow); a subnormal
  // becomes a number of about its size, infinity a finite number
  const uint32_t b = __float_as_uint(x);
  const double xd = __hiloint2double((int)(((b & 0x7FFFFFFFu) >> 3) + (896u << 20) + (b & 0x80000000u)), (int)(b << 29));
  const double t = (xd - xmax) * k1;
  const double m = t + kMagic;
  const int n = __double2loint(m);
  const double f = t - (m - kMagic);
  double p = fma(fma(fma(fma(c4, f, c3), f, c2), f, c1), f, 1.0);
  p *= table[n & 31];
  // * 2^(n >> 5) * 2^44, then to a whole number
  p = __hiloint2double(__double2hiint(p) + (((n >> 5) + 44) << 20), __double2loint(p));
  p += kMagic;
  return (((unsigned long long)(uint32_t)__double2hiint(p) << 32) | (uint32_t)__double2loint(p)) - 0x4338000000000000ull;
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

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// Bitonic sort of n (a power of two, at most 2 SMP_THREADS) values in shared
// memory, largest first; a pair a thread and step.  Up to 64 values are one
// warp's, which needs no barrier of the block.
__device__ __noinline__ void sort_descending(unsigned long long* a, uint32_t n) {
  __syncthreads();
  const bool one_warp = n <= 64;
  if (!one_warp || threadIdx.x < 32)
    for (uint32_t k = 2; k <= n; k *= 2)
      for (uint32_t j = k / 2; j > 0; j /= 2) {
        const uint32_t i = 2 * threadIdx.x - (threadIdx.x & (j - 1));
        if (i + j < n) {
          const unsigned long long x = a[i], y = a[i + j];
          if ((x < y) == ((i & k) == 0)) {
            a[i] = y;
            a[i + j] = x;
          }
        }
        if (one_warp) __syncwarp();
        else __syncthreads();
      }
  __syncthreads();
}

template <int N>
__device__ __forceinline__ float tree_sum(const float (&a)[N]) {
  if constexpr (N == 8) return ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
  else return (a[0] + a[1]) + (a[2] + a[3]);
}

// ---- passes over a warp's range [a, b) of vectors, results per lane

// Exact weight of the logits >= from.
template <typename Raw>
__device__ __noinline__ unsigned long long exact_sum(const uint4* vals, int a, int b, float from, double xmax,
                                                     double k1, const double* table) {
  using K = Key<Raw>;
  unsigned long long s = 0;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < from) continue;
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) s += weight_from(x[i], from, xmax, k1, table);
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

// Approximate weights of a vector's logits >= from; their sum, and the error
// bound of it in units of 2^-22 added to `err`.
template <typename Raw>
__device__ __forceinline__ float fast_vector(const uint4& q, float fc, float fm, float from,
                                             float (&w)[Key<Raw>::kPerVec], float& err) {
  using K = Key<Raw>;
  float x[K::kPerVec], e[K::kPerVec];
  K::unpack(q, x);
#pragma unroll
  for (int i = 0; i < K::kPerVec; ++i) {
    const float arg = fmaf(x[i], fc, fm);
    w[i] = x[i] >= from ? ex2_approx(arg) : 0.f;
    e[i] = w[i] * fmaxf(arg, -150.f);  // -inf: no weight
  }
  const float s = tree_sum(w);
  err += 1.75f * s - 0.35f * tree_sum(e);
  return s;
}
struct FastSum {
  unsigned long long s;
  float err;
};
template <typename Raw>
__device__ __noinline__ FastSum fast_sum(const uint4* vals, int a, int b, float fc, float fm, float from) {
  using K = Key<Raw>;
  FastSum r{0, 0.f};
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    float w[K::kPerVec];
    r.s += __float2ull_rn(fast_vector<Raw>(vals[v], fc, fm, from, w, r.err) * (float)SMP_FAST_ONE);
  }
  return r;
}

// Mass per bin of -log2 w, to the thread's own sums: w 2^(e + 23) <= 2^23,
// rounded to a whole number.  All logits, bins floor(-log2 w); or those within
// [flo, fhi], bins floor((-log2 w - a0) sc).
__device__ __forceinline__ void put_mass(uint32_t* mine, uint32_t b, uint32_t e, float arg) {
  const float m = fmaf(ex2_approx(arg), __uint_as_float((127u + 23u + e) << 23), 8388608.f);
  mine[b * SMP_THREADS] += __float_as_uint(m) - 0x4B000000u;
}
__device__ __forceinline__ float bin_of(float x, float fc, float fm, float a0, float sc) {  // + 2^23
  return __fadd_rd(fminf(fmaxf((-fmaf(x, fc, fm) - a0) * sc, 0.f), (float)(SMP_OCTAVES - 1)), 8388608.f);
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
      const uint32_t bin = __float_as_uint(__fadd_rd(fminf(-arg, (float)(SMP_OCTAVES - 1)), 8388608.f)) - 0x4B000000u;
      put_mass(mine, bin, bin, arg);
    }
  }
}
template <typename Raw>
__device__ __noinline__ void refine_sums(const uint4* vals, int a, int b, float fc, float fm, float a0, float sc,
                                         uint32_t oct, float flo, float fhi, uint32_t* mine) {
  using K = Key<Raw>;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < flo) continue;
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) {  // outside: no mass, without a branch
      const bool in = x[i] >= flo && x[i] <= fhi;
      put_mass(mine, __float_as_uint(bin_of(x[i], fc, fm, a0, sc)) - 0x4B000000u, oct,
               in ? fmaf(x[i], fc, fm) : -INFINITY);
    }
  }
}

// Tokens per bin of (key - lo) >> shift, keys in [lo, hi]; with shift > 0 and
// table, their weights too.
template <typename Raw>
__device__ __noinline__ void histogram(const uint4* vals, int a, int b, float flo, float fhi, uint32_t lo, int shift,
                                       uint32_t* count, unsigned long long* weight, double xmax, double k1,
                                       const double* table) {
  using K = Key<Raw>;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < flo) continue;
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i) {
      const uint32_t bin = (K::of(x[i]) - lo) >> shift;
      if (x[i] >= flo && x[i] <= fhi) {
        atomicAdd(&count[bin], 1u);
        if (weight != nullptr) atomicAdd(&weight[bin], exact_weight(x[i], xmax, k1, table));
      }
    }
  }
}

// Candidates >= xlo into this CTA's segment of the first CTA's list.
template <typename Raw>
__device__ __noinline__ void collect(const uint4* vals, int a, int b, int token0, float xlo, uint32_t* counter,
                                     unsigned long long* to, uint32_t segment) {
  using K = Key<Raw>;
  for (int v = a + (threadIdx.x & 31); v < b; v += 32) {
    const uint4 q = vals[v];
    if (K::largest(q) < xlo) continue;
    float x[K::kPerVec];
    K::unpack(q, x);
#pragma unroll
    for (int i = 0; i < K::kPerVec; ++i)
      if (x[i] >= xlo) {
        const uint32_t at = atomicAdd(counter, 1u);
        if (at < segment)
          to[at] = (unsigned long long)K::of(x[i]) << 32 | (0xFFFFFFFFu - (uint32_t)(token0 + v * K::kPerVec + i));
      }
  }
}

// Running sums of kept weight over the n <= 128 ranges: weight above tau and
// tokens at tau, of which the first `quota` count `wtau` each.  One warp; lane
// l holds entries [l per, (l + 1) per).  The lane whose entry passes u times
// the total returns entry >= 0, what is left of that target before the entry,
// and of the quota.
struct Found {
  int entry;
  unsigned long long t, total;
  uint32_t quota;
};
__device__ __noinline__ Found find_entry(const unsigned long long* wsum, const uint32_t* wties, int n, uint32_t quota,
                                         unsigned long long wtau, double u) {
  constexpr int MOST = SMP_RANGES / 32;
  const int lane = threadIdx.x & 31;
  const int per = (n + 31) / 32;
  unsigned long long s[MOST], mine = 0;
  uint32_t k[MOST], ties = 0;
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int i = lane * per + j;
    const bool in = j < per && i < n;
    s[j] = in ? wsum[i] : 0ull;
    k[j] = in && quota > 0 ? wties[i] : 0u;
    ties += k[j];
  }
  uint32_t before = quota > 0 ? warp_inclusive(ties, lane) - ties : 0u;
  Found f{-1, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const uint32_t left = quota > before ? quota - before : 0u;
    before += k[j];
    s[j] += (unsigned long long)min(left, k[j]) * wtau;
    k[j] = left;
    mine += s[j];
  }
  const unsigned long long inc = warp_inclusive(mine, lane);
  f.total = __shfl_sync(0xffffffffu, inc, 31);
  unsigned long long t = u > 0.0 ? (u < 1.0 ? (unsigned long long)(u * (double)f.total) : f.total - 1) : 0ull;
  if (t >= f.total) t = f.total - 1;
  unsigned long long run = inc - mine;
  if (run <= t && t < inc) {
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
      if (f.entry < 0) {
        if (t < run + s[j]) {
          f.entry = lane * per + j;
          f.t = t - run;
          f.quota = k[j];
        } else {
          run += s[j];
        }
      }
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
  return x == r.top || (!isinf(r.top) && exp(((double)x - r.xmax) * r.inv_t) >= r.min_w);
}

// Largest key in [lo, hi] at which `above` (the sum over keys larger than hi)
// plus the sum over keys from it to hi reaches a target: tokens, or their
// weights (W).  The target is `target`, or with below >= 0
// ceil(top_p (above + all of [lo, hi] + below)), at least 1.
struct Selected {
  bool ok;  // false: never reached
  uint32_t key, count;             // the key, tokens equal to it
  unsigned long long above, goal;  // sum over larger keys
};
template <typename Raw, bool W>
__device__ __noinline__ Selected select(SampleShared& sh, const uint4* vals, int v0, int v1, uint32_t lo, uint32_t hi,
                                        unsigned long long above, unsigned long long target, double below) {
  using K = Key<Raw>;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), tid = threadIdx.x;
  Selected r{false, 0, 0, above, target};
  if (lo > hi) return r;
  for (bool first = true;; first = false) {
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
    histogram<Raw>(vals, v0, v1, K::value(lo), K::value(hi), lo, shift, sh.count, weighted ? sh.weight : nullptr,
                   sh.row.xmax, sh.row.k1, sh.exp2_table);
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
    if (first && below >= 0.0)
      r.goal = (unsigned long long)fmax(1.0, ceil(sh.row.top_p * ((double)r.above + (double)ex.y + below)));
    if (r.above >= r.goal || r.above + ex.y < r.goal) {  // uniform over the cluster
      cluster.sync();
      return r;
    }
    unsigned long long before = r.above + ex.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (before < r.goal && before + val[j] >= r.goal) {
        sh.found_bin = b0 + PER - 1 - j;
        sh.found_above = before;
        sh.found_count = cnt[j];
      }
      before += val[j];
    }
    cluster.sync();  // the found bin, and every read of the bins
    const uint32_t b = sh.found_bin;
    r.above = sh.found_above;
    if (shift == 0) {
      r.ok = true;
      r.key = lo + b;
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

// top-p over the whole row: where its cut falls.  The mass per power of two of
// the weight (bins floor(-log2 w), the last one open), then, while the bin in
// which the cut falls holds many tokens, the mass of its sixteenths.
struct Nucleus {
  double above, err_above;  // keys > hi: mass (units of 1), its error
  double below, err_below;  // keys < lo
  uint32_t lo, hi;
  double tokens;            // at most so many tokens >= lo
};
template <typename Raw>
__device__ __noinline__ Nucleus find_nucleus(SampleShared& sh, const uint4* vals, int v0, int v1, int V) {
  using K = Key<Raw>;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float fc = sh.row.fc, fm = sh.row.fm;
  const double pd = sh.row.top_p;
  Nucleus r{0.0, 0.0, 0.0, 0.0, K::kNegInf + 1, sh.row.kmax, 1e30};
  float a0 = 0.f, sc = 1.f;
  int oct = 0;
  for (int level = 0;; ++level) {
#pragma unroll
    for (int b = 0; b < SMP_OCTAVES; ++b) sh.mine[b][tid] = 0;
    if (level == 0) octave_sums<Raw>(vals, v0, v1, fc, fm, &sh.mine[0][tid]);
    else refine_sums<Raw>(vals, v0, v1, fc, fm, a0, sc, (uint32_t)oct, K::value(r.lo), K::value(r.hi), &sh.mine[0][tid]);
    __syncthreads();
    {  // one warp a bin
      static_assert(SMP_WARPS == SMP_OCTAVES, "a warp a bin");
      unsigned long long m = 0;
#pragma unroll
      for (int i = 0; i < SMP_THREADS; i += 32) m += sh.mine[warp][i + lane];
      m = warp_add(m);
      if (lane < cs) cluster.map_shared_rank(&sh.octave[level & 1][0][0], lane)[rank * SMP_OCTAVES + warp] = m;
    }
    cluster.sync();
    // every warp, a lane a bin: mass, error, the bin in which the cut falls
    double mass = 0.0, err = 0.0;
    if (lane < SMP_OCTAVES) {
      unsigned long long m = 0;
      for (int c = 0; c < cs; ++c) m += sh.octave[level & 1][c][lane];
      const int e = level == 0 ? lane : oct;
      mass = (double)m * __hiloint2double((1023 - 23 - e) << 20, 0);
      // 2^-22 (ex2) + 2^-23 (rounded to a whole) + 2 * 2^-24 |arg| ln 2
      // (argument; the open bin: at most 46); its wholes are of its upper end
      err = mass * ((1.5 + 0.35 * (e == SMP_OCTAVES - 1 ? 46.0 : e + 1.0)) * (1.01 / 4194304.0)) +
            (e == SMP_OCTAVES - 1 ? (double)V * __hiloint2double((1023 - 24 - (SMP_OCTAVES - 1)) << 20, 0) : 0.0);
    }
    const double upto = warp_inclusive(mass, lane), err_upto = warp_inclusive(err, lane);
    const double all = __shfl_sync(0xffffffffu, upto, 31), err_all = __shfl_sync(0xffffffffu, err_upto, 31);
    // top_p (above + all + below) - above, and how far it may be off
    const double goal = pd * (r.above + all + r.below) - r.above;
    const double e = (1.0 - pd) * r.err_above + pd * (err_all + r.err_below) + err_all;
    const uint32_t past = __ballot_sync(0xffffffffu, lane < SMP_OCTAVES - 1 && upto >= goal);
    const uint32_t past0 = __ballot_sync(0xffffffffu, lane < SMP_OCTAVES - 1 && upto >= goal - e);
    const uint32_t past1 = __ballot_sync(0xffffffffu, lane < SMP_OCTAVES - 1 && upto >= goal + e);
    if (level > 0 && (past0 != past || past1 != past)) break;  // on a border: stay with the wider bin
    const int at = past ? __ffs(past) - 1 : SMP_OCTAVES - 1;
    const double here = __shfl_sync(0xffffffffu, upto, at), err_here = __shfl_sync(0xffffffffu, err_upto, at);
    const double in = __shfl_sync(0xffffffffu, mass, at), err_in = __shfl_sync(0xffffffffu, err, at);
    r.above += here - in;
    r.err_above += err_here - err_in;
    r.below += all - here;
    r.err_below += err_all - err_here;
    if (level == 0) {
      oct = at;
      const double n = warp_inclusive(lane < SMP_OCTAVES - 1 ? mass * (double)(2u << lane) * 1.001 : 1e30, lane);
      r.tokens = __shfl_sync(0xffffffffu, n, at);
    }
    // the bin's keys: bin_of does not rise with x
    if (warp < 2) {
      const float border = 8388608.f + (float)(at + 1 - warp);  // bins < at + 1; < at
      uint32_t k = warp == 0 ? r.lo : r.hi + 1;
      if (warp == 0 ? at < SMP_OCTAVES - 1 : at > 0)
        k = first_key(r.lo, r.hi, [&](uint32_t q) { return bin_of(K::value(q), fc, fm, a0, sc) < border; });
      if (lane == 0) sh.edge[warp] = k;
    }
    __syncthreads();
    r.lo = sh.edge[0];
    r.hi = sh.edge[1] - 1;
    const double tokens = oct == SMP_OCTAVES - 1 ? 1e30 : in * (double)(2u << oct);
    // (a bin per key takes 32-bit counts: cheaper than another level up to more tokens)
    if (r.tokens <= SMP_FEW || tokens <= (r.hi - r.lo < SMP_BINS ? 8192.0 : 1024.0) || r.lo >= r.hi || level == 3) break;
    a0 += (float)at / sc;
    sc *= level == 0 && oct == SMP_OCTAVES - 1 ? 0.5f : 16.f;
  }
  return r;
}

// The few candidates in sh.list, in segments of one CTA each: filters, draw.
// `below` and its error: mass (units of 1) of the lighter tokens, for a top-p
// over the whole row (below >= 0).  False: too near a border.
template <typename Raw>
__device__ __noinline__ bool finish_list(SampleShared& sh, const LLSample& p, int64_t row, int cs, uint32_t n,
                                         uint32_t limit, bool use_p, bool use_m, double below, double err) {
  using K = Key<Raw>;
  const int tid = threadIdx.x, segment = SMP_LIST / cs;
  uint32_t base = 0;
  for (int c = 0; c < cs; ++c) {
    const uint32_t m = sh.listed[c];
    for (uint32_t i = tid; i < m; i += SMP_THREADS) sh.flat[base + i] = sh.list[c * segment + i];
    base += m;
  }
  // two tokens a thread, in the order: weights and what is before them
  uint32_t size = 2;
  while (size < n) size *= 2;
  for (uint32_t i = n + tid; i < size; i += SMP_THREADS) sh.flat[i] = 0;
  sort_descending(sh.flat, size);
  limit = min(limit, n);
  unsigned long long c[2], w[2], before[2];
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const uint32_t i = 2 * tid + o;
    c[o] = i < n ? sh.flat[i] : 0ull;
    w[o] = i < limit ? weight_of(sh, K::value((uint32_t)(c[o] >> 32))) : 0ull;
  }
  ulonglong2 ex = block_exclusive(w[0] + w[1], sh.scan);
  before[0] = ex.x;
  before[1] = ex.x + w[0];
  double goal = 0.0, goal0 = 0.0, goal1 = 0.0;
  if (use_p) {
    const double pd = sh.row.top_p, s = (double)ex.y + (below > 0.0 ? below * sh.row.shift * SMP_ONE : 0.0);
    goal = goal0 = goal1 = fmax(1.0, ceil(pd * s));
    if (below >= 0.0) {
      const double e = pd * err * sh.row.shift * SMP_ONE + 2.0;
      goal0 = fmax(1.0, goal - e);
      goal1 = goal + e;
    }
  }
  bool near = false;
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const uint32_t i = 2 * tid + o;
    bool in = i < limit;
    if (in && use_p && i > 0) {
      near |= (double)before[o] >= goal0 && (double)before[o] < goal1;
      in = (double)before[o] < goal;
    }
    // the list ends above the lighter tokens: the cut must lie inside it
    if (below >= 0.0 && i == n - 1) near |= (double)(before[o] + w[o]) < goal1;
    if (in && use_m) in = heavy(sh.row, K::value((uint32_t)(c[o] >> 32)));
    if (!in) c[o] = 0;
  }
  if (__syncthreads_or(near && below >= 0.0)) return false;
  // the kept ones, which are the first: by index (~index, key), and their running sum
  const uint32_t kept = __syncthreads_count(c[0] != 0) + __syncthreads_count(c[1] != 0);
  size = 2;
  while (size < kept) size *= 2;
#pragma unroll
  for (int o = 0; o < 2; ++o)
    if (2 * tid + o < size) sh.flat[2 * tid + o] = c[o] << 32 | c[o] >> 32;
  sort_descending(sh.flat, size);
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    c[o] = 2 * tid + o < kept ? sh.flat[2 * tid + o] : 0ull;
    w[o] = c[o] != 0 ? weight_of(sh, K::value((uint32_t)c[o])) : 0ull;
  }
  ex = block_exclusive(w[0] + w[1], sh.scan);
  const double u = sh.row.u;
  unsigned long long t = u > 0.0 ? (u < 1.0 ? (unsigned long long)(u * (double)ex.y) : ex.y - 1) : 0ull;
  if (t >= ex.y) t = ex.y - 1;
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    if (ex.x <= t && t < ex.x + w[o]) {
      p.out[row] = (int)(0xFFFFFFFFu - (uint32_t)(c[o] >> 32));
      if (p.logprob) p.logprob[row] = log_share(sh.row, K::value((uint32_t)c[o]), (double)ex.y / SMP_ONE);
    }
    ex.x += w[o];
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

  pdl_trigger();
  if (tid < 32) sh.exp2_table[tid] = exp2((double)tid / 32.0);
  if (tid == 0) sh.redo = 0;
  pdl_wait();
  const float T = p.temperature ? p.temperature[row] : 1.f;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;
  const int k_of = T > 0.f && top_k > 0 && top_k < V ? top_k : 0;
  // few candidates: at least k_of tokens lie at or above the k_of-th largest
  // of the ranges' maxima; with r_want of them wanted from every range, at or
  // above the smallest of the ranges' r_want-th largest lane maxima
  const int r_want = k_of <= SMP_FEW ? (k_of + ranges - 1) / ranges : 0;

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
  if (tid == 0) {
    Row& r = sh.row;
    const bool inf = isinf(xmax);  // then all mass is on the infinities, alike
    r.top = xmax;
    r.kmax = K::of(xmax);
    r.xmax = (double)xmax;
    r.inv_t = 1.0 / (double)T;
    r.k1 = inf ? 0.0 : 46.16624130844683 * r.inv_t;  // 32 / ln 2
    // rounded up: no logit from it on is outside the polynomial's range
    float z = fminf(xmax, __double2float_ru(r.xmax - 31.2 * (double)T));
    z = inf ? xmax : K::up(z == kNone ? SMP_LOWEST : z);
    r.zero = z;
    r.fc = (float)(1.4426950408889634 * r.inv_t);
    r.fm = fmaf(-xmax, r.fc, -0.001953125f);  // every argument is below 0
    // 2^-(fm + xmax fc), the exponent within 2^-8: by its series
    const double d = -0.6931471805599453 * ((double)r.fm + r.xmax * (double)r.fc);
    r.shift = 1.0 + d * (1.0 + d * (0.5 + d * (1.0 / 6 + d * (1.0 / 24 + d * (1.0 / 120)))));
    if (inf) r.xmax = 0.0;  // (x - xmax) k1 = 0
    r.u = p.u[row];
    r.top_p = fmax((double)top_p, 0.0);
    r.min_w = fmin((double)min_p, 1.0);
  }
  // where the approximate sums' bound holds: no overflow or cancellation in
  // the arguments, fm rounded to 2^-12 at most
  const float fm_size = fabsf(xmax) / T * 1.4427f;
  const bool fast_ok = T >= 1e-3f && T <= 1e4f && fm_size <= 4000.f && V >= 2048;
  __syncthreads();

  const bool use_p = top_p < 1.f, use_m = min_p > 0.f;
  const bool nucleus = use_p && k_of == 0 && fast_ok;
  Nucleus nu{0.0, 0.0, -1.0, 0.0, K::kNegInf + 1, 0u, 1e30};
  if (nucleus) nu = find_nucleus<Raw>(sh, vals, v0, v1, V);

  // ---- few candidates: every token at or above `xlo`, finished by one CTA
  {
    float xlo = INFINITY;
    if (r_want == 1) {
      if (tid < ranges) {
        const float mine = sh.wmax[tid];
        int larger = 0;
#pragma unroll 8
        for (int i = 0; i < ranges; ++i) {
          const float o = sh.wmax[i];
          larger += o > mine || (o == mine && i < tid);
        }
        if (larger == k_of - 1) sh.bound = mine;
      }
      __syncthreads();
      xlo = sh.bound;
    } else if (r_want > 1) {
      float b = r_want <= 32 ? INFINITY : kNone;
      for (int i = lane; i < ranges; i += 32) b = fminf(b, sh.wkth[i]);
      xlo = -warp_max(-b);
    } else if (nucleus) {
      if (nu.tokens <= SMP_FEW) xlo = K::value(nu.lo);
    } else if (k_of == 0 && !use_p && min_p >= 1e-4f && !isinf(xmax)) {
      // a little below max + T log(min_p)
      xlo = __double2float_rd(sh.row.xmax + (double)T * (log(sh.row.min_w) - 1e-6) - 1e-6 * fabs(sh.row.xmax));
      xlo = K::up(fmaxf(xlo, SMP_LOWEST));
      if (!(xlo <= xmax)) xlo = xmax;
    }
    if (xlo != INFINITY || isinf(xmax)) {
      xlo = fmaxf(fminf(xlo, xmax), SMP_LOWEST);
      const uint32_t segment = SMP_LIST / cs;
      if (tid == 0) sh.count_here = 0;
      __syncthreads();
      collect<Raw>(vals, v0, v1, token0, xlo, &sh.count_here, cluster.map_shared_rank(sh.list, 0) + rank * segment,
                   segment);
      __syncthreads();
      if (tid < cs) cluster.map_shared_rank(sh.listed, tid)[rank] = sh.count_here;
      cluster.sync();
      uint32_t n = 0;
      bool fits = true;
      for (int c = 0; c < cs; ++c) {
        fits = fits && sh.listed[c] <= segment;
        n += sh.listed[c];
      }
      if (fits && n <= SMP_FEW) {
        if (rank == 0 && !finish_list<Raw>(sh, p, row, cs, n, k_of > 0 ? (uint32_t)k_of : n, use_p, use_m, nu.below,
                                           nu.err_below) &&
            tid < cs)
          *cluster.map_shared_rank(&sh.redo, tid) = 1;
        if (!nucleus) return;
        cluster.sync();
        if (!sh.redo) return;
      }
    }
  }

  // ---- many: what is kept is logits above tau, and the first `quota` equal to it
  float tau = kNone;
  uint32_t quota = 0;
  // The smallest logit above tau with weight; NaN where there is none.
  auto above_tau = [&](bool fast) {
    if (tau >= xmax) return __int_as_float(0x7FFFFFFF);
    const float next = tau == kNone ? SMP_LOWEST : K::value(K::of(tau) + 1);
    return fast ? next : fmaxf(next, sh.row.zero);
  };
  // Weight above tau and tokens at tau per warp range, to every CTA.
  auto sum_pass = [&](bool fast) {
    const float next = above_tau(fast);
    unsigned long long s;
    float err = 0.f;
    if (fast) {
      const FastSum f = fast_sum<Raw>(vals, v0, v1, sh.row.fc, sh.row.fm, next);
      s = f.s;
      err = warp_sum(f.err);
    } else {
      s = exact_sum<Raw>(vals, v0, v1, next, sh.row.xmax, sh.row.k1, sh.exp2_table);
    }
    s = warp_add(s);
    const uint32_t ties = quota > 0 ? __reduce_add_sync(0xffffffffu, count_equal<Raw>(vals, v0, v1, tau)) : 0u;
    if (lane < cs) {
      const int i = rank * SMP_WARPS + warp;
      cluster.map_shared_rank(sh.wsum, lane)[i] = s;
      cluster.map_shared_rank(sh.wties, lane)[i] = ties;
      cluster.map_shared_rank(sh.werr, lane)[i] = err;
    }
    cluster.sync();
  };
  if (k_of > 0) {
    const Selected r = select<Raw, false>(sh, vals, v0, v1, K::kNegInf + 1, sh.row.kmax, 0, (unsigned long long)k_of, -1.0);
    if (r.ok) {
      tau = K::value(r.key);
      quota = (uint32_t)(k_of - r.above);
    }
  }
  double kept_bound = k_of > 0 ? k_of : V;  // at most so many tokens are kept
  if (use_p) {
    const uint32_t floor_key = max(K::of(fmaxf(fmaxf(tau, SMP_LOWEST), sh.row.zero)), K::kNegInf + 1);
    // pass 0: from the approximate masses, if they leave one answer; 1: from
    // exact ones, within the same keys; 2: over all keys
    for (int pass = !nucleus ? 2 : (sh.redo ? 1 : 0); pass < 3; ++pass) {
      const float tau0 = tau;
      const uint32_t quota0 = quota;
      unsigned long long above = 0, goal = 0;
      double below = -1.0, e = 0.0;
      uint32_t lo = floor_key, hi = sh.row.kmax;
      if (pass < 2) {
        lo = max(lo, nu.lo);
        hi = nu.hi;
      }
      if (pass == 0) {
        above = (unsigned long long)(nu.above * sh.row.shift * SMP_ONE);
        below = nu.below * sh.row.shift * SMP_ONE;
        // of top_p (above + between + below) - above, and a unit's rounding
        e = ((1.0 - sh.row.top_p) * nu.err_above + sh.row.top_p * nu.err_below) * sh.row.shift * SMP_ONE + 2.0;
      } else {
        for (int part = pass == 1 ? 0 : 1; part < 2; ++part) {  // above the keys; all
          if (part == 0) {
            tau = K::value(hi);
            quota = 0;
          }
          sum_pass(false);
          if (warp == 0) {
            const Found f = find_entry(sh.wsum, sh.wties, ranges, quota, quota > 0 ? weight_of(sh, tau) : 0ull, 0.0);
            if (lane == 0) sh.total = f.total;
          }
          __syncthreads();
          if (part == 0) above = sh.total;
          else goal = (unsigned long long)fmax(1.0, ceil(sh.row.top_p * (double)sh.total));
          tau = tau0;
          quota = quota0;
          cluster.sync();  // every CTA has read its sums
        }
      }
      // predecessors' mass below top_p of all; the first token is always kept
      const Selected r = select<Raw, true>(sh, vals, v0, v1, lo, hi, above, goal, below);
      if (!r.ok) {
        if (pass < 2) continue;
        break;  // everything with weight is kept
      }
      const unsigned long long w = weight_of(sh, K::value(r.key));
      const unsigned long long n = (r.goal - r.above + w - 1) / w;
      if (pass == 0) {
        const double first = ceil(((double)r.goal - e - (double)r.above) / (double)w);
        const double last = ceil(((double)r.goal + e - (double)r.above) / (double)w);
        if (!(first == (double)n && last == (double)n && n <= r.count)) continue;  // too near a border
      }
      tau = K::value(r.key);
      quota = (uint32_t)min(n, (unsigned long long)r.count);
      kept_bound = (double)r.goal / (double)w;
      break;
    }
  }
  if (use_m) {
    if (warp == 0) {
      const uint32_t k = first_key(K::kNegInf + 1, sh.row.kmax, [&](uint32_t q) { return heavy(sh.row, K::value(q)); });
      if (lane == 0) sh.minp_key = k;
    }
    __syncthreads();
    const float below = K::value(sh.minp_key - 1);
    if (below >= tau) {
      tau = below;
      quota = 0;
    }
  }

  // ---- draw: the range in which the running sum passes u * S, then, by its
  // warp, the lane and the token
  for (int pass = fast_ok && kept_bound > 4096.0 ? 0 : 1; pass < 2; ++pass) {
    const bool fast = pass == 0;
    const float one = fast ? (float)SMP_FAST_ONE : (float)SMP_ONE;
    const unsigned long long wtau =
        quota == 0 ? 0ull
                   : (fast ? __float2ull_rn(ex2_approx(fmaf(tau, sh.row.fc, sh.row.fm)) * one) : weight_of(sh, tau));
    sum_pass(fast);
    if (warp == 0) {
      const Found f = find_entry(sh.wsum, sh.wties, ranges, quota, wtau, sh.row.u);
      if (f.entry >= 0) {
        sh.at_range = f.entry;
        sh.at_target = f.t;
        sh.at_ties = f.quota;
        sh.total = f.total;
      }
    }
    __syncthreads();
    if (sh.at_range == rank * SMP_WARPS + warp) {
      unsigned long long t = sh.at_target;
      uint32_t left = sh.at_ties;
      const float from = above_tau(fast);
      for (int vb = v0; vb < v1; vb += 32) {
        const int v = vb + lane;
        const uint4 q = v < v1 ? vals[v] : make_uint4(K::kFill, K::kFill, K::kFill, K::kFill);
        float wf[PV], err = 0.f, x[PV];
        unsigned long long s = 0;
        uint32_t ties = 0;
        K::unpack(q, x);
        if (fast) {
          s = __float2ull_rn(fast_vector<Raw>(q, sh.row.fc, sh.row.fm, from, wf, err) * one);
        } else {
#pragma unroll
          for (int i = 0; i < PV; ++i) s += weight_from(x[i], from, sh.row.xmax, sh.row.k1, sh.exp2_table);
        }
        uint32_t mine = 0, after = 0;  // ties this lane may keep; left after this step
        if (quota > 0) {
#pragma unroll
          for (int i = 0; i < PV; ++i) ties += x[i] == tau;
          const uint32_t tinc = warp_inclusive(ties, lane);
          mine = left > tinc - ties ? left - (tinc - ties) : 0;
          const uint32_t all = __shfl_sync(0xffffffffu, tinc, 31);
          after = left > all ? left - all : 0;
          s += (unsigned long long)min(mine, ties) * wtau;
        }
        const unsigned long long inc = warp_inclusive(s, lane);
        const unsigned long long all = __shfl_sync(0xffffffffu, inc, 31);
        if (t < all) {
          // how far an approximate running sum less u * S may be from the
          // exact one: (1 - u) times the error before, u times the error
          // after (the ties' weights: within 5e-6 of themselves and half a
          // unit; the vector's own sum: 2^-20)
          double margin = 0.0;
          if (fast) {
            float e0 = 0.f, e1 = 0.f;
            for (int i = lane; i < ranges; i += 32) {
              e0 += i <= sh.at_range ? sh.werr[i] : 0.f;
              e1 += i >= sh.at_range ? sh.werr[i] : 0.f;
            }
            const double uc = fmin(fmax(sh.row.u, 0.0), 1.0);
            margin = ((1.0 - uc) * (double)warp_sum(e0) + uc * (double)warp_sum(e1)) * (1.01 / 4194304.0 * SMP_FAST_ONE) +
                     nvec + (double)quota * (5e-6 * (double)wtau + 1.0) + 2.0 + (double)s * 9.5367431640625e-7;
          }
          if (inc - s <= t && t < inc) {
            unsigned long long run = inc - s, w_at = 0;
            int at = -1;
            float x_at = 0.f;
#pragma unroll
            for (int i = 0; i < PV; ++i) {
              if (at < 0) {
                unsigned long long w = 0;
                if (x[i] >= from)
                  w = fast ? __float2ull_rn(wf[i] * one) : exact_weight(x[i], sh.row.xmax, sh.row.k1, sh.exp2_table);
                else if (mine > 0 && x[i] == tau) {
                  w = wtau;
                  --mine;
                }
                if (t < run + w) {
                  at = i;
                  x_at = x[i];
                  w_at = w;
                } else {
                  run += w;
                }
              }
            }
            if (!fast || (at >= 0 && (double)(t - run) > margin && (double)(run + w_at - t) > margin)) {
              p.out[row] = token0 + v * PV + at;
              if (p.logprob)
                p.logprob[row] =
                    log_share(sh.row, x_at, (double)sh.total / (double)one * (fast ? sh.row.shift : 1.0));
            } else {
              for (int c = 0; c < cs; ++c) *cluster.map_shared_rank(&sh.redo, c) = 2;
            }
          }
          break;
        }
        t -= all;
        left = after;
      }
    }
    if (!fast) return;
    cluster.sync();
    if (sh.redo != 2) return;
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
