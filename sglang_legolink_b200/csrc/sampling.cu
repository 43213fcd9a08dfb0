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
// sorted: tau comes from radix selection on the values' order-preserving
// integer keys, with token counts (top-k) or weights (top-p) summed per bin.
//
// Weights are integers: w in units of 2^-44, from a double exponential.
// Integer sums do not depend on their order, so a row gives the same token
// whatever batch, cluster size or device it is drawn on, and the sums over a
// whole vocabulary (2^19 tokens at most: 2^63) are exact to 2^-45 of the
// largest weight per token.  A token below 2^-45 of it has weight 0 and is
// never drawn.
//
// A cluster of CTAs owns a row and holds it in shared memory as keys, so the
// logits are read from memory once; the passes over the row run on shared
// memory and exchange their sums through it (distributed shared memory).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "sampling.h"

namespace cg = cooperative_groups;

namespace ll {

constexpr int SMP_THREADS = 512;
constexpr int SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_MAX_CLUSTER = 8;
constexpr int SMP_BINS = 2048;
constexpr double SMP_ONE = 17592186044416.0;  // 2^44

// Order-preserving keys: larger value, larger key.  -0 and +0 share a key
// (they are equal values); NaN takes key 0, below -inf, so it is never drawn.
template <typename Raw>
struct Key;
template <>
struct Key<uint16_t> {
  static constexpr uint32_t kNegInf = 0x007Fu, kPosInf = 0xFF80u;
  static constexpr int kPerVec = 8;
  __device__ static uint32_t encode(uint32_t b) {
    if ((b & 0x7FFFu) > 0x7F80u) return 0;
    if (b == 0x8000u) b = 0;
    return (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
  }
  __device__ static float decode(uint32_t k) {
    const uint32_t b = (k & 0x8000u) ? (k & 0x7FFFu) : (~k & 0xFFFFu);
    return __uint_as_float(b << 16);
  }
};
template <>
struct Key<uint32_t> {
  static constexpr uint32_t kNegInf = 0x007FFFFFu, kPosInf = 0xFF800000u;
  static constexpr int kPerVec = 4;
  __device__ static uint32_t encode(uint32_t b) {
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0;
    if (b == 0x80000000u) b = 0;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  }
  __device__ static float decode(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
  }
};

struct SampleShared {
  unsigned long long best[SMP_MAX_CLUSTER];                 // (key, ~index) of each CTA's largest logit
  unsigned long long wsum[SMP_MAX_CLUSTER * SMP_WARPS];     // kept weight of each warp's range
  uint32_t wties[SMP_MAX_CLUSTER * SMP_WARPS];              // its tokens equal to tau
  unsigned long long scan[SMP_WARPS];
  unsigned long long found_above, total;
  unsigned long long at_target;
  uint32_t found_bin, found_count;
  uint32_t minp_key;
  int at_warp;
  uint32_t at_ties;
  uint32_t count[SMP_BINS];
  unsigned long long weight[SMP_BINS];
};

// w of a key, in units of 2^-44.
template <typename Raw>
struct Weight {
  double xmax, inv_t;
  uint32_t kmax;
  __device__ double y(uint32_t key) const { return ((double)Key<Raw>::decode(key) - xmax) * inv_t; }
  __device__ unsigned long long operator()(uint32_t key) const {
    if (key == kmax) return (unsigned long long)SMP_ONE;
    if (kmax == Key<Raw>::kPosInf) return 0;  // mass on the infinities alone
    const double v = y(key);
    if (v < -31.2) return 0;  // below half a unit
    return (unsigned long long)__double2ll_rn(exp(v) * SMP_ONE);
  }
};

// exclusive prefix over the block of one value per thread (thread order)
__device__ __forceinline__ unsigned long long block_exclusive(unsigned long long v, unsigned long long* scan,
                                                              unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();
  if (lane == 31) scan[warp] = inc;
  __syncthreads();
  unsigned long long before = 0;
  total = 0;
  for (int w = 0; w < SMP_WARPS; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  return before + inc - v;
}

template <typename Raw>
__global__ void __launch_bounds__(SMP_THREADS) sample_kernel(const LLSample p) {
  using K = Key<Raw>;
  constexpr int PV = K::kPerVec;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
  uint4* keys = reinterpret_cast<uint4*>(smem_raw + ((sizeof(SampleShared) + 15) & ~size_t(15)));

  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / cs;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = p.V;

  pdl_trigger();
  pdl_wait();

  // ---- load: keys to shared memory, the largest logit and its first index
  const Raw* src = reinterpret_cast<const Raw*>(p.logits) + row * p.stride;
  const int pad = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(Raw));  // elements before the row in its first vector
  const int nvec = (pad + V + PV - 1) / PV;
  const int per_cta = (nvec + cs - 1) / cs;
  const int cv0 = min(nvec, rank * per_cta), cv1 = min(nvec, cv0 + per_cta);
  const int per_warp = (per_cta + SMP_WARPS - 1) / SMP_WARPS;
  const int v0 = min(cv1, cv0 + warp * per_warp), v1 = min(cv1, v0 + per_warp);
  const uint4* vsrc = reinterpret_cast<const uint4*>(src - pad);

  auto unpack = [&](const uint4& q, uint32_t (&k)[PV]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (PV == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k[2 * i] = w[i] & 0xFFFFu;
        k[2 * i + 1] = w[i] >> 16;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = w[i];
    }
  };

  unsigned long long best = 0;
  for (int v = v0 + lane; v < v1; v += 32) {
    uint32_t k[PV];
    const int64_t e0 = (int64_t)v * PV - pad;  // token of the vector's first element
    if (e0 >= 0 && e0 + PV <= V) {
      uint32_t raw[PV];
      unpack(vsrc[v], raw);
#pragma unroll
      for (int i = 0; i < PV; ++i) k[i] = K::encode(raw[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PV; ++i) {
        const int64_t e = e0 + i;
        k[i] = (e >= 0 && e < V) ? K::encode((uint32_t)src[e]) : 0u;
      }
    }
    uint4 q;
    if constexpr (PV == 8) {
      q = make_uint4(k[0] | k[1] << 16, k[2] | k[3] << 16, k[4] | k[5] << 16, k[6] | k[7] << 16);
    } else {
      q = make_uint4(k[0], k[1], k[2], k[3]);
    }
    keys[v - cv0] = q;
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      const unsigned long long c = (unsigned long long)k[i] << 32 | (0xFFFFFFFFu - (uint32_t)(e0 + i));
      best = c > best ? c : best;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long t = __shfl_xor_sync(0xffffffffu, best, o);
    best = t > best ? t : best;
  }
  if (lane == 0) sh.scan[warp] = best;
  __syncthreads();
  if (tid < cs) {
    unsigned long long b = 0;
    for (int w = 0; w < SMP_WARPS; ++w) b = sh.scan[w] > b ? sh.scan[w] : b;
    cluster.map_shared_rank(sh.best, tid)[rank] = b;
  }
  cluster.sync();
  best = 0;
  for (int r = 0; r < cs; ++r) best = sh.best[r] > best ? sh.best[r] : best;
  const uint32_t kmax = (uint32_t)(best >> 32);

  const float T = p.temperature ? p.temperature[row] : 1.f;
  const bool greedy = !(T > 0.f);
  if (kmax <= K::kNegInf || greedy) {  // nothing to draw, or the largest logit
    if (rank == 0 && tid == 0) {
      const bool none = kmax <= K::kNegInf;
      p.out[row] = none ? -1 : (int)(0xFFFFFFFFu - (uint32_t)best);
      if (p.logprob) p.logprob[row] = none ? -INFINITY : 0.f;
    }
    return;
  }

  Weight<Raw> wt;
  wt.kmax = kmax;
  wt.xmax = (double)K::decode(kmax);
  wt.inv_t = 1.0 / (double)T;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;

  // Largest key at which the sum over keys >= it reaches `target` (tokens, or
  // their weights); `above` is the sum over larger keys, `c` the tokens equal
  // to it.  Only keys in [lo, kmax] count.  False: the sum never reaches it.
  auto select = [&](auto weighted, uint32_t lo, unsigned long long target, uint32_t& key, unsigned long long& above,
                    uint32_t& c) -> bool {
    constexpr bool W = decltype(weighted)::value;
    uint32_t hi = kmax;
    above = 0;
    while (true) {
      const uint32_t span = hi - lo;
      const int shift = span < (uint32_t)SMP_BINS ? 0 : 32 - __clz(span) - 11;
      for (int i = tid; i < SMP_BINS; i += SMP_THREADS) {
        sh.count[i] = 0;
        if constexpr (W) sh.weight[i] = 0;
      }
      __syncthreads();
      for (int v = v0 + lane; v < v1; v += 32) {
        uint32_t k[PV];
        unpack(keys[v - cv0], k);
#pragma unroll
        for (int i = 0; i < PV; ++i)
          if (k[i] >= lo && k[i] <= hi) {
            const uint32_t b = (k[i] - lo) >> shift;
            atomicAdd(&sh.count[b], 1u);
            if constexpr (W)
              if (shift > 0) atomicAdd(&sh.weight[b], wt(k[i]));
          }
      }
      cluster.sync();
      // thread t merges bins [B-1-4t-3, B-1-4t], largest first
      constexpr int PER = SMP_BINS / SMP_THREADS;
      uint32_t cnt[PER];
      unsigned long long val[PER], mine = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int b = SMP_BINS - 1 - tid * PER - j;
        uint32_t n = 0;
        unsigned long long w = 0;
        for (int r = 0; r < cs; ++r) {
          n += cluster.map_shared_rank(sh.count, r)[b];
          if constexpr (W)
            if (shift > 0) w += cluster.map_shared_rank(sh.weight, r)[b];
        }
        cnt[j] = n;
        if constexpr (!W) w = n;
        else if (shift == 0 && n > 0) w = n * wt(lo + b);
        val[j] = w;
        mine += w;
      }
      unsigned long long total;
      unsigned long long before = above + block_exclusive(mine, sh.scan, total);
      if (above + total < target) {  // uniform over the cluster
        cluster.sync();
        return false;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (before < target && before + val[j] >= target) {
          sh.found_bin = SMP_BINS - 1 - tid * PER - j;
          sh.found_above = before;
          sh.found_count = cnt[j];
        }
        before += val[j];
      }
      cluster.sync();  // the found bin, and every read of the bins
      const uint32_t b = sh.found_bin;
      above = sh.found_above;
      if (shift == 0) {
        key = lo + b;
        c = sh.found_count;
        return true;
      }
      const uint32_t nlo = lo + (b << shift);
      hi = min(hi, nlo + ((1u << shift) - 1));
      lo = nlo;
    }
  };

  // Weight of what (tau, quota) keeps, per warp range, in every CTA.
  auto sum_pass = [&](uint32_t tau) {
    unsigned long long s = 0;
    uint32_t ties = 0;
    for (int v = v0 + lane; v < v1; v += 32) {
      uint32_t k[PV];
      unpack(keys[v - cv0], k);
#pragma unroll
      for (int i = 0; i < PV; ++i) {
        if (k[i] > tau) s += wt(k[i]);
        ties += k[i] == tau;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      ties += __shfl_xor_sync(0xffffffffu, ties, o);
    }
    if (lane < cs) {
      cluster.map_shared_rank(sh.wsum, lane)[rank * SMP_WARPS + warp] = s;
      cluster.map_shared_rank(sh.wties, lane)[rank * SMP_WARPS + warp] = ties;
    }
    cluster.sync();
  };
  auto total_of = [&](uint32_t tau, uint32_t quota) {
    unsigned long long s = 0;
    uint32_t ties = 0;
    for (int i = 0; i < cs * SMP_WARPS; ++i) {
      s += sh.wsum[i];
      ties += sh.wties[i];
    }
    if (quota > 0) s += (unsigned long long)min(ties, quota) * wt(tau);
    return s;
  };

  uint32_t tau = K::kNegInf, quota = 0;
  if (top_k > 0 && top_k < V) {
    uint32_t key, c;
    unsigned long long above;
    if (select(std::false_type{}, K::kNegInf + 1, (unsigned long long)top_k, key, above, c)) {
      tau = key;
      quota = (uint32_t)(top_k - above);
    }
  }
  if (top_p < 1.f) {
    sum_pass(tau);
    const unsigned long long s1 = total_of(tau, quota);
    // predecessors' mass below top_p * s1; the first token is always kept
    const double target = ceil((double)top_p * (double)s1);
    const unsigned long long goal = target >= 1.0 ? min(s1, (unsigned long long)target) : 1ull;
    uint32_t key, c;
    unsigned long long above;
    if (select(std::true_type{}, max(tau, K::kNegInf + 1), goal, key, above, c)) {
      const unsigned long long w = wt(key);
      tau = key;
      quota = (uint32_t)((goal - above + w - 1) / w);
    }
  }
  if (min_p > 0.f) {
    // smallest key whose weight is at least min_p: 32-ary search, one warp
    if (warp == 0) {
      const double m = fmin((double)min_p, 1.0);
      uint32_t lo = K::kNegInf + 1, hi = kmax;  // kmax qualifies
      while (lo < hi) {
        const uint32_t step = (hi - lo) / 32 + 1;
        const uint32_t probe = (uint32_t)min((unsigned long long)hi, (unsigned long long)lo + (unsigned long long)lane * step);
        const bool in = probe == kmax || (kmax != K::kPosInf && exp(wt.y(probe)) >= m);
        const uint32_t ok = __ballot_sync(0xffffffffu, in);
        const int f = __ffs(ok) - 1;  // first probe inside; none: beyond the last one
        const uint32_t base = lo;
        if (f < 0) {
          lo = base + 31 * step + 1;
        } else {
          hi = (uint32_t)min((unsigned long long)hi, (unsigned long long)base + (unsigned long long)f * step);
          if (f > 0) lo = base + (f - 1) * step + 1;
        }
      }
      if (lane == 0) sh.minp_key = lo;
    }
    __syncthreads();
    if (sh.minp_key > tau) {
      tau = sh.minp_key - 1;
      quota = 0;
    }
  }

  // ---- draw: the warp range in which the running sum passes u * S
  sum_pass(tau);
  if (tid == 0) {
    const unsigned long long total = total_of(tau, quota);
    const double u = p.u[row];
    unsigned long long t = u > 0.0 ? (u < 1.0 ? (unsigned long long)(u * (double)total) : total - 1) : 0ull;
    if (t >= total) t = total - 1;
    const unsigned long long wtau = quota > 0 ? wt(tau) : 0;
    unsigned long long run = 0;
    uint32_t ties = 0;
    int at = 0;
    for (int i = 0; i < cs * SMP_WARPS; ++i) {
      const uint32_t left = quota > ties ? quota - ties : 0;
      const unsigned long long s = sh.wsum[i] + (unsigned long long)min(left, sh.wties[i]) * wtau;
      at = i;
      if (run + s > t) break;
      run += s;
      ties += sh.wties[i];
    }
    sh.at_warp = at;
    sh.at_target = t - run;
    sh.at_ties = quota > ties ? quota - ties : 0;
    sh.total = total;
  }
  __syncthreads();
  if (sh.at_warp != rank * SMP_WARPS + warp) return;
  const unsigned long long wtau = quota > 0 ? wt(tau) : 0;
  unsigned long long t = sh.at_target;
  uint32_t left = sh.at_ties;
  for (int vb = v0; vb < v1; vb += 32) {
    const int v = vb + lane;
    uint32_t k[PV];
    uint32_t ties = 0;
#pragma unroll
    for (int i = 0; i < PV; ++i) k[i] = 0;
    if (v < v1) unpack(keys[v - cv0], k);
#pragma unroll
    for (int i = 0; i < PV; ++i) ties += k[i] == tau;
    uint32_t tinc = ties;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, tinc, o);
      if (lane >= o) tinc += x;
    }
    uint32_t mine = left > tinc - ties ? left - (tinc - ties) : 0;  // ties this lane may keep
    unsigned long long w[PV], s = 0;
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      w[i] = 0;
      if (k[i] > tau) {
        w[i] = wt(k[i]);
      } else if (k[i] == tau && mine > 0) {
        w[i] = wtau;
        --mine;
      }
      s += w[i];
    }
    unsigned long long inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    const unsigned long long all = __shfl_sync(0xffffffffu, inc, 31);
    if (t < all) {
      if (inc - s <= t && t < inc) {
        unsigned long long run = inc - s;
        int at = 0;
        for (int i = 0; i < PV; ++i) {
          at = i;
          if (run + w[i] > t) break;
          run += w[i];
        }
        p.out[row] = (int)((int64_t)v * PV - pad + at);
        if (p.logprob) {
          uint32_t key = 0;
#pragma unroll
          for (int i = 0; i < PV; ++i)
            if (i == at) key = k[i];
          const double y = key == kmax ? 0.0 : wt.y(key);
          p.logprob[row] = (float)(y - log((double)sh.total / SMP_ONE));
        }
      }
      return;
    }
    t -= all;
    const uint32_t alln = __shfl_sync(0xffffffffu, tinc, 31);
    left = left > alln ? left - alln : 0;
  }
}

// CTAs per row: enough that a row fits in their shared memory; more while
// the batch leaves SMs idle and a CTA keeps at least a vector per thread.
template <typename Raw>
static int sample_launch(const LLSample& p, cudaStream_t stream) {
  constexpr int PV = Key<Raw>::kPerVec;
  const int nvec = (p.V + PV - 1) / PV + 1;  // + 1: a row that starts inside a vector
  const size_t fixed = (sizeof(SampleShared) + 15) & ~size_t(15);
  const size_t limit = 227 * 1024;
  auto bytes = [&](int cs) { return fixed + (size_t)((nvec + cs - 1) / cs) * 16; };
  int cs = 1;
  while (cs < SMP_MAX_CLUSTER && bytes(cs) > limit) cs *= 2;
  if (bytes(cs) > limit) return -4;
  while (cs < SMP_MAX_CLUSTER && (int64_t)p.B * cs * 2 <= 148 && nvec / (2 * cs) >= SMP_THREADS) cs *= 2;
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
