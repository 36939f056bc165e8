// sample_requests.cu — a token for each request of a step, with its own temperature, top-k, top-p,
// min-p and random number (gq_sample_requests).
//
//   w_i = e^((l_i - max l) / T)
//   in the order of the logits (largest first, ties to the smaller id): the first top_k; of those the
//   shortest run that holds top_p of their mass; of those the ones with w_i >= min_p
//   token: in the order of the ids, the first kept one at which the running sum of w passes u * (their sum)
//
// All three options keep a beginning of the order, so what is left is one border: a logit and an id.
// It is found without sorting, by radix selection over (logit, id) keys of 64 bits: counts for top-k,
// masses for top-p. Masses are whole numbers, w * 2^44 rounded: their sums (vocab <= 2^19) fit 64 bits,
// and do not depend on the order of additions, so atomics may add them up. The weights are made in f64:
// with f32's 2^-24 a draw over 262144 tokens would land on a neighbour of the right token every few
// hundred rows; 2^-45 leaves less than one in 10^6.
//
// A row is kept in the shared memory of a cluster of CTAs, each with a share of its columns: the logits
// are read once, and every pass over them is on chip.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "gq_internal.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kBits = 11, kBins = 1 << kBits;
constexpr int kOne = 44;                  // w = 1 is 2^44
constexpr int kMaxShare = 32768;          // columns of a CTA
constexpr int64_t kMaxVocab = (int64_t)kMaxShare * kMaxCluster;

struct Args {
  const float *logits;
  int64_t ld;
  int vocab, share;  // share: columns of a CTA, a multiple of 4
  const float *temperature, *top_p, *min_p;
  const int32_t *top_k;
  const double *uniforms;
  uint64_t *rng;
  int32_t *tokens;
  float *probs;
};

// Order of the logits as an order of numbers (no logit is NaN here, and no zero negative).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
// Of a logit and its id: larger logits first, then smaller ids.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t id) { return ((uint64_t)key_of(v) << 32) | (uint32_t)~id; }

// w * 2^44 to the nearest whole number; `scale` is log2(e) / T.
__device__ __forceinline__ uint64_t mass_of(float v, float top, double scale) {
  if (v == top) return 1ull << kOne;
  if (v == -INFINITY) return 0;
  const double x = ((double)v - (double)top) * scale;
  return x >= -(kOne + 2.0) ? __double2ull_rn(exp2(x + kOne)) : 0;
}

struct Shared {
  uint64_t hist[kBins];
  uint64_t warp_sum[kWarps];
  uint64_t cta_sum[kMaxCluster];  // written by every CTA of the cluster
  float top[kMaxCluster];
  uint32_t first[kMaxCluster];
  uint64_t prefix, need;          // written by the first CTA of the cluster
  float warp_top[kWarps];
};

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t up = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += up;
  }
  return v;
}

struct Row {
  const float *vals;  // this CTA's columns
  int n;
  uint32_t id0;
  float top;
  double scale;
};

// The border of the shortest beginning of the order (of what is at or above `above`) whose mass, or
// count, reaches `share` of the whole, or `count`: the key of its last member.
template <bool MASS>
__device__ uint64_t find_border(cg::cluster_group &cluster, Shared &s, const Row &row, uint64_t above, double share, uint64_t count) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t prefix = 0, need = count;
  for (int shift = 64 - kBits, bits = kBits;;) {
    for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < row.n; i += kThreads) {
      const float v = row.vals[i];
      const uint64_t k = rank_key(v, row.id0 + i);
      if (k < above || (shift + bits < 64 && (k >> (shift + bits)) != prefix)) continue;
      const uint64_t w = MASS ? mass_of(v, row.top, row.scale) : 1ull;
      if (w) atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[(k >> shift) & ((1u << bits) - 1)]), (unsigned long long)w);
    }
    cluster.sync();
    if (cluster.block_rank() == 0) {
      // thread t has bins from the top: kBins - 1 - 2 t and the one below
      uint64_t w[2] = {0, 0};
      for (int r = 0; r < (int)cluster.num_blocks(); ++r) {
        const uint64_t *h = cluster.map_shared_rank(s.hist, r);
        w[0] += h[kBins - 1 - 2 * tid];
        w[1] += h[kBins - 2 - 2 * tid];
      }
      uint64_t incl = warp_scan(w[0] + w[1]);
      if (lane == 31) s.warp_sum[warp] = incl;
      __syncthreads();
      uint64_t total = 0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) incl += s.warp_sum[i];
        total += s.warp_sum[i];
      }
      uint64_t want = need;
      if (MASS && shift + bits == 64) {
        const double x = ceil(share * (double)total);
        want = x >= 1.0 ? (uint64_t)x : 1ull;
      }
      want = min(want, total);
      const uint64_t before = incl - w[0] - w[1];
      if (want > before && want <= incl) {
        const bool second = want > before + w[0];
        s.prefix = (prefix << bits) | (uint64_t)(kBins - 1 - 2 * tid - second);
        s.need = want - before - (second ? w[0] : 0);
      }
      __syncthreads();
      if (tid < (int)cluster.num_blocks() && tid > 0) {
        *cluster.map_shared_rank(&s.prefix, tid) = s.prefix;
        *cluster.map_shared_rank(&s.need, tid) = s.need;
      }
    }
    cluster.sync();
    prefix = s.prefix;
    need = s.need;
    if (shift == 0) return prefix;
    bits = min(kBits, shift);
    shift -= bits;
  }
}

__device__ __forceinline__ double next_f64(uint64_t z) {  // of the advanced state
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  z ^= z >> 31;
  return (double)(z >> 11) / (double)(1ull << 53);
}
constexpr uint64_t kStep = 0x9e3779b97f4a7c15ull;

__global__ void __launch_bounds__(kThreads) sample_requests_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int64_t r = blockIdx.x / ctas;
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  float *vals = reinterpret_cast<float *>(smem);
  Row row;
  row.vals = vals;
  row.id0 = (uint32_t)rank * a.share;
  row.n = min(max(a.vocab - rank * a.share, 0), a.share);
  const float *from = a.logits + r * a.ld + row.id0;
  float top = -INFINITY;
  for (int i = tid; i < row.n; i += kThreads) {
    float v = from[i];
    v = v != v ? -INFINITY : v + 0.0f;  // (a NaN is never drawn; -0 counts as 0)
    vals[i] = v;
    top = fmaxf(top, v);
  }
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.warp_top[warp] = top;
  __syncthreads();
  if (tid < 32) {
    top = s.warp_top[lane];
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane < ctas) *cluster.map_shared_rank(&s.top[rank], lane) = top;
  }
  const float t = a.temperature ? a.temperature[r] : 1.0f;
  uint64_t state = a.rng ? a.rng[r] : 0;
  cluster.sync();
  for (int i = 0; i < ctas; ++i) top = fmaxf(top, s.top[i]);
  row.top = top;
  const bool greedy = !(t > 0.0f);
  uint64_t above = 0, least = 1;
  double u = 0.0;
  row.scale = greedy ? 0.0 : 1.4426950408889634074 / (double)t;
  if (greedy) {
    above = rank_key(top, 0) & ~0xffffffffull;  // all that are as large as the largest: the first is drawn, with u = 0
  } else {
    if (a.rng) {
      state += kStep;
      u = next_f64(state);
    } else {
      u = a.uniforms[r];
    }
    u = u >= 0.0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
    const int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    if (k > 0 && k < a.vocab) above = find_border<false>(cluster, s, row, 0, 0.0, (uint64_t)k);
    if (p < 1.0f && top > -INFINITY) above = find_border<true>(cluster, s, row, above, fmax((double)p, 0.0), 0);
    const float low = a.min_p ? a.min_p[r] : 0.0f;
    if (low > 0.0f) least = max(least, (uint64_t)ceil(fmin((double)low, 1.0) * (double)(1ull << kOne)));
  }
  auto kept = [&](int i) -> uint64_t {
    const float v = vals[i];
    if (v == -INFINITY || rank_key(v, row.id0 + i) < above) return 0;
    const uint64_t w = mass_of(v, top, row.scale);
    return w >= least ? w : 0;
  };
  // a warp sums a run of columns, the same runs that are searched below
  const int run = (a.share + kThreads - 1) / kThreads * 32;
  const int c0 = min(warp * run, row.n), c1 = min(c0 + run, row.n);
  uint64_t mine = 0;
  for (int i = c0 + lane; i < c1; i += 32) mine += kept(i);
  mine = warp_sum(mine);
  if (lane == 0) s.warp_sum[warp] = mine;
  __syncthreads();
  if (tid < 32) {
    const uint64_t sum = warp_sum(s.warp_sum[lane]);
    if (lane < ctas) *cluster.map_shared_rank(&s.cta_sum[rank], lane) = sum;
  }
  cluster.sync();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < ctas; ++i) {
    total += s.cta_sum[i];
    if (i < rank) before += s.cta_sum[i];
  }
  if (rank == 0 && tid == 0) {
    if (a.rng && !greedy) a.rng[r] = state;
    if (total == 0) {  // nothing that can be drawn
      a.tokens[r] = -1;
      if (a.probs) a.probs[r] = 0.0f;
    }
  }
  uint64_t at = (uint64_t)(u * (double)total);
  if (total > 0) at = min(at, total - 1);
  for (int i = 0; i < warp; ++i) before += s.warp_sum[i];
  if (at < before || at >= before + s.warp_sum[warp]) return;
  for (int i0 = c0; i0 < c1; i0 += 32) {
    const int i = i0 + lane;
    const uint64_t w = i < c1 ? kept(i) : 0;
    const uint64_t incl = warp_scan(w) + before;
    const uint32_t past = __ballot_sync(0xffffffffu, incl > at);
    if (past) {
      if (lane == __ffs(past) - 1) {
        a.tokens[r] = (int32_t)(row.id0 + i);
        if (a.probs) a.probs[r] = greedy ? 1.0f : (float)((double)w / (double)total);
      }
      return;
    }
    before = __shfl_sync(0xffffffffu, incl, 31);
  }
}

}  // namespace

extern "C" int gq_sample_requests(gq_ctx *ctx, const float *logits, int64_t m, int64_t vocab, int64_t ld, const float *temperature,
                                  const int32_t *top_k, const float *top_p, const float *min_p, const double *uniforms,
                                  uint64_t *rng_state, int32_t *tokens, float *probs) {
  if (!ctx) return GQ_ERR_INVALID_ARGUMENT;
  const int rc = gq_enter_ctx(ctx);
  if (rc != GQ_OK) return rc;
  if (ld == 0) ld = vocab;
  if (m < 0 || vocab < 1 || ld < vocab) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "sample_requests: bad m, vocab or ld");
  if (vocab > kMaxVocab || m > INT32_MAX / kMaxCluster)
    return gq_fail(ctx, GQ_ERR_UNSUPPORTED, "sample_requests: vocab above 524288, or too many rows");
  if (m == 0) return GQ_OK;
  if (!logits || !tokens) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "sample_requests: null pointer");
  if (!uniforms == !rng_state)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "sample_requests: either uniforms or rng_state, one of them");
  int cluster = kMaxCluster;
  Args a{};
  a.logits = logits;
  a.ld = ld;
  a.vocab = (int)vocab;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.uniforms = uniforms;
  a.rng = rng_state;
  a.tokens = tokens;
  a.probs = probs;
  while (cluster > 1 && (vocab + cluster / 2 - 1) / (cluster / 2) <= kMaxShare && m * cluster > ctx->num_sms) cluster >>= 1;
  a.share = (int)((vocab + cluster - 1) / cluster + 3) / 4 * 4;
  static bool attr_set[64] = {};
  if (!attr_set[ctx->device & 63]) {
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_requests_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShare * 4));
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_requests_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_set[ctx->device & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(m * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)a.share * 4;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctx->pdl ? 2 : 1;
  GQ_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, sample_requests_kernel, (const Args)a));
  return GQ_OK;
}
