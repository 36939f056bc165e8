// sample_requests.cu — a token for each request of a step, with its own temperature, top-k, top-p,
// min-p and random number (gq_sample_requests).
//
//   w_i = e^((l_i - max l) / T)
//   in the order of the logits (largest first, ties to the smaller id): the first top_k; of those the
//   shortest run that holds top_p of their mass; of those the ones with w_i >= min_p
//   token: in the order of the ids, the first kept one at which the running sum of w passes u * (their sum)
//
// All three options keep a beginning of the order, so what is left is one border: a logit and an id,
// together a key of 64 bits. It is found without sorting the row: a histogram of counts (top-k) or masses
// (top-p) says in which of 2048 bins the border lies, and the keys of that bin alone are sorted; where
// they are too many (equal logits, far outliers) the bin's keys are cut into 2048 bins again.
// Masses are whole numbers, w * 2^44 rounded: their sums (vocab <= 2^19) fit 64 bits and do not depend on
// the order of additions, so atomics may add them up. The weights are made in f64: with f32's 2^-24 a
// draw over 262144 tokens would land on a neighbour of the right token every few hundred rows; 2^-45
// leaves less than one in 10^6.
//
// A row is kept in the shared memory of a cluster of CTAs, each with a share of its columns: the logits
// are read once, and every pass over them is on chip.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "gq_internal.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kBins = 2048;
constexpr int kOne = 44;          // w = 1 is 2^44
constexpr int kLimb = 15;         // bits of a mass that one 32-bit sum takes: a CTA has at most 2^15 columns
constexpr int kMaxShare = 32768;  // columns of a CTA
constexpr int kTwoPerSm = 16384;  // columns of a CTA that leave room for two on an SM
constexpr int kList = 2048;       // keys that are sorted
constexpr int kTable = 128;
constexpr int64_t kMaxVocab = (int64_t)kMaxShare * kMaxCluster;

struct Args {
  const float *logits;
  int64_t ld;
  int vocab, share;  // share: columns of a CTA
  int run;           // columns of a warp, a multiple of 128; kWarps * run >= share
  int wide;          // rows are read 16 bytes at a time
  const float *temperature, *top_p, *min_p;
  const int32_t *top_k;
  const double *uniforms;
  uint64_t *rng;
  int32_t *tokens;
  float *probs;
};

struct Shared {
  union {
    uint32_t limb[3][kBins];  // sums of a mass's bits 0-14, 15-29 and 30-44 (counts: the first)
    uint64_t bin[kBins];      // the same as one number
    uint64_t list[kList];     // of the first CTA: the keys of the border's bin
  };
  double table[kTable];           // 2^(j / 128)
  uint64_t warp_sum[kWarps];
  // written by every CTA of the cluster, in every CTA:
  uint64_t cta_sum[2][kMaxCluster], low[kMaxCluster], high[kMaxCluster];
  float top[kMaxCluster], bottom[kMaxCluster];
  // written by one CTA, in every CTA:
  uint64_t border, need;
  uint32_t bin_at;
  uint32_t listed;  // of the first CTA: keys of the border's bin
  float warp_top[kWarps], warp_bottom[kWarps];
  uint64_t warp_low[kWarps], warp_high[kWarps];
};

// Order of the logits as an order of numbers (no logit is NaN here, and no zero negative).
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}
// Of a logit and its id: larger logits first, then smaller ids.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t id) { return ((uint64_t)key_of(v) << 32) | (uint32_t)~id; }

struct Row {
  float top, bins_per_logit;
  double scale;  // 128 log2(e) / T
};

// w * 2^44 to the nearest whole number: 2^(t / 128), t = j + r with |r| <= 1/2, is 2^(j / 128) from a table
// times a Taylor polynomial (its next term is below 2^-48).
__device__ __forceinline__ uint64_t mass_of(const Shared &s, const Row &row, float v) {
  if (v == row.top) return 1ull << kOne;  // (infinities too)
  const double t = ((double)v - (double)row.top) * row.scale;
  if (!(t > -128.0 * (kOne + 2))) return 0;  // (-inf; a NaN of two infinities)
  constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
  const double shifted = t + kRound;
  const int j = __double2loint(shifted);
  const double x = (t - (shifted - kRound)) * (0.69314718055994530942 / 128);
  double p = fma(x, 1.0 / 24, 1.0 / 6);
  p = fma(x, p, 0.5);
  p = fma(x, p, 1.0);
  p = fma(x, p, 1.0);
  p *= s.table[j & (kTable - 1)];
  p = __hiloint2double(__double2hiint(p) + ((j >> 7) + kOne) * (1 << 20), __double2loint(p));
  const double whole = p + 4503599627370496.0;  // 2^52: the sum's fraction is p rounded
  return ((uint64_t)(__double2hiint(whole) & 0xfffff) << 32) | (uint32_t)__double2loint(whole);
}

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
// Inclusive scan over the block; sums[] of scratch. The total too.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *sums, uint64_t &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan(v);
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) v += sums[i];
    total += sums[i];
  }
  __syncthreads();
  return v;
}

// Descending sort of n (a power of two) keys by all threads.
__device__ void sort_down(uint64_t *k, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const uint64_t x = k[lo], y = k[hi];
        if ((x < y) == ((lo & size) == 0)) {
          k[lo] = y;
          k[hi] = x;
        }
      }
    }
  __syncthreads();
}

// This CTA's columns, four at a time: f(logit, id) in the order of the warp's run, lanes in turn.
template <typename F>
__device__ __forceinline__ void each(const Args &a, const float *vals, uint32_t id0, F f) {
  const int lane = threadIdx.x & 31, c0 = (threadIdx.x >> 5) * a.run + lane * 4;
  for (int c = 0; c < a.run; c += 128) {
    const float4 v = *reinterpret_cast<const float4 *>(vals + c0 + c);
    f(v.x, id0 + c0 + c);
    f(v.y, id0 + c0 + c + 1);
    f(v.z, id0 + c0 + c + 2);
    f(v.w, id0 + c0 + c + 3);
  }
}

// The border of the shortest beginning of the order (of the keys from `above` on) whose mass reaches `share`
// of the whole, or whose number reaches `count`: the key of its last member.
template <bool MASS>
__device__ uint64_t find_border(cg::cluster_group &cluster, Shared &s, const Args &a, const Row &row, const float *vals, uint32_t id0,
                                uint64_t above, double share, uint64_t count) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  uint64_t low = above, high = ~0ull, need = count;
  int shift = -1;  // -1: bins by the distance from the largest logit; else by (key - low) >> shift, the largest first
  for (;;) {
    for (int i = tid; i < kBins * (MASS ? 3 : 1); i += kThreads) (&s.limb[0][0])[i] = 0;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    auto bin_of = [&](float v, uint64_t key) -> uint32_t {
      if (shift < 0) {
        const float d = (row.top - v) * row.bins_per_logit;  // (NaN: two infinities)
        return d > 0.0f ? (uint32_t)fminf(d, (float)(kBins - 1)) : 0u;
      }
      return (uint32_t)((high - key) >> shift);
    };
    each(a, vals, id0, [&](float v, uint32_t id) {
      const uint64_t key = rank_key(v, id);
      if (key < low || key > high || v == -INFINITY) return;
      const uint32_t b = bin_of(v, key);
      if constexpr (MASS) {
        const uint64_t w = mass_of(s, row, v);
        if (w == 0) return;
        atomicAdd(&s.limb[0][b], (uint32_t)w & ((1u << kLimb) - 1));
        const uint32_t rest = (uint32_t)(w >> kLimb);
        if (rest & ((1u << kLimb) - 1)) atomicAdd(&s.limb[1][b], rest & ((1u << kLimb) - 1));
        if (rest >> kLimb) atomicAdd(&s.limb[2][b], rest >> kLimb);
      } else {
        atomicAdd(&s.limb[0][b], 1u);
      }
    });
    __syncthreads();
    {  // one number for each bin
      uint64_t w[kBins / kThreads];
#pragma unroll
      for (int i = 0; i < kBins / kThreads; ++i) {
        const int b = tid + i * kThreads;
        w[i] = MASS ? s.limb[0][b] + ((uint64_t)s.limb[1][b] << kLimb) + ((uint64_t)s.limb[2][b] << (2 * kLimb)) : s.limb[0][b];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kBins / kThreads; ++i) s.bin[tid + i * kThreads] = w[i];
    }
    cluster.sync();
    // every CTA adds up a share of the bins: thread t has one of them, or none
    const int per = (kBins + ctas - 1) / ctas;  // (a power of two: 128 to 2048)
    uint64_t w[kBins / kThreads];
    uint64_t mine = 0;
    const int each_bins = (per + kThreads - 1) / kThreads;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      w[i] = 0;
      const int in = tid * each_bins + i;
      if (i < each_bins && in < per)
        for (int r = 0; r < ctas; ++r) w[i] += cluster.map_shared_rank(s.bin, r)[rank * per + in];
      mine += w[i];
    }
    uint64_t total;
    uint64_t incl = block_scan(mine, s.warp_sum, total);
    if (tid < ctas) cluster.map_shared_rank(s.cta_sum[0], tid)[rank] = total;
    cluster.sync();
    uint64_t before = 0, all = 0;
    for (int r = 0; r < ctas; ++r) {
      if (r < rank) before += s.cta_sum[0][r];
      all += s.cta_sum[0][r];
    }
    if (shift < 0) {
      if constexpr (MASS) {
        const double x = ceil(share * (double)all);
        need = x >= 1.0 ? (uint64_t)x : 1ull;
      }
      need = min(need, all);
    }
    uint64_t at = before + incl - mine;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      if (need > at && need <= at + w[i]) {
        for (int r = 0; r < ctas; ++r) {
          *cluster.map_shared_rank(&s.bin_at, r) = (uint32_t)(rank * per + tid * each_bins + i);
          *cluster.map_shared_rank(&s.need, r) = need - at;
        }
      }
      at += w[i];
    }
    cluster.sync();
    const uint32_t bin = s.bin_at;
    need = s.need;
    // the bin's keys to the first CTA, and the smallest and largest of them
    uint64_t lo = ~0ull, hi = 0;
    uint64_t *list = cluster.map_shared_rank(s.list, 0);
    uint32_t *listed = cluster.map_shared_rank(&s.listed, 0);
    each(a, vals, id0, [&](float v, uint32_t id) {
      const uint64_t key = rank_key(v, id);
      const bool in = key >= low && key <= high && v != -INFINITY && bin_of(v, key) == bin;
      const uint32_t who = __ballot_sync(0xffffffffu, in);
      if (who == 0) return;
      uint32_t i = 0;
      if (lane == __ffs(who) - 1) i = atomicAdd(listed, (uint32_t)__popc(who));
      i = __shfl_sync(0xffffffffu, i, __ffs(who) - 1) + __popc(who & ((1u << lane) - 1));
      if (in) {
        lo = min(lo, key);
        hi = max(hi, key);
        if (i < (uint32_t)kList) list[i] = key;
      }
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (lane == 0) {
      s.warp_low[warp] = lo;
      s.warp_high[warp] = hi;
    }
    __syncthreads();
    if (tid < ctas) {
      for (int i = 0; i < kWarps; ++i) {
        lo = min(lo, s.warp_low[i]);
        hi = max(hi, s.warp_high[i]);
      }
      cluster.map_shared_rank(s.low, tid)[rank] = lo;
      cluster.map_shared_rank(s.high, tid)[rank] = hi;
    }
    cluster.sync();
    const uint32_t n = *listed;
    if (n <= (uint32_t)kList) {
      if (rank == 0) {
        int n2 = 1;
        while (n2 < (int)n) n2 <<= 1;
        for (int i = n + tid; i < n2; i += kThreads) s.list[i] = 0;
        sort_down(s.list, n2);
        // thread t has neighbouring keys; the one whose sum reaches what is needed says so
        const int e = (n2 + kThreads - 1) / kThreads;
        uint64_t sum = 0;
        for (int i = 0; i < e; ++i) {
          const int p = tid * e + i;
          if (p < (int)n) sum += MASS ? mass_of(s, row, logit_of(s.list[p])) : 1ull;
        }
        uint64_t whole;
        uint64_t run = block_scan(sum, s.warp_sum, whole) - sum;
        if (need > run && need <= run + sum)
          for (int i = 0; i < e; ++i) {
            const int p = tid * e + i;
            run += MASS ? mass_of(s, row, logit_of(s.list[p])) : 1ull;
            if (run >= need) {
              for (int r = 0; r < ctas; ++r) *cluster.map_shared_rank(&s.border, r) = s.list[p];
              break;
            }
          }
      }
      cluster.sync();
      return s.border;
    }
    for (int r = 0; r < ctas; ++r) {
      lo = min(lo, s.low[r]);
      hi = max(hi, s.high[r]);
    }
    cluster.sync();  // everyone has read what the next round writes
    low = lo;
    high = hi;
    shift = max(0, 64 - __clzll((long long)(hi - lo)) - 11);
  }
}

__device__ __forceinline__ double next_f64(uint64_t z) {  // of the advanced state
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  z ^= z >> 31;
  return (double)(z >> 11) / (double)(1ull << 53);
}
constexpr uint64_t kStep = 0x9e3779b97f4a7c15ull;

__global__ void __launch_bounds__(kThreads, 2) sample_requests_kernel(const Args a) {
  extern __shared__ __align__(16) float vals[];  // [kWarps * run]: this CTA's columns, -inf past them
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int64_t r = blockIdx.x / ctas;
  if (tid < kTable) s.table[tid] = exp2((double)tid / kTable);
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const float t = a.temperature ? a.temperature[r] : 1.0f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  const float low_p = a.min_p ? a.min_p[r] : 0.0f;
  uint64_t state = a.rng ? a.rng[r] : 0;
  const double given = a.uniforms ? a.uniforms[r] : 0.0;
  const uint32_t id0 = (uint32_t)rank * a.share;
  const int n = min(max(a.vocab - (int)id0, 0), a.share);
  float top = -INFINITY, bottom = INFINITY;  // of the numbers
  {
    const float *from = a.logits + r * a.ld + id0;
    auto take = [&](float v) {
      v = v != v ? -INFINITY : v + 0.0f;  // (a NaN is never drawn; -0 counts as 0)
      top = fmaxf(top, v);
      if (v > -INFINITY) bottom = fminf(bottom, v);
      return v;
    };
    for (int c = warp * a.run + lane * 4; c < (warp + 1) * a.run; c += 128) {
      float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (a.wide && c + 3 < n) {
        v = __ldcs(reinterpret_cast<const float4 *>(from + c));
      } else {
        if (c < n) v.x = from[c];
        if (c + 1 < n) v.y = from[c + 1];
        if (c + 2 < n) v.z = from[c + 2];
        if (c + 3 < n) v.w = from[c + 3];
      }
      *reinterpret_cast<float4 *>(vals + c) = make_float4(take(v.x), take(v.y), take(v.z), take(v.w));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bottom = fminf(bottom, __shfl_xor_sync(0xffffffffu, bottom, o));
  }
  if (lane == 0) {
    s.warp_top[warp] = top;
    s.warp_bottom[warp] = bottom;
  }
  __syncthreads();
  if (tid < ctas) {
    for (int i = 0; i < kWarps; ++i) {
      top = fmaxf(top, s.warp_top[i]);
      bottom = fminf(bottom, s.warp_bottom[i]);
    }
    cluster.map_shared_rank(s.top, tid)[rank] = top;
    cluster.map_shared_rank(s.bottom, tid)[rank] = bottom;
  }
  cluster.sync();
  for (int i = 0; i < ctas; ++i) {
    top = fmaxf(top, s.top[i]);
    bottom = fminf(bottom, s.bottom[i]);
  }
  const bool greedy = !(t > 0.0f);
  Row row;
  row.top = top;
  row.scale = greedy ? 0.0 : kTable * 1.4426950408889634074 / (double)t;
  uint64_t above = 0, least = 1;
  double u = 0.0;
  if (greedy) {
    above = (uint64_t)key_of(top) << 32;  // all that are as large as the largest: the first is drawn, with u = 0
  } else {
    if (a.rng) {
      state += kStep;
      u = next_f64(state);
    } else {
      u = given;
    }
    u = u >= 0.0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
    if (top > -INFINITY) {
      // bins over the row's numbers, for masses over those that have any
      const float span = top - bottom, heavy = 32.0f * t;
      row.bins_per_logit = (float)(kBins - 1) / span;
      if (k > 0 && k < a.vocab) above = find_border<false>(cluster, s, a, row, vals, id0, 0, 0.0, (uint64_t)k);
      row.bins_per_logit = (float)(kBins - 1) / fminf(span, heavy);
      if (p < 1.0f) above = find_border<true>(cluster, s, a, row, vals, id0, above, fmax((double)p, 0.0), 0);
    }
    if (low_p > 0.0f) least = max(least, (uint64_t)ceil(fmin((double)low_p, 1.0) * (double)(1ull << kOne)));
  }
  auto kept = [&](float v, uint32_t id) -> uint64_t {
    if (v == -INFINITY || rank_key(v, id) < above) return 0;
    const uint64_t w = mass_of(s, row, v);
    return w >= least ? w : 0;
  };
  uint64_t sum = 0;
  each(a, vals, id0, [&](float v, uint32_t id) { sum += kept(v, id); });
  sum = warp_sum(sum);
  if (lane == 0) s.warp_sum[warp] = sum;
  __syncthreads();
  if (tid < ctas) {
    uint64_t whole = 0;
    for (int i = 0; i < kWarps; ++i) whole += s.warp_sum[i];
    cluster.map_shared_rank(s.cta_sum[1], tid)[rank] = whole;
  }
  cluster.sync();
  uint64_t total = 0, before = 0;
  for (int i = 0; i < ctas; ++i) {
    total += s.cta_sum[1][i];
    if (i < rank) before += s.cta_sum[1][i];
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
  // the warp in whose run the sum passes `at`
  for (int c = warp * a.run + lane * 4; c < (warp + 1) * a.run; c += 128) {
    const float4 v = *reinterpret_cast<const float4 *>(vals + c);
    const uint64_t w[4] = {kept(v.x, id0 + c), kept(v.y, id0 + c + 1), kept(v.z, id0 + c + 2), kept(v.w, id0 + c + 3)};
    const uint64_t four = w[0] + w[1] + w[2] + w[3];
    const uint64_t incl = warp_scan(four) + before;
    const uint32_t past = __ballot_sync(0xffffffffu, incl > at);
    if (past) {
      if (lane == __ffs(past) - 1) {
        uint64_t run = incl - four;
        for (int i = 0; i < 4; ++i) {
          run += w[i];
          if (run > at) {
            a.tokens[r] = (int32_t)(id0 + c + i);
            if (a.probs) a.probs[r] = greedy ? 1.0f : (float)((double)w[i] / (double)total);
            break;
          }
        }
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
  a.wide = (uintptr_t)logits % 16 == 0 && ld % 4 == 0;
  // CTAs of a row: as few as hold it at two CTAs per SM, more while a share is large and the GPU not full
  int cluster = 1;
  while (cluster < kMaxCluster && (vocab > (int64_t)cluster * kTwoPerSm || (vocab > cluster * 2048 && m * cluster * 2 <= 2 * ctx->num_sms)))
    cluster *= 2;
  a.share = (int)((vocab + cluster - 1) / cluster + 3) / 4 * 4;
  a.run = (a.share + kWarps * 128 - 1) / (kWarps * 128) * 128;
  static bool attr_set[64] = {};
  if (!attr_set[ctx->device & 63]) {
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_requests_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxShare + 4 * kWarps * 128) * 4));
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_requests_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    attr_set[ctx->device & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(m * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)a.run * kWarps * 4;
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
