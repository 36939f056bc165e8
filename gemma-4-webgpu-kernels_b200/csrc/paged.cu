// paged.cu — pages of a key-value cache shared by many requests: taking pages for a
// step's new tokens (gq_paged_reserve), giving them back (gq_paged_release) and
// writing key and value rows into them (gq_paged_append).
//
// Reserve and release are prefix sums over the requests followed by independent work
// per token (or per page). Every CTA makes the whole prefix sum itself in shared
// memory (a few microseconds of L2 reads at the 16384-request limit, one load round
// trip at ordinary batches) and then takes its share of the tokens: one launch, no
// pass through memory between the two steps. Outputs that may alias inputs (lengths,
// the free count) are written by the last CTA to arrive, when every CTA has read them.
// What bounds them is the chain of loads (lengths, then table or list, then the arrival):
// replayed, 3.8 us for 64 requests of one token, 6.7 us for 131,000 tokens of 512
// requests, 4.5 and 6.6 us to give back 3,000 and 180,000 pages. One request per thread
// and round, with 64-bit divisions, took 10.1 us for the last.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanEach = 4;  // neighbouring requests per thread and round of loads
constexpr int kMaxBatch = 16384;

struct PlanArgs {
  int64_t batch, table_stride, n_pages, max_tokens;
  uint32_t page_size;
  const int32_t *seq_lens, *other_lens;  // other: new (reserve) or kept (release) tokens
  int32_t *table;                        // reserve writes it, release reads it
  int32_t *free_pages;                   // reserve reads it, release writes it
  const int32_t *free_count;
  int32_t *free_left;
  int64_t *slots;
  int32_t *positions, *owners, *totals;
  uint32_t *ctr, *err;
};

__device__ __forceinline__ int64_t len_of(const int32_t *p, int64_t b) {
  const int32_t v = p[b];
  return v > 0 ? (int64_t)v : 0;
}
// (two lengths add up to less than 2^32: the short division)
__device__ __forceinline__ int64_t pages_of(int64_t tokens, uint32_t page_size) {
  const uint32_t t = (uint32_t)tokens, full = t / page_size;
  return full + (t != full * page_size);
}

// Inclusive scan over the block of two sums at once; red is 2 * 32 entries of scratch.
__device__ __forceinline__ void block_scan2(int64_t &a, int64_t &b, int64_t (*red)[32], int64_t &ta, int64_t &tb) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += ua;
      b += ub;
    }
  }
  if (lane == 31) {
    red[0][warp] = a;
    red[1][warp] = b;
  }
  __syncthreads();
  int64_t pa = 0, pb = 0;
  ta = tb = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) {
      pa += red[0][w];
      pb += red[1][w];
    }
    ta += red[0][w];
    tb += red[1][w];
  }
  a += pa;
  b += pb;
  __syncthreads();  // red may be written again
}

// First index whose inclusive prefix sum exceeds v (sums non-decreasing, v < the last).
__device__ __forceinline__ int owner_of(const int32_t *ends, int n, int32_t v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > v) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// True in every thread of the last CTA of the grid to get here (after all others'
// reads of the inputs); puts the counter back to zero.
__device__ __forceinline__ bool last_cta(uint32_t *ctr) {
  __shared__ int last;
  __syncthreads();
  if (gridDim.x == 1) return true;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(ctr, 1u) == gridDim.x - 1;
    if (last) {
      *ctr = 0u;
      __threadfence();
    }
  }
  __syncthreads();
  return last != 0;
}

__global__ void __launch_bounds__(kPlanThreads) paged_reserve_kernel(const PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  __shared__ int64_t red[2][32];
  const int n = (int)a.batch, tid = threadIdx.x;
  int32_t *ends = plan_smem;       // tokens of requests 0 .. b
  int32_t *first = plan_smem + n;  // pages taken by requests before b
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int64_t listed = a.free_count[0];
  const int64_t count = min(max(listed, (int64_t)0), a.n_pages);
  int64_t tokens = 0, taken = 0;
  bool bad = listed != count;
  for (int b0 = 0; b0 < n; b0 += kPlanThreads * kPlanEach) {
    int64_t add[kPlanEach], need[kPlanEach], sa = 0, sn = 0, ta, tn;
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) {
      const int b = b0 + tid * kPlanEach + i;
      add[i] = need[i] = 0;
      if (b < n) {
        const int64_t len = len_of(a.seq_lens, b);
        add[i] = len_of(a.other_lens, b);
        const int64_t have = pages_of(len + add[i], a.page_size);
        need[i] = have - pages_of(len, a.page_size);
        bad |= have > a.table_stride || len + add[i] > INT32_MAX;
      }
      sa += add[i];
      sn += need[i];
    }
    const int64_t mine_a = sa, mine_n = sn;
    block_scan2(sa, sn, red, ta, tn);
    sa += tokens - mine_a;  // of the requests before this thread's
    sn += taken - mine_n;
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) {
      const int b = b0 + tid * kPlanEach + i;
      sa += add[i];
      if (b < n) {  // (sums past 31 bits end up refused below: max_tokens and n_pages are smaller)
        ends[b] = (int32_t)min(sa, (int64_t)INT32_MAX);
        first[b] = (int32_t)min(sn, (int64_t)INT32_MAX);
      }
      sn += need[i];
    }
    tokens += ta;
    taken += tn;
  }
  bad = __syncthreads_or(bad) || tokens > a.max_tokens || taken > count;
  bool wrong = false;  // a page id outside the pool
  for (int64_t t = blockIdx.x * (int64_t)kPlanThreads + tid; t < a.max_tokens; t += (int64_t)gridDim.x * kPlanThreads) {
    int64_t slot = -1;
    int32_t pos32 = 0, owner = -1;
    if (!bad && t < tokens) {
      owner = owner_of(ends, n, (int32_t)t);
      const int64_t len = len_of(a.seq_lens, owner);
      const int64_t pos = len + (t - (owner ? ends[owner - 1] : 0));
      const int64_t p = (uint32_t)pos / a.page_size, row = pos - p * a.page_size, had = pages_of(len, a.page_size);
      int32_t *entry = a.table + owner * a.table_stride + p;
      int32_t page;
      if (p < had) {
        page = *entry;
      } else {
        page = a.free_pages[count - 1 - (first[owner] + (p - had))];
        // a new page starts past the old tokens, so its row 0 is one of this step's tokens
        if (row == 0) *entry = page;
      }
      if (page >= 0 && page < a.n_pages) slot = (int64_t)page * a.page_size + row;
      else wrong = true;
      pos32 = (int32_t)pos;
    }
    a.slots[t] = slot;
    a.positions[t] = pos32;
    a.owners[t] = owner;
  }
  if (wrong) gqd::report(a.err, GQ_DEVERR_PAGES);
  if (last_cta(a.ctr)) {
    for (int b = tid; b < n; b += kPlanThreads) {
      const int64_t len = len_of(a.seq_lens, b);
      a.totals[b] = (int32_t)min(bad ? len : len + len_of(a.other_lens, b), (int64_t)INT32_MAX);
    }
    if (tid == 0) {
      a.free_left[0] = (int32_t)(bad ? count : count - taken);
      if (bad) gqd::report(a.err, GQ_DEVERR_PAGES);
    }
  }
}

__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(const PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  __shared__ int64_t red[2][32];
  const int n = (int)a.batch, tid = threadIdx.x;
  int32_t *ends = plan_smem;        // pages given back by requests 0 .. b
  int32_t *start = plan_smem + n;   // first table entry that request b gives back
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int64_t listed = a.free_count[0];
  const int64_t count = min(max(listed, (int64_t)0), a.n_pages);
  int64_t given = 0;
  bool bad = listed != count;
  for (int b0 = 0; b0 < n; b0 += kPlanThreads * kPlanEach) {
    int64_t back[kPlanEach], sb = 0, unused = 0, tb, tu;
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) {
      const int b = b0 + tid * kPlanEach + i;
      back[i] = 0;
      if (b < n) {
        const int64_t len = len_of(a.seq_lens, b);
        const int64_t had = pages_of(len, a.page_size), keep = pages_of(min(len_of(a.other_lens, b), len), a.page_size);
        back[i] = had - keep;
        start[b] = (int32_t)keep;
        bad |= had > a.table_stride;
      }
      sb += back[i];
    }
    const int64_t mine = sb;
    block_scan2(sb, unused, red, tb, tu);
    sb += given - mine;
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) {
      const int b = b0 + tid * kPlanEach + i;
      sb += back[i];
      if (b < n) ends[b] = (int32_t)min(sb, (int64_t)INT32_MAX);
    }
    given += tb;
  }
  bad = __syncthreads_or(bad) || count + given > a.n_pages;
  bool wrong = false;  // a page id outside the pool
  if (!bad)
    for (int64_t i0 = blockIdx.x * (int64_t)kPlanThreads + tid; i0 < given; i0 += (int64_t)gridDim.x * kPlanThreads * kPlanEach) {
      int32_t page[kPlanEach];
#pragma unroll
      for (int k = 0; k < kPlanEach; ++k) {
        const int64_t i = i0 + (int64_t)k * gridDim.x * kPlanThreads;
        page[k] = 0;
        if (i >= given) continue;
        const int b = owner_of(ends, n, (int32_t)i);
        page[k] = a.table[b * a.table_stride + start[b] + (i - (b ? ends[b - 1] : 0))];
      }
#pragma unroll
      for (int k = 0; k < kPlanEach; ++k) {
        const int64_t i = i0 + (int64_t)k * gridDim.x * kPlanThreads;
        if (i >= given) break;
        a.free_pages[count + given - 1 - i] = page[k];
        wrong |= page[k] < 0 || page[k] >= a.n_pages;
      }
    }
  if (wrong) gqd::report(a.err, GQ_DEVERR_PAGES);
  if (last_cta(a.ctr)) {
    for (int b = tid; b < n; b += kPlanThreads) {
      const int64_t len = len_of(a.seq_lens, b);
      a.totals[b] = (int32_t)(bad ? len : min(len_of(a.other_lens, b), len));
    }
    if (tid == 0) {
      a.free_left[0] = (int32_t)(bad ? count : count + given);
      if (bad) gqd::report(a.err, GQ_DEVERR_PAGES);
    }
  }
}

// ---- append -----------------------------------------------------------------------

struct AppendArgs {
  const float *src[2];  // k, v
  void *dst[2];
  int64_t src_stride[2];
  const int64_t *slots;
  int64_t tokens, page_size, page_stride, n_slots;
  int heads, head_dim;
  float inv_scale[2];
  uint32_t *err;
};

// Four values to the pages' type, rounded to nearest even.
template <int TYPE>
__device__ __forceinline__ void store4(void *base, int64_t elem, const float4 v, float inv_scale) {
  if constexpr (TYPE == GQ_KV_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(base) + elem) = v;
  } else if constexpr (TYPE == GQ_KV_F16) {
    const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(static_cast<__half *>(base) + elem) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
  } else if constexpr (TYPE == GQ_KV_BF16) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(base) + elem) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
  } else {
    // saturating conversion: finite values past the largest code become it; an infinity too
    const float2 a = make_float2(v.x * inv_scale, v.y * inv_scale), b = make_float2(v.z * inv_scale, v.w * inv_scale);
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(base) + elem) = lo | (hi << 16);
  }
}

// A warp writes one token's row of keys (or values): what it needs of the slot is worked
// out once, and a lane's kAppendLoads loads of 16 bytes are in flight together. Rows are
// taken in turn by a grid of eight CTAs per SM, of which some 48 registers a thread let
// five be resident; the arguments that are indexed by key or value lie in local memory (a
// frame of 112 bytes). HBM-bound: 16411 rows of 512 to e4m3, 84 MB, 17.5 us, 4.8 TB/s (a
// thread per 4 values, each with its own slot and divisions: 34 us).
constexpr int kAppendThreads = 256, kAppendLoads = 4;

template <int TYPE>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int per_head = a.head_dim / 4, pieces = a.heads * per_head;
  const int64_t rows = 2 * a.tokens, step = (int64_t)gridDim.x * (kAppendThreads / 32);
  if (pieces <= 32) {
    // A row is one load per lane at most, so kAppendLoads rows are taken at a time to have
    // as many loads in flight: f32, 59672 rows of 128, 123 MB, 25.0 us, 4.9 TB/s (one at a
    // time, as below: 37.7 us). Longer rows have that many loads of their own.
    const int h = lane / per_head;
    const int64_t in_row = (h * (int64_t)a.page_size) * a.head_dim + (lane - h * per_head) * 4;
    for (int64_t r0 = (blockIdx.x * (int64_t)(kAppendThreads / 32) + threadIdx.x / 32) * kAppendLoads; r0 < rows;
         r0 += step * kAppendLoads) {
      int64_t slot[kAppendLoads];
      float4 v[kAppendLoads];
#pragma unroll
      for (int i = 0; i < kAppendLoads; ++i) {
        const int64_t t = (r0 + i) >> 1;  // r0 is even: row i is of keys or of values as i is
        slot[i] = r0 + i < rows ? a.slots[t] : -1;
        if (r0 + i < rows && lane < pieces)
          v[i] = __ldcs(reinterpret_cast<const float4 *>(a.src[i & 1] + t * a.src_stride[i & 1]) + lane);
      }
#pragma unroll
      for (int i = 0; i < kAppendLoads; ++i) {
        if (slot[i] < 0) continue;
        if (slot[i] >= a.n_slots) {
          if (lane == 0) gqd::report(a.err, GQ_DEVERR_PAGES);
          continue;
        }
        const int64_t page =
            (slot[i] >> 32) == 0 ? (int64_t)((uint32_t)slot[i] / (uint32_t)a.page_size) : slot[i] / a.page_size;
        if (lane < pieces)
          store4<TYPE>(a.dst[i & 1], page * a.page_stride + (slot[i] - page * a.page_size) * a.head_dim + in_row, v[i],
                       a.inv_scale[i & 1]);
      }
    }
    return;
  }
  for (int64_t r = blockIdx.x * (int64_t)(kAppendThreads / 32) + threadIdx.x / 32; r < rows; r += step) {
    const int64_t t = r >> 1;
    const int kv = (int)(r & 1);
    const int64_t slot = a.slots[t];
    if (slot < 0) continue;
    if (slot >= a.n_slots) {
      if (lane == 0) gqd::report(a.err, GQ_DEVERR_PAGES);
      continue;
    }
    const int64_t page = (slot >> 32) == 0 ? (int64_t)((uint32_t)slot / (uint32_t)a.page_size) : slot / a.page_size;
    const int64_t base = page * a.page_stride + (slot - page * a.page_size) * a.head_dim;
    const int64_t head = a.page_size * a.head_dim;  // elements between heads
    const float4 *src = reinterpret_cast<const float4 *>(a.src[kv] + t * a.src_stride[kv]);
    void *dst = a.dst[kv];
    const float inv = a.inv_scale[kv];
    for (int c0 = lane; c0 < pieces; c0 += 32 * kAppendLoads) {
      float4 v[kAppendLoads];
#pragma unroll
      for (int i = 0; i < kAppendLoads; ++i)
        if (c0 + 32 * i < pieces) v[i] = __ldcs(src + c0 + 32 * i);
#pragma unroll
      for (int i = 0; i < kAppendLoads; ++i) {
        const int c = c0 + 32 * i;
        if (c >= pieces) break;
        const int h = a.heads == 1 ? 0 : c / per_head;
        store4<TYPE>(dst, base + h * head + (c - h * per_head) * 4, v[i], inv);
      }
    }
  }
}

int plan_launch(gq_ctx *ctx, bool reserve, PlanArgs &a, int64_t work) {
  a.ctr = ctx->counters;
  a.err = ctx->dev_err;
  const size_t smem = (size_t)a.batch * 8;
  static bool attr_set[64] = {};
  if (smem > 32768 && !attr_set[ctx->device & 63]) {
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(paged_reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBatch * 8));
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(paged_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBatch * 8));
    attr_set[ctx->device & 63] = true;
  }
  const int64_t grid = std::min<int64_t>(std::max<int64_t>(1, (work + 2 * kPlanThreads - 1) / (2 * kPlanThreads)), ctx->num_sms);
  GQ_CUDA_TRY(ctx, gq_launch(ctx, reserve ? paged_reserve_kernel : paged_release_kernel, dim3((unsigned)grid),
                             dim3(kPlanThreads), smem, a));
  return GQ_OK;
}

#define ENTER(ctx)                              \
  do {                                          \
    if (!(ctx)) return GQ_ERR_INVALID_ARGUMENT; \
    int _rc = gq_enter_ctx(ctx);                \
    if (_rc != GQ_OK) return _rc;               \
  } while (0)

int check_plan(gq_ctx *ctx, const char *op, int64_t batch, int64_t page_size, int64_t table_stride, int64_t n_pages) {
  if (batch < 0 || page_size < 1 || page_size > 65536 || table_stride < 0 || n_pages < 0 || n_pages > INT32_MAX)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, std::string(op) + ": bad batch, page_size, table_stride or n_pages");
  if (batch > kMaxBatch) return gq_fail(ctx, GQ_ERR_UNSUPPORTED, std::string(op) + ": more than 16384 requests");
  return GQ_OK;
}

}  // namespace

int gq_check_kv_pages(gq_ctx *ctx, const char *op, const gq_kv_pages *p) {
  const std::string who(op);
  if (!p) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, who + ": null pages");
  if (p->type < GQ_KV_F32 || p->type > GQ_KV_E2M1) return gq_fail(ctx, GQ_ERR_UNSUPPORTED, who + ": unknown page type");
  if (p->n_pages < 0 || p->n_pages > INT32_MAX || p->page_size < 1 || p->page_size > 65536 || p->heads < 1 ||
      p->heads > 65535 || p->head_dim < 1)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, who + ": bad n_pages, page_size, heads or head_dim");
  if (p->head_dim % 4 != 0 || p->head_dim > 512)
    return gq_fail(ctx, GQ_ERR_UNSUPPORTED, who + ": head_dim must be a multiple of 4, at most 512");
  if (p->type == GQ_KV_E2M1 && p->head_dim % 16 != 0)
    return gq_fail(ctx, GQ_ERR_UNSUPPORTED, who + ": head_dim of e2m1 pages must be a multiple of 16");
  const int64_t packed = p->heads * p->page_size * gq_kv_row(p), stride = gq_kv_page_stride(p);
  if (stride < packed || (p->type != GQ_KV_E2M1 && stride % 4 != 0))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, who + ": page_stride below a page's size, or not a multiple of 4");
  if (p->n_pages > 0 && (!p->k || !p->v)) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, who + ": null page pool");
  if (((uintptr_t)p->k | (uintptr_t)p->v) % 16 != 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, who + ": k and v pages must be 16-byte aligned");
  const bool scaled = p->type == GQ_KV_E4M3 || p->type == GQ_KV_E2M1;
  for (const float s : {p->k_scale, p->v_scale})
    if (!(s > 0.0f) || !std::isfinite(s) || !std::isfinite(1.0f / s) || (!scaled && s != 1.0f))
      return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT,
                     who + ": scales must be positive, finite with a finite reciprocal, and 1 unless the type is e4m3 or e2m1");
  return GQ_OK;
}

extern "C" int gq_paged_reserve(gq_ctx *ctx, int64_t batch, int64_t page_size, const int32_t *seq_lens,
                                const int32_t *new_lens, int32_t *block_table, int64_t table_stride,
                                const int32_t *free_pages, int64_t n_pages, const int32_t *free_count,
                                int32_t *free_left, int64_t max_tokens, int64_t *slots, int32_t *positions,
                                int32_t *owners, int32_t *totals) {
  ENTER(ctx);
  int rc = check_plan(ctx, "paged_reserve", batch, page_size, table_stride, n_pages);
  if (rc != GQ_OK) return rc;
  if (max_tokens < 0 || max_tokens > INT32_MAX - 1)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_reserve: max_tokens must be below 2^31 - 1");
  if (!free_count || !free_left || (n_pages > 0 && !free_pages) || (batch > 0 && (!seq_lens || !new_lens || !totals)) ||
      (batch > 0 && table_stride > 0 && !block_table) || (max_tokens > 0 && (!slots || !positions || !owners)))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_reserve: null pointer");
  PlanArgs a{};
  a.batch = batch;
  a.page_size = (uint32_t)page_size;
  a.table_stride = table_stride;
  a.n_pages = n_pages;
  a.max_tokens = max_tokens;
  a.seq_lens = seq_lens;
  a.other_lens = new_lens;
  a.table = block_table;
  a.free_pages = const_cast<int32_t *>(free_pages);
  a.free_count = free_count;
  a.free_left = free_left;
  a.slots = slots;
  a.positions = positions;
  a.owners = owners;
  a.totals = totals;
  return plan_launch(ctx, true, a, max_tokens);
}

extern "C" int gq_paged_release(gq_ctx *ctx, int64_t batch, int64_t page_size, const int32_t *seq_lens,
                                const int32_t *keep_lens, const int32_t *block_table, int64_t table_stride,
                                int32_t *free_pages, int64_t n_pages, const int32_t *free_count, int32_t *free_left,
                                int32_t *totals) {
  ENTER(ctx);
  int rc = check_plan(ctx, "paged_release", batch, page_size, table_stride, n_pages);
  if (rc != GQ_OK) return rc;
  if (!free_count || !free_left || (n_pages > 0 && !free_pages) || (batch > 0 && (!seq_lens || !keep_lens || !totals)) ||
      (batch > 0 && table_stride > 0 && !block_table))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_release: null pointer");
  PlanArgs a{};
  a.batch = batch;
  a.page_size = (uint32_t)page_size;
  a.table_stride = table_stride;
  a.n_pages = n_pages;
  a.seq_lens = seq_lens;
  a.other_lens = keep_lens;
  a.table = const_cast<int32_t *>(block_table);
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.free_left = free_left;
  a.totals = totals;
  // the pages given back are known on the device only: at most every entry of the pool or the table
  return plan_launch(ctx, false, a, std::min(n_pages, batch * std::min<int64_t>(table_stride, INT32_MAX)));
}

extern "C" int gq_paged_append(gq_ctx *ctx, const gq_kv_pages *pages, const float *k, const float *v, int64_t t,
                               int64_t k_tok_stride, int64_t v_tok_stride, const int64_t *slots) {
  ENTER(ctx);
  int rc = gq_check_kv_pages(ctx, "paged_append", pages);
  if (rc != GQ_OK) return rc;
  const int64_t row = pages->heads * pages->head_dim;
  if (k_tok_stride == 0) k_tok_stride = row;
  if (v_tok_stride == 0) v_tok_stride = row;
  if (t < 0 || k_tok_stride < row || v_tok_stride < row || k_tok_stride % 4 != 0 || v_tok_stride % 4 != 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_append: bad token count, or a token stride below a row or not a multiple of 4");
  if (t == 0) return GQ_OK;
  if (!k || !v || !slots) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_append: null pointer");
  if (((uintptr_t)k | (uintptr_t)v) % 16 != 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_append: k and v must be 16-byte aligned");
  if (pages->type == GQ_KV_E2M1) return gq_paged_append_e2m1(ctx, pages, k, v, t, k_tok_stride, v_tok_stride, slots);
  AppendArgs a{};
  a.src[0] = k;
  a.src[1] = v;
  a.dst[0] = pages->k;
  a.dst[1] = pages->v;
  a.src_stride[0] = k_tok_stride;
  a.src_stride[1] = v_tok_stride;
  a.slots = slots;
  a.tokens = t;
  a.page_size = pages->page_size;
  a.page_stride = pages->page_stride ? pages->page_stride : row * pages->page_size;
  a.n_slots = pages->n_pages * pages->page_size;
  a.heads = (int)pages->heads;
  a.head_dim = (int)pages->head_dim;
  a.inv_scale[0] = 1.0f / pages->k_scale;
  a.inv_scale[1] = 1.0f / pages->v_scale;
  a.err = ctx->dev_err;
  const dim3 grid((unsigned)std::min<int64_t>((2 * t + kAppendThreads / 32 - 1) / (kAppendThreads / 32), (int64_t)ctx->num_sms * 8));
  switch (pages->type) {
    case GQ_KV_F32: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_append_kernel<GQ_KV_F32>, grid, dim3(kAppendThreads), 0, a)); break;
    case GQ_KV_F16: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_append_kernel<GQ_KV_F16>, grid, dim3(kAppendThreads), 0, a)); break;
    case GQ_KV_BF16: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_append_kernel<GQ_KV_BF16>, grid, dim3(kAppendThreads), 0, a)); break;
    default: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_append_kernel<GQ_KV_E4M3>, grid, dim3(kAppendThreads), 0, a)); break;
  }
  return GQ_OK;
}
