// paged_attn.cu — attention of one new token per request over a paged key-value cache
// (gq_paged_attention).
//
//   out_h = sum_j p_j v_j / sum_j p_j,  p_j = e^(s_j - m),  s_j = cap(scale q_h . k_j)
//
// with m the running maximum: tiles of keys are read once, and when a tile raises m the
// sum and the output so far are scaled by e^(m_old - m). What bounds it: the bytes of
// the visible keys and values, each read once (the up to 8 query heads of a key-value
// head share the read).
//
// paged_rows_kernel serves every head_dim, page size and type with plain loads and
// CUDA-core products.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "paged_attn.cuh"

// paged_attn_tc.cu
bool gq_paged_attn_tc_supported(const gq_kv_pages *pages, int64_t page_stride);
int gq_paged_attn_tc_launch(gq_ctx *ctx, const gq_kv_pages *pages, pattn::Args &a);

namespace {

using namespace pattn;

constexpr int kRowThreads = 128;
constexpr int kRowTile = 64;
// CTAs per SM: a warp has one key's loads in flight, so warps make up for it. Two against
// four, replayed, 64 requests of up to 4096 keys: e4m3 rows of 64 184.9 / 116.7 us, bf16
// rows of 96 371.7 / 205.5, bf16 rows of 512 on pages of 24 575.3 / 316.9; 225 of up to 62
// keys, 8 heads of 96 in bf16, 160.7 / 129.1; one of 333 keys 27.5 / 27.4.
constexpr int kRowPerSm = 4;
static_assert(kRowPerSm <= kMostPerSm, "memory for the parts");

template <int TYPE>
__device__ __forceinline__ float4 load4(const void *base, int64_t elem) {
  if constexpr (TYPE == GQ_KV_F32) {
    return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + elem);
  } else if constexpr (TYPE == GQ_KV_E4M3) {
    const uint32_t u = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(base) + elem);
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> 16), __NV_E4M3);
    const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
    return make_float4(a.x, a.y, b.x, b.y);
  } else {
    const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + elem);
    if constexpr (TYPE == GQ_KV_BF16) {
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xffff0000u));
    } else {
      const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
      return make_float4(a.x, a.y, b.x, b.y);
    }
  }
}

// Scores: a warp per key, 4 columns per lane and step. Softmax: 16 threads per head.
// Output: thread t owns columns 4t .. 4t + 3 of all 8 heads.
template <int TYPE>
__global__ void __launch_bounds__(kRowThreads) paged_rows_kernel(const Args a) {
  __shared__ __align__(16) float q[kHeads][512];
  __shared__ float s[kHeads][kRowTile];
  __shared__ int64_t elem[kRowTile];  // first element of a key's row, -1: zero row
  __shared__ float fix[kHeads], sum[kHeads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const Cut cut = find_cut<kRowThreads, kRowTile>(a);
  if (cut.w0 >= cut.w1) {
    if (tid == 0) a.cut_units[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  int b = cut.b, u = cut.u, t = cut.t;
  for (int64_t w = cut.w0;;) {
    const Range r = range_of<kRowTile>(a, visible(a, b));
    if (t < 0) {  // the place ahead of the unit's tiles
      t = 0;
      if (++w == cut.w1) {  // its tiles are the next CTA's
        if (tid == 0) a.cut_units[blockIdx.x] = make_int4(0, 0, 0, 0);
        return;
      }
    }
    const int tiles = (int)min((int64_t)(r.nt - t), cut.w1 - w);
    int head0, nh, kvh;
    unit_heads(a, u, head0, nh, kvh);
    __syncthreads();  // q and s of the unit before are read
    for (int i = tid; i < kHeads * a.dim; i += kRowThreads) {
      const int h = i / a.dim, c = i - h * a.dim;
      q[h][c] = h < nh ? a.q[b * a.q_stride + (int64_t)(head0 + h) * a.dim + c] : 0.0f;
    }
    const int sh = tid >> 4, sl = tid & 15;  // softmax: head, lane of 16
    float m = -INFINITY, l = 0.0f;
    float4 o[kHeads];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) o[h] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < tiles; ++i) {
      const int j0 = (r.tile0 + t + i) * kRowTile;
      if (tid < kRowTile) {
        const int j = j0 + tid;
        int64_t e = -1;
        if (j >= r.lo && j < r.hi) {
          const int page = a.table[b * a.table_stride + j / a.page_size];
          if (page >= 0 && page < a.n_pages)
            e = page * a.page_stride + ((int64_t)kvh * a.page_size + j % a.page_size) * a.dim;
          else
            gqd::report(a.err, GQ_DEVERR_PAGES);
        }
        elem[tid] = e;
      }
      __syncthreads();
      for (int kk = warp; kk < kRowTile; kk += kRowThreads / 32) {
        const int64_t e = elem[kk];
        float dot[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) dot[h] = 0.0f;
        if (e >= 0)
          for (int c = lane * 4; c < a.dim; c += 128) {
            const float4 k = load4<TYPE>(a.k, e + c);
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
              const float4 qv = *reinterpret_cast<const float4 *>(&q[h][c]);
              dot[h] = fmaf(qv.x, k.x, fmaf(qv.y, k.y, fmaf(qv.z, k.z, fmaf(qv.w, k.w, dot[h]))));
            }
          }
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
#pragma unroll
          for (int off = 16; off >= 1; off >>= 1) dot[h] += __shfl_xor_sync(0xffffffffu, dot[h], off);
        if (lane == 0)
#pragma unroll
          for (int h = 0; h < kHeads; ++h) s[h][kk] = dot[h];
      }
      __syncthreads();
      float x[kRowTile / 16], top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kRowTile / 16; ++k) {
        const int j = j0 + k * 16 + sl;
        x[k] = j >= r.lo && j < r.hi ? score_of(a, s[sh][k * 16 + sl]) : -INFINITY;
        top = fmaxf(top, x[k]);
      }
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float mn = fmaxf(m, top);
      const float base = mn == -INFINITY ? 0.0f : mn;  // (no visible key yet)
      const float f = exp_of(m - base);
      l *= f;
#pragma unroll
      for (int k = 0; k < kRowTile / 16; ++k) {
        const float p = exp_of(x[k] - base);
        s[sh][k * 16 + sl] = p;
        l += p;
      }
      m = mn;
      if (sl == 0) fix[sh] = f;
      __syncthreads();
      if (tid * 4 < a.dim) {
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const float g = fix[h];
          o[h].x *= g;
          o[h].y *= g;
          o[h].z *= g;
          o[h].w *= g;
        }
        for (int kk = 0; kk < kRowTile; ++kk) {
          const int64_t e = elem[kk];
          if (e < 0) continue;
          const float4 v = load4<TYPE>(a.v, e + tid * 4);
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            const float p = s[h][kk];
            o[h].x = fmaf(p, v.x, o[h].x);
            o[h].y = fmaf(p, v.y, o[h].y);
            o[h].z = fmaf(p, v.z, o[h].z);
            o[h].w = fmaf(p, v.w, o[h].w);
          }
        }
      }
      __syncthreads();  // s and elem are free
    }
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const bool whole = tiles == r.nt;
    const int64_t s0 = w - t;
    const int slot = whole ? 0 : slot_of(cut, s0);
    if (sl == 0) {
      sum[sh] = l;
      if (!whole) {
        a.part_ml[(slot * kHeads + sh) * 2] = m;
        a.part_ml[(slot * kHeads + sh) * 2 + 1] = l;
      }
    }
    __syncthreads();
    if (tid * 4 < a.dim) {
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        if (whole) {
          const float f = inv_or_zero(sum[h]) * a.v_scale;
          if (h < nh)
            *reinterpret_cast<float4 *>(a.out + ((int64_t)b * a.hq + head0 + h) * a.dim + tid * 4) =
                make_float4(o[h].x * f, o[h].y * f, o[h].z * f, o[h].w * f);
        } else {
          *reinterpret_cast<float4 *>(a.part_o + ((int64_t)slot * kHeads + h) * a.dim + tid * 4) = o[h];
        }
      }
    }
    w += tiles;
    if (w == cut.w1) {
      if (tid == 0) put_cut_unit(a, cut, b, u, s0, r.nt);
      return;
    }
    t = -1;
    if (++u == a.units_per_req) {
      u = 0;
      ++b;
    }
  }
}

// Adds up the parts of cut units. A CTA takes (unit, `wide` float4 columns of its heads)
// in turn; its threads are wide columns times 256 / wide groups that share the parts, and
// the groups' sums are added in order. wide is the most that leaves a thread no more parts
// of the longest unit than it loads at once: one round of loads per item, and few items
// (with items of 128 columns for all, 64 units of 5 parts took 11 us at head_dim 512).
// A join inside the first launch was built two ways and was slower: by the last CTA of a
// unit to arrive (up to 40 us after the last tile for a unit of 99 parts of 16 KB), and
// by all CTAs of a cooperative launch, each waiting for its units' parts and joining a
// share of their columns (4 us for 6 parts, 10-14 us for 300).
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinBatch = 8;

__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const Args a, int grid) {
  constexpr int kEach = (kMaxGrid + kJoinThreads - 1) / kJoinThreads;
  __shared__ int4 units[kMaxGrid];
  __shared__ int counts[kJoinWarps], longest[kJoinWarps];
  __shared__ float4 sums[kJoinThreads];
  __shared__ float2 sum_ml[kJoinThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  // the list of cut units, in order of the CTAs they begin in
  int4 mine[kEach];
  int have = 0, most = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int c = tid * kEach + i;
    mine[i] = c < grid ? __ldcg(a.cut_units + c) : make_int4(0, 0, 0, 0);
    have += mine[i].z > 0;
    most = max(most, mine[i].z);
  }
  int incl = have;
  most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) {
    counts[warp] = incl;
    longest[warp] = most;
  }
  __syncthreads();
  int n = 0, at = incl - have;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    if (w < warp) at += counts[w];
    n += counts[w];
    most = max(most, longest[w]);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (mine[i].z > 0) units[at++] = mine[i];
  __syncthreads();

  int groups = 1;
  while (groups * kJoinBatch < most && groups < kJoinThreads / 8) groups <<= 1;
  const int wide = kJoinThreads / groups, group = tid / wide, cols = a.dim / 4;
  const int slices = (kHeads * cols + wide - 1) / wide;
  for (int item = blockIdx.x; item < n * slices; item += gridDim.x) {
    const int4 unit = units[item / slices];
    const int at = (item % slices) * wide + tid % wide, h = at / cols, col = at - h * cols;
    int head0, nh, kvh;
    unit_heads(a, unit.y, head0, nh, kvh);
    const bool real = h < nh;
    const int parts = real ? unit.z : 0, first = unit.w, next = (first & ~1) + 2;  // slots: first, next, next + 2, ...
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml);
    const float4 *part = reinterpret_cast<const float4 *>(a.part_o);
    // each group adds its parts to a maximum of its own, kJoinBatch parts' loads at a time
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = group; p0 < parts; p0 += groups * kJoinBatch) {
      float2 x[kJoinBatch];
      float4 v[kJoinBatch];
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        const int p = p0 + k * groups;
        x[k] = make_float2(-INFINITY, 0.0f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < parts) {
          const int64_t s = (int64_t)(p == 0 ? first : next + 2 * (p - 1)) * kHeads + h;
          x[k] = __ldcg(ml + s);
          v[k] = __ldcg(part + s * cols + col);
        }
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) top = fmaxf(top, x[k].x);
      const float f = m == -INFINITY ? 0.0f : exp_of(m - top);
      l *= f;
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        const float w = x[k].x == -INFINITY ? 0.0f : exp_of(x[k].x - top);
        l = fmaf(w, x[k].y, l);
        o.x = fmaf(w, v[k].x, o.x);
        o.y = fmaf(w, v[k].y, o.y);
        o.z = fmaf(w, v[k].z, o.z);
        o.w = fmaf(w, v[k].w, o.w);
      }
      m = top;
    }
    __syncthreads();  // the sums of the item before are read
    sums[tid] = o;
    sum_ml[tid] = make_float2(m, l);
    __syncthreads();
    if (group == 0 && real) {
      for (int k = 1; k < groups; ++k) m = fmaxf(m, sum_ml[k * wide + tid].x);
      l = 0.0f;
      o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < groups; ++k) {
        const float2 x = sum_ml[k * wide + tid];
        const float4 v = sums[k * wide + tid];
        const float f = x.x == -INFINITY ? 0.0f : exp_of(x.x - m);
        l = fmaf(f, x.y, l);
        o.x = fmaf(f, v.x, o.x);
        o.y = fmaf(f, v.y, o.y);
        o.z = fmaf(f, v.z, o.z);
        o.w = fmaf(f, v.w, o.w);
      }
      const float s = inv_or_zero(l) * a.v_scale;
      *reinterpret_cast<float4 *>(a.out + ((int64_t)unit.x * a.hq + head0 + h) * a.dim + col * 4) =
          make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
    }
  }
}

template <int TYPE>
cudaError_t rows_launch(gq_ctx *ctx, int grid, const Args &a) {
  return gq_launch(ctx, paged_rows_kernel<TYPE>, dim3(grid), dim3(kRowThreads), 0, a);
}

}  // namespace

int gq_paged_join_launch(gq_ctx *ctx, const Args &a, int grid) {
  if (grid <= 1) return GQ_OK;  // nothing can be cut
  // two CTAs per SM, fewer where even the narrowest items of all possible cuts are fewer
  const int64_t most = (int64_t)(grid - 1) * ((kHeads * a.dim / 4 + 7) / 8);
  const int items = (int)std::min<int64_t>(most, 2 * (int64_t)ctx->num_sms);
  GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_join_kernel, dim3(items), dim3(kJoinThreads), 0, a, grid));
  return GQ_OK;
}

extern "C" int gq_paged_attention(gq_ctx *ctx, const gq_kv_pages *pages, const float *q, int64_t batch, int64_t hq,
                                  int64_t q_tok_stride, const int32_t *block_table, int64_t table_stride,
                                  const int32_t *seq_lens, float scale, uint32_t sliding_window, float attn_softcap,
                                  float *out) {
  if (!ctx) return GQ_ERR_INVALID_ARGUMENT;
  int rc = gq_enter_ctx(ctx);
  if (rc != GQ_OK) return rc;
  rc = gq_check_kv_pages(ctx, "paged_attention", pages);
  if (rc != GQ_OK) return rc;
  if (batch < 0 || batch > INT32_MAX || hq < 1 || hq % pages->heads != 0 || table_stride < 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_attention: bad batch or table_stride, or hq not a multiple of the pages' heads");
  if (hq / pages->heads > 64)
    return gq_fail(ctx, GQ_ERR_UNSUPPORTED, "paged_attention: more than 64 query heads per key-value head");
  if (q_tok_stride == 0) q_tok_stride = hq * pages->head_dim;
  if (q_tok_stride < hq * pages->head_dim || q_tok_stride % 4 != 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_attention: q_tok_stride below a row, or not a multiple of 4");
  if (batch == 0) return GQ_OK;
  if (!q || !out || !seq_lens || (table_stride > 0 && !block_table))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
  if (((uintptr_t)q | (uintptr_t)out) % 16 != 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_attention: q and out must be 16-byte aligned");
  Args a{};
  a.q = q;
  a.out = out;
  a.k = pages->k;
  a.v = pages->v;
  a.table = block_table;
  a.lens = seq_lens;
  a.q_stride = q_tok_stride;
  a.table_stride = table_stride;
  a.page_stride = pages->page_stride ? pages->page_stride : pages->heads * pages->page_size * pages->head_dim;
  a.n_pages = pages->n_pages;
  // (the last tile's keys are numbered in 32 bits; the product is kept inside 64)
  a.room = std::min<int64_t>(std::min<int64_t>(table_stride, INT32_MAX) * pages->page_size, INT32_MAX - 1024);
  a.batch = (int)batch;
  a.hq = (int)hq;
  a.heads = (int)pages->heads;
  a.group = (int)(hq / pages->heads);
  a.sub = (a.group + kHeads - 1) / kHeads;
  a.units_per_req = a.heads * a.sub;
  a.dim = (int)pages->head_dim;
  a.page_size = (int)pages->page_size;
  a.window = (int32_t)std::min<uint32_t>(sliding_window, INT32_MAX);
  a.scale = scale * pages->k_scale;
  a.softcap = attn_softcap;
  a.inv_softcap = attn_softcap > 0.0f ? 1.0f / attn_softcap : 0.0f;
  a.v_scale = pages->v_scale;
  a.err = ctx->dev_err;
  if (gq_paged_attn_tc_supported(pages, a.page_stride)) return gq_paged_attn_tc_launch(ctx, pages, a);
  const int grid = grid_for(a, kRowTile, kRowPerSm * ctx->num_sms);
  rc = bind_parts(ctx, grid, a);
  if (rc != GQ_OK) return rc;
  switch (pages->type) {
    case GQ_KV_F32: GQ_CUDA_TRY(ctx, rows_launch<GQ_KV_F32>(ctx, grid, a)); break;
    case GQ_KV_F16: GQ_CUDA_TRY(ctx, rows_launch<GQ_KV_F16>(ctx, grid, a)); break;
    case GQ_KV_BF16: GQ_CUDA_TRY(ctx, rows_launch<GQ_KV_BF16>(ctx, grid, a)); break;
    default: GQ_CUDA_TRY(ctx, rows_launch<GQ_KV_E4M3>(ctx, grid, a)); break;
  }
  return gq_paged_join_launch(ctx, a, grid);
}
