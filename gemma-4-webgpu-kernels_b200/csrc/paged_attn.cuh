// paged_attn.cuh — the parts that the kernels of gq_paged_attention share: how the work
// is cut over the grid, and how the parts of a cut request are joined.
//
// Work: a unit is one request and one block of up to 8 query heads that read the same
// key-value head; it is a run of tiles of T keys. All units' tiles in a row (request by
// request) are cut into one equal piece per CTA, so every CTA streams the same number
// of keys whatever the requests' lengths; a CTA may end one unit, do some whole and
// begin another. The lengths are on the device, so each CTA makes the cut itself.
//
// Joining: softmax over a cut unit needs each part's maximum m, sum l and unnormalised
// output o: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i, m = max m_i. Parts go
// to a workspace slot; the last CTA of a group of about sqrt(n) parts to arrive joins
// the group, the last group joins the groups, always in part order, so the result does
// not depend on who came last. Two levels because one CTA reads about 100 GB/s: the
// 296 parts of one long request (8 KB each at head_dim 256) would take it 24 us, two
// levels of 17 take 3.
#pragma once

#include <algorithm>

#include "paged.cuh"

namespace pattn {

constexpr int kHeads = 8;       // query heads per unit
constexpr int kMaxGrid = 1000;  // 4 counters per CTA
constexpr int kCtrBase = 64;    // (paged.cu uses the counters below)
constexpr int kOneLevel = 8;    // up to this many parts are joined at once
constexpr int kMaxJoin = 32;    // >= ceil(sqrt(kMaxGrid))
static_assert(kCtrBase + 4 * kMaxGrid <= (int)kCtxCounters, "counters");
static_assert(kMaxJoin * kMaxJoin >= kMaxGrid, "two levels must reach every part");

constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const float *q;
  float *out;
  const void *k, *v;
  const int32_t *table, *lens;
  int64_t q_stride, table_stride, page_stride, n_pages;
  int batch, hq, heads, group, sub, units_per_req;  // group = hq / heads, sub = blocks of 8 per key-value head
  int dim, page_size, page_shift;                   // page_shift: log2 page_size (tiled kernels)
  int32_t window;
  float scale, softcap, v_scale;  // scale: of the scores, the keys' scale included
  float *part_o, *part_ml;        // [2 grid][8][dim], [2 grid][8][2]
  uint32_t *ctr, *err;
};

struct Range {
  int lo, hi;    // visible keys
  int tile0, nt; // tiles that hold them (at least one, so that every unit has an owner)
};

__device__ __forceinline__ int visible(const Args &a, int b) {
  const int64_t len = max(a.lens[b], 0), room = a.table_stride * a.page_size;
  return (int)min(len, room);
}
template <int T>
__device__ __forceinline__ Range range_of(const Args &a, int b) {
  Range r;
  r.hi = visible(a, b);
  r.lo = a.window > 0 && r.hi > a.window ? r.hi - a.window : 0;
  r.tile0 = r.lo / T;
  r.nt = max(1, (int)(((uint32_t)r.hi + T - 1) / T) - r.tile0);
  return r;
}

// This CTA's piece [w0, w1) of all tiles, and the unit and tile w0 lies in. The grid may
// be larger than the work: CTAs at or past `grid` have none.
struct Cut {
  int64_t total, w0, w1;
  int grid, b, u, t;  // request, unit of the request, tile of the unit
  __device__ __forceinline__ int64_t start(int c) const { return c * total / grid; }
  // the CTA whose piece holds tile w
  __device__ __forceinline__ int at(int64_t w) const { return (int)(((w + 1) * grid - 1) / total); }
};

// Threads 0 .. NT - 1 (a whole block) take neighbouring requests each.
template <int NT, int T>
__device__ __forceinline__ Cut find_cut(const Args &a) {
  __shared__ int64_t sums[NT / 32];
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch + NT - 1) / NT;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  int64_t mine = 0;
  bool past = false;
  for (int b = b0; b < b1; ++b) {
    mine += (int64_t)range_of<T>(a, b).nt * a.units_per_req;
    past |= a.lens[b] > a.table_stride * a.page_size;
  }
  if (past && blockIdx.x == 0) gqd::report(a.err, GQ_DEVERR_PAGES);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  Cut cut;
  cut.total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) incl += sums[w];
    cut.total += sums[w];
  }
  cut.grid = (int)min((int64_t)gridDim.x, cut.total);
  const int c = blockIdx.x;
  cut.w0 = c < cut.grid ? cut.start(c) : cut.total;
  cut.w1 = c < cut.grid ? cut.start(c + 1) : cut.total;
  if (cut.w0 >= incl - mine && cut.w0 < incl) {
    int64_t at = incl - mine;
    for (int b = b0; b < b1; ++b) {
      const int nt = range_of<T>(a, b).nt;
      const int64_t next = at + (int64_t)nt * a.units_per_req;
      if (cut.w0 < next) {
        found[0] = b;
        found[1] = (int)((cut.w0 - at) / nt);
        found[2] = (int)((cut.w0 - at) % nt);
        break;
      }
      at = next;
    }
  }
  __syncthreads();
  cut.b = found[0];
  cut.u = found[1];
  cut.t = found[2];
  return cut;
}

// Query heads of unit u: its first head, how many, and its key-value head.
__device__ __forceinline__ void unit_heads(const Args &a, int u, int &head0, int &n, int &kv) {
  kv = u / a.sub;
  const int s = u - kv * a.sub;
  head0 = kv * a.group + s * kHeads;
  n = min(kHeads, a.group - s * kHeads);
}

// Barrier of the NT threads that compute (the first NT of the block).
template <int NT>
__device__ __forceinline__ void sync_compute() {
  asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
}

// Join `n` parts (part i in slot slots(i)) and hand each (head, 4 columns) sum with its
// maximum and sum of weights to `put`.
template <int NT, typename Slots, typename Put>
__device__ __forceinline__ void join(const Args &a, int n, Slots slots, Put put) {
  __shared__ float wgt[kMaxJoin][kHeads];
  __shared__ float ms[kHeads], ls[kHeads];
  const int tid = threadIdx.x;
  for (int i = tid; i < n * kHeads; i += NT) wgt[i / kHeads][i % kHeads] = __ldcg(a.part_ml + (slots(i / kHeads) * kHeads + i % kHeads) * 2);
  sync_compute<NT>();
  if (tid < kHeads) {
    float m = -INFINITY, l = 0.0f;
    for (int i = 0; i < n; ++i) m = fmaxf(m, wgt[i][tid]);
    for (int i = 0; i < n; ++i) {
      const float mi = wgt[i][tid];
      const float w = mi == -INFINITY ? 0.0f : exp2f(mi - m);
      l = fmaf(w, __ldcg(a.part_ml + (slots(i) * kHeads + tid) * 2 + 1), l);
      wgt[i][tid] = w;
    }
    ms[tid] = m;
    ls[tid] = l;
  }
  sync_compute<NT>();
  const int per = a.dim / 4;
  for (int i = tid; i < kHeads * per; i += NT) {
    const int h = i / per, c = (i - h * per) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < n; ++p) {
      const float w = wgt[p][h];
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(a.part_o + ((int64_t)slots(p) * kHeads + h) * a.dim + c));
      o.x = fmaf(w, x.x, o.x);
      o.y = fmaf(w, x.y, o.y);
      o.z = fmaf(w, x.z, o.z);
      o.w = fmaf(w, x.w, o.w);
    }
    put(h, c, o, ms[h], ls[h]);
  }
}

// True in every thread of the CTA that arrives last of n at the counter.
template <int NT>
__device__ __forceinline__ bool arrive_last(uint32_t *ctr, int n) {
  __shared__ int last;
  sync_compute<NT>();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(ctr, 1u) == (uint32_t)n - 1;
    if (last) {
      *ctr = 0u;
      __threadfence();
    }
  }
  sync_compute<NT>();
  return last != 0;
}

__device__ __forceinline__ float inv_or_zero(float l) { return l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l); }

// Slot of CTA c's part of the unit that starts at tile s0: a CTA has at most two parts
// of cut units, the one it begins in the middle of (or begins with) and its last.
__device__ __forceinline__ int slot_of(const Cut &cut, int c, int64_t s0) { return 2 * c + (cut.start(c) < s0 ? 1 : 0); }

// The NT computing threads of CTA blockIdx.x, after its part of unit (b, u) (tiles s0 .. s0 + nt of
// the whole row of tiles) is in its slot: join when this CTA is the last.
template <int NT>
__device__ __forceinline__ void finish_part(const Args &a, const Cut &cut, int b, int u, int64_t s0, int nt) {
  const int c0 = cut.at(s0), n = cut.at(s0 + nt - 1) - c0 + 1;
  const int g = n > kOneLevel ? (int)ceilf(sqrtf((float)n)) : n;
  const int groups = (n + g - 1) / g, j = ((int)blockIdx.x - c0) / g;
  const int first = c0 + j * g, members = min(g, n - j * g);
  if (!arrive_last<NT>(a.ctr + 2 * slot_of(cut, first, s0), members)) return;
  if (groups > 1) {
    const int to = slot_of(cut, first, s0);
    // the sums replace the group's first part, column by column where that was just read
    join<NT>(a, members, [&](int i) { return slot_of(cut, first + i, s0); },
             [&](int h, int c, float4 o, float m, float l) {
               *reinterpret_cast<float4 *>(a.part_o + ((int64_t)to * kHeads + h) * a.dim + c) = o;
               if (c == 0) {
                 a.part_ml[(to * kHeads + h) * 2] = m;
                 a.part_ml[(to * kHeads + h) * 2 + 1] = l;
               }
             });
    if (!arrive_last<NT>(a.ctr + 2 * slot_of(cut, c0, s0) + 1, groups)) return;
  }
  int head0, nh, kv;
  unit_heads(a, u, head0, nh, kv);
  float *out = a.out + ((int64_t)b * a.hq + head0) * a.dim;
  join<NT>(a, groups > 1 ? groups : n, [&](int i) { return slot_of(cut, c0 + (groups > 1 ? i * g : i), s0); },
           [&](int h, int c, float4 o, float, float l) {
             if (h >= nh) return;
             const float s = inv_or_zero(l) * a.v_scale;
             *reinterpret_cast<float4 *>(out + (int64_t)h * a.dim + c) = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
           });
}

// Score of one visible key in units of log2: the scaled, optionally capped product.
__device__ __forceinline__ float score_log2(const Args &a, float dot) {
  float s = dot * a.scale;
  if (a.softcap > 0.0f) s = a.softcap * tanhf(__fdiv_rn(s, a.softcap));
  return s * kLog2e;
}

// ---- host side

// CTAs to launch: at most `most`, and no more than there can be tiles (the table bounds
// the lengths, which the host does not know).
inline int grid_for(const Args &a, int tile, int most) {
  int64_t keys = std::min<int64_t>(a.table_stride * a.page_size, INT32_MAX);
  if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + tile);
  const int64_t tiles = (int64_t)a.batch * a.units_per_req * std::max<int64_t>(1, (keys + tile - 1) / tile);
  return (int)std::min<int64_t>(tiles, std::min(kMaxGrid, most));
}

// Workspace for the parts: two per CTA.
inline int bind_workspace(gq_ctx *ctx, int grid, Args &a) {
  void *ws = nullptr;
  const int rc = gq_workspace(ctx, (size_t)grid * 2 * kHeads * (a.dim + 2) * 4, &ws);
  a.part_o = static_cast<float *>(ws);
  a.part_ml = a.part_o + (size_t)grid * 2 * kHeads * a.dim;
  return rc;
}

}  // namespace pattn
