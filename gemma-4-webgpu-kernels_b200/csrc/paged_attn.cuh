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
// output o: out = sum_i e^(m_i - m) o_i / sum_i e^(m_i - m) l_i, m = max m_i. Parts go
// to workspace slots and the second launch of the call, paged_join_kernel, adds them up
// in part order, whichever CTA made them (results do not vary from run to run). A join
// inside the first launch, by the last CTA to arrive, was measured slower: one CTA reads
// its parts at some 15-100 GB/s, so the 99 parts of a 131072-key request (16 KB each)
// kept it 40 us after the last key; the join kernel spreads them over the GPU.
#pragma once

#include <algorithm>

#include "paged.cuh"

namespace pattn {

constexpr int kHeads = 8;       // query heads per unit
constexpr int kMaxGrid = 640;
constexpr int kMostPerSm = 4;   // CTAs per SM of any of the kernels

constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const float *q;
  float *out;
  const void *k, *v;
  const int32_t *table, *lens;
  int64_t q_stride, table_stride, page_stride, n_pages;
  int64_t room;                                     // tokens that a table row can hold
  int cluster;                                      // CTAs per unit (one cluster), 0: units cut by find_cut
  int batch, hq, heads, group, sub, units_per_req;  // group = hq / heads, sub = blocks of 8 per key-value head
  int dim, page_size, page_shift;                   // page_shift: log2 page_size (tiled kernels)
  int row;                                          // elements from a row of a page to the next (bytes of e2m1 rows)
  int32_t window;
  float scale, softcap, inv_softcap, v_scale;  // scale: of the scores, the keys' scale included
  float *part_o, *part_ml;        // [2 grid][8][dim], [2 grid][8][2]
  int4 *cut_units;                // [grid]: the cut unit that begins in a CTA: request, unit, parts (0: none), first slot
  uint32_t *err;
};

struct Range {
  int lo, hi;    // visible keys
  int tile0, nt; // tiles that hold them (at least one, so that every unit has an owner)
};

__device__ __forceinline__ int visible(const Args &a, int b) {
  return (int)min((int64_t)max(a.lens[b], 0), a.room);
}
template <int T>
__device__ __forceinline__ Range range_of(const Args &a, int keys) {
  Range r;
  r.hi = keys;
  r.lo = a.window > 0 && r.hi > a.window ? r.hi - a.window : 0;
  r.tile0 = r.lo / T;
  r.nt = max(1, (int)(((uint32_t)r.hi + T - 1) / T) - r.tile0);
  return r;
}

__device__ __forceinline__ int64_t div_of(int64_t x, int64_t y) {  // x, y >= 0; the short division where it will do
  return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}

// This CTA's piece [w0, w1) of all places, and the unit and tile w0 lies in (a unit is nt
// + 1 places: t = -1 is the place ahead of its tiles). The first
// `more` of `grid` pieces hold each + 1 tiles, the others each. (The grid may be larger
// than the work: CTAs past `grid` have none.)
struct Cut {
  int64_t total, each, w0, w1;
  int grid, more;
  int b, u, t, keys;  // request, unit of the request, tile of the unit; the request's keys
  __device__ __forceinline__ int64_t start(int c) const { return c * each + min(c, more); }
  // the CTA whose piece holds place w
  __device__ __forceinline__ int at(int64_t w) const {
    const int64_t big = more * (each + 1);
    return (int)(w < big ? div_of(w, each + 1) : more + div_of(w - big, each));
  }
};

// Threads 0 .. NT - 1 (a whole block) take neighbouring requests each.
template <int NT, int T>
__device__ __forceinline__ Cut find_cut(const Args &a) {
  __shared__ int64_t sums[NT / 32];
  __shared__ int found[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch + NT - 1) / NT;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  int64_t mine = 0;
  bool past = false;
  for (int b = b0; b < b1; ++b) {
    mine += (int64_t)(range_of<T>(a, visible(a, b)).nt + 1) * a.units_per_req;
    past |= a.lens[b] > a.room;
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
  cut.each = div_of(cut.total, cut.grid);
  cut.more = (int)(cut.total - cut.each * cut.grid);
  const int c = blockIdx.x;
  cut.w0 = c < cut.grid ? cut.start(c) : cut.total;
  cut.w1 = c < cut.grid ? cut.start(c + 1) : cut.total;
  if (cut.w0 >= incl - mine && cut.w0 < incl) {
    int64_t at = incl - mine;
    for (int b = b0; b < b1; ++b) {
      const int keys = visible(a, b), places = range_of<T>(a, keys).nt + 1;
      const int64_t next = at + (int64_t)places * a.units_per_req;
      if (cut.w0 < next) {
        const int u = (int)div_of(cut.w0 - at, places);
        found[0] = b;
        found[1] = u;
        found[2] = (int)(cut.w0 - at - (int64_t)u * places) - 1;
        found[3] = keys;
        break;
      }
      at = next;
    }
  }
  __syncthreads();
  cut.b = found[0];
  cut.u = found[1];
  cut.t = found[2];
  cut.keys = found[3];
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

__device__ __forceinline__ float inv_or_zero(float l) { return l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l); }

// Slot of this CTA's part of a cut unit whose first tile is at place s0: a CTA has at most
// two parts of cut units, the one it begins in the middle of (or begins with) and its last.
__device__ __forceinline__ int slot_of(const Cut &cut, int64_t s0) { return 2 * blockIdx.x + (cut.w0 < s0 ? 1 : 0); }

// One thread of each CTA says which cut unit's first tile is in it (nt tiles from place
// s0 on), or that none is. The unit's other parts are in the slots 2 c of the
// CTAs that follow.
__device__ __forceinline__ void put_cut_unit(const Args &a, const Cut &cut, int b, int u, int64_t s0, int nt) {
  const bool begins = cut.w0 <= s0 && s0 < cut.w1 && s0 + nt > cut.w1;
  const int parts = begins ? cut.at(s0 + nt - 1) - (int)blockIdx.x + 1 : 0;
  a.cut_units[blockIdx.x] = make_int4(b, u, parts, slot_of(cut, s0));
}

// e^x of a difference x <= 0 of two scores; -inf gives 0. (The difference is taken before it
// is brought to powers of 2: of scores near the maximum, which weigh most, it is exact.
// What is below 2^-126 counts as 0; the instruction's error is 2^-22.)
__device__ __forceinline__ float exp_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * kLog2e));
  return y;
}

// Score of one visible key: the scaled, optionally capped product.
__device__ __forceinline__ float score_of(const Args &a, float dot) {
  const float s = dot * a.scale;
  return a.softcap > 0.0f ? a.softcap * tanhf(s * a.inv_softcap) : s;
}

// ---- host side

// Most tiles a unit can have.
inline int64_t most_tiles(const Args &a, int tile) {
  const int64_t keys = a.window > 0 ? std::min<int64_t>(a.room, (int64_t)a.window + tile - 1) : a.room;
  return std::max<int64_t>(1, (keys + tile - 1) / tile);
}

// CTAs to launch: at most `slots`, and no more than there can be tiles (the table bounds
// the lengths, which the host does not know).
inline int grid_for(const Args &a, int tile, int slots) {
  const int64_t tiles = (int64_t)a.batch * a.units_per_req * most_tiles(a, tile);
  return (int)std::min<int64_t>(tiles, std::min(kMaxGrid, slots));
}

// Memory for the parts (two per CTA) and the list of cut units: one block of the largest
// size, made by the context's first call and kept, so that a recorded graph's addresses
// stay good whatever is called after it (20 MB on 148 SMs: four CTAs per SM, the most any
// kernel has, at head_dim 512).
inline int bind_parts(gq_ctx *ctx, int grid, Args &a) {
  constexpr size_t kPerCta = 2 * kHeads * (512 + 2) * 4 + sizeof(int4);
  const size_t bytes = (size_t)std::min(kMaxGrid, kMostPerSm * ctx->num_sms) * kPerCta;
  if ((size_t)grid * (2 * kHeads * (a.dim + 2) * 4 + sizeof(int4)) > bytes)
    return gq_fail(ctx, GQ_ERR_UNSUPPORTED, "paged_attention: more partial results than there is memory for");
  if (!ctx->paged_ws) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    GQ_CUDA_TRY(ctx, cudaStreamIsCapturing(ctx->stream, &st));
    if (st != cudaStreamCaptureStatusNone)
      return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_attention: run the call once before recording (it allocates)");
    GQ_CUDA_TRY(ctx, cudaMalloc(&ctx->paged_ws, bytes));
  }
  a.cut_units = static_cast<int4 *>(ctx->paged_ws);
  a.part_o = reinterpret_cast<float *>(a.cut_units + grid);
  a.part_ml = a.part_o + (size_t)grid * 2 * kHeads * a.dim;
  return GQ_OK;
}

}  // namespace pattn

// The second launch: joins the units that the first one (of `grid` CTAs) cut.
int gq_paged_join_launch(gq_ctx *ctx, const pattn::Args &a, int grid);
