// paged_attn_q4.cu — gq_paged_attention over pages of 4-bit values (GQ_KV_E2M1) on the tensor cores.
//
// A value is a code of 4 bits times its block's e4m3 scale, exact in f16; the query and the weights
// (f32) are cut into two f16 parts (22 bits). Rows of 9/16 byte a value make the instructions per
// value, not the bytes, what bounds this kernel: at 6.5 TB/s a scheduler has one instruction of a warp
// for 10 values. Hence:
//   * A warp does everything for its 32 keys: both products and the softmax between them, in registers.
//     Warps meet at the end of a request only.
//   * Scores S = q K^T with the 8 heads as rows 0-7 and the second parts of the same heads as rows 8-15 of
//     the m16n8k16 instruction: no row is idle. Its result is laid out as the second operand of
//     O^T = V^T P^T wants the weights, so they stay where they are.
//   * Codes go from shared memory to fragments without a transposing load: which keys and columns an
//     instruction's rows stand for is free, so a lane reads 8 bytes of one key (4 of 64 columns) and
//     uses all of them. For V the codes of two keys are put side by side (one byte, two keys) before they become f16.
//   * A key that is not visible gets the scale 0 (a code is never NaN): nothing is cleared.
// Copies are untiled bulk copies, one per page (or part of a page) of 32 keys, into a ring of each team's
// own: a team is one warp, or D / 128 of 128 columns each, which add up their parts of the scores (256
// columns a warp leave registers for three warps to a scheduler: 50.0 us in place of 47.8 for 64 requests
// of up to 4096 keys of 512).
//
// 64 requests of up to 4096 keys of 512 (80 MB): 47 us; 23 of up to 10007, 4 key-value heads of 128, capped
// scores (72 MB): 39 us; 4 of up to 131072 of 512 (205 MB): 76 us, 2.7 TB/s. No unit is full: issue slots are 52-60%
// taken, conversions 36-39%, the matrix pipe 25-32%. 128 registers a thread (and 8 to 100 bytes of each instance
// spilled) leave 16 warps per SM, too few to hide a tile's dependent steps, of which it has many: a warp executes 830
// instructions for 32 keys of 128 columns, 320 of them conversions, products with scales and matrix products. Some
// 12 us of a call are not keys: the cut 2, code that is run once, parts brought together 2, the join's launch 5.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "e2m1.cuh"
#include "paged_attn.cuh"

namespace {

using namespace pattn;

constexpr int kKeys = 32;  // keys of a tile

template <int D>
struct Conf {
  static constexpr int PS = D > 128 ? D / 128 : 1;  // warps that share a tile's columns (a team)
  static constexpr int DW = D / PS;              // columns of a warp
  static constexpr int kRow = D / 16 * 9;        // bytes of a key's row
  static constexpr int CB = DW / 16;             // bytes of codes that a lane takes at once
  static constexpr int NC = DW / (8 * CB);       // times it does for K
  static constexpr int W = CB / 4;               // words of it: 2, or 1 of 64 columns
  static constexpr int kWarps = D > 128 ? 8 : 4;
  static constexpr int kTeams = kWarps / PS;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kSlot = 2 * kKeys * kRow;
  static constexpr int kStages = 2;
  static constexpr int kPerSm = D > 128 ? 2 : 4;
  static constexpr int kQBytes = D / 16 * 32 * 16;
  static constexpr int kSwap = PS > 1 ? kTeams * 2 * PS * 32 * 8 * 4 : 0;
  static constexpr int kSmem = kTeams * kStages * kSlot + kQBytes + kSwap;
  static_assert(kSlot >= 8 * D * 4, "a team's part of the output fits a slot");
  static_assert(W <= 2, "a lane's codes have one scale");
};

// The key that stands at place n of the r-th 8 keys: rows of the 8 lanes that load together (K: keys of
// neighbouring n; V: every other key) then lie on different banks.
template <int D>
__device__ __forceinline__ int key_at(int r, int n) {
  const int e = n < 4 ? n : n ^ 1;
  if constexpr (D == 512) return 8 * r + e;
  if constexpr (D == 256) return 16 * (r >> 1) + (r & 1) + 2 * e;
  if constexpr (D == 128) return r + 4 * e;
  return r + 4 * n;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Eight codes to f16: pair i from byte i.
__device__ __forceinline__ void e2m1_word(uint32_t u, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(u));
}
// Two e4m3 codes (low 16 bits of u) to a pair of f16.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t u) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(u));
  return r;
}
__device__ __forceinline__ uint32_t mul2(uint32_t x, uint32_t y) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2 *>(&x), *reinterpret_cast<__half2 *>(&y));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void split_f16(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  hi = *reinterpret_cast<const uint32_t *>(&h);
  lo = pack2(x - __low2float(h), y - __high2float(h));
}
// The bits of x where the mask has ones, of y where it has none.
__device__ __forceinline__ uint32_t select(uint32_t mask, uint32_t x, uint32_t y) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xca;" : "=r"(r) : "r"(mask), "r"(x), "r"(y));
  return r;
}
template <int W>
__device__ __forceinline__ void lds(const uint8_t *p, uint32_t (&w)[W]) {
  if constexpr (W == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  }
}
template <int PS>
__device__ __forceinline__ void team_sync(int team) {
  if constexpr (PS == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(PS * 32) : "memory");
}

// Wait of a whole warp; false in all its lanes where one's gave up, or did not wait because another's
// had. It is reported, and the CTA runs to its end without waiting (what it computes is dropped by the
// error); its warps ask for no more copies.
__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort, uint32_t *err) {
  bool ok = !*abort;
  if (ok) {
    ok = gqd::mbar_wait_bounded(bar, parity);
    if (!ok) {
      *abort = 1;
      gqd::report(err, GQ_DEVERR_WAIT_TIMEOUT);
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Join the parts of a cluster's unit, each in its CTA's shared memory (mine [8][D] and its maxima and
// sums): every CTA adds up a share of the columns, in rank order.
template <int D, int NT>
__device__ __forceinline__ void join_cluster(const Args &a, const float *mine, const float2 *mine_ml, int b, int head0, int nh) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int n = a.cluster, rank = (int)cluster.block_rank(), items = nh * (D / 4);
  cluster.sync();  // every part is written
  for (int at = items * rank / n + (int)threadIdx.x; at < items * (rank + 1) / n; at += NT) {
    const int h = at / (D / 4);
    float m = -INFINITY, l = 0.0f;
    float2 ml[8];
    float4 v[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      v[p] = p < n ? reinterpret_cast<const float4 *>(cluster.map_shared_rank(mine, p))[at] : make_float4(0.f, 0.f, 0.f, 0.f);
      ml[p] = p < n ? cluster.map_shared_rank(mine_ml, p)[h] : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, ml[p].x);
    }
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      // (a part whose largest is -inf has no visible key, and zeros, or scores that are no numbers: its NaNs are kept)
      const float w = ml[p].x == -INFINITY ? 0.0f : exp_of(ml[p].x - m);
      l = fmaf(w, ml[p].y, l);
      o.x = fmaf(w, v[p].x, o.x);
      o.y = fmaf(w, v[p].y, o.y);
      o.z = fmaf(w, v[p].z, o.z);
      o.w = fmaf(w, v[p].w, o.w);
    }
    const float s = inv_or_zero(l) * a.v_scale;
    reinterpret_cast<float4 *>(a.out + ((int64_t)b * a.hq + head0) * D)[at] = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
  }
  cluster.sync();  // no CTA's memory goes away while it is read
}

// The power of two that brings a number whose bits these are to 2^13 .. 2^14, 0 where that has no answer.
__device__ __forceinline__ int up_of(uint32_t bits) {
  const int e = (int)(bits >> 23);
  return e > 0 && e < 255 ? min(max(140 - e, -126), 126) : 0;
}

template <int D>
__global__ void __launch_bounds__(Conf<D>::kThreads, Conf<D>::kPerSm) paged_q4_kernel(const Args a) {
  using C = Conf<D>;
  constexpr int PS = C::PS, DW = C::DW, CB = C::CB, NC = C::NC, W = C::W, TEAMS = C::kTeams, S = C::kStages, ROW = C::kRow;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[TEAMS][S];
  __shared__ uint32_t head_top[kHeads];  // the largest |q| of a head (bits)
  __shared__ float2 ml[TEAMS][kHeads], share_ml[kHeads];
  __shared__ int part_slot[TEAMS];  // the slot of a team's part, -1: none
  __shared__ int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int team = warp / PS, half = warp - team * PS;
  const int g = lane >> 2, q4 = lane & 3;
  uint8_t *ring = smem + team * (S * C::kSlot);
  uint4 *qs = reinterpret_cast<uint4 *>(smem + TEAMS * S * C::kSlot);  // [half][step][lane]
  float4 *swap = reinterpret_cast<float4 *>(smem + TEAMS * S * C::kSlot + C::kQBytes);
  if (tid == 0) {
    for (int t = 0; t < TEAMS; ++t)
      for (int i = 0; i < S; ++i) gqd::mbar_init(&full[t][i], 1);
    gqd::fence_mbar_init();
    abort_flag = 0;
  }
  if (tid < kHeads) head_top[tid] = 0;
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  Cut cut;
  if (a.cluster) {
    // a unit of few tiles: its cluster's CTAs take neighbouring tiles (the last may get none)
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
    cut.b = unit / a.units_per_req;
    cut.u = unit - cut.b * a.units_per_req;
    cut.keys = visible(a, cut.b);
    const int nt = range_of<kKeys>(a, cut.keys).nt, each = (nt + a.cluster - 1) / a.cluster;
    cut.t = min(rank * each, nt);
    cut.w0 = 0;
    cut.w1 = min(each, nt - cut.t);
    if (tid == 0 && rank == 0 && a.lens[cut.b] > a.room) gqd::report(a.err, GQ_DEVERR_PAGES);
    __syncthreads();  // the mbarriers
  } else {
    cut = find_cut<C::kThreads, kKeys>(a);  // (its barriers also publish the mbarriers)
    if (cut.w0 >= cut.w1) {
      if (tid == 0) a.cut_units[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
  }
  const int rows_shift = min(a.page_shift, 5), rows = 1 << rows_shift;  // keys that one copy brings
  const int boxes = kKeys >> rows_shift;

  // ---- loads (the team's first warp): a cursor that walks every TEAMS-th tile of this CTA's piece. Lane
  // i owns a tile's i-th copy; its table entry is read a tile before the copy is asked for.
  int lb = cut.b, lu = cut.u, lt = cut.t;
  int64_t lw = cut.w0;
  Range lr = range_of<kKeys>(a, cut.keys);
  bool more = true;        // the cursor is on a tile
  bool has = false;        // this lane has a copy of it
  int page = 0, row = 0;   // of this lane's copy
  int lhead = (lu / a.sub) << a.page_shift;  // the first row of the unit's key-value head in a page
  auto step = [&](int n) {  // n tiles on
    if (lt < 0) {
      lt = 0;
      ++lw;
    }
    while (lw < cut.w1 && n >= lr.nt - lt) {
      n -= lr.nt - lt;
      lw += lr.nt - lt + 1;
      lt = 0;
      if (lw >= cut.w1) break;
      if (++lu == a.units_per_req) {
        lu = 0;
        lr = range_of<kKeys>(a, visible(a, ++lb));
      }
      lhead = (lu / a.sub) << a.page_shift;
    }
    lt += n;
    lw += n;
    more = lw < cut.w1;
    has = false;
    if (!more) return;
    const int j = (lr.tile0 + lt) * kKeys + (lane << rows_shift);
    if (lane < boxes && j < lr.hi && j + rows > lr.lo) {
      row = lhead + (j & (a.page_size - 1));
      page = a.table[lb * a.table_stride + (j >> a.page_shift)];  // (not looked at before its copy is due)
      has = true;
    }
  };
  uint32_t issued = 0;
  auto issue = [&]() {  // the cursor's tile to the next slot, and on to the next tile
    if (!more) return;
    const int slot = issued % S;
    uint8_t *to = ring + slot * C::kSlot;
    const uint32_t bytes = (uint32_t)rows * ROW;
    const bool good = has && page >= 0 && page < a.n_pages;
    const int copies = __popc(__ballot_sync(0xffffffffu, good));
    const uint32_t bad = __ballot_sync(0xffffffffu, has && !good);
    if (bad) {  // rows of zeros
      if (lane == 0) gqd::report(a.err, GQ_DEVERR_PAGES);
      for (int i = 0; i < boxes; ++i)
        if (bad >> i & 1)
          for (int at = lane * 4; at < (int)bytes; at += 128) {
            *reinterpret_cast<uint32_t *>(to + i * bytes + at) = 0;
            *reinterpret_cast<uint32_t *>(to + kKeys * ROW + i * bytes + at) = 0;
          }
      __syncwarp();
    }
    if (lane == 0) gqd::mbar_arrive_expect_tx(&full[team][slot], (uint32_t)copies * 2 * bytes);
    __syncwarp();
    if (good) {
      const int64_t at = page * a.page_stride + (int64_t)row * ROW;
      gqd::bulk_g2s(to + lane * bytes, static_cast<const uint8_t *>(a.k) + at, bytes, &full[team][slot]);
      gqd::bulk_g2s(to + kKeys * ROW + lane * bytes, static_cast<const uint8_t *>(a.v) + at, bytes, &full[team][slot]);
    }
    ++issued;
    step(TEAMS);
  };

  if (half == 0) step(team);

  // ---- compute
  uint32_t n = 0;    // tiles that this team has read
  int count = 0;     // tiles of this CTA's piece so far (all teams)
  bool begun = false;
  int b = cut.b, u = cut.u, t = cut.t, keys = cut.keys;
  for (int64_t w = cut.w0;;) {
    const Range r = range_of<kKeys>(a, keys);
    if (t < 0) {  // the place ahead of the unit's tiles
      t = 0;
      if (++w == cut.w1) {  // its tiles are the next CTA's
        if (tid == 0) a.cut_units[blockIdx.x] = make_int4(0, 0, 0, 0);
        break;
      }
    }
    const int tiles = (int)min((int64_t)(r.nt - t), cut.w1 - w);
    int head0, nh, kvh;
    unit_heads(a, u, head0, nh, kvh);

    // ---- q: per head scaled to 2^13 .. 2^14, so that the second part stays normal, and cut in two. Asked
    // for before the first keys, which come later.
    constexpr int kItems = D / 16 * 32 / C::kThreads;
    const int ig = (tid >> 2) & 7;  // the head of this thread's items: 4 columns each
    float4 qv[kItems];
    {
      const float *qg = a.q + b * a.q_stride + (int64_t)(head0 + ig) * D + (tid & 3) * (2 * CB);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int st = (tid >> 5) + i * C::kWarps, k = st % (DW / 16);
        qv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ig < nh) qv[i] = *reinterpret_cast<const float4 *>(qg + st / (DW / 16) * DW + k / (CB / 2) * (8 * CB) + k % (CB / 2) * 4);
      }
    }
    if (!begun) {
      begun = true;
      if (half == 0)
        for (int i = 0; i < S; ++i) issue();
    }
    {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < kItems; ++i)
        top = fmaxf(top, fmaxf(fmaxf(fabsf(qv[i].x), fabsf(qv[i].y)), fmaxf(fabsf(qv[i].z), fabsf(qv[i].w))));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (q4 == 0) atomicMax(&head_top[ig], __float_as_uint(top));
    }
    __syncthreads();  // (also: everyone is done with the unit before)
    {
      const float f = __uint_as_float((uint32_t)(127 + up_of(head_top[ig])) << 23);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        uint4 v;
        split_f16(qv[i].x * f, qv[i].y * f, v.x, v.y);
        split_f16(qv[i].z * f, qv[i].w * f, v.z, v.w);
        qs[tid + i * C::kThreads] = v;
      }
    }
    const float un = __uint_as_float((uint32_t)(127 - up_of(head_top[g])) << 23) * a.scale;
    __syncthreads();

    float acc[CB][4];
#pragma unroll
    for (int i = 0; i < CB; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int mine = -1;  // the last slot read: kept for this team's part of the unit
    // the team's tiles: every TEAMS-th of the piece
    for (int i = (team - count % TEAMS + TEAMS) % TEAMS; i < tiles; i += TEAMS) {
      const int j0 = (r.tile0 + t + i) * kKeys, slot = n % S;
      uint8_t *kt = ring + slot * C::kSlot;
      if (!wait_or_abort(&full[team][slot], (n / S) & 1, &abort_flag, a.err)) more = false;
      // ---- scores of head g and the keys at places 2 q4 and 2 q4 + 1 of each 8
      float x[4][2];
      {
        float c[4][4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          x[y][0] = x[y][1] = 0.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k) c[y][k] = 0.0f;
        }
#pragma unroll
        for (int cc = 0; cc < NC; ++cc) {
          uint32_t kw[4][W], sc[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const uint8_t *kr = kt + key_at<D>(y, g) * ROW;
            lds<W>(kr + half * (DW / 2) + cc * (4 * CB) + q4 * CB, kw[y]);
            const uint8_t *ks = kr + D / 2 + half * (DW / 16);
            const uint32_t one = e4m3_pair(ks[(cc * 4 + q4) * CB / 8]);
            sc[y] = __byte_perm(one, one, 0x1010);
          }
#pragma unroll
          for (int wd = 0; wd < W; ++wd) {
            const int st = cc * (CB / 2) + wd * 2;
            const uint4 q0 = qs[(half * (DW / 16) + st) * 32 + lane], q1 = qs[(half * (DW / 16) + st + 1) * 32 + lane];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              uint32_t h[4];
              e2m1_word(kw[y][wd], h);
              const uint32_t f = sc[y];
              mma_f16(c[y], q0.x, q0.y, q0.z, q0.w, mul2(h[0], f), mul2(h[1], f));
              mma_f16(c[y], q1.x, q1.y, q1.z, q1.w, mul2(h[2], f), mul2(h[3], f));
              // (the instruction truncates its sums: four are added up in it, the rest here)
              if (wd % 2 == 1 || W == 1) {
                x[y][0] += c[y][0];
                x[y][1] += c[y][1];
                c[y][0] = c[y][1] = 0.0f;
              }
            }
          }
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          x[y][0] += c[y][2];
          x[y][1] += c[y][3];
        }
      }
      if constexpr (PS > 1) {  // the other warps' columns
        float4 *at = swap + (team * 2 + (n & 1)) * (PS * 64) + lane;
        at[half * 64] = make_float4(x[0][0], x[0][1], x[1][0], x[1][1]);
        at[half * 64 + 32] = make_float4(x[2][0], x[2][1], x[3][0], x[3][1]);
        team_sync<PS>(team);  // (the team is done with the tile before, too)
        // (in the same order in every warp: their weights are the same)
#pragma unroll
        for (int h = 0; h < PS; ++h) {
          const float4 o0 = at[h * 64], o1 = at[h * 64 + 32];
          if (h == 0) {
            x[0][0] = o0.x, x[0][1] = o0.y, x[1][0] = o0.z, x[1][1] = o0.w;
            x[2][0] = o1.x, x[2][1] = o1.y, x[3][0] = o1.z, x[3][1] = o1.w;
          } else {
            x[0][0] += o0.x, x[0][1] += o0.y, x[1][0] += o0.z, x[1][1] += o0.w;
            x[2][0] += o1.x, x[2][1] += o1.y, x[3][0] += o1.z, x[3][1] += o1.w;
          }
        }
        if (mine >= 0 && half == 0) {
          gqd::fence_proxy_async_smem();
          __syncwarp();
          issue();
        }
      }
      mine = slot;
      ++n;

      // ---- weights
      const bool ragged = j0 < r.lo || j0 + kKeys > r.hi;
      float top = -INFINITY;
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int e = 0; e < 2; ++e) x[y][e] = a.softcap * tanhf(x[y][e] * un * a.inv_softcap);
      } else {
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int e = 0; e < 2; ++e) x[y][e] *= un;
      }
      if (ragged) {
        asm volatile("");  // (a branch: most tiles are whole)
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = j0 + key_at<D>(y, 2 * q4 + e);
            if (j < r.lo || j >= r.hi) x[y][e] = -INFINITY;
          }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) top = fmaxf(top, fmaxf(x[y][0], x[y][1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn, f = exp_of(m - base);
      m = mn;
      l *= f;
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        // times 2^14, a common factor of every weight and sum: the second part stays normal
        const float p0 = 16384.0f * exp_of(x[y][0] - base), p1 = 16384.0f * exp_of(x[y][1] - base);
        l += p0 + p1;
        split_f16(p0, p1, ph[y], pl[y]);
      }
      const float f0 = __shfl_sync(0xffffffffu, f, q4 * 8), f1 = __shfl_sync(0xffffffffu, f, q4 * 8 + 4);

      // ---- output: 16 columns by 8 heads per instruction, over 16 keys
      const uint8_t *vt = kt + kKeys * ROW;
      uint32_t vw[8][W], sb[8], sp[4];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const uint8_t *vr = vt + key_at<D>(y >> 1, 2 * q4 + (y & 1)) * ROW;
        lds<W>(vr + half * (DW / 2) + g * CB, vw[y]);
        const uint8_t *vs = vr + D / 2 + half * (DW / 16);
        sb[y] = vs[g * CB / 8];
      }
      if (ragged) {
        asm volatile("");
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const int j = j0 + key_at<D>(y >> 1, 2 * q4 + (y & 1));
          if (j < r.lo || j >= r.hi) sb[y] = 0;
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) sp[y] = e4m3_pair(__byte_perm(sb[2 * y], sb[2 * y + 1], 0x5140));
#pragma unroll
      for (int wd = 0; wd < W; ++wd) {
        float c[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) c[k][0] = c[k][1] = c[k][2] = c[k][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t ev[2][4], od[2][4];  // columns 2 k and 2 k + 1 of two keys, twice
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t v0 = vw[4 * ks + 2 * y][wd], v1 = vw[4 * ks + 2 * y + 1][wd];
            e2m1_word(select(0x0f0f0f0fu, v0, v1 << 4), ev[y]);
            e2m1_word(select(0x0f0f0f0fu, v0 >> 4, v1), od[y]);
            const uint32_t s = sp[2 * ks + y];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              ev[y][k] = mul2(ev[y][k], s);
              od[y][k] = mul2(od[y][k], s);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_f16(c[k], ev[0][k], od[0][k], ev[1][k], od[1][k], pl[2 * ks], pl[2 * ks + 1]);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_f16(c[k], ev[0][k], od[0][k], ev[1][k], od[1][k], ph[2 * ks], ph[2 * ks + 1]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float (&o)[4] = acc[4 * wd + k];
          o[0] = fmaf(o[0], f0, c[k][0]);
          o[1] = fmaf(o[1], f1, c[k][1]);
          o[2] = fmaf(o[2], f0, c[k][2]);
          o[3] = fmaf(o[3], f1, c[k][3]);
        }
      }
      if (PS == 1 && i + TEAMS < tiles) {  // the slot is read (a unit's last one is kept)
        gqd::fence_proxy_async_smem();
        __syncwarp();
        issue();
      }
    }

    // ---- the unit's output, or this CTA's part of it: teams' parts are brought to a common maximum and
    // added up through their last slots
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (half == 0 && q4 == 0) ml[team][g] = make_float2(m, l);
    if (half == 0 && lane == 0) part_slot[team] = mine;
    __syncthreads();
    if (mine >= 0) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float most = -INFINITY;
#pragma unroll
        for (int y = 0; y < TEAMS; ++y) most = fmaxf(most, ml[y][2 * q4 + e].x);
        f[e] = most == -INFINITY ? 0.0f : exp_of(ml[team][2 * q4 + e].x - most);
      }
      float *to = reinterpret_cast<float *>(ring + mine * C::kSlot) + half * DW + g * (2 * CB);
#pragma unroll
      for (int i = 0; i < CB; ++i) {
        *reinterpret_cast<float2 *>(to + (2 * q4) * D + 2 * i) = make_float2(acc[i][0] * f[0], acc[i][2] * f[0]);
        *reinterpret_cast<float2 *>(to + (2 * q4 + 1) * D + 2 * i) = make_float2(acc[i][1] * f[1], acc[i][3] * f[1]);
      }
    }
    __syncthreads();
    const bool shared = a.cluster > 1, whole = !shared && tiles == r.nt;
    const int64_t s0 = w - t;
    const int part = whole || shared ? 0 : slot_of(cut, s0);
    float4 *base = reinterpret_cast<float4 *>(shared  ? reinterpret_cast<float *>(smem)
                                              : whole ? a.out + ((int64_t)b * a.hq + head0) * D
                                                      : a.part_o + (int64_t)part * kHeads * D);
    for (int at = tid; at < (whole ? nh : kHeads) * (D / 4); at += C::kThreads) {
      const int h = at / (D / 4);
      float most = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int y = 0; y < TEAMS; ++y) most = fmaxf(most, ml[y][h].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int y = 0; y < TEAMS; ++y) {
        if (part_slot[y] < 0) continue;
        const float4 v = reinterpret_cast<const float4 *>(smem + (y * S + part_slot[y]) * C::kSlot)[at];
        const float2 x = ml[y][h];
        sum += x.x == -INFINITY ? 0.0f : exp_of(x.x - most) * x.y;
        o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
      }
      if (whole) {
        const float s = inv_or_zero(sum) * a.v_scale;
        o = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
      } else if (at % (D / 4) == 0) {
        if (shared) share_ml[h] = make_float2(most, sum);
        else *reinterpret_cast<float2 *>(a.part_ml + ((int64_t)part * kHeads + h) * 2) = make_float2(most, sum);
      }
      base[at] = o;
    }
    if (shared) {
      join_cluster<D, C::kThreads>(a, reinterpret_cast<const float *>(smem), share_ml, b, head0, nh);
      break;
    }
    if (a.cluster) break;
    w += tiles;
    count += tiles;
    if (w == cut.w1) {
      if (tid == 0) put_cut_unit(a, cut, b, u, s0, r.nt);
      break;
    }
    if (tid < kHeads) head_top[tid] = 0;
    __syncthreads();  // the parts are read
    if (mine >= 0 && half == 0) {
      gqd::fence_proxy_async_smem();
      __syncwarp();
      issue();
    }
    t = -1;
    if (++u == a.units_per_req) {
      u = 0;
      keys = visible(a, ++b);
    }
  }
  if (half == 0 && lane == 0 && *(volatile int *)&abort_flag)
    // copies still in flight end before the CTA's memory goes away
    for (uint32_t i = issued > S ? issued - S : 0; i < issued; ++i)
      (void)gqd::mbar_wait_bounded(&full[team][i % S], (i / S) & 1, 100000000ull);
}

template <int D>
int launch(gq_ctx *ctx, Args &a) {
  using C = Conf<D>;
  static bool attr_set[64] = {};
  if (!attr_set[ctx->device & 63]) {
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(paged_q4_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    attr_set[ctx->device & 63] = true;
  }
  // Units that cannot have many tiles get a cluster of CTAs each: no cut, no join. (One request of 333 keys 6.9 us,
  // cut 10.2; 64 of 512 keys in a window 13.4 and 18.6; 225 of up to 62 keys, 8 heads, 20 and 25.) Where units are long
  // or uneven a cluster waits for its longest: 64 of up to 4096 keys 59 us, cut 47. Hence 8 tiles of a CTA at the
  // most, and not many more than equal pieces had.
  const int64_t units = (int64_t)a.batch * a.units_per_req, tiles = most_tiles(a, kKeys);
  const int slots = C::kPerSm * ctx->num_sms;
  int cluster = 8;
  while (cluster > 1 && (units * cluster > slots || cluster >= 2 * tiles)) cluster >>= 1;
  const int64_t each = (tiles + cluster - 1) / cluster;
  const int64_t equal = (units * tiles + slots - 1) / slots;
  if (each <= 8 && each <= equal + 2 && units * cluster <= INT32_MAX) {
    a.cluster = cluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * cluster));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
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
    GQ_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, paged_q4_kernel<D>, (const Args)a));
    return GQ_OK;
  }
  const int grid = grid_for(a, kKeys, slots);
  const int rc = bind_parts(ctx, grid, a);
  if (rc != GQ_OK) return rc;
  GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_q4_kernel<D>, dim3(grid), dim3(C::kThreads), C::kSmem, a));
  return gq_paged_join_launch(ctx, a, grid);
}

}  // namespace

// Head_dims of the instantiated kernels, and pages of which a tile has a whole number or the other way round, in copies
// that begin and end on 16 bytes: a power of two of rows, 8 at least (a row may be 36 bytes), and pages a multiple of 16
// bytes apart. What is left goes to the kernel that takes keys one by one: 4 requests of up to 131072 keys of 512 733 us,
// here 76.
bool gq_paged_attn_q4_supported(const gq_kv_pages *p) {
  const int64_t d = p->head_dim, stride = gq_kv_page_stride(p);
  return p->type == GQ_KV_E2M1 && (d == 64 || d == 128 || d == 256 || d == 512) && p->page_size >= 8 &&
         (p->page_size & (p->page_size - 1)) == 0 && stride % 16 == 0 && p->heads * p->page_size <= INT32_MAX;
}

int gq_paged_attn_q4_launch(gq_ctx *ctx, const gq_kv_pages *p, Args &a) {
  while ((int64_t(1) << a.page_shift) < p->page_size) ++a.page_shift;
  switch (p->head_dim) {
    case 64: return launch<64>(ctx, a);
    case 128: return launch<128>(ctx, a);
    case 256: return launch<256>(ctx, a);
    default: return launch<512>(ctx, a);
  }
}
