// paged_attn_tc.cu — the tiled kernel of gq_paged_attention: pages by TMA, products on
// the tensor cores, f32 results.
//
// A tile is T keys of one unit (one request, up to 8 query heads of one key-value head).
// Pages (or parts of pages) come by one 4-D TMA copy each into a ring of tiles (128-byte
// swizzle, so the fragment loads below have no bank conflicts), issued by warp 0 as ring
// slots become free. Four warps compute:
//   S^T = K q^T        m16 = keys, n8 = heads, over head_dim: keys split over the warps
//                      (and head_dim over KS warps where q would not fit the registers)
//   p = e^(s - m)      16 threads per head; running maximum and sum
//   O^T += V^T p^T     m16 = head_dim columns, n8 = heads, over the T keys: columns
//                      split over the warps
// with the scores of tile i + 1 in the tensor pipe while the weights of tile i are made:
// one barrier per tile. Transposed, the 8 heads fill the instruction's n = 8 exactly: no
// product is wasted, and a key-value head's cache is read once for all of them. More than 8
// heads are more units, each of which reads it (L2 may still have it: 64 requests of up to
// 4096 keys in bf16, 8 against 16 heads of 512 59 / 91 us, 8 against 64 heads of 128 24 / 121
// us, replayed). The m16n8 instructions
// (mma.sync) are used, not tcgen05: at n = 8 the work is 16 products per cached value,
// and the ring, not the tensor pipe, is the limit; a 128-row accumulator tile in tensor
// memory would add a round trip per tile for a softmax over its rows.
//
// f32 results from 16-bit products: q and p (f32) are cut into parts that each fit the
// type and add up to the number: bf16 3 parts (24 bits); f16 2 parts (22 bits, q scaled
// per head to 2^13..2^14 and p to 2^14 so the second part stays normal); f32 pages use
// tf32 with both operands in 2 parts, the product of the two low parts (2^-22) left out.
// The cached 16- and 8-bit values are exact in their type (e4m3 in f16), products are
// exact in f32, and sums are f32: relative errors of 0.3-0.8e-6 against 64 bits, as plain
// f32 arithmetic has. The extra instructions are free here: 3 per 16 x 16
// cached values, a fifth to a third of the legacy tensor pipe at the rates below.
//
// Measured (B200, a call among others, both launches): 64 requests of up to 4096 keys,
// head_dim 512, bf16, 279 MB: 59 us, 4.7 TB/s, the tiles themselves 41 us at 6.8 TB/s
// (the rest: 4 us from the start to the first keys, which come through two dependent
// loads, lengths and table, and 12 us for the join and two kernel boundaries). 3 requests
// of up to 131072 keys, e4m3, 249 MB: 58 us. 23 requests of up to 2501, f32, 4 heads of
// 128, soft-cap, 127 MB: 34 us. With plain loads and CUDA-core products
// (paged_rows_kernel, replayed): 318, 528 and 202 us. One request of 333 keys (a cluster of 8): 6.7
// us replayed.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "paged_attn.cuh"
#include "tc_common.cuh"

namespace {

using namespace pattn;

constexpr int kComputeWarps = 4;
constexpr int kCompute = kComputeWarps * 32;
constexpr int kMaxSlots = 8;

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          gqd::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(gqd::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ float lds32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// v = hi + lo: hi the nearest tf32 number (two integer operations; the conversion
// instruction costs four), lo exact (the tensor instruction reads its top 11 bits).
__device__ __forceinline__ void split_tf32(float v, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(v) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(v - __uint_as_float(hi));
}
template <typename H2>
__device__ __forceinline__ uint32_t bits(H2 v) {
  return *reinterpret_cast<uint32_t *>(&v);
}
// Parts of a pair of f32 numbers as packed pairs.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&part)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    part[i] = bits(h);
    x -= __low2float(h);
    y -= __high2float(h);
  }
}
__device__ __forceinline__ void split_f16(float x, float y, uint32_t (&part)[2]) {
  const __half2 h = __floats2half2_rn(x, y);
  part[0] = bits(h);
  part[1] = bits(__floats2half2_rn(x - __low2float(h), y - __high2float(h)));
}
// Two e4m3 codes (low 16 bits of u) to a pair of f16.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t u) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(u));
  return r;
}

// What a type and head_dim fix.
template <int TYPE, int D>
struct Tile {
  static constexpr int kSize = TYPE == GQ_KV_F32 ? 4 : TYPE == GQ_KV_E4M3 ? 1 : 2;
  static constexpr int kRow = D * kSize;          // bytes of a key
  static constexpr int kChunks = kRow / 128;      // 128-byte pieces of a key
  // head_dim is split over KS warps where the q fragments of one warp would not fit its
  // registers (2 parts of 256 columns or 3 of 256 at 16 bits, 2 of 128 at 32)
  static constexpr int KS = TYPE == GQ_KV_F32 ? (D > 128 ? D / 128 : 1) : (D > 256 ? D / 256 : 1);
  // 16-key tiles per warp: two where one would make a tile small beside what it costs
  // whatever its size (barrier, softmax), and two leave room for three slots
  static constexpr int MT = 16 * kComputeWarps / KS * kRow <= (KS > 1 ? 16384 : 8192) ? 2 : 1;
  static constexpr int T = 16 * kComputeWarps * MT / KS;
  static constexpr int kSlot = T * kRow;
  // CTAs per SM: three where rows are short, a tile is little work and 168 registers will
  // do (225 requests of up to 62 keys, 8 heads of 64, bf16: 31.4 us with two, 24.5 with
  // three; 10 of up to 40000, one head of 128: 35.3 and 33.8; e4m3 rows of 256 spill with
  // three and lose 20 %). (With two, e4m3 rows of 512 spill 16 bytes at the head.)
  static constexpr int kPerSm = kRow <= 256 && D <= 128 ? 3 : 2;
  static constexpr int kSmemBytes = (kPerSm == 3 ? 72 : 110) * 1024;
  static constexpr int kParts = TYPE == GQ_KV_BF16 ? 3 : 2;
  static constexpr int kStep = TYPE == GQ_KV_F32 ? 8 : 16;      // head_dim columns (keys) per instruction
  static constexpr int kQSteps = D / KS / kStep;
  static constexpr int kMTiles = D / kComputeWarps / 16;        // 16-column tiles of the output per warp
  static constexpr int kSStride = T + 4;                        // floats between heads' scores
  static constexpr int kSFloats = KS * kHeads * kSStride;
  static constexpr int kPStride = TYPE == GQ_KV_F32 ? (T + 4) * 4 : T * 2 + 16;  // bytes between heads' weights
  static constexpr int kPBytes = (TYPE == GQ_KV_F32 ? 1 : kParts) * kHeads * kPStride;
  static constexpr int kRest = 1024 + 2 * (kSFloats * 4 + kPBytes);  // scores and weights of two tiles
  static constexpr int kSlots = std::min(kMaxSlots, (kSmemBytes - kRest) / kSlot);
  static constexpr int kSmem = kRest + kSlots * kSlot;
  static constexpr int kTShift = T == 128 ? 7 : T == 64 ? 6 : T == 32 ? 5 : 4;
  static_assert(kQSteps % 4 == 0, "whole groups of products");
  static_assert(kRow % 128 == 0 && kSlots >= 3 && (1 << kTShift) == T && kPBytes % 16 == 0, "tile");
};

// Wait of a whole warp; false in all its lanes where one's gave up, or did not wait because
// another's had. It is reported, and the CTA runs to its end without waiting (what it
// computes is dropped by the error). Warp 0 then asks for no more copies: the slot's last
// one may still be in flight, and its barrier's phase is not over. (The vote in place of a
// warp barrier: 64 requests of up to 4096 keys in bf16 58.3 -> 58.4 us; the vote in each
// tile's block barrier, or on the flag before each copy, 58.7 and 58.8.)
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


// Join the parts of a cluster's unit, each in its CTA's shared memory (mine [8][D] and its
// maxima and sums): every CTA adds up a share of the columns, in rank order.
template <int D>
__device__ __forceinline__ void join_cluster(const Args &a, const float *mine, const float2 *mine_ml, int b, int head0, int nh) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int n = a.cluster, rank = (int)cluster.block_rank(), items = nh * (D / 4);
  cluster.sync();  // every part is written
  for (int at = items * rank / n + (int)threadIdx.x; at < items * (rank + 1) / n; at += kCompute) {
    const int h = at / (D / 4);
    float m = -INFINITY, l = 0.0f;
    float2 ml[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      ml[p] = p < n ? cluster.map_shared_rank(mine_ml, p)[h] : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, ml[p].x);
    }
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      if (ml[p].x == -INFINITY) continue;  // no CTA, or one without a visible key: its columns are not written
      const float4 v = reinterpret_cast<const float4 *>(cluster.map_shared_rank(mine, p))[at];
      const float w = exp_of(ml[p].x - m);
      l = fmaf(w, ml[p].y, l);
      o.x = fmaf(w, v.x, o.x);
      o.y = fmaf(w, v.y, o.y);
      o.z = fmaf(w, v.z, o.z);
      o.w = fmaf(w, v.w, o.w);
    }
    const float s = inv_or_zero(l) * a.v_scale;
    reinterpret_cast<float4 *>(a.out + ((int64_t)b * a.hq + head0) * D)[at] = make_float4(o.x * s, o.y * s, o.z * s, o.w * s);
  }
  cluster.sync();  // no CTA's memory goes away while it is read
}

// One tile of this CTA, as warp 0 sees it: lane i owns the tile's i-th copy.
struct TileRef {
  int page, row;      // of this lane's copy; page -1: nothing to load
  bool valid, first;  // first: begins a unit's part
};

template <int TYPE, int D>
__global__ void __launch_bounds__(kCompute, (Tile<TYPE, D>::kPerSm))
    paged_tiles_kernel(const Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = Tile<TYPE, D>;
  constexpr int T = C::T, KS = C::KS, MT = C::MT;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kMaxSlots];
  __shared__ float fix[2][kHeads], sum[kHeads];
  __shared__ float2 share_ml[kHeads];
  __shared__ int abort_flag;
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *sS = reinterpret_cast<float *>(ring + C::kSlots * C::kSlot);       // [2][KS][head][key]
  uint8_t *sP = reinterpret_cast<uint8_t *>(sS + 2 * C::kSFloats);          // [2][part][head][key]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < C::kSlots; ++i) gqd::mbar_init(&full[i], 1);
    gqd::fence_mbar_init();
    abort_flag = 0;
  }
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  Cut cut;
  if (a.cluster) {
    // a unit of few tiles: its cluster's CTAs take neighbouring tiles (the last may get none)
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
    cut.b = unit / a.units_per_req;
    cut.u = unit - cut.b * a.units_per_req;
    cut.keys = visible(a, cut.b);
    const int nt = range_of<T>(a, cut.keys).nt, each = (nt + a.cluster - 1) / a.cluster;
    cut.t = min(rank * each, nt);
    cut.w0 = 0;
    cut.w1 = min(each, nt - cut.t);
    if (tid == 0 && rank == 0 && a.lens[cut.b] > a.room) gqd::report(a.err, GQ_DEVERR_PAGES);
    __syncthreads();  // the mbarriers
  } else {
    cut = find_cut<kCompute, T>(a);  // (its barriers also publish the mbarriers)
  }
  if (!a.cluster && cut.w0 >= cut.w1) {
    if (tid == 0) a.cut_units[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  const int rows_shift = min(a.page_shift, C::kTShift), rows = 1 << rows_shift;  // keys that one copy brings
  const int boxes = T >> rows_shift;

  // ---- loads (warp 0). Order of the ring: the first keys of a part, then for each tile
  // the next tile's keys and its own values. A tile's table entries are read two tiles
  // before its copies are issued.
  int lb = cut.b, lu = cut.u, lt = cut.t;
  int64_t lw = cut.w0;
  Range lr = range_of<T>(a, cut.keys);
  auto advance = [&](bool begin) {
    TileRef x;
    x.valid = false;
    x.first = begin;
    x.page = -1;
    x.row = 0;
    if (!begin) {
      if (lw >= cut.w1) return x;
      ++lw;
      ++lt;
      if (lt == lr.nt) {
        lt = -1;
        if (lw >= cut.w1) return x;
        if (++lu == a.units_per_req) {
          lu = 0;
          lr = range_of<T>(a, visible(a, ++lb));
        }
      }
    }
    if (lt < 0) {  // the place ahead of a unit's tiles
      lt = 0;
      ++lw;
      x.first = true;
    }
    if (lw >= cut.w1) return x;
    x.valid = true;
    const int j = (lr.tile0 + lt) * T + (lane << rows_shift);
    if (lane < boxes && j < lr.hi && j + rows > lr.lo) {
      x.row = ((lu / a.sub) << a.page_shift) + (j & (a.page_size - 1));
      x.page = a.table[lb * a.table_stride + (j >> a.page_shift)];
      if (x.page < 0 || x.page >= a.n_pages) {
        gqd::report(a.err, GQ_DEVERR_PAGES);
        x.page = (int)a.n_pages;  // out of the tensor's bounds: reads as zeros
      }
    }
    return x;
  };
  TileRef cur = {}, nxt = {};
  uint32_t issued = 0;  // ring positions filled
  int stage = 0;        // of the current tile: 0 its keys (if first), 1 the next tile's keys, 2 its values
  auto copy = [&](const TileRef &x, const CUtensorMap *map) {
    const int slot = issued % C::kSlots;
    const int copies = __popc(__ballot_sync(0xffffffffu, x.page >= 0));
    if (lane == 0) gqd::mbar_arrive_expect_tx(&full[slot], (uint32_t)(copies * rows * C::kRow));
    __syncwarp();
    if (x.page >= 0)
      tma_load_4d(ring + slot * C::kSlot + lane * rows * C::kRow, map, 0, x.row, 0, x.page, &full[slot]);
    ++issued;
  };
  auto fill = [&](uint32_t limit) {  // issue what there is, up to ring position `limit`
    while (issued < limit && cur.valid) {
      if (stage == 0) {
        stage = 1;
        if (cur.first) {
          copy(cur, &kmap);
          continue;
        }
      }
      if (stage == 1) {
        stage = 2;
        if (nxt.valid && !nxt.first) {
          copy(nxt, &kmap);
          continue;
        }
      }
      copy(cur, &vmap);
      cur = nxt;
      nxt = advance(false);
      stage = 0;
    }
  };
  // The first fill comes after the first unit's q is requested: the ring holds some 3 us
  // of this SM's share of the bandwidth, and what is asked for later arrives later.
  bool filled = false;
  auto first_fill = [&]() {
    if (filled) return;
    filled = true;
    if (warp == 0) {
      cur = advance(true);
      cur.first = true;
      nxt = advance(false);
      fill(C::kSlots);
    }
  };

  // ---- compute
  const int g = lane >> 2, q4 = lane & 3;  // fragment row / column group
  const int ks = warp % KS, mt = warp / KS * MT;
  const int sh = tid >> 4, sl = tid & 15;  // softmax: head, thread of 16
  constexpr int KPT = T / 16;              // keys per softmax thread
  const uint32_t ring_u = gqd::smem_u32(ring);
  const uint32_t box_bytes = (uint32_t)rows * C::kRow;
  // byte of row `key` of a tile (first 128-byte piece); pieces are rows * 128 bytes apart
  auto row_at = [&](int key) { return (uint32_t)(key >> rows_shift) * box_bytes + (uint32_t)(key & (rows - 1)) * 128u; };
  const uint32_t piece = (uint32_t)rows * 128u;

  uint32_t n = 0;  // ring position of the next tile to read
  int b = cut.b, u = cut.u, t = cut.t, keys = cut.keys;
  for (int64_t w = cut.w0;;) {
    const Range r = range_of<T>(a, keys);
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

    // q fragments of this warp's columns (head g of the unit), in parts
    uint32_t qf[C::kQSteps][C::kParts][2];
    float unscale0 = 1.0f, unscale1 = 1.0f;  // of heads 2 q4 and 2 q4 + 1
    {
      const float *qg = a.q + b * a.q_stride + (int64_t)(head0 + min(g, nh - 1)) * D + ks * (D / KS);
      const bool real = g < nh;
      if constexpr (TYPE == GQ_KV_F32) {
        float v[C::kQSteps][2];
#pragma unroll
        for (int s = 0; s < C::kQSteps; ++s) {
          v[s][0] = real ? qg[s * 8 + q4] : 0.0f;
          v[s][1] = real ? qg[s * 8 + q4 + 4] : 0.0f;
        }
        first_fill();
#pragma unroll
        for (int s = 0; s < C::kQSteps; ++s) {
          split_tf32(v[s][0], qf[s][0][0], qf[s][1][0]);
          split_tf32(v[s][1], qf[s][0][1], qf[s][1][1]);
        }
      } else {
        float2 v[C::kQSteps][2];
#pragma unroll
        for (int s = 0; s < C::kQSteps; ++s) {
          // e4m3: a thread's 4 bytes of a fragment are neighbours, so columns 4 q4 .. 4 q4 + 3
          const int c0 = s * 16 + (TYPE == GQ_KV_E4M3 ? 4 * q4 : 2 * q4), c1 = c0 + (TYPE == GQ_KV_E4M3 ? 2 : 8);
          v[s][0] = real ? *reinterpret_cast<const float2 *>(qg + c0) : make_float2(0.f, 0.f);
          v[s][1] = real ? *reinterpret_cast<const float2 *>(qg + c1) : make_float2(0.f, 0.f);
        }
        first_fill();
        if constexpr (TYPE != GQ_KV_BF16) {
          float top = 0.0f;
#pragma unroll
          for (int s = 0; s < C::kQSteps; ++s)
            top = fmaxf(top, fmaxf(fmaxf(fabsf(v[s][0].x), fabsf(v[s][0].y)), fmaxf(fabsf(v[s][1].x), fabsf(v[s][1].y))));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // 2^e with top * 2^e in [2^13, 2^14); 1 where that has no answer
          const int e = (int)((__float_as_uint(top) >> 23) & 255u);
          const int up = e > 0 && e < 255 ? min(max(140 - e, -126), 126) : 0;
          const float f = __uint_as_float((uint32_t)(127 + up) << 23), inv = __uint_as_float((uint32_t)(127 - up) << 23);
          unscale0 = __shfl_sync(0xffffffffu, inv, q4 * 8);  // lane of head 2 q4: group 2 q4
          unscale1 = __shfl_sync(0xffffffffu, inv, q4 * 8 + 4);
#pragma unroll
          for (int s = 0; s < C::kQSteps; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t part[2];
              split_f16(v[s][i].x * f, v[s][i].y * f, part);
              qf[s][0][i] = part[0];
              qf[s][1][i] = part[1];
            }
        } else {
#pragma unroll
          for (int s = 0; s < C::kQSteps; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t part[3];
              split_bf16(v[s][i].x, v[s][i].y, part);
#pragma unroll
              for (int p = 0; p < 3; ++p) qf[s][p % C::kParts][i] = part[p];
            }
        }
      }
    }
    float acc[C::kMTiles][4];
#pragma unroll
    for (int i = 0; i < C::kMTiles; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[i][k] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    if (tiles > 0) {  // (a cluster's last CTAs may have none)
    // Products of this warp's keys and columns with q. The instruction truncates its sums:
    // the large products (with q's first part) are added up four instructions at a time
    // in 0, and those sums, rounded, in 2; the small ones go to 1.
    float c[MT][3][4];
    auto products = [&]() {
      const int slot = n % C::kSlots;
      if (!wait_or_abort(&full[slot], (n / C::kSlots) & 1, &abort_flag, a.err)) cur.valid = false;
      ++n;
#pragma unroll
      for (int x = 0; x < MT; ++x) {
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
          for (int k = 0; k < 4; ++k) c[x][p][k] = 0.0f;
        // 16-byte pieces s * 2 and s * 2 + 1 of the rows; a piece's place in its 128 bytes is
        // its number xor the row's, so steps of whole bits can be xor-ed on afterwards
        const int krow = (mt + x) * 16 + (lane & 15);
        const uint32_t at = ring_u + slot * C::kSlot + row_at(krow) + (uint32_t)(ks * (C::kChunks / KS)) * piece +
                            (((uint32_t)(lane >> 4) ^ (uint32_t)(krow & 7)) << 4);
#pragma unroll
        for (int s = 0; s < (TYPE == GQ_KV_E4M3 ? C::kQSteps / 2 : C::kQSteps); ++s) {
          uint32_t k4[4];
          ldsm4(k4, (at ^ (uint32_t)((s * 2 & 7) << 4)) + (uint32_t)(s >> 2) * piece);
          if constexpr (TYPE == GQ_KV_F32) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) split_tf32(__uint_as_float(k4[y]), hi[y], lo[y]);
            mma_tf32(c[x][0], hi, qf[s][0][0], qf[s][0][1]);
            mma_tf32(c[x][1], hi, qf[s][1][0], qf[s][1][1]);
            mma_tf32(c[x][1], lo, qf[s][0][0], qf[s][0][1]);
          } else if constexpr (TYPE == GQ_KV_E4M3) {
            const uint32_t a0[4] = {e4m3_pair(k4[0]), e4m3_pair(k4[1]), e4m3_pair(k4[0] >> 16), e4m3_pair(k4[1] >> 16)};
            const uint32_t a1[4] = {e4m3_pair(k4[2]), e4m3_pair(k4[3]), e4m3_pair(k4[2] >> 16), e4m3_pair(k4[3] >> 16)};
            mma_f16(c[x][0], a0, qf[2 * s][0][0], qf[2 * s][0][1]);
            mma_f16(c[x][1], a0, qf[2 * s][1][0], qf[2 * s][1][1]);
            mma_f16(c[x][0], a1, qf[2 * s + 1][0][0], qf[2 * s + 1][0][1]);
            mma_f16(c[x][1], a1, qf[2 * s + 1][1][0], qf[2 * s + 1][1][1]);
          } else if constexpr (TYPE == GQ_KV_F16) {
            mma_f16(c[x][0], k4, qf[s][0][0], qf[s][0][1]);
            mma_f16(c[x][1], k4, qf[s][1][0], qf[s][1][1]);
          } else {
            mma_bf16(c[x][0], k4, qf[s][0][0], qf[s][0][1]);
#pragma unroll
            for (int p = 1; p < C::kParts; ++p) mma_bf16(c[x][1], k4, qf[s][p][0], qf[s][p][1]);
          }
          if (s % (TYPE == GQ_KV_E4M3 ? 2 : 4) == (TYPE == GQ_KV_E4M3 ? 1 : 3))
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              c[x][2][k] += c[x][0][k];
              c[x][0][k] = 0.0f;
            }
        }
      }
    };
    auto put_scores = [&](int buf) {
#pragma unroll
      for (int x = 0; x < MT; ++x) {
        float *to = sS + buf * C::kSFloats + ks * kHeads * C::kSStride + 2 * q4 * C::kSStride + (mt + x) * 16 + g;
        to[0] = (c[x][2][0] + c[x][1][0]) * unscale0;
        to[C::kSStride] = (c[x][2][1] + c[x][1][1]) * unscale1;
        to[8] = (c[x][2][2] + c[x][1][2]) * unscale0;
        to[C::kSStride + 8] = (c[x][2][3] + c[x][1][3]) * unscale1;
      }
    };

    products();
    put_scores(0);
    sync_compute<kCompute>();
    if (warp == 0) {  // every warp is done with what lies before ring position n
      gqd::fence_proxy_async_smem();
      fill(n + C::kSlots);
    }

    for (int i = 0; i < tiles; ++i) {
      const int j0 = (r.tile0 + t + i) * T, buf = i & 1;
      const bool more = i + 1 < tiles;
      if (more) products();  // of tile i + 1

      // ---- weights of tile i
      const bool ragged = j0 < r.lo || j0 + T > r.hi;
      {
        const float *from = sS + buf * C::kSFloats + sh * C::kSStride + sl * KPT;
        float x[KPT], top = -INFINITY;
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
          float s = from[k];
#pragma unroll
          for (int p = 1; p < KS; ++p) s += from[p * kHeads * C::kSStride + k];
          const int j = j0 + sl * KPT + k;
          s = score_of(a, s);
          x[k] = ragged && (j < r.lo || j >= r.hi) ? -INFINITY : s;
          top = fmaxf(top, x[k]);
        }
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float mn = fmaxf(m, top);
        const float base = mn == -INFINITY ? 0.0f : mn;  // (no visible key yet)
        const float f = exp_of(m - base);
        // p = e^(x - m), times 2^14 for the f16 parts (a common factor of every weight and sum)
        constexpr float kUp = TYPE == GQ_KV_F16 || TYPE == GQ_KV_E4M3 ? 16384.0f : 1.0f;
        float p[KPT];
        l *= f;
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
          p[k] = kUp * exp_of(x[k] - base);
          l += p[k];
        }
        m = mn;
        if (sl == 0) fix[buf][sh] = f;
        uint8_t *to = sP + buf * C::kPBytes + sh * C::kPStride;
        if constexpr (TYPE == GQ_KV_F32) {
#pragma unroll
          for (int k = 0; k < KPT; ++k) reinterpret_cast<float *>(to)[sl * KPT + k] = p[k];
        } else {
          static_assert(KPT % 2 == 0 || TYPE == GQ_KV_F32, "pairs of keys");
#pragma unroll
          for (int k = 0; k + 1 < KPT; k += 2) {
            if constexpr (TYPE == GQ_KV_BF16) {
              uint32_t part[3];
              split_bf16(p[k], p[k + 1], part);
#pragma unroll
              for (int y = 0; y < 3; ++y)
                *reinterpret_cast<uint32_t *>(to + y * kHeads * C::kPStride + (sl * KPT + k) * 2) = part[y];
            } else {
              uint32_t part[2];
              split_f16(p[k], p[k + 1], part);
#pragma unroll
              for (int y = 0; y < 2; ++y)
                *reinterpret_cast<uint32_t *>(to + y * kHeads * C::kPStride + (sl * KPT + k) * 2) = part[y];
            }
          }
        }
      }
      if (more) put_scores(buf ^ 1);
      const int vslot = n % C::kSlots;
      if (!wait_or_abort(&full[vslot], (n / C::kSlots) & 1, &abort_flag, a.err)) cur.valid = false;
      const uint32_t vat = ring_u + vslot * C::kSlot;
      if (ragged) {
        // rows that are not visible hold anything, NaN too, or an earlier tile: make them 0
        for (int e = tid; e < T * C::kChunks * 8; e += kCompute) {
          const int key = e / (C::kChunks * 8), ch = e - key * (C::kChunks * 8);
          if (j0 + key >= r.lo && j0 + key < r.hi) continue;
          *reinterpret_cast<uint4 *>(ring + vslot * C::kSlot + row_at(key) + (ch >> 3) * piece + (ch & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        }
        gqd::fence_proxy_async_smem();  // before the slot's next copy
      }
      sync_compute<kCompute>();
      if (warp == 0) {  // every warp is done with what lies before the values of tile i
        gqd::fence_proxy_async_smem();
        fill(n + C::kSlots);
      }
      ++n;

      // ---- output columns warp * D/4 ..: o = o e^(m_old - m) + V^T p. The instruction
      // truncates its sums, so it adds up one tile only; tiles are added in registers.
      {
        const float f0 = fix[buf][2 * q4], f1 = fix[buf][2 * q4 + 1];
        const uint8_t *pg = sP + buf * C::kPBytes + g * C::kPStride;
        constexpr int kSteps = T / C::kStep;
        uint32_t pf[kSteps][C::kParts][2];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          if constexpr (TYPE == GQ_KV_F32) {
            const float2 p = *reinterpret_cast<const float2 *>(pg + (s * 8 + 2 * q4) * 4);
            split_tf32(p.x, pf[s][0][0], pf[s][1][0]);
            split_tf32(p.y, pf[s][0][1], pf[s][1][1]);
          } else {
#pragma unroll
            for (int y = 0; y < C::kParts; ++y) {
              pf[s][y][0] = *reinterpret_cast<const uint32_t *>(pg + y * kHeads * C::kPStride + (s * 16 + 2 * q4) * 2);
              pf[s][y][1] = *reinterpret_cast<const uint32_t *>(pg + y * kHeads * C::kPStride + (s * 16 + 2 * q4 + 8) * 2);
            }
          }
        }
        // columns in groups of G 16-column tiles: their sums are independent, which hides
        // the instruction's latency
        constexpr int G = std::min(C::kMTiles, 4);
#pragma unroll
        for (int x0 = 0; x0 < C::kMTiles; x0 += G) {
          float c[G][4] = {};
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            if constexpr (TYPE == GQ_KV_F32) {
              // the instruction's keys t, t + 4 are rows 2t, 2t + 1: four rows two apart lie on
              // different banks. Columns g and g + 8 of tile x are 16-byte pieces 4x + g/4 and
              // two on of the warp's.
              const int k0 = s * 8 + 2 * q4;
              constexpr int kWarpPieces = D / kComputeWarps / 4;
              const uint32_t wp = (uint32_t)(warp * kWarpPieces), in = (wp >> 3) * piece + (uint32_t)(g & 3) * 4;
              const uint32_t r0 = vat + row_at(k0) + in, r1 = vat + row_at(k0 + 1) + in;
              const uint32_t c0 = (wp & 7) | (uint32_t)(g >> 2), z0 = (uint32_t)(2 * q4), z1 = z0 + 1;
              const uint32_t at[4] = {r0 + ((c0 ^ z0) << 4), r0 + (((c0 ^ 2) ^ z0) << 4), r1 + ((c0 ^ z1) << 4),
                                      r1 + (((c0 ^ 2) ^ z1) << 4)};
#pragma unroll
              for (int x = 0; x < G; ++x) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                  split_tf32(lds32((at[y] ^ (uint32_t)(((x0 + x) & 1) << 6)) + (uint32_t)((x0 + x) >> 1) * piece), hi[y], lo[y]);
                mma_tf32(c[x], lo, pf[s][0][0], pf[s][0][1]);
                mma_tf32(c[x], hi, pf[s][1][0], pf[s][1][1]);
                mma_tf32(c[x], hi, pf[s][0][0], pf[s][0][1]);
              }
            } else if constexpr (TYPE == GQ_KV_E4M3) {
              // two 16-column tiles per load: keys 0-7 and 8-15 of each. A transposed 8 x 8
              // of byte pairs gives columns 2g and 2g + 1 of two keys: row g of the
              // instruction is column 2g, row g + 8 column 2g + 1.
              const int key = s * 16 + (lane & 15);
              constexpr int kWarpPieces = D / kComputeWarps / 16;
              const uint32_t wp = (uint32_t)(warp * kWarpPieces);
              const uint32_t at = vat + row_at(key) + (wp >> 3) * piece + ((((wp & 7) | (uint32_t)(lane >> 4)) ^ (uint32_t)(key & 7)) << 4);
              uint32_t af[G][4];
#pragma unroll
              for (int x = 0; x < G; x += 2) {
                uint32_t v4[4];
                ldsm4_t(v4, at ^ (uint32_t)((x0 + x) << 4));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t e = __byte_perm(v4[2 * h], 0, 0x3120), f = __byte_perm(v4[2 * h + 1], 0, 0x3120);
                  af[x + h][0] = e4m3_pair(e);
                  af[x + h][1] = e4m3_pair(e >> 16);
                  af[x + h][2] = e4m3_pair(f);
                  af[x + h][3] = e4m3_pair(f >> 16);
                }
              }
#pragma unroll
              for (int y = C::kParts - 1; y >= 0; --y)
#pragma unroll
                for (int x = 0; x < G; ++x) mma_f16(c[x], af[x], pf[s][y][0], pf[s][y][1]);
            } else {
              const int key = s * 16 + (lane & 7) + (lane >> 4) * 8;
              constexpr int kWarpPieces = D / kComputeWarps / 8;
              const uint32_t wp = (uint32_t)(warp * kWarpPieces);
              const uint32_t at = vat + row_at(key) + (wp >> 3) * piece + ((((wp & 7) | (uint32_t)((lane >> 3) & 1)) ^ (uint32_t)(key & 7)) << 4);
              uint32_t v4[G][4];
#pragma unroll
              for (int x = 0; x < G; ++x) {
                ldsm4_t(v4[x], (at ^ (uint32_t)(((x0 + x) * 2 & 7) << 4)) + (uint32_t)((x0 + x) >> 2) * piece);
              }
#pragma unroll
              for (int y = C::kParts - 1; y >= 0; --y)
#pragma unroll
                for (int x = 0; x < G; ++x) {
                  if constexpr (TYPE == GQ_KV_BF16) mma_bf16(c[x], v4[x], pf[s][y][0], pf[s][y][1]);
                  else mma_f16(c[x], v4[x], pf[s][y][0], pf[s][y][1]);
                }
            }
          }
#pragma unroll
          for (int x = 0; x < G; ++x) {
            acc[x0 + x][0] = fmaf(acc[x0 + x][0], f0, c[x][0]);
            acc[x0 + x][1] = fmaf(acc[x0 + x][1], f1, c[x][1]);
            acc[x0 + x][2] = fmaf(acc[x0 + x][2], f0, c[x][2]);
            acc[x0 + x][3] = fmaf(acc[x0 + x][3], f1, c[x][3]);
          }
        }
      }
    }

    }

    // ---- the unit's output, or this CTA's part of it
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const bool shared = a.cluster > 1, whole = !shared && tiles == r.nt;
    const int64_t s0 = w - t;
    const int slot = whole || shared ? 0 : slot_of(cut, s0);
    if (sl == 0) {
      sum[sh] = l;
      if (shared) {
        share_ml[sh] = make_float2(m, l);
      } else if (!whole) {
        a.part_ml[(slot * kHeads + sh) * 2] = m;
        a.part_ml[(slot * kHeads + sh) * 2 + 1] = l;
      }
    }
    sync_compute<kCompute>();
    {
      // (the ring's tiles are read: a cluster's part takes its place)
      float *base = shared  ? reinterpret_cast<float *>(ring)
                    : whole ? a.out + ((int64_t)b * a.hq + head0) * D
                            : a.part_o + (int64_t)slot * kHeads * D;
      const float f0 = whole ? inv_or_zero(sum[2 * q4]) * a.v_scale : 1.0f;
      const float f1 = whole ? inv_or_zero(sum[2 * q4 + 1]) * a.v_scale : 1.0f;
      const int most = whole ? nh : kHeads;
#pragma unroll
      for (int x = 0; x < C::kMTiles; ++x) {
        const int col = warp * (D / kComputeWarps) + x * 16;
        const int ca = TYPE == GQ_KV_E4M3 ? col + 2 * g : col + g, cb = TYPE == GQ_KV_E4M3 ? ca + 1 : ca + 8;
        if (2 * q4 < most) {
          base[(2 * q4) * D + ca] = acc[x][0] * f0;
          base[(2 * q4) * D + cb] = acc[x][2] * f0;
        }
        if (2 * q4 + 1 < most) {
          base[(2 * q4 + 1) * D + ca] = acc[x][1] * f1;
          base[(2 * q4 + 1) * D + cb] = acc[x][3] * f1;
        }
      }
    }
    if (shared) {
      join_cluster<D>(a, reinterpret_cast<const float *>(ring), share_ml, b, head0, nh);
      break;
    }
    if (a.cluster) break;
    w += tiles;
    if (w == cut.w1) {
      if (tid == 0) put_cut_unit(a, cut, b, u, s0, r.nt);
      break;
    }
    t = -1;
    if (++u == a.units_per_req) {
      u = 0;
      keys = visible(a, ++b);
    }
  }
  if (warp == 0 && lane == 0 && *(volatile int *)&abort_flag)
    // copies still in flight end before the CTA's memory goes away
    for (uint32_t i = issued > C::kSlots ? issued - C::kSlots : 0; i < issued; ++i)
      (void)gqd::mbar_wait_bounded(&full[i % C::kSlots], (i / C::kSlots) & 1, 100000000ull);
}

int log2_of(int64_t v) {
  int s = 0;
  while ((int64_t(1) << s) < v) ++s;
  return s;
}

// A layer's pages as a 4-D tensor: 128-byte pieces of a row, rows of all heads of a
// page, pieces of a row, pages. One copy brings `rows` rows whole, laid out piece by
// piece with the 128-byte swizzle.
int encode(gq_ctx *ctx, const gq_kv_pages *p, const void *base, int64_t page_stride, int rows, CUtensorMap *map) {
  auto fn = gq_encode_fn();
  if (!fn) return gq_fail(ctx, GQ_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled is not available");
  const int size = gq_kv_size(p->type);
  const int64_t row = p->head_dim * size;
  const cuuint64_t dims[4] = {(cuuint64_t)(128 / size), (cuuint64_t)(p->heads * p->page_size), (cuuint64_t)(row / 128),
                              (cuuint64_t)p->n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)row, 128, (cuuint64_t)(page_stride * size)};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / size), (cuuint32_t)rows, (cuuint32_t)(row / 128), 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = size == 4   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : size == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                               : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUresult e = fn(map, type, 4, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e != CUDA_SUCCESS) return gq_fail(ctx, GQ_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed");
  return GQ_OK;
}

template <int TYPE, int D>
int launch(gq_ctx *ctx, const gq_kv_pages *p, Args &a) {
  using C = Tile<TYPE, D>;
  static bool attr_set[64] = {};
  if (!attr_set[ctx->device & 63]) {
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(paged_tiles_kernel<TYPE, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    attr_set[ctx->device & 63] = true;
  }
  a.page_shift = log2_of(p->page_size);
  CUtensorMap kmap, vmap;
  const int rows = (int)std::min<int64_t>(p->page_size, C::T);
  int rc = encode(ctx, p, p->k, a.page_stride, rows, &kmap);
  if (rc == GQ_OK) rc = encode(ctx, p, p->v, a.page_stride, rows, &vmap);
  if (rc != GQ_OK) return rc;
  // Units that cannot have many tiles (a sliding window, a short table) get a cluster of
  // CTAs each, as large as fills the GPU: no cut to work out, and a join in shared memory
  // (some 4 us less, the time of two tiles). What it can cost is uneven work: tiles beyond
  // an equal share, and lengths that differ (a window evens them out). The bounds below come
  // from head_dim 256 in bf16 (tiles of 64 keys), cluster against cut, us: window 512 and 1,
  // 8, 64, 200, 500 requests 6.9 / 9.6, 9.2 / 12.4, 13.2 / 17.2, 28.4 / 34.5, 56 / 60; up to
  // 1024 keys and 1, 16, 64 requests 8.7 / 10.0, 9.4 / 12.8, 15.3 / 17.6; up to 2048 keys
  // 13.1 / 10.0, 13.7 / 13.0, 26.5 / 24.1. (150 requests with the window, where a cluster is
  // one CTA and half the GPU is idle: 27.5 / 27.0.) Elsewhere, where they choose clusters:
  // 225 requests of up to 62 keys, 8 heads of 64, bf16 24.7 / 26.8; 256 of up to 60, 4 heads
  // of 128 16.1 / 19.1; 200 of up to 200, 8 heads of 128 35.1 / 37.1; 53 of one key, 8 heads
  // of 512, f16 11.1 / 14.3; 100 of up to 300, 8 heads of 64, f32 29.3 / 29.0, of 128, e4m3
  // 21.2 / 23.8; 39 of up to 2017, one head of 64, f32 13.8 / 14.7; 64 of up to 1024,
  // head_dim 256, e4m3 14.7 / 16.6; 256 of up to 100, head_dim 256, bf16 9.5 / 17.3.
  const int64_t units = (int64_t)a.batch * a.units_per_req, tiles = most_tiles(a, C::T);
  const int slots = C::kPerSm * ctx->num_sms;
  int cluster = 8;
  while (cluster > 1 && (units * cluster > slots || cluster >= 2 * tiles)) cluster >>= 1;
  const int64_t each = (tiles + cluster - 1) / cluster;
  const int64_t equal = (units * tiles + slots - 1) / slots;
  const bool even = a.window > 0;
  if (each <= (even ? 9 : 4) && each <= equal + (even ? 2 : 1) && units * cluster <= INT32_MAX) {
    a.cluster = cluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * cluster));
    cfg.blockDim = dim3(kCompute);
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
    GQ_CUDA_TRY(ctx, cudaLaunchKernelEx(&cfg, paged_tiles_kernel<TYPE, D>, (const Args)a, (const CUtensorMap)kmap, (const CUtensorMap)vmap));
    return GQ_OK;
  }
  const int grid = grid_for(a, C::T, slots);
  rc = bind_parts(ctx, grid, a);
  if (rc != GQ_OK) return rc;
  GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_tiles_kernel<TYPE, D>, dim3(grid), dim3(kCompute), C::kSmem, a, kmap, vmap));
  return gq_paged_join_launch(ctx, a, grid);
}

template <int TYPE>
int launch_dim(gq_ctx *ctx, const gq_kv_pages *p, Args &a) {
  switch (p->head_dim) {
    case 64:
      if constexpr (TYPE != GQ_KV_E4M3) return launch<TYPE, 64>(ctx, p, a);
      break;
    case 128: return launch<TYPE, 128>(ctx, p, a);
    case 256: return launch<TYPE, 256>(ctx, p, a);
    case 512: return launch<TYPE, 512>(ctx, p, a);
  }
  return gq_fail(ctx, GQ_ERR_UNSUPPORTED, "paged_attention: no tiled kernel");
}

}  // namespace

// Rows of whole 128-byte pieces at the instantiated head_dims, and pages that a tile is
// a whole number of (or that are a whole number of tiles).
bool gq_paged_attn_tc_supported(const gq_kv_pages *p, int64_t page_stride) {
  const int size = gq_kv_size(p->type);
  const int64_t d = p->head_dim;
  return (d == 64 || d == 128 || d == 256 || d == 512) && d * size % 128 == 0 && p->page_size >= 8 &&
         (p->page_size & (p->page_size - 1)) == 0 && page_stride * size % 16 == 0 &&
         page_stride < (int64_t(1) << 36) && p->heads * p->page_size <= INT32_MAX && p->n_pages > 0;
}

int gq_paged_attn_tc_launch(gq_ctx *ctx, const gq_kv_pages *p, Args &a) {
  switch (p->type) {
    case GQ_KV_F32: return launch_dim<GQ_KV_F32>(ctx, p, a);
    case GQ_KV_F16: return launch_dim<GQ_KV_F16>(ctx, p, a);
    case GQ_KV_BF16: return launch_dim<GQ_KV_BF16>(ctx, p, a);
    default: return launch_dim<GQ_KV_E4M3>(ctx, p, a);
  }
}
