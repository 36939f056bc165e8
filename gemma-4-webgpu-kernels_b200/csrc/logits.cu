// logits.cu — penalties for repeated tokens, biases and grammar masks on a step's
// logits (gq_process_logits), one pass over the rows.
//
// What bounds it: 8 bytes per logit (read and written once); the histories, biases
// and mask bits are small beside that. The counts of a row's earlier tokens are made
// where they are needed, in shared memory: a cluster of kCluster CTAs owns
// kCluster * kCols neighbouring columns of a row, its CTAs share the scan of the
// row's history, each adding a token to the counter of the CTA that owns its column
// (distributed shared memory). A row's history is so read once per cluster instead of
// once per CTA, and no count table goes through memory. Counts are whole numbers, so
// the order of the atomic additions changes nothing.
#include <cooperative_groups.h>

#include <algorithm>

#include "gq_internal.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256;
constexpr int kVecs = 8;                        // float4 per thread
constexpr int kCols = kThreads * kVecs * 4;     // columns per CTA
constexpr int kCluster = 8;
constexpr uint32_t kSeen = 0x80000000u;         // the token is in the prompt; below: times generated

struct LogitArgs {
  const float *x;
  float *y;
  int64_t vocab, ld, ldy;
  const int32_t *tokens, *prompt_lens, *lens;
  int64_t tok_stride;
  const float *penalties;
  const int32_t *bias_ids, *bias_offsets;
  const float *bias_values;
  const uint32_t *masks;
  const int32_t *mask_rows;
  int64_t n_masks, mask_stride;
};

__device__ __forceinline__ float penalised(float l, uint32_t w, float rep, float presence, float frequency) {
  if (w == 0) return l;
  l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
  const uint32_t n = w & ~kSeen;
  if (n) l = __fsub_rn(__fsub_rn(l, __fmul_rn(frequency, (float)n)), presence);
  return l;
}

// Bits of columns c .. c + 3 of a mask (only columns inside [0, vocab) are looked up).
__device__ __forceinline__ uint32_t mask_bits4(const uint32_t *mask, int64_t c, int64_t vocab) {
  if (!mask) return 15u;
  const int64_t c0 = c < 0 ? 0 : c, c1 = min(c + 3, vocab - 1);
  const int64_t w0 = c0 >> 5, w1 = c1 >> 5;
  const uint64_t both = (uint64_t)mask[w0] | ((uint64_t)(w1 != w0 ? mask[w1] : 0u) << 32);
  const uint32_t bits = (uint32_t)(both >> (c0 & 31));
  return c < 0 ? bits << (uint32_t)(-c) : bits;
}

// Grid: x = pieces of a row (a whole number of clusters), y = rows. Columns are
// numbered from the 16-byte boundary at or before the row's first logit, so that
// rows of any stride are read in whole 16-byte pieces; `lead` columns are before the row.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) __cluster_dims__(kCluster, 1, 1) logits_kernel(const LogitArgs a) {
  __shared__ __align__(16) uint32_t words[kCols];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  const float *x = a.x + row * a.ld;
  float *y = a.y + row * a.ldy;
  const int lead = VEC ? (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3u) : 0;
  const int64_t col0 = (int64_t)blockIdx.x * kCols - lead;  // column of words[0]
  for (int i = tid; i < kCols / 4; i += kThreads) reinterpret_cast<uint4 *>(words)[i] = make_uint4(0, 0, 0, 0);
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();

  // the logits are requested first: the counting below runs while they arrive
  float4 v[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int64_t c = col0 + (int64_t)(j * kThreads + tid) * 4;
    v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC && c >= 0 && c + 3 < a.vocab) {
      v[j] = *reinterpret_cast<const float4 *>(x + c);
    } else {
      if (c >= 0 && c < a.vocab) v[j].x = x[c];
      if (c + 1 >= 0 && c + 1 < a.vocab) v[j].y = x[c + 1];
      if (c + 2 >= 0 && c + 2 < a.vocab) v[j].z = x[c + 2];
      if (c + 3 >= 0 && c + 3 < a.vocab) v[j].w = x[c + 3];
    }
  }

  float rep = 1.0f, presence = 0.0f, frequency = 0.0f;
  if (a.tokens) {
    rep = a.penalties[row * 3];
    presence = a.penalties[row * 3 + 1];
    frequency = a.penalties[row * 3 + 2];
    const int64_t len = min((int64_t)a.lens[row], a.tok_stride);
    const int64_t prompt = a.prompt_lens[row];
    const int rank = (int)cluster.block_rank();
    const int64_t first = col0 - (int64_t)rank * kCols;  // of the cluster
    const int32_t *tok = a.tokens + row * a.tok_stride;
    cluster.sync();  // every CTA's counters are zero
    for (int64_t i = rank * kThreads + tid; i < len; i += kCluster * kThreads) {
      const int32_t t = tok[i];
      const int64_t at = t - first;
      if (t < 0 || t >= a.vocab || at < 0 || at >= (int64_t)kCluster * kCols) continue;
      uint32_t *w = cluster.map_shared_rank(words, (unsigned)(at / kCols)) + at % kCols;
      if (i < prompt) atomicOr(w, kSeen);
      else atomicAdd(w, 1u);
    }
    cluster.sync();  // every count has arrived, and no CTA leaves before the others' additions
  }

  const uint32_t *mask = nullptr;
  if (a.masks) {
    const int64_t mr = a.mask_rows ? (int64_t)a.mask_rows[row] : row;
    if (mr >= 0 && mr < a.n_masks) mask = a.masks + mr * a.mask_stride;
  }
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int at = (j * kThreads + tid) * 4;
    const int64_t c = col0 + at;
    if (c + 3 < 0 || c >= a.vocab) continue;
    const uint4 w = *reinterpret_cast<const uint4 *>(words + at);
    if (w.x | w.y | w.z | w.w) {
      v[j].x = penalised(v[j].x, w.x, rep, presence, frequency);
      v[j].y = penalised(v[j].y, w.y, rep, presence, frequency);
      v[j].z = penalised(v[j].z, w.z, rep, presence, frequency);
      v[j].w = penalised(v[j].w, w.w, rep, presence, frequency);
    }
    const uint32_t bits = mask_bits4(mask, c, a.vocab);
    if (!(bits & 1u)) v[j].x = -INFINITY;
    if (!(bits & 2u)) v[j].y = -INFINITY;
    if (!(bits & 4u)) v[j].z = -INFINITY;
    if (!(bits & 8u)) v[j].w = -INFINITY;
    if (VEC && c >= 0 && c + 3 < a.vocab) {
      *reinterpret_cast<float4 *>(y + c) = v[j];
    } else {
      if (c >= 0 && c < a.vocab) y[c] = v[j].x;
      if (c + 1 >= 0 && c + 1 < a.vocab) y[c + 1] = v[j].y;
      if (c + 2 >= 0 && c + 2 < a.vocab) y[c + 2] = v[j].z;
      if (c + 3 >= 0 && c + 3 < a.vocab) y[c + 3] = v[j].w;
    }
  }

  if (a.bias_offsets) {
    // words now says which entry of the row's list owns a column: the last one
    const int64_t b0 = a.bias_offsets[row], b1 = a.bias_offsets[row + 1];
    if (b0 >= b1) return;
    const int64_t lo = max(col0, (int64_t)0), hi = min(col0 + kCols, a.vocab);
    __syncthreads();
    for (int64_t i = b0 + tid; i < b1; i += kThreads) {
      const int32_t id = a.bias_ids[i];
      if (id >= lo && id < hi) words[id - col0] = 0;
    }
    __syncthreads();
    for (int64_t i = b0 + tid; i < b1; i += kThreads) {
      const int32_t id = a.bias_ids[i];
      if (id >= lo && id < hi) atomicMax(&words[id - col0], (uint32_t)(i - b0 + 1));
    }
    __syncthreads();
    for (int64_t i = b0 + tid; i < b1; i += kThreads) {
      const int32_t id = a.bias_ids[i];
      if (id < lo || id >= hi || words[id - col0] != (uint32_t)(i - b0 + 1)) continue;
      // a masked column stays -inf whatever its bias (-inf + inf would be NaN)
      if (mask && !((mask[id >> 5] >> (id & 31)) & 1u)) continue;
      y[id] = __fadd_rn(y[id], a.bias_values[i]);
    }
  }
}

}  // namespace

extern "C" int gq_process_logits(gq_ctx *ctx, const float *logits, int64_t m, int64_t vocab, int64_t ld,
                                 const int32_t *tokens, int64_t tok_stride, const int32_t *prompt_lens,
                                 const int32_t *lens, const float *penalties, const int32_t *bias_ids,
                                 const float *bias_values, const int32_t *bias_offsets, const uint32_t *masks,
                                 int64_t n_masks, int64_t mask_stride, const int32_t *mask_rows, float *y, int64_t ldy) {
  if (!ctx) return GQ_ERR_INVALID_ARGUMENT;
  int rc = gq_enter_ctx(ctx);
  if (rc != GQ_OK) return rc;
  if (ld == 0) ld = vocab;
  if (ldy == 0) ldy = vocab;
  if (m < 0 || vocab < 0 || ld < vocab || ldy < vocab)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "process_logits: negative size, or a row stride below vocab");
  if (vocab >= (1 << 28) || m > 65535)
    return gq_fail(ctx, GQ_ERR_UNSUPPORTED, "process_logits: vocab must be below 2^28 and m at most 65535");
  if (m == 0 || vocab == 0) return GQ_OK;
  if (!logits || !y) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "process_logits: null logits or output");
  if (tokens && (!prompt_lens || !lens || !penalties || tok_stride < 0))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "process_logits: tokens need prompt_lens, lens, penalties and a stride");
  if (bias_offsets && (!bias_ids || !bias_values))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "process_logits: bias_offsets need bias_ids and bias_values");
  if (masks && (n_masks < 0 || mask_stride < (vocab + 31) / 32 || (!mask_rows && n_masks < m)))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT,
                   "process_logits: a mask row holds ceil(vocab / 32) words, and without mask_rows every row needs one");
  if (y == logits && ldy != ld)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "process_logits: in place, the row strides must be equal");
  LogitArgs a{};
  a.x = logits;
  a.y = y;
  a.vocab = vocab;
  a.ld = ld;
  a.ldy = ldy;
  a.tokens = tokens;
  a.tok_stride = tok_stride;
  a.prompt_lens = prompt_lens;
  a.lens = lens;
  a.penalties = penalties;
  a.bias_ids = bias_ids;
  a.bias_values = bias_values;
  a.bias_offsets = bias_offsets;
  a.masks = masks;
  a.n_masks = n_masks;
  a.mask_stride = mask_stride;
  a.mask_rows = mask_rows;
  // 16-byte pieces need input and output rows on the same phase of a 16-byte boundary
  const bool vec = ((uintptr_t)logits - (uintptr_t)y) % 16 == 0 && (m == 1 || (ld - ldy) % 4 == 0);
  const int64_t pieces = (vocab + 3 + kCols - 1) / kCols;
  const dim3 grid((unsigned)((pieces + kCluster - 1) / kCluster * kCluster), (unsigned)m);
  GQ_CUDA_TRY(ctx, vec ? gq_launch(ctx, logits_kernel<true>, grid, dim3(kThreads), 0, a)
                       : gq_launch(ctx, logits_kernel<false>, grid, dim3(kThreads), 0, a));
  return GQ_OK;
}
