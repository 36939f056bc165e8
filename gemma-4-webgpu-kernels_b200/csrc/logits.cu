// logits.cu — penalties for repeated tokens, biases and grammar masks on a step's
// logits (gq_process_logits), one pass over the rows.
//
// What it has to move: 8 bytes per logit (read and written once). The histories, biases and
// mask bits are small beside that, but what bounds it is the latency of what they cost: the
// look at each earlier token by each CTA of the row, and chains of dependent loads. So a
// CTA owns many columns (16384): it copies them masked, which waits for nothing, while it
// marks and counts the tokens of its columns in shared memory (whole numbers: the order
// of the atomic operations changes nothing), and then rewrites the few columns that a
// penalty or a bias changes, one thread each, from a list.
// Measured on 64 rows of 262144, histories up to 8192, 300 biases a row: penalties
// applied where all columns are written, 47-67 us (their divisions run in nearly every
// warp for a lane or two, and the logits wait in registers for the counts); a cluster of
// 4 or 8 CTAs sharing the scan of the history, 38-53 us (cluster scheduling and barriers);
// this way 34.8 us (floor 20.8; 23.4 without history, biases and masks).
#include <algorithm>

#include "gq_internal.cuh"

namespace {

constexpr uint32_t kOwner = 0x80000000u;  // a word that holds a bias entry, not a count (below 2^30, as tok_stride)
constexpr int kListed = 2048;  // columns of a CTA's list; past that it looks at every column

struct LogitArgs {
  const float *x;
  float *y;
  int64_t vocab, ld, ldy;
  const int32_t *tokens, *prompt_lens, *lens;
  int64_t tok_stride;
  const float *penalties;
  const int32_t *bias_ids, *bias_offsets;
  const float *bias_values;
  int n_bias;  // entries of bias_ids, where the call is told (COUNTED)
  const uint32_t *masks;
  const int32_t *mask_rows;
  int64_t n_masks, mask_stride;
};

// A logit whose token was seen, n times among the generated ones.
__device__ __forceinline__ float penalised(float l, uint32_t n, float rep, float presence, float frequency) {
  l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
  if (n) l = __fsub_rn(__fsub_rn(l, __fmul_rn(frequency, (float)n)), presence);
  return l;
}

// Bits of columns c .. c + 3 of a mask (only columns inside [0, vocab) are looked up).
__device__ __forceinline__ uint32_t mask_bits4(const uint32_t *mask, int c, int vocab) {
  const int c0 = max(c, 0), c1 = min(c + 3, vocab - 1);
  const int w0 = c0 >> 5, w1 = c1 >> 5;
  const uint64_t both = (uint64_t)mask[w0] | ((uint64_t)(w1 != w0 ? mask[w1] : 0u) << 32);
  const uint32_t bits = (uint32_t)(both >> (c0 & 31));
  return c < 0 ? bits << (uint32_t)(-c) : bits;
}

// A masked column is -inf whatever it was (a NaN, or -inf + inf, too).
__device__ __forceinline__ void mask4(float4 &v, uint32_t bits) {
  if (!(bits & 1u)) v.x = -INFINITY;
  if (!(bits & 2u)) v.y = -INFINITY;
  if (!(bits & 4u)) v.z = -INFINITY;
  if (!(bits & 8u)) v.w = -INFINITY;
}

// Grid: x = chunks of a row, y = rows; NT threads of V pieces of 4 columns. Columns are
// counted from the 16-byte boundary at or before the row's first logit, so that rows of
// any stride are read in whole 16-byte pieces; `lead` columns lie before the row.
// COUNTED: the number of bias entries is an argument, not the last offset (which costs a
// branch and a load: 64 rows 34.6 / 34.8 us; without any bound 34.2).
template <int NT, int V, bool VEC, bool COUNTED>
__global__ void __launch_bounds__(NT, 1024 / NT) logits_kernel(const LogitArgs a) {
  constexpr int kCols = NT * V * 4, kLoads = V < 4 ? V : 4, kTokens = 4;
  static_assert(V % kLoads == 0 && kCols <= 65536, "whole batches, 16-bit columns");
  static_assert(NT * 4 % 32 == 0, "a thread's pieces lie at the same place of a mask word");
  extern __shared__ __align__(16) uint32_t words[];  // [kCols] counts, later owners of biases
  __shared__ uint32_t seen[kCols / 32];              // bit: the column's token was seen
  __shared__ uint16_t listed[kListed];               // the first kListed of them
  __shared__ int n_seen;
  const int tid = threadIdx.x, vocab = (int)a.vocab;
  const int64_t row = blockIdx.y;
  const float *x = a.x + row * a.ld;
  float *y = a.y + row * a.ldy;
  const int lead = VEC ? (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3u) : 0;
  const int col0 = (int)blockIdx.x * kCols - lead;  // column of words[0]
  const int lo = max(col0, 0), span = max(min(col0 + kCols, vocab) - lo, 0);
  // (ids below lo, negative ones too, wrap past span: lo + span < 2^28)
  auto here = [&](int id) { return (uint32_t)id - (uint32_t)lo < (uint32_t)span; };
  if (a.tokens || a.bias_offsets) {
#pragma unroll
    for (int i = 0; i < V; ++i) reinterpret_cast<uint4 *>(words)[i * NT + tid] = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < kCols / 32; i += NT) seen[i] = 0;
    if (tid == 0) n_seen = 0;
  }
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();

  // every chain of dependent loads begins here
  int len = 0, prompt = 0, b0 = 0, biases = 0;
  float rep = 1.0f, presence = 0.0f, frequency = 0.0f;
  const uint32_t *mask = nullptr;
  if (a.tokens) {
    len = a.lens[row];
    prompt = a.prompt_lens[row];
    rep = a.penalties[row * 3];
    presence = a.penalties[row * 3 + 1];
    frequency = a.penalties[row * 3 + 2];
  }
  if (a.bias_offsets) {
    // (offsets are cut to the entries there are: nothing past bias_ids is read)
    const int entries = COUNTED ? a.n_bias : min(max(a.bias_offsets[gridDim.y], 0), INT32_MAX / 2);
    b0 = min(max(a.bias_offsets[row], 0), entries);
    biases = min(max(a.bias_offsets[row + 1], 0), entries) - b0;
  }
  if (a.masks) {
    const int64_t mr = a.mask_rows ? (int64_t)a.mask_rows[row] : row;
    if (mr >= 0 && mr < a.n_masks) mask = a.masks + mr * a.mask_stride;
  }
  const bool inside = VEC && col0 >= 0 && col0 + kCols <= vocab;  // every piece is whole
  const int c0 = col0 + tid * 4;
  float4 v[kLoads];
  uint32_t bits[kLoads];
  const uint32_t *mask0 = mask + (c0 >> 5);  // (read only where columns are inside the row)
  auto fetch = [&](int j0) {  // pieces j0 .. of this thread, and their mask bits
    if (inside) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) v[j] = *reinterpret_cast<const float4 *>(x + c0 + (j0 + j) * NT * 4);
      if (mask && lead == 0)  // a piece's bits lie in one word, at the same place for all of a thread's pieces
#pragma unroll
        for (int j = 0; j < kLoads; ++j) bits[j] = mask0[(j0 + j) * (NT / 8)] >> (c0 & 31);
      else if (mask)
#pragma unroll
        for (int j = 0; j < kLoads; ++j) bits[j] = mask_bits4(mask, c0 + (j0 + j) * NT * 4, vocab);
    } else {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int c = c0 + (j0 + j) * NT * 4;
        v[j].x = c >= 0 && c < vocab ? x[c] : 0.0f;
        v[j].y = c + 1 >= 0 && c + 1 < vocab ? x[c + 1] : 0.0f;
        v[j].z = c + 2 >= 0 && c + 2 < vocab ? x[c + 2] : 0.0f;
        v[j].w = c + 3 >= 0 && c + 3 < vocab ? x[c + 3] : 0.0f;
        bits[j] = !mask || c + 3 < 0 || c >= vocab ? 15u : mask_bits4(mask, c, vocab);
      }
    }
  };
  auto put = [&](int j0) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int c = c0 + (j0 + j) * NT * 4;
      if (mask) mask4(v[j], bits[j]);
      if (inside) {
        *reinterpret_cast<float4 *>(y + c) = v[j];
      } else {
        if (c >= 0 && c < vocab) y[c] = v[j].x;
        if (c + 1 >= 0 && c + 1 < vocab) y[c + 1] = v[j].y;
        if (c + 2 >= 0 && c + 2 < vocab) y[c + 2] = v[j].z;
        if (c + 3 >= 0 && c + 3 < vocab) y[c + 3] = v[j].w;
      }
    }
  };
  // the first logits are requested, then the history is counted while they arrive
  fetch(0);
  const int32_t *ids = a.bias_ids + b0;
  const int id0 = tid < biases ? ids[tid] : -1;  // this thread's first entry
  if (a.tokens) {
    len = (int)min((int64_t)len, a.tok_stride);
    const int32_t *tok = a.tokens + row * a.tok_stride;
    __syncthreads();  // the counters are zero
    for (int i = tid; i < len; i += NT * kTokens) {
      uint32_t t[kTokens];  // column in the chunk's part of the row
#pragma unroll
      for (int k = 0; k < kTokens; ++k) t[k] = i + k * NT < len ? (uint32_t)tok[i + k * NT] - (uint32_t)lo : ~0u;
#pragma unroll
      for (int k = 0; k < kTokens; ++k) {
        if (t[k] >= (uint32_t)span) continue;
        const int at = (int)t[k] + lo - col0;
        atomicOr(&seen[at >> 5], 1u << (at & 31));
        if (i + k * NT >= prompt) atomicAdd(&words[at], 1u);
      }
    }
  }
#pragma unroll
  for (int j0 = 0; j0 < V; j0 += kLoads) {
    put(j0);
    if (j0 + kLoads < V) fetch(j0 + kLoads);
  }

  if (a.tokens) {
    __syncthreads();  // counts are made, columns are written
    for (int i = tid; i < kCols / 32; i += NT) {
      uint32_t set = seen[i];
      if (!set) continue;
      int p = atomicAdd(&n_seen, __popc(set));
      for (; set; set &= set - 1, ++p)
        if (p < kListed) listed[p] = (uint16_t)(i * 32 + __ffs(set) - 1);
    }
    __syncthreads();
    const int n = n_seen;
    auto rewrite = [&](int at) {
      // (in place x[c] is what was just written: itself, unless it is masked)
      const int c = col0 + at;
      if (!mask || ((mask[c >> 5] >> (c & 31)) & 1u)) y[c] = penalised(x[c], words[at], rep, presence, frequency);
    };
    if (n <= kListed) {
      for (int i = tid; i < n; i += NT) rewrite(listed[i]);
    } else {  // more than the list holds: look at every column
      for (int at = tid; at < kCols; at += NT)
        if ((seen[at >> 5] >> (at & 31)) & 1u) rewrite(at);
    }
  }
  if (biases > 0) {
    // words now says which entry of the row's list owns a column: the last one
    auto each = [&](auto f) {
      if (here(id0)) f(tid, id0);
      for (int i = tid + NT; i < biases; i += NT) {
        const int id = ids[i];
        if (here(id)) f(i, id);
      }
    };
    __syncthreads();  // counts are read, y is written
    each([&](int i, int id) { atomicMax(&words[id - col0], kOwner + (uint32_t)i); });
    __syncthreads();
    each([&](int i, int id) {
      // a masked column stays -inf whatever its bias (-inf + inf would be NaN)
      if (words[id - col0] == kOwner + (uint32_t)i && (!mask || ((mask[id >> 5] >> (id & 31)) & 1u)))
        y[id] = __fadd_rn(y[id], a.bias_values[b0 + i]);
    });
  }
}

template <int NT, int V, bool VEC, bool COUNTED>
int logits_launch(gq_ctx *ctx, const LogitArgs &a, int64_t m, int64_t most_lead) {
  constexpr int kCols = NT * V * 4;
  static bool attr_set[64] = {};
  if (kCols * 4 > 32768 && !attr_set[ctx->device & 63]) {
    GQ_CUDA_TRY(ctx, cudaFuncSetAttribute(logits_kernel<NT, V, VEC, COUNTED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCols * 4));
    attr_set[ctx->device & 63] = true;
  }
  const dim3 grid((unsigned)((a.vocab + most_lead + kCols - 1) / kCols), (unsigned)m);
  GQ_CUDA_TRY(ctx, gq_launch(ctx, logits_kernel<NT, V, VEC, COUNTED>, grid, dim3(NT), kCols * 4, a));
  return GQ_OK;
}

template <bool VEC, bool COUNTED>
int logits_dispatch(gq_ctx *ctx, const LogitArgs &a, int64_t m, int64_t most_lead) {
  // Chunks of 2048 columns while chunks of 4096 would not give every SM one (rows of 262144:
  // up to 2): more SMs take part, but each looks at its rows' whole histories. 2048 against
  // 16384, us replayed, 300 biases, histories up to 900: 1 row 3.4 / 4.8, 2 3.6 / 4.8, 3
  // 3.9 / 5.0, 4 4.0 / 4.8, 8 6.9 / 5.3, 16 13.9 / 9.0, 64 47.2 / 29.0; up to 8192: 5.9 / 6.5,
  // 6.2 / 6.5, 6.3 / 6.5, 6.6 / 6.5, 10.6 / 6.7, 20.7 / 10.6, 77.2 / 33.9.
  if (m * ((a.vocab + 4095) / 4096) < ctx->num_sms) return logits_launch<256, 2, VEC, COUNTED>(ctx, a, m, most_lead);
  return logits_launch<512, 8, VEC, COUNTED>(ctx, a, m, most_lead);
}

int process_logits(gq_ctx *ctx, const float *logits, int64_t m, int64_t vocab, int64_t ld, const int32_t *tokens,
                   int64_t tok_stride, const int32_t *prompt_lens, const int32_t *lens, const float *penalties,
                   const int32_t *bias_ids, const float *bias_values, const int32_t *bias_offsets, int64_t n_bias,
                   const uint32_t *masks, int64_t n_masks, int64_t mask_stride, const int32_t *mask_rows, float *y,
                   int64_t ldy) {
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
  if (tokens && (!prompt_lens || !lens || !penalties || tok_stride < 0 || tok_stride > INT32_MAX / 2))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "process_logits: tokens need prompt_lens, lens, penalties and a stride below 2^30");
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
  a.n_bias = (int)n_bias;
  a.bias_offsets = bias_offsets;
  a.masks = masks;
  a.n_masks = n_masks;
  a.mask_stride = mask_stride;
  a.mask_rows = mask_rows;
  // 16-byte pieces need input and output rows on the same phase of a 16-byte boundary
  const bool vec = ((uintptr_t)logits - (uintptr_t)y) % 16 == 0 && (m == 1 || (ld - ldy) % 4 == 0);
  const int64_t most_lead = (uintptr_t)logits % 16 == 0 && (m == 1 || ld % 4 == 0) ? 0 : 3;
  if (n_bias >= 0) return vec ? logits_dispatch<true, true>(ctx, a, m, most_lead) : logits_dispatch<false, true>(ctx, a, m, 0);
  return vec ? logits_dispatch<true, false>(ctx, a, m, most_lead) : logits_dispatch<false, false>(ctx, a, m, 0);
}

}  // namespace

extern "C" int gq_process_logits(gq_ctx *ctx, const float *logits, int64_t m, int64_t vocab, int64_t ld,
                                 const int32_t *tokens, int64_t tok_stride, const int32_t *prompt_lens,
                                 const int32_t *lens, const float *penalties, const int32_t *bias_ids,
                                 const float *bias_values, const int32_t *bias_offsets, const uint32_t *masks,
                                 int64_t n_masks, int64_t mask_stride, const int32_t *mask_rows, float *y, int64_t ldy) {
  return process_logits(ctx, logits, m, vocab, ld, tokens, tok_stride, prompt_lens, lens, penalties, bias_ids, bias_values,
                        bias_offsets, -1, masks, n_masks, mask_stride, mask_rows, y, ldy);
}

extern "C" int gq_process_logits_bounded(gq_ctx *ctx, const float *logits, int64_t m, int64_t vocab, int64_t ld,
                                         const int32_t *tokens, int64_t tok_stride, const int32_t *prompt_lens,
                                         const int32_t *lens, const float *penalties, const int32_t *bias_ids,
                                         const float *bias_values, const int32_t *bias_offsets, int64_t n_bias,
                                         const uint32_t *masks, int64_t n_masks, int64_t mask_stride,
                                         const int32_t *mask_rows, float *y, int64_t ldy) {
  if (ctx && (n_bias < 0 || n_bias > INT32_MAX / 2))
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "process_logits: the number of bias entries must be below 2^30");
  return process_logits(ctx, logits, m, vocab, ld, tokens, tok_stride, prompt_lens, lens, penalties, bias_ids, bias_values,
                        bias_offsets, n_bias, masks, n_masks, mask_stride, mask_rows, y, ldy);
}
