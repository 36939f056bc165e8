// paged_rows.cu — rows of a paged key-value cache: written as 4-bit values (gq_paged_append to
// GQ_KV_E2M1 pages) and read back from pages of any type (gq_paged_read).
//
// A block of 16 values becomes a scale s and 16 codes:
//   x = v * (1 / pool scale),  s = the e4m3 number nearest max|x| / 6 (at most 448),
//   code = the e2m1 number nearest x / s (at most 6 in size),   ties to even in both.
// Both quotients are rounded as they are, not as f32 holds them: a number next to the middle of two
// codes is not moved onto it. Neither quotient is computed exactly for that. An interval that holds it
// is rounded at both ends, and where the ends differ the number is compared with the middle of the
// two, multiplied out, which is exact in f32 (few bits times few bits).
#include <cuda_bf16.h>

#include <algorithm>

#include "e2m1.cuh"
#include "paged.cuh"

namespace {

// Two f32 to the byte of their codes, x in the low half; past 6 they become 6.
__device__ __forceinline__ uint32_t to_e2m1(float x, float y) {
  uint32_t r;
  asm("{\n\t.reg .b8 b, z;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\tmov.b32 %0, {b, 0, 0, 0};\n\t}" : "=r"(r) : "f"(x), "f"(y));
  return r & 255u;
}

// The code of |x| / s by comparison: the middles of neighbouring codes times s are exact.
__device__ __forceinline__ uint32_t code_of(float x, float s) {
  const float a = fabsf(x);
  uint32_t c = a > 0.25f * s;  // (0.25, 1.25, 2.5 and 5 go down to the even code, 0.75, 1.75 and 3.5 up)
  c += a >= 0.75f * s;
  c += a > 1.25f * s;
  c += a >= 1.75f * s;
  c += a > 2.5f * s;
  c += a >= 3.5f * s;
  c += a > 5.0f * s;
  return c | (__float_as_uint(x) >> 31 << 3);
}

constexpr float kUp = 1.0f + 0x1p-21f, kDown = 1.0f - 0x1p-21f;  // more than what two f32 roundings move

// Four neighbouring values of a lane, a quarter of a block (its lanes are 4 i .. 4 i + 3, all of them
// here): their codes, and the block's scale.
__device__ __forceinline__ uint32_t quantise(const float4 x, uint32_t lanes, uint32_t &scale) {
  // largest size as bits: a NaN is above every number
  uint32_t top = max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu),
                     max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
  top = max(top, __shfl_xor_sync(lanes, top, 1));
  top = max(top, __shfl_xor_sync(lanes, top, 2));
  const float a = __uint_as_float(top), sixth = a * (1.0f / 6.0f);
  const uint32_t ends = __nv_cvt_float2_to_fp8x2(make_float2(sixth * kDown, sixth * kUp), __NV_SATFINITE, __NV_E4M3);
  const uint32_t lo = ends & 255u, hi = ends >> 8;
  const float below = e4m3_value((uint8_t)lo), above = e4m3_value((uint8_t)hi), middle = 3.0f * (below + above);
  const bool up = a > middle || (a == middle && (lo & 1u));
  scale = up ? hi : lo;
  const float s = up ? above : below;
  if (top > 0x7f800000u) scale = 0x7fu;  // a NaN among them: the block is NaN, its codes are 0
  const float r = s > 0.0f ? 1.0f / s : 0.0f, r0 = r * kDown, r1 = r * kUp;
  const uint32_t near = to_e2m1(x.x * r0, x.y * r0) | (to_e2m1(x.z * r0, x.w * r0) << 8);
  const uint32_t far = to_e2m1(x.x * r1, x.y * r1) | (to_e2m1(x.z * r1, x.w * r1) << 8);
  if (near == far && top <= 0x7f800000u) return near;
  return code_of(x.x, s) | (code_of(x.y, s) << 4) | (code_of(x.z, s) << 8) | (code_of(x.w, s) << 12);
}

struct RowArgs {
  float *rows[2];  // k, v (read: written; append: read)
  uint8_t *pool[2];
  int64_t stride[2];
  const int64_t *slots;
  int64_t tokens, page_size, page_bytes, n_slots;
  int heads, head_dim, row_bytes, wide;
  float scale[2];  // append: 1 / the pool's scale
  uint32_t *err;
};

constexpr int kThreads = 256, kWarps = kThreads / 32;

__global__ void __launch_bounds__(kThreads) append_e2m1_kernel(const RowArgs a) {
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int lane = threadIdx.x & 31, per_head = a.head_dim / 4, pieces = a.heads * per_head;
  for (int64_t r = blockIdx.x * (int64_t)kWarps + threadIdx.x / 32; r < 2 * a.tokens; r += (int64_t)gridDim.x * kWarps) {
    const int64_t t = r >> 1, slot = a.slots[t];
    const bool v = r & 1;
    if (slot < 0) continue;
    if (slot >= a.n_slots) {
      if (lane == 0) gqd::report(a.err, GQ_DEVERR_PAGES);
      continue;
    }
    const int64_t page = slot / a.page_size;
    uint8_t *to = (v ? a.pool[1] : a.pool[0]) + page * a.page_bytes + (slot - page * a.page_size) * a.row_bytes;
    const float4 *from = reinterpret_cast<const float4 *>((v ? a.rows[1] : a.rows[0]) + t * (v ? a.stride[1] : a.stride[0]));
    const float inv = v ? a.scale[1] : a.scale[0];
    for (int c0 = 0; c0 < pieces; c0 += 32) {
      const int c = c0 + lane;
      const uint32_t lanes = __ballot_sync(0xffffffffu, c < pieces);  // whole blocks: pieces is a multiple of 4
      if (c >= pieces) continue;
      float4 x = __ldcs(from + c);
      x = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
      uint32_t scale;
      const uint32_t codes = quantise(x, lanes, scale);
      const int h = c / per_head, in = c - h * per_head;
      uint8_t *row = to + h * a.page_size * a.row_bytes;
      row[2 * in] = (uint8_t)codes;
      row[2 * in + 1] = (uint8_t)(codes >> 8);
      if ((in & 3) == 0) row[a.head_dim / 2 + in / 4] = (uint8_t)scale;
    }
  }
}

template <int TYPE>
__device__ __forceinline__ float4 value4(const uint8_t *row, int c, int dim, float scale) {
  float4 v = {};
  if constexpr (TYPE == GQ_KV_F32) {
    return reinterpret_cast<const float4 *>(row)[c];
  } else if constexpr (TYPE == GQ_KV_E2M1) {
    const uint32_t u = row[2 * c] | ((uint32_t)row[2 * c + 1] << 8);
    const float s = e4m3_value(row[dim / 2 + c / 4]);
    const float2 a = __half22float2(e2m1_pair(u)), b = __half22float2(e2m1_pair(u >> 8));
    v = make_float4(a.x * s, a.y * s, b.x * s, b.y * s);
  } else if constexpr (TYPE == GQ_KV_E4M3) {
    const uint32_t u = reinterpret_cast<const uint32_t *>(row)[c];
    const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u & 0xffffu), __NV_E4M3)));
    const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> 16), __NV_E4M3)));
    v = make_float4(a.x, a.y, b.x, b.y);
  } else {
    const uint2 u = reinterpret_cast<const uint2 *>(row)[c];
    if constexpr (TYPE == GQ_KV_BF16)
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xffff0000u));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  return make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const RowArgs a) {
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int lane = threadIdx.x & 31, per_head = a.head_dim / 4, pieces = a.heads * per_head;
  for (int64_t r = blockIdx.x * (int64_t)kWarps + threadIdx.x / 32; r < 2 * a.tokens; r += (int64_t)gridDim.x * kWarps) {
    const int64_t t = r >> 1, slot = a.slots[t];
    const bool v = r & 1;
    if (slot < 0) continue;
    if (slot >= a.n_slots) {
      if (lane == 0) gqd::report(a.err, GQ_DEVERR_PAGES);
      continue;
    }
    const int64_t page = slot / a.page_size;
    const uint8_t *from = (v ? a.pool[1] : a.pool[0]) + page * a.page_bytes + (slot - page * a.page_size) * a.row_bytes;
    float4 *to = reinterpret_cast<float4 *>((v ? a.rows[1] : a.rows[0]) + t * (v ? a.stride[1] : a.stride[0]));
    for (int c = lane; c < pieces; c += 32) {
      const int h = c / per_head, in = c - h * per_head;
      to[c] = value4<TYPE>(from + h * a.page_size * a.row_bytes, in, a.head_dim, v ? a.scale[1] : a.scale[0]);
    }
  }
}

RowArgs args_of(gq_ctx *ctx, const gq_kv_pages *p, float *k, float *v, int64_t t, int64_t k_stride, int64_t v_stride,
                const int64_t *slots) {
  const int size = p->type == GQ_KV_E2M1 ? 1 : gq_kv_size(p->type);
  RowArgs a{};
  a.rows[0] = k;
  a.rows[1] = v;
  a.pool[0] = static_cast<uint8_t *>(p->k);
  a.pool[1] = static_cast<uint8_t *>(p->v);
  a.stride[0] = k_stride;
  a.stride[1] = v_stride;
  a.slots = slots;
  a.tokens = t;
  a.page_size = p->page_size;
  a.page_bytes = gq_kv_page_stride(p) * size;
  a.n_slots = p->n_pages * p->page_size;
  a.heads = (int)p->heads;
  a.head_dim = (int)p->head_dim;
  a.row_bytes = (int)gq_kv_row(p) * size;
  a.scale[0] = p->k_scale;
  a.scale[1] = p->v_scale;
  a.err = ctx->dev_err;
  return a;
}

dim3 grid_of(gq_ctx *ctx, int64_t t) {
  return dim3((unsigned)std::min<int64_t>((2 * t + kWarps - 1) / kWarps, (int64_t)ctx->num_sms * 8));
}

}  // namespace

int gq_paged_append_e2m1(gq_ctx *ctx, const gq_kv_pages *pages, const float *k, const float *v, int64_t t,
                         int64_t k_tok_stride, int64_t v_tok_stride, const int64_t *slots) {
  RowArgs a = args_of(ctx, pages, const_cast<float *>(k), const_cast<float *>(v), t, k_tok_stride, v_tok_stride, slots);
  a.scale[0] = 1.0f / pages->k_scale;
  a.scale[1] = 1.0f / pages->v_scale;
  GQ_CUDA_TRY(ctx, gq_launch(ctx, append_e2m1_kernel, grid_of(ctx, t), dim3(kThreads), 0, a));
  return GQ_OK;
}

extern "C" int gq_paged_read(gq_ctx *ctx, const gq_kv_pages *pages, const int64_t *slots, int64_t t, float *k, float *v,
                             int64_t k_tok_stride, int64_t v_tok_stride) {
  if (!ctx) return GQ_ERR_INVALID_ARGUMENT;
  int rc = gq_enter_ctx(ctx);
  if (rc != GQ_OK) return rc;
  rc = gq_check_kv_pages(ctx, "paged_read", pages);
  if (rc != GQ_OK) return rc;
  const int64_t row = pages->heads * pages->head_dim;
  if (k_tok_stride == 0) k_tok_stride = row;
  if (v_tok_stride == 0) v_tok_stride = row;
  if (t < 0 || k_tok_stride < row || v_tok_stride < row || k_tok_stride % 4 != 0 || v_tok_stride % 4 != 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_read: bad token count, or a token stride below a row or not a multiple of 4");
  if (t == 0) return GQ_OK;
  if (!k || !v || !slots) return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_read: null pointer");
  if (((uintptr_t)k | (uintptr_t)v) % 16 != 0)
    return gq_fail(ctx, GQ_ERR_INVALID_ARGUMENT, "paged_read: k and v must be 16-byte aligned");
  const RowArgs a = args_of(ctx, pages, k, v, t, k_tok_stride, v_tok_stride, slots);
  const dim3 grid = grid_of(ctx, t);
  switch (pages->type) {
    case GQ_KV_F32: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_read_kernel<GQ_KV_F32>, grid, dim3(kThreads), 0, a)); break;
    case GQ_KV_F16: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_read_kernel<GQ_KV_F16>, grid, dim3(kThreads), 0, a)); break;
    case GQ_KV_BF16: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_read_kernel<GQ_KV_BF16>, grid, dim3(kThreads), 0, a)); break;
    case GQ_KV_E4M3: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_read_kernel<GQ_KV_E4M3>, grid, dim3(kThreads), 0, a)); break;
    default: GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_read_kernel<GQ_KV_E2M1>, grid, dim3(kThreads), 0, a)); break;
  }
  return GQ_OK;
}
