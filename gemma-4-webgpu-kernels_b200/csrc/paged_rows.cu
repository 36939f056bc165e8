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
//
// Both directions wait for memory (issue slots 50-58% taken; 2.9 stalls on loads per issue when writing, 6.6 when
// reading). With pieces of four 4-bit values a lane and 16-byte accesses they took a third more. 16411 tokens' rows of 512
// written and read back 33 us (144 MB, 4.4 TB/s; the first kernels, a piece at a time, 54), 32771 tokens' read 28 us
// (153 MB, 5.4 TB/s; 43). Rows of whole bytes are read in pieces of four values, four of them in flight, which is near the
// bytes' time as it is: 16411 rows of 512 in f32 24.4 us (135 MB, 5.5 TB/s; 20.5 at the copy rate), f16 and bf16 18.7
// (15.4), e4m3 15.9 (12.8), 4-bit 15.6 (11.7); 4 heads of 128 take 7 to 12% more. A few rows take the time of their
// launches: 5 us.
#include <cuda_bf16.h>

#include <algorithm>

#include "e2m1.cuh"
#include "paged.cuh"

namespace {

// Eight f32 to their codes, the first in the lowest four bits; past 6 they become 6.
__device__ __forceinline__ uint32_t to_e2m1(const float (&x)[8], float r) {
  uint32_t c;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tcvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\tmov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(c)
      : "f"(x[0] * r), "f"(x[1] * r), "f"(x[2] * r), "f"(x[3] * r), "f"(x[4] * r), "f"(x[5] * r), "f"(x[6] * r), "f"(x[7] * r));
  return c;
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

// More than what is lost on the way: a reciprocal within 2^-23 and two f32 roundings, 2^-24 each.
constexpr float kUp = 1.0f + 0x1p-21f, kDown = 1.0f - 0x1p-21f;

// Eight neighbouring values of a lane, half a block (the other half is the lane's beside it; both are
// here): their codes, and the block's scale.
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], uint32_t &scale) {
  uint32_t top = 0;  // largest size as bits: a NaN is above every number
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const float a = __uint_as_float(top), sixth = a * (1.0f / 6.0f);
  const uint32_t ends = __nv_cvt_float2_to_fp8x2(make_float2(sixth * kDown, sixth * kUp), __NV_SATFINITE, __NV_E4M3);
  const uint32_t lo = ends & 255u, hi = ends >> 8;
  const float below = e4m3_value((uint8_t)lo), above = e4m3_value((uint8_t)hi), middle = 3.0f * (below + above);
  const bool up = a > middle || (a == middle && (lo & 1u));
  scale = up ? hi : lo;
  const float s = up ? above : below;
  if (top > 0x7f800000u) scale = 0x7fu;  // a NaN among them: the block is NaN, its codes are 0 or -0
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  r = s > 0.0f ? r : 0.0f;
  const uint32_t near = to_e2m1(x, r * kDown), far = to_e2m1(x, r * kUp);
  if (near == far && top <= 0x7f800000u) return near;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) codes |= code_of(x[i], s) << (4 * i);
  return codes;
}

struct RowArgs {
  float *rows[2];  // k, v (read: written; append: read)
  uint8_t *pool[2];
  int64_t stride[2];
  const int64_t *slots;
  int64_t tokens, page_size, page_bytes, n_slots;
  int heads, head_dim, row_bytes;
  int wide;  // e2m1: the pages' codes are words of an aligned address
  int broad; // the rows of f32 begin on 32 bytes
  float scale[2];  // append: 1 / the pool's scale
  uint32_t *err;
};

constexpr int kThreads = 256, kWarps = kThreads / 32;

// Values of a piece, a lane's share of a row at a time, and pieces of key and value rows in flight: a warp
// takes a token's two rows, its lanes pieces in turn, or kPieces tokens' where a row has one piece per lane
// at most. The next tokens' slots are read meanwhile.
template <int TYPE>
constexpr int kValues = TYPE == GQ_KV_E2M1 ? 8 : 4;
template <int TYPE>
constexpr int kPieces = TYPE == GQ_KV_E2M1 ? 2 : 4;

// Eight f32 as one access of 32 bytes where the rows begin on such.
__device__ __forceinline__ void load8(const RowArgs &a, const float *p, float (&x)[8]) {
  if (a.broad) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "l"(p));
  } else {
    const float4 lo = __ldcs(reinterpret_cast<const float4 *>(p)), hi = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
  }
}
__device__ __forceinline__ void store8(const RowArgs &a, float *p, const float (&x)[8]) {
  if (a.broad) {
    asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
                 "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]), "l"(p)
                 : "memory");
  } else {
    __stcs(reinterpret_cast<float4 *>(p), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4 *>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
  }
}

// Where a token's rows lie: bytes from the pool's start on, -1 where it has none.
__device__ __forceinline__ int64_t row_at(const RowArgs &a, int64_t slot, int lane) {
  if (slot < 0) return -1;
  if (slot >= a.n_slots) {
    if (lane == 0) gqd::report(a.err, GQ_DEVERR_PAGES);
    return -1;
  }
  const int64_t page = (slot >> 32) == 0 ? (int64_t)((uint32_t)slot / (uint32_t)a.page_size) : slot / a.page_size;
  return page * a.page_bytes + (slot - page * a.page_size) * a.row_bytes;
}

// Scales x, and puts its codes and its block's scale in place.
__device__ __forceinline__ void put(const RowArgs &a, uint8_t *row, int in, float (&x)[8], float inv, bool has) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= inv;
  uint32_t scale;
  const uint32_t codes = quantise(x, scale);
  if (!has) return;
  if (a.wide) {
    reinterpret_cast<uint32_t *>(row)[in] = codes;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) row[4 * in + i] = (uint8_t)(codes >> (8 * i));
  }
  if ((in & 1) == 0) row[a.head_dim / 2 + in / 2] = (uint8_t)scale;
}

__global__ void __launch_bounds__(kThreads) append_e2m1_kernel(const RowArgs a) {
  constexpr int N = kPieces<GQ_KV_E2M1>;
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int lane = threadIdx.x & 31, per_head = a.head_dim / 8, pieces = a.heads * per_head;
  const int64_t first = blockIdx.x * (int64_t)kWarps + threadIdx.x / 32, step = (int64_t)gridDim.x * kWarps;
  const int64_t head_bytes = a.page_size * a.row_bytes;
  if (pieces <= 32) {
    const int h = lane / per_head, in = lane - h * per_head;
    const bool has = lane < pieces;
    for (int64_t t0 = first * N; t0 < a.tokens; t0 += step * N) {
      int64_t slot[N];
      float x[N][2][8] = {};
#pragma unroll
      for (int i = 0; i < N; ++i) slot[i] = t0 + i < a.tokens ? a.slots[t0 + i] : -1;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          if (has && t0 + i < a.tokens) load8(a, a.rows[v] + (t0 + i) * a.stride[v] + 8 * lane, x[i][v]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t at = row_at(a, slot[i], lane);
        if (at < 0) continue;
#pragma unroll
        for (int v = 0; v < 2; ++v) put(a, a.pool[v] + at + h * head_bytes, in, x[i][v], a.scale[v], has);
      }
    }
    return;
  }
  int64_t slot = first < a.tokens ? a.slots[first] : -1;
  for (int64_t t = first; t < a.tokens; t += step) {
    const int64_t at = row_at(a, slot, lane);
    if (t + step < a.tokens) slot = a.slots[t + step];
    if (at < 0) continue;
    for (int c0 = 0; c0 < pieces; c0 += 32 * N) {
      float x[2][N][8] = {};
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (c0 + i * 32 + lane < pieces) load8(a, a.rows[v] + t * a.stride[v] + 8 * (c0 + i * 32 + lane), x[v][i]);
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = c0 + i * 32 + lane, h = a.heads == 1 ? 0 : c / per_head;
          if (c0 + i * 32 < pieces)  // (the same for the whole warp)
            put(a, a.pool[v] + at + h * head_bytes, c - h * per_head, x[v][i], a.scale[v], c < pieces);
        }
    }
  }
}

// A piece as it is stored: four values, or the codes of eight and their scale.
template <int TYPE>
struct Piece {
  float4 f;
  uint2 h;
  uint32_t u, s;
  __device__ __forceinline__ void load(const RowArgs &a, const uint8_t *row, int c) {
    if constexpr (TYPE == GQ_KV_F32) {
      f = reinterpret_cast<const float4 *>(row)[c];
    } else if constexpr (TYPE == GQ_KV_E2M1) {
      u = a.wide ? reinterpret_cast<const uint32_t *>(row)[c]
                 : row[4 * c] | ((uint32_t)row[4 * c + 1] << 8) | ((uint32_t)row[4 * c + 2] << 16) | ((uint32_t)row[4 * c + 3] << 24);
      s = row[a.head_dim / 2 + c / 2];
    } else if constexpr (TYPE == GQ_KV_E4M3) {
      u = reinterpret_cast<const uint32_t *>(row)[c];
    } else {
      h = reinterpret_cast<const uint2 *>(row)[c];
    }
  }
  __device__ __forceinline__ void store(const RowArgs &a, float *to, float scale) const {
    if constexpr (TYPE == GQ_KV_E2M1) {
      const __half2 block = __half2half2(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)s, __NV_E4M3)));
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 two = __half22float2(__hmul2(e2m1_pair(u >> (8 * i)), block));  // (exact)
        x[2 * i] = two.x * scale;
        x[2 * i + 1] = two.y * scale;
      }
      store8(a, to, x);
    } else {
      float4 x;
      if constexpr (TYPE == GQ_KV_F32) {
        x = f;
      } else if constexpr (TYPE == GQ_KV_BF16) {
        x = make_float4(__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16),
                        __uint_as_float(h.y & 0xffff0000u));
      } else if constexpr (TYPE == GQ_KV_F16) {
        const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&h.x));
        const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
        x = make_float4(lo.x, lo.y, hi.x, hi.y);
      } else {
        const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u & 0xffffu), __NV_E4M3)));
        const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> 16), __NV_E4M3)));
        x = make_float4(lo.x * scale, lo.y * scale, hi.x * scale, hi.y * scale);
      }
      __stcs(reinterpret_cast<float4 *>(to), x);
    }
  }
};

template <int TYPE>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(const RowArgs a) {
  constexpr int V = kValues<TYPE>, N = kPieces<TYPE>;
  gqd::griddep_wait();
  gqd::griddep_launch_dependents();
  const int lane = threadIdx.x & 31, per_head = a.head_dim / V, pieces = a.heads * per_head;
  const int64_t first = blockIdx.x * (int64_t)kWarps + threadIdx.x / 32, step = (int64_t)gridDim.x * kWarps;
  const int64_t head_bytes = a.page_size * a.row_bytes;
  if (pieces <= 32) {
    const int h = lane / per_head, in = lane - h * per_head;
    const bool has = lane < pieces;
    for (int64_t t0 = first * N; t0 < a.tokens; t0 += step * N) {
      int64_t at[N];
      Piece<TYPE> x[N][2];
#pragma unroll
      for (int i = 0; i < N; ++i) at[i] = t0 + i < a.tokens ? a.slots[t0 + i] : -1;
#pragma unroll
      for (int i = 0; i < N; ++i) at[i] = row_at(a, at[i], lane);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          if (has && at[i] >= 0) x[i][v].load(a, a.pool[v] + at[i] + h * head_bytes, in);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          if (has && at[i] >= 0) x[i][v].store(a, a.rows[v] + (t0 + i) * a.stride[v] + V * lane, a.scale[v]);
    }
    return;
  }
  int64_t slot = first < a.tokens ? a.slots[first] : -1;
  for (int64_t t = first; t < a.tokens; t += step) {
    const int64_t at = row_at(a, slot, lane);
    if (t + step < a.tokens) slot = a.slots[t + step];
    if (at < 0) continue;
    for (int c0 = lane; c0 < pieces; c0 += 32 * N) {
      Piece<TYPE> x[2][N];
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = c0 + i * 32, h = a.heads == 1 ? 0 : c / per_head;
          if (c < pieces) x[v][i].load(a, a.pool[v] + at + h * head_bytes, c - h * per_head);
        }
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (c0 + i * 32 < pieces) x[v][i].store(a, a.rows[v] + t * a.stride[v] + V * (c0 + i * 32), a.scale[v]);
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
  a.wide = (a.row_bytes | a.page_bytes) % 4 == 0;
  a.broad = (((uintptr_t)k | (uintptr_t)v) % 32 | (k_stride | v_stride) % 8) == 0;
  a.err = ctx->dev_err;
  return a;
}

dim3 grid_of(gq_ctx *ctx, const RowArgs &a, int values, int pieces) {
  const int64_t each = kWarps * (a.heads * a.head_dim <= 32 * values ? pieces : 1);  // tokens of a CTA's round
  return dim3((unsigned)std::min<int64_t>((a.tokens + each - 1) / each, (int64_t)ctx->num_sms * 8));
}

template <int TYPE>
int read_rows(gq_ctx *ctx, const RowArgs &a) {
  GQ_CUDA_TRY(ctx, gq_launch(ctx, paged_read_kernel<TYPE>, grid_of(ctx, a, kValues<TYPE>, kPieces<TYPE>), dim3(kThreads), 0, a));
  return GQ_OK;
}

}  // namespace

int gq_paged_append_e2m1(gq_ctx *ctx, const gq_kv_pages *pages, const float *k, const float *v, int64_t t,
                         int64_t k_tok_stride, int64_t v_tok_stride, const int64_t *slots) {
  RowArgs a = args_of(ctx, pages, const_cast<float *>(k), const_cast<float *>(v), t, k_tok_stride, v_tok_stride, slots);
  a.scale[0] = 1.0f / pages->k_scale;
  a.scale[1] = 1.0f / pages->v_scale;
  GQ_CUDA_TRY(ctx, gq_launch(ctx, append_e2m1_kernel, grid_of(ctx, a, kValues<GQ_KV_E2M1>, kPieces<GQ_KV_E2M1>), dim3(kThreads), 0, a));
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
  switch (pages->type) {
    case GQ_KV_F32: return read_rows<GQ_KV_F32>(ctx, a);
    case GQ_KV_F16: return read_rows<GQ_KV_F16>(ctx, a);
    case GQ_KV_BF16: return read_rows<GQ_KV_BF16>(ctx, a);
    case GQ_KV_E4M3: return read_rows<GQ_KV_E4M3>(ctx, a);
    default: return read_rows<GQ_KV_E2M1>(ctx, a);
  }
}
