// paged.cuh — what the kernels over paged key-value caches share.
#pragma once

#include "gq_internal.cuh"

// Bytes of one stored value of a GQ_KV_* type (of the types whose values are whole bytes).
inline int gq_kv_size(int32_t type) { return type == GQ_KV_F32 ? 4 : type == GQ_KV_E4M3 ? 1 : 2; }

// Elements from one row of a page to the next: values, or the bytes of a GQ_KV_E2M1 row (head_dim / 2
// of codes, then head_dim / 16 of scales).
inline int64_t gq_kv_row(const gq_kv_pages *p) { return p->type == GQ_KV_E2M1 ? p->head_dim / 16 * 9 : p->head_dim; }
inline int64_t gq_kv_page_stride(const gq_kv_pages *p) {
  return p->page_stride ? p->page_stride : p->heads * p->page_size * gq_kv_row(p);
}

// Refuse a page description the kernels cannot read (gq_last_error names `op`).
int gq_check_kv_pages(gq_ctx *ctx, const char *op, const gq_kv_pages *p);

// gq_paged_append to GQ_KV_E2M1 pages (arguments checked, strides not 0).
int gq_paged_append_e2m1(gq_ctx *ctx, const gq_kv_pages *pages, const float *k, const float *v, int64_t t,
                         int64_t k_tok_stride, int64_t v_tok_stride, const int64_t *slots);
