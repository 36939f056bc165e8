// paged.cuh — what the kernels over paged key-value caches share.
#pragma once

#include "gq_internal.cuh"

// Bytes of one stored value of a GQ_KV_* type.
inline int gq_kv_size(int32_t type) { return type == GQ_KV_F32 ? 4 : type == GQ_KV_E4M3 ? 1 : 2; }

// Refuse a page description the kernels cannot read (gq_last_error names `op`).
int gq_check_kv_pages(gq_ctx *ctx, const char *op, const gq_kv_pages *p);
