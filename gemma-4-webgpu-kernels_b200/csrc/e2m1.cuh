// e2m1.cuh — rows of 4-bit values in the pages of a key-value cache (GQ_KV_E2M1): codes of two
// exponent and one fraction bit (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and an e4m3 scale
// for every 16 of them. A code times a scale has at most 6 significant bits and lies in
// [2^-10, 2688]: it is exact in f16, which the tensor kernels make use of.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

// Two codes (the low byte of u, the first in its low half) to f16.
__device__ __forceinline__ __half2 e2m1_pair(uint32_t u) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}" : "=r"(r) : "r"(u));
  return *reinterpret_cast<__half2 *>(&r);
}
__device__ __forceinline__ float e4m3_value(uint8_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}
