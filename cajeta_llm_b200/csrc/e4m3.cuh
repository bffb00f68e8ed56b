// What the kernels of the 8-bit cache share: exponents of blocks and of queries, codes to f16.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace cj {

// 2^e for e in [-126, 127]
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// The smallest e with most <= 448 2^e, within [-100, 119] (below: zeros and what is next to them; above: 448 2^119 is the last
// that float32 holds).  most >= 0; 448 = 1.75 2^8.
__device__ __forceinline__ int block_exponent(float most) {
    const uint32_t bits = __float_as_uint(most);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, -100), 119);
}

// The power of two that brings the largest entry of a query head to [2^7, 2^8) (0 entries, and what is beyond float32's reach
// after it, keep a finite one)
__device__ __forceinline__ int query_exponent(float most) {
    const int e = 7 - ((int)(__float_as_uint(most) >> 23) - 127);
    return min(max(e, -100), 100);
}

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// four codes as two pairs of f16 (every e4m3 number is an f16 number)
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}

}  // namespace cj
