// 4-bit weights: the layout that both products read, and what turns codes into bfloat16 numbers.
//
// A weight [features, K] is cut into tiles of 128 features x 64 of K, those of a feature block one after the other along K.  A tile is
// eight pieces of 16 features: 512 bytes of codes, then the scales.  Lane (g, t) = lane / 4, lane % 4 of a warp owns 16 bytes of a
// piece's codes: features g (first eight bytes) and g + 8, of each the entries 16 j + 4 t + {0, 1, 2, 3} of the four steps j of 16 -
// the first operand of a 16 x 16 product, its K in an order that the second operand's 8-byte loads keep.  A word holds two steps,
// nibble n the entry that pair() finds: n and n + 4 come out together.  The scales: for every group of the tile (one, or two of 32),
// bfloat16 pairs of the features g and g + 8.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace q4 {

__host__ __device__ constexpr int piece_bytes(bool half) { return 512 + (half ? 64 : 32); }
__host__ __device__ constexpr int tile_bytes(bool half) { return 8 * piece_bytes(half); }

// nibbles 0 and 4 of w (codes + 8) as two bfloat16 numbers -8 .. 7: 0x4300 is 128, whose last bit counts one
__device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t v = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*(const __nv_bfloat162*)&v, __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));
    return *(const uint32_t*)&r;
}

// the smallest number of five significant bits that is at least s (s >= 0, finite); what is under float32's normal numbers is 0
__device__ __forceinline__ float scale_up(float s) {
    const uint32_t b = __float_as_uint(s);
    if (b < 0x00800000u) return 0.0f;
    return __uint_as_float((b + 0x0007ffffu) & 0xfff80000u);
}

__device__ __forceinline__ uint4 ldg_codes(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

}  // namespace q4
