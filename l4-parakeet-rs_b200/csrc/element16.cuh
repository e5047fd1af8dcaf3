// The two 16-bit element types of the language-model operators behind one set of names.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace pk100 {

__device__ __forceinline__ float2 floats_of(uint32_t packed, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&packed)); }
__device__ __forceinline__ float2 floats_of(uint32_t packed, __nv_bfloat16) {
    return make_float2(__uint_as_float(packed << 16), __uint_as_float(packed & 0xffff0000u));
}
__device__ __forceinline__ uint32_t packed_of(float lo, float hi, __half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t packed_of(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The same, rounded towards zero.
__device__ __forceinline__ uint32_t packed_below(float lo, float hi, __half) {
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t packed_below(float lo, float hi, __nv_bfloat16) {
    uint32_t r;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 8 elements of a row from `column` on, packed; those at or behind `width` read as zero.  vec: 16-byte aligned and whole.
template <typename T>
__device__ __forceinline__ uint4 load8(const T* row, int column, int width, bool vec) {
    if (vec) return column < width ? *reinterpret_cast<const uint4*>(row + column) : make_uint4(0, 0, 0, 0);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = column + 2 * i;
        const uint32_t lo = c < width ? reinterpret_cast<const uint16_t*>(row)[c] : 0;
        const uint32_t hi = c + 1 < width ? reinterpret_cast<const uint16_t*>(row)[c + 1] : 0;
        w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int column, int width, bool vec, uint4 v) {
    if (vec) {
        if (column < width) *reinterpret_cast<uint4*>(row + column) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (column + i < width) reinterpret_cast<uint16_t*>(row)[column + i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)));
}

}  // namespace pk100
