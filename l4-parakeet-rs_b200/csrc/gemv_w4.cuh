// Shared by the kernels for products of a few rows with INT4 group-128 weights.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include <atomic>

#include "pk100_internal.h"

namespace pk100 {

constexpr int kGroup = 128;

struct GemvParams {
    int m, n, k;
    const __half* a; long long lda;
    const uint8_t* codes;             // [n, k / 2]
    const __half* group_scales;       // [k / 128, n]
    const float* row_scales; float row_scale;
    const float* col_scales; const float* bias;
    int act;
    const __half* residual; long long ld_res;
    float alpha; int valid_rows;
    void* out; long long ld_out; int out_type;
    int* status;                      // of the wide kernel's waits
    unsigned long long wait_ns;       // their limit
};

// 8 codes of a word -> 4 pairs of weights f16(code * scale), pair i = codes (i, i + 4).  With its sign bit flipped a code
// is code + 8; in the low mantissa bits behind the exponent of 1024 it is 1024 + code + 8, four bits higher 1024 +
// 16 (code + 8), and one subtraction or multiply-add gives the code, exactly.
struct CodeMasks {
    uint32_t low, low_magic, high, high_magic;
    // (unknown to the compiler, which would otherwise split (a & low) ^ magic into two instructions with a constant each)
    __device__ __forceinline__ CodeMasks() {
        asm volatile("mov.b32 %0, 0x000f000f;\n\tmov.b32 %1, 0x64086408;\n\tmov.b32 %2, 0x00f000f0;\n\tmov.b32 %3, 0x64806480;"
                     : "=r"(low), "=r"(low_magic), "=r"(high), "=r"(high_magic));
    }
};
__device__ __forceinline__ __half2 and_xor(uint32_t a, uint32_t mask, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(a), "r"(mask), "r"(magic));
    return *reinterpret_cast<const __half2*>(&r);
}
__device__ __forceinline__ void weights_of(uint32_t word, __half2 scale, const CodeMasks& m, uint32_t (&w)[4]) {
    const __half2 low = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));        // 1032
    const __half2 shift = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));      // 1 / 16
    const __half2 high = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));       // -72
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t bits = word >> (4 * i);
        const __half2 even = __hmul2(__hsub2(and_xor(bits, m.low, m.low_magic), low), scale);
        const __half2 odd = __hmul2(__hfma2(and_xor(bits, m.high, m.high_magic), shift, high), scale);
        w[i] = *reinterpret_cast<const uint32_t*>(&even);
        w[i + 1] = *reinterpret_cast<const uint32_t*>(&odd);
    }
}

// Epilogue and store of one sum.
__device__ __forceinline__ void gemv_store(const GemvParams& p, float v, int m, int n) {
    v *= p.row_scales != nullptr ? p.row_scales[m] : p.row_scale;
    if (p.col_scales != nullptr) v *= p.col_scales[n];
    if (p.bias != nullptr) v += p.bias[n];
    if (p.act == PK100_ACT_SILU) v = v / (1.0f + __expf(-v));
    else if (p.act == PK100_ACT_RELU) v = fmaxf(v, 0.0f);
    v = p.residual != nullptr ? fmaf(p.alpha, v, __half2float(p.residual[m * p.ld_res + n])) : p.alpha * v;
    if (m >= p.valid_rows) v = 0.0f;
    if (p.out_type == PK100_OUT_F16) static_cast<__half*>(p.out)[m * p.ld_out + n] = __float2half_rn(v);
    else static_cast<float*>(p.out)[m * p.ld_out + n] = v;
}

// The kernel for many weight rows (gemv_w4_tcgen05.cu); the largest k that it takes.
int gemv_wide_limit();
int launch_gemv_wide(const GemvParams& p, cudaStream_t stream);

}  // namespace pk100
