// Products of a few rows with INT4 group-128 weights: D[m, n] = epilogue(A[m, k] . W[n, k]^T), W = f16(code * scale),
// m <= 16.
#include <cuda_fp16.h>

#include "pk100_internal.h"
#include "ptx_sm100.cuh"

namespace pk100 {

constexpr int kGroup = 128;
constexpr int kGemvWarps = 8, kGemvThreads = kGemvWarps * 32;

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
};

__device__ __forceinline__ void cp_async_16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int Left>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(Left) : "memory"); }

// D (16 x 8, fp32) += A (16 x 16) . B (16 x 8), fp16
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8 codes of a word -> 4 pairs of weights f16(code * scale), pair i = codes (i, i + 4).  A code with its sign bit
// flipped is code + 8; behind the exponent of 1024 it is 1024 + code + 8, exactly.
__device__ __forceinline__ void weights_of(uint32_t word, __half2 scale, uint32_t (&w)[4]) {
    const uint32_t flipped = word ^ 0x88888888u;
    const __half2 zero = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));       // 1032
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bits = ((flipped >> (4 * i)) & 0x000f000fu) | 0x64006400u;
        const __half2 v = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&bits), zero), scale);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}

template <int RowTiles, int Tiles, int Stages>
struct GemvSmem {
    uint4 ring[Stages][2 * Tiles][kGemvThreads];                       // codes, each piece private to its thread
    float sums[kGemvWarps][16 * Tiles][8 * RowTiles + 1];
};

// The weights are the A operand of the tensor instruction (16 weight rows x 16 k), the activations its B operand (up
// to 8 rows each), so a product of 1 to 8 rows costs one instruction per 256 codes and the time is that of reading
// and converting the codes.  The k order inside a group is free: a thread takes 32 consecutive codes of a row (one
// 16-byte load) and pairs them as the nibbles fall, and the activations follow it.  A block owns 16 * Tiles weight
// rows; its warps take the groups in turn and their sums are joined in a fixed order.  Codes come by asynchronous
// copies into a ring in which every thread reads what it has copied itself: no barrier in the loop.
template <int RowTiles, int Tiles, int Stages>
__global__ void __launch_bounds__(kGemvThreads)
gemv_w4g128_kernel(const GemvParams p) {
    extern __shared__ uint8_t gemv_raw[];
    using Smem = GemvSmem<RowTiles, Tiles, Stages>;
    Smem& sm = *reinterpret_cast<Smem*>(gemv_raw);
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, c = lane % 4;
    const int n0 = blockIdx.x * 16 * Tiles, groups = p.k / kGroup;
    grid_dependents_launch();
    grid_dependency_wait();

    // weight rows of this thread: g and g + 8 of every tile (those behind the last one repeat it and are not stored)
    long long code_at[2 * Tiles];
    int scale_at[2 * Tiles];
#pragma unroll
    for (int i = 0; i < 2 * Tiles; ++i) {
        const int n = min(n0 + (i / 2) * 16 + (i % 2) * 8 + g, p.n - 1);
        code_at[i] = static_cast<long long>(n) * (p.k / 2) + 16 * c;
        scale_at[i] = n;
    }
    auto fetch = [&](int group, int stage) {
        if (group < groups) {
#pragma unroll
            for (int i = 0; i < 2 * Tiles; ++i) cp_async_16(&sm.ring[stage][i][tid], p.codes + code_at[i] + static_cast<long long>(group) * (kGroup / 2));
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < Stages - 1; ++s) fetch(warp + s * kGemvWarps, s);

    float acc[Tiles][RowTiles][4];
#pragma unroll
    for (int i = 0; i < Tiles; ++i)
#pragma unroll
        for (int j = 0; j < RowTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.0f;

    int stage = 0;
#pragma unroll 1
    for (int group = warp; group < groups; group += kGemvWarps) {
        uint4 x[RowTiles][4];
#pragma unroll
        for (int j = 0; j < RowTiles; ++j) {
            const int m = 8 * j + g;
            const uint4* src = reinterpret_cast<const uint4*>(p.a + m * p.lda + group * kGroup + 32 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = m < p.m ? src[i] : make_uint4(0, 0, 0, 0);
        }
        __half2 scale[2 * Tiles];
#pragma unroll
        for (int i = 0; i < 2 * Tiles; ++i)
            scale[i] = __half2half2(p.group_scales[static_cast<long long>(group) * p.n + scale_at[i]]);
        cp_async_wait<Stages - 2>();
#pragma unroll
        for (int w = 0; w < 4; ++w) {                                  // words of 8 codes
            uint32_t b[RowTiles][4];
#pragma unroll
            for (int j = 0; j < RowTiles; ++j) {
                b[j][0] = __byte_perm(x[j][w].x, x[j][w].z, 0x5410);   // (0, 4)
                b[j][1] = __byte_perm(x[j][w].x, x[j][w].z, 0x7632);   // (1, 5)
                b[j][2] = __byte_perm(x[j][w].y, x[j][w].w, 0x5410);   // (2, 6)
                b[j][3] = __byte_perm(x[j][w].y, x[j][w].w, 0x7632);   // (3, 7)
            }
#pragma unroll
            for (int i = 0; i < Tiles; ++i) {
                uint32_t lo[4], hi[4];                                 // rows g and g + 8
                weights_of(reinterpret_cast<const uint32_t*>(&sm.ring[stage][2 * i][tid])[w], scale[2 * i], lo);
                weights_of(reinterpret_cast<const uint32_t*>(&sm.ring[stage][2 * i + 1][tid])[w], scale[2 * i + 1], hi);
                const uint32_t first[4] = {lo[0], hi[0], lo[1], hi[1]}, second[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                for (int j = 0; j < RowTiles; ++j) {
                    mma_16x8x16(acc[i][j], first, b[j][0], b[j][1]);
                    mma_16x8x16(acc[i][j], second, b[j][2], b[j][3]);
                }
            }
        }
        const int next = stage == 0 ? Stages - 1 : stage - 1;          // the stage read a group ago
        fetch(group + (Stages - 1) * kGemvWarps, next);
        stage = stage + 1 == Stages ? 0 : stage + 1;
    }
    cp_async_wait<0>();

#pragma unroll
    for (int i = 0; i < Tiles; ++i)
#pragma unroll
        for (int j = 0; j < RowTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sm.sums[warp][16 * i + g + (e / 2) * 8][8 * j + 2 * c + e % 2] = acc[i][j][e];
    __syncthreads();
    for (int o = tid; o < 16 * Tiles * p.m; o += kGemvThreads) {
        const int row = o % (16 * Tiles), m = o / (16 * Tiles), n = n0 + row;
        if (n >= p.n) continue;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kGemvWarps; ++w) v += sm.sums[w][row][m];
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
}

template <int RowTiles, int Tiles, int Stages>
static int launch_gemv(const GemvParams& p, cudaStream_t stream) {
    constexpr auto kernel = gemv_w4g128_kernel<RowTiles, Tiles, Stages>;
    constexpr int bytes = sizeof(GemvSmem<RowTiles, Tiles, Stages>);
    const cudaError_t granted = pk100_grant_smem<kernel>(bytes);
    if (granted != cudaSuccess) return static_cast<int>(granted);
    pk100_launch_chained(kernel, dim3((p.n + 16 * Tiles - 1) / (16 * Tiles)), dim3(kGemvThreads), bytes, stream, p);
    return pk100_launch_status();
}

}  // namespace pk100

using namespace pk100;

extern "C" int pk100_gemv_w4g128(void* stream_v, const pk100_gemm_args* a) {
    if (a == nullptr) return PK100_ERR_NULL;
    if (a->kind != PK100_KIND_F16_W4G128 || a->epilogue != PK100_EPI_LINEAR) return PK100_ERR_UNSUPPORTED;
    if (a->act < PK100_ACT_NONE || a->act > PK100_ACT_RELU) return PK100_ERR_UNSUPPORTED;
    if (a->out_type != PK100_OUT_F16 && a->out_type != PK100_OUT_F32) return PK100_ERR_UNSUPPORTED;
    if (a->m < 0 || a->n <= 0 || a->k <= 0 || a->k % kGroup != 0) return PK100_ERR_SHAPE;
    if (a->m > 16) return PK100_ERR_LIMIT;
    if (a->m == 0) return PK100_OK;
    if (a->a == nullptr || a->b == nullptr || a->out == nullptr || a->b_group_scales == nullptr) return PK100_ERR_NULL;
    // (a single row has no distance)
    if (a->m > 1 && (a->lda < a->k || a->lda % 8 != 0 || a->ld_out < a->n || (a->residual != nullptr && a->ld_res < a->n))) return PK100_ERR_SHAPE;
    auto off = [](const void* ptr, unsigned bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes != 0; };
    if (off(a->a, 16) || off(a->b, 16) || off(a->b_group_scales, 2) || off(a->residual, 2) || off(a->row_scales, 4) ||
        off(a->col_scales, 4) || off(a->bias, 4) || off(a->out, a->out_type == PK100_OUT_F16 ? 2 : 4))
        return PK100_ERR_ALIGN;
    GemvParams p{};
    p.m = a->m; p.n = a->n; p.k = a->k;
    p.a = static_cast<const __half*>(a->a); p.lda = a->lda;
    p.codes = static_cast<const uint8_t*>(a->b);
    p.group_scales = static_cast<const __half*>(a->b_group_scales);
    p.row_scales = a->row_scales; p.row_scale = a->row_scale;
    p.col_scales = a->col_scales; p.bias = a->bias; p.act = a->act;
    p.residual = static_cast<const __half*>(a->residual); p.ld_res = a->ld_res;
    p.alpha = a->alpha; p.valid_rows = a->valid_rows <= 0 ? a->m : a->valid_rows;
    p.out = a->out; p.ld_out = a->ld_out; p.out_type = a->out_type;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    // 64 weight rows a block share the activations that they read; 16 where that leaves SMs without a block
    const bool wide = a->n >= 64 * pk100_sm_count();
    if (a->m <= 8) return wide ? launch_gemv<1, 4, 4>(p, stream) : launch_gemv<1, 1, 6>(p, stream);
    return wide ? launch_gemv<2, 4, 4>(p, stream) : launch_gemv<2, 1, 6>(p, stream);
}
