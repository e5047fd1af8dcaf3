// Products of a few rows with INT4 group-128 weights: D[m, n] = epilogue(A[m, k] . W[n, k]^T), W = f16(code * scale),
// m <= 16.
#include <type_traits>

#include "gemv_w4.cuh"
#include "ptx_sm100.cuh"

namespace pk100 {

constexpr int kGemvWarps = 12, kGemvThreads = kGemvWarps * 32;

__device__ __forceinline__ void cp_async_16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int Left>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(Left) : "memory"); }

// D (16 x 8, fp32) += A (16 x 16) . B (16 x 8), fp16
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kWideRows = 16384;      // weight rows from which the wide kernel takes them
constexpr int kGemvTiles = 4;         // 16-row tiles of weights that a block takes at a time

template <int RowTiles>
struct GemvSmem {
    static constexpr int kStages = 3;
    uint4 ring[kStages][2 * kGemvTiles][kGemvThreads];                 // codes, each piece private to its thread
    float sums[kGemvWarps][16 * kGemvTiles][8 * RowTiles + 1];
};

// The weights are the A operand of the tensor instruction (16 weight rows x 16 k), the activations its B operand (up
// to 8 rows each), so a product of 1 to 8 rows costs one instruction per 256 codes and the time is that of reading
// and converting the codes.  The k order inside a group is free: a thread takes 32 consecutive codes of a row (one
// 16-byte load) and pairs them as the nibbles fall, and the activations follow it.
// One block an SM owns a contiguous share of the 16-row tiles and takes them in chunks of up to four, which share the
// activations that they read; its warps take the groups in turn and their sums are joined in a fixed order.  Codes
// come by asynchronous copies, up to 96 KB of them in flight, into a ring in which every thread reads what it has
// copied itself: no barrier in the loop, and the next chunk is on its way while this one is joined.  Activations and
// scales of the next group are requested a group ahead.
// One row by 8192 x 4096 (17 MB): 6.8 us; 1024 x 4096: 4.0 us.  Bound by the conversion and by mma.sync, whose ten issue
// cycles nothing else fills; small products by their chain of load, conversion and join.
template <int RowTiles>
__global__ void __launch_bounds__(kGemvThreads, 1)
gemv_w4g128_kernel(const GemvParams p) {
    extern __shared__ uint8_t gemv_raw[];
    using Smem = GemvSmem<RowTiles>;
    constexpr int kStages = Smem::kStages;
    Smem& sm = *reinterpret_cast<Smem*>(gemv_raw);
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, c = lane % 4;
    const int groups = p.k / kGroup, all = (p.n + 15) / 16;
    const int first = static_cast<int>(static_cast<long long>(all) * blockIdx.x / gridDim.x);
    const int last = static_cast<int>(static_cast<long long>(all) * (blockIdx.x + 1) / gridDim.x);
    // chunks of nearly equal size, the larger ones first
    const int chunks = (last - first + kGemvTiles - 1) / kGemvTiles, each = (last - first) / chunks, larger = last - first - each * chunks;
    auto chunk_at = [&](int chunk) { return first + chunk * each + min(chunk, larger); };
    grid_dependents_launch();
    grid_dependency_wait();

    const CodeMasks masks;
    // what the ring is filled with next: a group of a chunk, rows g + 8 i < limit of it
    const long long row_step = 8ll * (p.k / 2);
    int f_chunk = -1, f_group = groups, f_limit = 0;
    const uint8_t* f_src = nullptr;
    auto fetch = [&](int stage) {
        if (f_group >= groups) {                                       // (a warp without groups fetches nothing)
            f_chunk = warp < groups ? f_chunk + 1 : chunks;
            f_group = warp;
            if (f_chunk < chunks) {
                const int row = chunk_at(f_chunk) * 16 + g;
                f_limit = min(chunk_at(f_chunk + 1) * 16, p.n) - row;
                f_src = p.codes + static_cast<long long>(row) * (p.k / 2) + warp * (kGroup / 2) + 16 * c;
            }
        }
        if (f_chunk < chunks) {
            const uint8_t* src = f_src;
#pragma unroll
            for (int i = 0; i < 2 * kGemvTiles; ++i, src += row_step)
                if (8 * i < f_limit) cp_async_16(&sm.ring[stage][i][tid], src);      // (rows that are not there keep what the ring holds)
            f_group += kGemvWarps;
            f_src += kGemvWarps * (kGroup / 2);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) fetch(s);

    int stage = 0;
#pragma unroll 1
    for (int chunk = 0; chunk < chunks; ++chunk) {
        const int at = chunk_at(chunk), tiles = chunk_at(chunk + 1) - at, limit = min((at + tiles) * 16, p.n) - (at * 16 + g);
        float acc[kGemvTiles][RowTiles][4];
#pragma unroll
        for (int i = 0; i < kGemvTiles; ++i)
#pragma unroll
            for (int j = 0; j < RowTiles; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.0f;
        uint4 x_next[RowTiles][4];
        __half scale_next[2 * kGemvTiles];
#pragma unroll
        for (int j = 0; j < RowTiles; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) x_next[j][i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2 * kGemvTiles; ++i) scale_next[i] = __half();
        const __half* x_src = p.a + g * p.lda + warp * kGroup + 32 * c;
        const __half* scale_src = p.group_scales + static_cast<long long>(warp) * p.n + at * 16 + g;
        // activations and scales, a group ahead (plain loads: the kernel in front may still be writing them when this one starts)
        auto request = [&](int group) {
            if (group >= groups) return;
#pragma unroll
            for (int j = 0; j < RowTiles; ++j)
                if (8 * j + g < p.m) {
                    const uint4* src = reinterpret_cast<const uint4*>(x_src + 8 * j * p.lda);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x_next[j][i] = src[i];
                }
#pragma unroll
            for (int i = 0; i < 2 * kGemvTiles; ++i)
                if (8 * i < limit) scale_next[i] = scale_src[8 * i];
            x_src += kGemvWarps * kGroup;
            scale_src += static_cast<long long>(kGemvWarps) * p.n;
        };
        request(warp);
        uint32_t x[RowTiles][4][4];
        __half scale[2 * kGemvTiles];
        auto products = [&](auto count) {
#pragma unroll
            for (int i = 0; i < decltype(count)::value; ++i) {
                const uint4 lo_codes = sm.ring[stage][2 * i][tid], hi_codes = sm.ring[stage][2 * i + 1][tid];    // rows g and g + 8
                const uint32_t lo_words[4] = {lo_codes.x, lo_codes.y, lo_codes.z, lo_codes.w}, hi_words[4] = {hi_codes.x, hi_codes.y, hi_codes.z, hi_codes.w};
                const __half2 lo_scale = __half2half2(scale[2 * i]), hi_scale = __half2half2(scale[2 * i + 1]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t lo[4], hi[4];
                    weights_of(lo_words[w], lo_scale, masks, lo);
                    weights_of(hi_words[w], hi_scale, masks, hi);
                    const uint32_t near[4] = {lo[0], hi[0], lo[1], hi[1]}, far[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                    for (int j = 0; j < RowTiles; ++j) mma_16x8x16(acc[i][j], near, x[j][w][0], x[j][w][1]);
#pragma unroll
                    for (int j = 0; j < RowTiles; ++j) mma_16x8x16(acc[i][j], far, x[j][w][2], x[j][w][3]);
                }
            }
        };
#pragma unroll 1
        for (int group = warp; group < groups; group += kGemvWarps) {
#pragma unroll
            for (int j = 0; j < RowTiles; ++j)
#pragma unroll
                for (int w = 0; w < 4; ++w) {                          // pairs (0, 4), (1, 5), (2, 6), (3, 7)
                    x[j][w][0] = __byte_perm(x_next[j][w].x, x_next[j][w].z, 0x5410);
                    x[j][w][1] = __byte_perm(x_next[j][w].x, x_next[j][w].z, 0x7632);
                    x[j][w][2] = __byte_perm(x_next[j][w].y, x_next[j][w].w, 0x5410);
                    x[j][w][3] = __byte_perm(x_next[j][w].y, x_next[j][w].w, 0x7632);
                }
#pragma unroll
            for (int i = 0; i < 2 * kGemvTiles; ++i) scale[i] = scale_next[i];
            request(group + kGemvWarps);
            cp_async_wait<kStages - 2>();
            // (straight code for each count, so that the conversions of one tile fill the waits of another's products)
            if (tiles == 4) products(std::integral_constant<int, 4>());
            else if (tiles == 3) products(std::integral_constant<int, 3>());
            else if (tiles == 2) products(std::integral_constant<int, 2>());
            else products(std::integral_constant<int, 1>());
            fetch(stage == 0 ? kStages - 1 : stage - 1);               // the stage read a group ago
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }

        if (chunk > 0) __syncthreads();                                // the sums of the chunk before have been read
#pragma unroll
        for (int i = 0; i < kGemvTiles; ++i)
#pragma unroll
            for (int j = 0; j < RowTiles; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sm.sums[warp][16 * i + g + (e / 2) * 8][8 * j + 2 * c + e % 2] = acc[i][j][e];
        __syncthreads();
        for (int o = tid; o < 16 * kGemvTiles * p.m; o += kGemvThreads) {
            const int row = o % (16 * kGemvTiles), m = o / (16 * kGemvTiles), n = at * 16 + row;
            if (row >= 16 * tiles || n >= p.n) continue;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kGemvWarps; ++w) v += sm.sums[w][row][m];
            gemv_store(p, v, m, n);
        }
    }
    cp_async_wait<0>();
}

template <int RowTiles>
static int launch_gemv(const GemvParams& p, cudaStream_t stream) {
    constexpr auto kernel = gemv_w4g128_kernel<RowTiles>;
    constexpr int bytes = sizeof(GemvSmem<RowTiles>);
    const cudaError_t granted = pk100_grant_smem<kernel>(bytes);
    if (granted != cudaSuccess) return static_cast<int>(granted);
    const int tiles = (p.n + 15) / 16, sms = pk100_cta_budget();
    pk100_launch_chained(kernel, dim3(tiles < sms ? tiles : sms), dim3(kGemvThreads), bytes, stream, p);
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
    if (a->m > 16 || a->n > 1 << 30) return PK100_ERR_LIMIT;             // (rows of weights are counted in 32 bits, whole tiles of them)
    if (a->m == 0) return PK100_OK;
    if (a->a == nullptr || a->b == nullptr || a->out == nullptr || a->b_group_scales == nullptr) return PK100_ERR_NULL;
    // (a single row has no distance)
    if (a->m > 1 && (a->lda < a->k || a->lda % 8 != 0 || a->ld_out < a->n || (a->residual != nullptr && a->ld_res < a->n))) return PK100_ERR_SHAPE;
    auto off = [](const void* ptr, unsigned bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes != 0; };
    if (off(a->a, 16) || off(a->b, 16) || off(a->b_group_scales, 2) || off(a->residual, 2) || off(a->row_scales, 4) ||
        off(a->col_scales, 4) || off(a->bias, 4) || off(a->status, 4) || off(a->out, a->out_type == PK100_OUT_F16 ? 2 : 4))
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
    p.status = a->status;
    p.wait_ns = pk100_wait_limit();
    // From 16 384 weight rows on (almost four tiles a cluster) the wide kernel: 13 rows by 28 672 x 8192 in 36 us against 50, x 1024
    // in 11.2 against 15.0, 16 384 x 4096 in 15.2 against 18.0; one row by 28 672 x 8192 in 33.5 against 36.4.  Below, one row by 8192 x 4096 takes
    // 9.3 us there against 6.8 here, 13 rows 9.8 against 9.4 (4096 x 14 336 14.5 against 15.2, 12 288 x 4096 12.1 against 15.6).
    if (a->n >= kWideRows && a->k <= gemv_wide_limit()) {
        const int rc = launch_gemv_wide(p, stream);
        if (rc != PK100_ERR_UNSUPPORTED) return rc;                    // (the device holds no such cluster)
    }
    return a->m <= 8 ? launch_gemv<1>(p, stream) : launch_gemv<2>(p, stream);
}
