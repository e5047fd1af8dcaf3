// Residual addition + root-mean-square norm with the output encodings of the 8-bit products.
#include <cuda_fp8.h>

#include <type_traits>

#include "element16.cuh"
#include "pk100_internal.h"
#include "ptx_sm100.cuh"

namespace pk100 {

struct RmsNormParams {
    int rows, width, threads;         // threads: of a row
    const void* input;    long long ld_in;
    const void* residual; long long ld_res;
    void* residual_out;   long long ld_res_out;
    const void* gamma;
    float eps, inv_scale;
    void* output;         long long ld_out;
    float* scales;
    bool vec_in, vec_res, vec_res_out, vec_gamma, vec_out;      // 16-byte (8-bit output: 8-byte) rows
};

__device__ __forceinline__ void store_codes(uint8_t* row, int column, int width, bool vec, uint2 v) {
    if (vec) {
        if (column < width) *reinterpret_cast<uint2*>(row + column) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (column + i < width) row[column + i] = static_cast<uint8_t>((i < 4 ? v.x : v.y) >> (8 * (i % 4)));
}

// y / c = s * gamma * (limit / max |s * gamma|): the root cancels, the product of two 16-bit numbers is exact in fp32, and the
// row's factor comes in two numbers, high + low.  One rounding is left of the quotient; five, with y and c rounded in between,
// moved codes of values half-way between two.
__device__ __forceinline__ float quotient(float product, float high, float low) { return fmaf(product, high, product * low); }

__device__ __forceinline__ float widest_or_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(fabsf(b)));
    return d;
}

// The nearest integers (ties to even) of limit * product / top as bytes, 0 of NaN.  Where a rounded quotient is half-way, which
// side the exact one lies on is decided in 64 bits.
__device__ __forceinline__ uint2 nearest_bytes(const float (&product)[8], float high, float low, float top, float limit) {
    constexpr float kMagic = 12582912.0f;               // 1.5 * 2^23: a quotient is 127 at most
    float n[8], off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = quotient(product[i], high, low);
        n[i] = q + kMagic;
        off = widest_or_nan(off, q - (n[i] - kMagic));
    }
    if (!(off < 0.5f)) {                                // (one of a million)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = quotient(product[i], high, low);
            if (fabsf(q - (n[i] - kMagic)) < 0.5f) continue;
            const double beyond = static_cast<double>(limit) * product[i] - static_cast<double>(q) * top;
            if (beyond != 0.0) n[i] = (q + (beyond > 0.0 ? 0.5f : -0.5f)) + kMagic;
            if (q != q) n[i] = kMagic;
        }
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = __byte_perm(__byte_perm(__float_as_uint(n[4 * i]), __float_as_uint(n[4 * i + 1]), 0x0040),
                           __byte_perm(__float_as_uint(n[4 * i + 2]), __float_as_uint(n[4 * i + 3]), 0x0040), 0x5410);
    return make_uint2(w[0], w[1]);
}

// A row belongs to a warp (8 rows a block) or to a whole block; every thread keeps Chunks x 8 of its elements, so
// the row is read once.  Mean square and max |s * gamma| leave in ONE reduction: max |y| = rstd * max |s * gamma|.
// Sums are fp32 in a fixed order.  The codes are formed from the fp32 y: rounding it to 16 bits first would cost
// bf16 rows a bit of their 7-bit codes.  Bound by HBM for many rows (16 384 x 4096 bf16 to E4M3, 470 MB: 75 to 82 us, 5.7 to 6.2 TB/s),
// by the latency of load, reduction and store for a few.
template <typename T, int Mode, int Chunks, int Block>
__global__ void __launch_bounds__(Block, 1024 / Block)
add_rms_norm_kernel(const RmsNormParams p) {
    __shared__ float part_sum[32], part_max[32];
    grid_dependents_launch();
    grid_dependency_wait();
    const int per_block = blockDim.x / p.threads;
    const int row = blockIdx.x * per_block + threadIdx.x / p.threads, t = threadIdx.x % p.threads;
    if (row >= p.rows) return;                          // (whole warps; blocks of one row have none)
    const T* in = static_cast<const T*>(p.input) + row * p.ld_in;
    const T* gamma = static_cast<const T*>(p.gamma);
    uint4 s[Chunks];
#pragma unroll
    for (int c = 0; c < Chunks; ++c) s[c] = load8(in, (c * p.threads + t) * 8, p.width, p.vec_in);
    if (p.residual != nullptr) {
        const T* res = static_cast<const T*>(p.residual) + row * p.ld_res;
        uint4 r[Chunks];
#pragma unroll
        for (int c = 0; c < Chunks; ++c) r[c] = load8(res, (c * p.threads + t) * 8, p.width, p.vec_res);
#pragma unroll
        for (int c = 0; c < Chunks; ++c) {
            uint32_t* a = reinterpret_cast<uint32_t*>(&s[c]);
            const uint32_t* b = reinterpret_cast<const uint32_t*>(&r[c]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = floats_of(a[i], T()), y = floats_of(b[i], T());
                a[i] = packed_of(x.x + y.x, x.y + y.y, T());
            }
        }
    }
    if (p.residual_out != nullptr) {
        T* o = static_cast<T*>(p.residual_out) + row * p.ld_res_out;
#pragma unroll
        for (int c = 0; c < Chunks; ++c) store8(o, (c * p.threads + t) * 8, p.width, p.vec_res_out, s[c]);
    }
    constexpr bool kRowScale = Mode == PK100_LN_E4M3_ROW || Mode == PK100_LN_S8_ROW;
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int c = 0; c < Chunks; ++c) {
        const uint32_t* a = reinterpret_cast<const uint32_t*>(&s[c]);
        const uint4 g = kRowScale ? load8(gamma, (c * p.threads + t) * 8, p.width, p.vec_gamma) : make_uint4(0, 0, 0, 0);
        const uint32_t* b = reinterpret_cast<const uint32_t*>(&g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = floats_of(a[i], T());
            sum = fmaf(x.x, x.x, sum);
            sum = fmaf(x.y, x.y, sum);
            if constexpr (kRowScale) {
                const float2 y = floats_of(b[i], T());
                top = fmaxf(top, fmaxf(fabsf(x.x * y.x), fabsf(x.y * y.y)));       // (NaN counts for nothing)
            }
        }
    }
    // over the row, to all of its threads
    auto reduce = [&] {
#pragma unroll
        for (int off = 16; off > 0; off /= 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if constexpr (kRowScale) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        }
        if (p.threads == 32) return;                    // (otherwise the block is one row)
        const int warps = p.threads / 32, warp = t / 32, lane = t % 32;
        if (lane == 0) {
            part_sum[warp] = sum;
            part_max[warp] = top;
        }
        __syncthreads();
        sum = lane < warps ? part_sum[lane] : 0.0f;
        top = kRowScale && lane < warps ? part_max[lane] : 0.0f;
#pragma unroll
        for (int off = 16; off > 0; off /= 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if constexpr (kRowScale) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        }
    };
    reduce();
    const float rstd = rsqrtf(sum / p.width + p.eps);
    bool finite = true;
    if (kRowScale && top == INFINITY) {                 // (rare) the maximum over what is a number
        finite = false;
        top = 0.0f;
#pragma unroll
        for (int c = 0; c < Chunks; ++c) {
            const uint32_t* a = reinterpret_cast<const uint32_t*>(&s[c]);
            const uint4 g = load8(gamma, (c * p.threads + t) * 8, p.width, p.vec_gamma);
            const uint32_t* b = reinterpret_cast<const uint32_t*>(&g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = floats_of(a[i], T()), y = floats_of(b[i], T());
                const float u = fabsf(x.x * y.x), v = fabsf(x.y * y.y);
                if (u < INFINITY) top = fmaxf(top, u);
                if (v < INFINITY) top = fmaxf(top, v);
            }
        }
        if (p.threads > 32) __syncthreads();            // (the parts have been read)
        reduce();                                       // (the sum has done its work)
    }
    constexpr float kLimit = Mode == PK100_LN_E4M3_ROW ? 448.0f : 127.0f;
    float scale = 1.0f, high = 0.0f, low = 0.0f;
    bool by_products = false;                           // the row's codes: all of it is numbers, within range
    if constexpr (kRowScale) {
        const float peak = top * rstd;
        if (peak > 0.0f && peak < INFINITY) {
            scale = __fdiv_rn(peak, kLimit);
            by_products = finite && top > 1e-30f && top < 1e30f;
        }
        high = __fdiv_rn(kLimit, top);
        low = __fdiv_rn(fmaf(-high, top, kLimit), top);
        if (t == 0) p.scales[row] = scale;
    }
    auto write = [&](auto products) {
#pragma unroll
        for (int c = 0; c < Chunks; ++c) {
            const int column = (c * p.threads + t) * 8;
            const uint32_t* a = reinterpret_cast<const uint32_t*>(&s[c]);
            const uint4 g = load8(gamma, column, p.width, p.vec_gamma);        // (again, from the L1: registers are blocks in flight)
            const uint32_t* b = reinterpret_cast<const uint32_t*>(&g);
            float y[8];                                  // or s * gamma
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = floats_of(a[i], T()), w = floats_of(b[i], T());
                y[2 * i] = decltype(products)::value ? x.x * w.x : x.x * rstd * w.x;
                y[2 * i + 1] = decltype(products)::value ? x.y * w.y : x.y * rstd * w.y;
            }
            if constexpr (Mode == PK100_LN_F16) {
                T* o = static_cast<T*>(p.output) + row * p.ld_out;
                store8(o, column, p.width, p.vec_out, make_uint4(packed_of(y[0], y[1], T()), packed_of(y[2], y[3], T()),
                                                                 packed_of(y[4], y[5], T()), packed_of(y[6], y[7], T())));
            } else {
                uint2 codes;
                if constexpr (Mode == PK100_LN_S8_ROW && decltype(products)::value) {
                    codes = nearest_bytes(y, high, low, top, kLimit);
                } else {
                    uint32_t w[2] = {0, 0};
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        float lo, hi;
                        if constexpr (decltype(products)::value) {
                            lo = quotient(y[i], high, low);
                            hi = quotient(y[i + 1], high, low);
                        } else if constexpr (kRowScale) {
                            lo = y[i] / scale;
                            hi = y[i + 1] / scale;
                        } else {
                            lo = y[i] * p.inv_scale;
                            hi = y[i + 1] * p.inv_scale;
                        }
                        uint32_t pair;
                        if constexpr (Mode == PK100_LN_S8_ROW) {
                            const int u = max(-127, min(127, __float2int_rn(lo))), v = max(-127, min(127, __float2int_rn(hi)));
                            pair = static_cast<uint32_t>((u & 255) | ((v & 255) << 8));
                        } else {
                            pair = __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
                        }
                        w[i / 4] |= pair << (8 * (i % 4));
                    }
                    codes = make_uint2(w[0], w[1]);
                }
                store_codes(static_cast<uint8_t*>(p.output) + row * p.ld_out, column, p.width, p.vec_out, codes);
            }
        }
    };
    if constexpr (kRowScale) {                          // (a branch a row)
        if (by_products) write(std::true_type());
        else write(std::false_type());
    } else {
        write(std::false_type());
    }
}

template <typename T, int Mode>
static void launch_rms_norm(const RmsNormParams& p, int chunks, int blocks, int block, cudaStream_t stream) {
    if (chunks == 1) pk100_launch_chained(add_rms_norm_kernel<T, Mode, 1, 1024>, dim3(blocks), dim3(block), 0, stream, p);
    else if (chunks == 2) pk100_launch_chained(add_rms_norm_kernel<T, Mode, 2, 1024>, dim3(blocks), dim3(block), 0, stream, p);
    else if (block <= 256) pk100_launch_chained(add_rms_norm_kernel<T, Mode, 4, 256>, dim3(blocks), dim3(block), 0, stream, p);
    else pk100_launch_chained(add_rms_norm_kernel<T, Mode, 4, 1024>, dim3(blocks), dim3(block), 0, stream, p);
}

template <typename T>
static void launch_rms_norm(const RmsNormParams& p, int mode, int chunks, int blocks, int block, cudaStream_t stream) {
    if (mode == PK100_LN_F16) launch_rms_norm<T, PK100_LN_F16>(p, chunks, blocks, block, stream);
    else if (mode == PK100_LN_E4M3_FIXED) launch_rms_norm<T, PK100_LN_E4M3_FIXED>(p, chunks, blocks, block, stream);
    else if (mode == PK100_LN_E4M3_ROW) launch_rms_norm<T, PK100_LN_E4M3_ROW>(p, chunks, blocks, block, stream);
    else launch_rms_norm<T, PK100_LN_S8_ROW>(p, chunks, blocks, block, stream);
}

}  // namespace pk100

using namespace pk100;

extern "C" int pk100_add_rms_norm(void* stream, const pk100_rms_norm_args* a) {
    if (a == nullptr) return PK100_ERR_NULL;
    if (a->type != PK100_TYPE_F16 && a->type != PK100_TYPE_BF16) return PK100_ERR_UNSUPPORTED;
    if (a->mode < PK100_LN_F16 || a->mode > PK100_LN_S8_ROW) return PK100_ERR_UNSUPPORTED;
    if (a->rows < 0 || a->width <= 0) return PK100_ERR_SHAPE;
    if (a->width > 32768) return PK100_ERR_LIMIT;
    if (a->rows == 0) return PK100_OK;
    const bool row_scale = a->mode == PK100_LN_E4M3_ROW || a->mode == PK100_LN_S8_ROW;
    if (a->input == nullptr || a->gamma == nullptr || a->output == nullptr || (row_scale && a->scales == nullptr)) return PK100_ERR_NULL;
    const long long least = a->rows > 1 ? a->width : 0;             // (a single row has no distance)
    if (a->ld_in < least || a->ld_out < least || (a->residual != nullptr && a->ld_res < least) ||
        (a->residual_out != nullptr && a->ld_res_out < least))
        return PK100_ERR_SHAPE;
    auto odd = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 1u) != 0; };
    if (odd(a->input) || odd(a->gamma) || odd(a->residual) || odd(a->residual_out) || (a->mode == PK100_LN_F16 && odd(a->output)) ||
        (reinterpret_cast<uintptr_t>(a->scales) & 3u))
        return PK100_ERR_ALIGN;
    // rows of 8 elements at a time: whole chunks, and every row starts on their boundary
    auto vec = [&](const void* ptr, long long ld, unsigned bytes) {
        return a->width % 8 == 0 && (reinterpret_cast<uintptr_t>(ptr) % bytes) == 0 && (a->rows == 1 || ld % 8 == 0);
    };
    RmsNormParams p{};
    p.rows = a->rows; p.width = a->width;
    p.input = a->input; p.ld_in = a->ld_in;
    p.residual = a->residual; p.ld_res = a->ld_res;
    p.residual_out = a->residual_out; p.ld_res_out = a->ld_res_out;
    p.gamma = a->gamma; p.eps = a->eps; p.inv_scale = a->inv_scale;
    p.output = a->output; p.ld_out = a->ld_out; p.scales = a->scales;
    p.vec_in = vec(a->input, a->ld_in, 16);
    p.vec_res = vec(a->residual, a->ld_res, 16);
    p.vec_res_out = vec(a->residual_out, a->ld_res_out, 16);
    p.vec_gamma = vec(a->gamma, 8, 16);
    p.vec_out = vec(a->output, a->ld_out, a->mode == PK100_LN_F16 ? 16 : 8);
    // As few chunks a thread as have all rows resident at once, the shortest chain (777 x 2560: 4.5 us with two, 5.4
    // with one, 6.6 with four); more rows: four in flight a thread (16 384 x 4096 to E4M3 in 75 us; two: 86, one: 124).  A row that 32 threads hold
    // goes to a warp, without the exchange through shared memory.
    const int need = (a->width + 7) / 8;
    int chunks = 1;
    while (chunks < 4 && static_cast<long long>(a->rows) * ((need + chunks - 1) / chunks) > 1536ll * pk100_sm_count()) chunks *= 2;
    while (chunks > 1 && need <= 16 * chunks) chunks /= 2;             // (half of them would do for a warp)
    while (chunks < 4 && (need + chunks - 1) / chunks > 1024) chunks *= 2;
    p.threads = ((need + chunks - 1) / chunks + 31) / 32 * 32;
    const int block = p.threads == 32 ? 256 : p.threads;
    const int blocks = (a->rows + block / p.threads - 1) / (block / p.threads);
    if (a->type == PK100_TYPE_F16) launch_rms_norm<__half>(p, a->mode, chunks, blocks, block, static_cast<cudaStream_t>(stream));
    else launch_rms_norm<__nv_bfloat16>(p, a->mode, chunks, blocks, block, static_cast<cudaStream_t>(stream));
    return pk100_launch_status();
}
