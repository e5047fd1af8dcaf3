// Shared by the kernels of attention over a paged cache: parameters, geometry of a request, tensor-map loads.
#pragma once

#include <cuda.h>

#include "element16.cuh"
#include "pk100_internal.h"
#include "ptx_sm100.cuh"

namespace pk100 {

struct PagedParams {
    const void* query; long long ld_query;
    void* out; long long ld_out;
    float* lse;
    const int* starts; const int* lengths; const int* table;
    int tokens, requests, heads, kv_heads, group;      // group: query heads of a key-value head
    int pages, page_shift, max_pages, causal, window;  // window: 0 or up to 2^30
    float scale_log2;                                  // scale * log2(e)
    int few_rows;                                      // requests of up to this many (token, head) rows belong to the few-row kernel
    int* status;
    unsigned long long wait_ns;                        // limit of a wait
};

constexpr float kLn2 = 0.6931471805599453f;

// A request as the kernels see it: whatever the arrays hold, no row lies outside the batch, no key outside the table.
struct PagedRequest {
    int row0, n, len;
    bool cut;
    __device__ __forceinline__ PagedRequest(int row0_, int n_, int len_, bool cut_) : row0(row0_), n(n_), len(len_), cut(cut_) {}
    __device__ __forceinline__ PagedRequest(const PagedParams& p, int r) {
        const int first = p.starts[r], end = p.starts[r + 1], length = p.lengths[r];
        row0 = min(max(first, 0), p.tokens);
        n = max(min(end, p.tokens) - row0, 0);
        const int capacity = p.max_pages << p.page_shift;
        len = min(max(length, 0), capacity);
        cut = length != len || first < 0 || end > p.tokens;
    }
    // keys that the i-th new token sees: [lo, hi)
    __device__ __forceinline__ int hi(const PagedParams& p, int i) const { return p.causal ? max(min(len - n + i + 1, len), 0) : len; }
    __device__ __forceinline__ int lo(const PagedParams& p, int i) const { return p.window > 0 ? max(len - n + i - p.window + 1, 0) : 0; }
};

// 4-D tiled load (feature, token in page, head, page); the feature coordinate is a multiple of 64 here.
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t c0, int32_t c1, int32_t c2, int32_t c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// log2 of a factor that the weights P of a softmax get for the tensor cores: what fp16 has room for above the largest, so that
// few of the small ones fall below its range.  Without it a key of 2^-25.5 had a weight in the sum but none in the output,
// and 2^17 of them behind one dominating key took 3e-3 from a row.  bf16 reaches to 2^-133.
template <typename T> __host__ __device__ constexpr int weight_bits(int largest) { return 0; }
template <> __host__ __device__ constexpr int weight_bits<__half>(int largest) { return 14 - largest; }

// sum = sum * factor + more, `excess` what the sum has too much from its roundings (W. Kahan, CACM 8, 1965)
__device__ __forceinline__ void add_compensated(float& sum, float& excess, float factor, float more) {
    const float before = sum * factor, part = fmaf(-excess, factor, more);
    sum = before + part;
    excess = (sum - before) - part;
}

// Keys that the chunk kernel adds up in tensor memory; the sums of more are kept in kept_ml and kept_out.
constexpr int kFoldKeys = 16384;

// The kernel for requests of more than p.few_rows rows (paged_attention_tcgen05.cu): `pairs` numbers of pairs of tiles
// (tokens * group / pair_rows + requests).  Where the pairs are few, a row's keys are shared out to up to `shares`; how many it came
// to goes to share_count, their parts to part_ml [shares, tokens, heads] and part_out [shares, tokens, heads, head_dim], and
// paged_attention_join adds them up (shares == 1: none of that).  Where max_pages hold more than half of kFoldKeys, kept_ml [shares,
// tokens, heads, 2] and kept_out [shares, tokens, heads, head_dim] are there.
constexpr int pair_rows(int head_dim) { return head_dim == 128 ? 256 : 128; }
int paged_attention_chunks(int type, int head_dim, const PagedParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, int pairs, int shares,
                           int* share_count, float2* part_ml, float* part_out, float2* kept_ml, float* kept_out, cudaStream_t stream);
int paged_attention_join(int type, int head_dim, const PagedParams& p, const int* share_count, const float2* part_ml, const float* part_out, cudaStream_t stream);

}  // namespace pk100
