// One step's bookkeeping of a paged key-value cache: block tables, starts, lengths, positions and slots.
#include "pk100_internal.h"
#include "ptx_sm100.cuh"

namespace pk100 {

constexpr int kPlanThreads = 512;
constexpr int kPlanTokens = 4;                // of a lane at a time
constexpr int kPlanShare = PK100_PLAN_MAX_REQUESTS / kPlanThreads;

// Every block forms the prefix sums over all requests for itself (reading 8 bytes a request is less than a second
// launch), then takes its share of the tokens and of the requests' new pages.  All blocks come to the same verdict
// on the step, so a refused one changes nothing without any block waiting for another.  The page of a token comes
// from the old part of the table or straight from the free list: no block reads what another writes.
// Bound by latencies, one behind the other: the lengths, the scan, the pages, the stores.  7 requests of one token 3.4 us, 1000
// requests with 530 000 tokens (6.5 MB) 9.3 us.
__global__ void __launch_bounds__(kPlanThreads)
paged_plan_kernel(const pk100_paged_plan_args p) {
    extern __shared__ int plan_shared[];                      // three numbers a request, of as many as there are
    int* first = plan_shared;                                 // row of a request's first token
    int* taken = first + p.requests + 1;                      // pages taken in front of it
    int* cached = taken + p.requests;
    __shared__ long long warp_tokens[kPlanThreads / 32], warp_pages[kPlanThreads / 32];
    __shared__ int refused;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    grid_dependents_launch();
    if (tid == 0) refused = 0;
    grid_dependency_wait();
    __syncthreads();

    // (lengths and page sizes are below 2^31: their sum fits.  Sizes that are powers of two are not divided by.)
    const unsigned size = p.page_size;
    const int shift = (size & (size - 1)) == 0 ? __ffs(size) - 1 : -1;
    auto page_of = [&](unsigned position) { return static_cast<int>(shift >= 0 ? position >> shift : position / size); };
    auto pages_of = [&](unsigned length) { return page_of(length + size - 1); };
    // a thread's requests: `share` consecutive ones
    const int share = (p.requests + kPlanThreads - 1) / kPlanThreads, r0 = tid * share;
    long long tokens = 0, pages = 0;
    int fresh[kPlanShare], extra[kPlanShare];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kPlanShare; ++i) {
        fresh[i] = extra[i] = 0;
        const int r = r0 + i;
        if (i >= share || r >= p.requests) continue;
        const long long c = p.cached[r], n = p.new_tokens[r];
        cached[r] = static_cast<int>(c);
        if (c < 0 || n < 0 || n > p.tokens || c + n > 0x7fffffffll) { bad = true; continue; }
        const int had = pages_of(static_cast<unsigned>(c)), has = pages_of(static_cast<unsigned>(c + n));
        if (has > p.max_pages) { bad = true; continue; }
        fresh[i] = static_cast<int>(n);
        extra[i] = has - had;
        tokens += n;
        pages += has - had;
    }
    long long token_sum = tokens, page_sum = pages;             // inclusive over the warp
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const long long t = __shfl_up_sync(0xffffffffu, token_sum, off), g = __shfl_up_sync(0xffffffffu, page_sum, off);
        if (lane >= off) { token_sum += t; page_sum += g; }
    }
    if (lane == 31) { warp_tokens[warp] = token_sum; warp_pages[warp] = page_sum; }
    if (bad) refused = 1;
    __syncthreads();
    long long before_tokens = token_sum - tokens, before_pages = page_sum - pages, all_tokens = 0, all_pages = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) { before_tokens += warp_tokens[w]; before_pages += warp_pages[w]; }
        all_tokens += warp_tokens[w];
        all_pages += warp_pages[w];
    }
    const int free_count = p.free_pages != nullptr ? min(*p.free_count, p.free_capacity) : 0;
    const bool no = refused != 0 || all_tokens > p.tokens || all_pages > free_count;
    const bool leader = blockIdx.x == 0;
#pragma unroll
    for (int i = 0; i < kPlanShare; ++i) {
        const int r = r0 + i;
        if (i >= share || r >= p.requests) continue;
        first[r] = no ? 0 : static_cast<int>(before_tokens);
        taken[r] = no ? 0 : static_cast<int>(before_pages);
        before_tokens += fresh[i];
        before_pages += extra[i];
        if (leader) {
            p.starts[r] = first[r];
            p.lengths[r] = cached[r] + (no ? 0 : fresh[i]);
        }
    }
    const int total = no ? 0 : static_cast<int>(all_tokens);
    if (tid == 0) {
        first[p.requests] = total;
        if (leader) {
            p.starts[p.requests] = total;
            *p.used = no ? 0 : static_cast<int>(all_pages);
            if (no && p.status != nullptr) atomicOr(p.status, PK100_STATUS_PLAN);
        }
    }
    __syncthreads();

    const int threads = gridDim.x * kPlanThreads, me = blockIdx.x * kPlanThreads + tid;
    if (!no) {                                                  // a warp per request writes its new pages
        for (int r = me / 32; r < p.requests; r += threads / 32) {
            const int had = pages_of(cached[r]), extra_r = pages_of(static_cast<unsigned>(cached[r]) + first[r + 1] - first[r]) - had;
            for (int i = lane; i < extra_r; i += 32)
                p.block_table[static_cast<long long>(r) * p.max_pages + had + i] = p.free_pages[taken[r] + i];
        }
    }
    // a warp takes a run of tokens, a lane every 32nd of it: stores are whole lines, and a token's request is mostly that
    // of the one before
    const int warps = threads / 32, run = (p.tokens + warps - 1) / warps, from = min(me / 32 * run, p.tokens), to = min(from + run, p.tokens);
    int r = 0;
    for (int base = from; base < to; base += 32 * kPlanTokens) {
        int position[kPlanTokens], id[kPlanTokens], offset[kPlanTokens];
#pragma unroll
        for (int i = 0; i < kPlanTokens; ++i) {
            const int t = base + 32 * i + lane;
            position[i] = -1;
            id[i] = offset[i] = 0;
            if (t >= min(total, to)) continue;
            if (t >= first[r + 1]) {                            // the last request with first <= t
                int lo = r + 1, hi = p.requests;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if (first[mid] <= t) lo = mid;
                    else hi = mid;
                }
                r = lo;
            }
            const int had = pages_of(cached[r]);
            position[i] = cached[r] + t - first[r];
            const int page = page_of(position[i]);
            offset[i] = static_cast<unsigned>(position[i]) - static_cast<unsigned>(page) * size;
            id[i] = page < had ? p.block_table[static_cast<long long>(r) * p.max_pages + page] : p.free_pages[taken[r] + page - had];
        }
#pragma unroll
        for (int i = 0; i < kPlanTokens; ++i) {
            const int t = base + 32 * i + lane;
            if (t >= to) continue;
            p.positions[t] = position[i];
            p.slots[t] = position[i] < 0 ? -1 : static_cast<long long>(id[i]) * p.page_size + offset[i];
        }
    }
}

}  // namespace pk100

using namespace pk100;

extern "C" int pk100_paged_plan(void* stream, const pk100_paged_plan_args* a) {
    if (a == nullptr) return PK100_ERR_NULL;
    if (a->requests < 0 || a->tokens < 0 || a->page_size <= 0 || a->max_pages <= 0 || a->free_capacity < 0) return PK100_ERR_SHAPE;
    if (a->requests > PK100_PLAN_MAX_REQUESTS || a->tokens > 1 << 30) return PK100_ERR_LIMIT;      // (rows are counted in 32 bits)
    if (a->starts == nullptr || a->used == nullptr || a->free_count == nullptr) return PK100_ERR_NULL;
    if (a->requests > 0 && (a->cached == nullptr || a->new_tokens == nullptr || a->block_table == nullptr || a->lengths == nullptr))
        return PK100_ERR_NULL;
    if (a->tokens > 0 && (a->positions == nullptr || a->slots == nullptr)) return PK100_ERR_NULL;
    if (a->requests > 0 && (a->lengths == a->cached || a->lengths == a->new_tokens)) return PK100_ERR_UNSUPPORTED;      // blocks read what others would have written
    const uintptr_t words = reinterpret_cast<uintptr_t>(a->cached) | reinterpret_cast<uintptr_t>(a->new_tokens) | reinterpret_cast<uintptr_t>(a->free_pages) |
                            reinterpret_cast<uintptr_t>(a->free_count) | reinterpret_cast<uintptr_t>(a->block_table) | reinterpret_cast<uintptr_t>(a->starts) |
                            reinterpret_cast<uintptr_t>(a->lengths) | reinterpret_cast<uintptr_t>(a->positions) | reinterpret_cast<uintptr_t>(a->used) |
                            reinterpret_cast<uintptr_t>(a->status);
    if ((words & 3u) != 0 || (reinterpret_cast<uintptr_t>(a->slots) & 7u) != 0) return PK100_ERR_ALIGN;
    const long long wanted = (static_cast<long long>(a->tokens) + kPlanThreads - 1) / kPlanThreads, most = pk100_sm_count();
    const int blocks = static_cast<int>(wanted < 1 ? 1 : (wanted > most ? most : wanted));
    constexpr int most_bytes = (3 * PK100_PLAN_MAX_REQUESTS + 1) * 4;
    const cudaError_t granted = pk100_grant_smem<paged_plan_kernel>(most_bytes);
    if (granted != cudaSuccess) return static_cast<int>(granted);
    pk100_launch_chained(paged_plan_kernel, dim3(blocks), dim3(kPlanThreads), (3 * a->requests + 1) * 4, static_cast<cudaStream_t>(stream), *a);
    return pk100_launch_status();
}
