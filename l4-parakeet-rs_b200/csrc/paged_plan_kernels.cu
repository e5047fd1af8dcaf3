// One step's bookkeeping of a paged key-value cache: block tables, starts, lengths, positions and slots.
#include "pk100_internal.h"
#include "ptx_sm100.cuh"

namespace pk100 {

constexpr int kPlanThreads = 512;
constexpr int kPlanShare = PK100_PLAN_MAX_REQUESTS / kPlanThreads;

// Every block forms the prefix sums over all requests for itself (reading 8 bytes a request is less than a second
// launch), then takes its share of the tokens and of the requests' new pages.  All blocks come to the same verdict
// on the step, so a refused one changes nothing without any block waiting for another.  The page of a token comes
// from the old part of the table or straight from the free list: no block reads what another writes.
// Bound by the latency of the lengths and of the scan (a few microseconds), then by 12 bytes a token.
__global__ void __launch_bounds__(kPlanThreads)
paged_plan_kernel(const pk100_paged_plan_args p) {
    __shared__ int first[PK100_PLAN_MAX_REQUESTS + 1];        // row of a request's first token
    __shared__ int taken[PK100_PLAN_MAX_REQUESTS];            // pages taken in front of it
    __shared__ long long warp_tokens[kPlanThreads / 32], warp_pages[kPlanThreads / 32];
    __shared__ int refused;
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    grid_dependents_launch();
    if (tid == 0) refused = 0;
    grid_dependency_wait();
    __syncthreads();

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
        if (c < 0 || n < 0 || n > p.tokens || c + n > 0x7fffffffll) { bad = true; continue; }
        const long long had = (c + p.page_size - 1) / p.page_size, has = (c + n + p.page_size - 1) / p.page_size;
        if (has > p.max_pages) { bad = true; continue; }
        fresh[i] = static_cast<int>(n);
        extra[i] = static_cast<int>(has - had);
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
            p.lengths[r] = p.cached[r] + (no ? 0 : fresh[i]);
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

    auto pages_of = [&](long long length) { return static_cast<int>((length + p.page_size - 1) / p.page_size); };
    const int threads = gridDim.x * kPlanThreads, me = blockIdx.x * kPlanThreads + tid;
    if (!no) {                                                  // a warp per request writes its new pages
        for (int r = me / 32; r < p.requests; r += threads / 32) {
            const int had = pages_of(p.cached[r]), extra_r = pages_of(static_cast<long long>(p.cached[r]) + first[r + 1] - first[r]) - had;
            for (int i = lane; i < extra_r; i += 32)
                p.block_table[static_cast<long long>(r) * p.max_pages + had + i] = p.free_pages[taken[r] + i];
        }
    }
    for (int t = me; t < p.tokens; t += threads) {
        int position = -1;
        long long slot = -1;
        if (t < total) {
            int lo = 0, hi = p.requests;                        // the last request with first <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (first[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int r = lo, had = pages_of(p.cached[r]);
            position = p.cached[r] + t - first[r];
            const int page = position / p.page_size;
            const int id = page < had ? p.block_table[static_cast<long long>(r) * p.max_pages + page] : p.free_pages[taken[r] + page - had];
            slot = static_cast<long long>(id) * p.page_size + position % p.page_size;
        }
        p.positions[t] = position;
        p.slots[t] = slot;
    }
}

}  // namespace pk100

using namespace pk100;

extern "C" int pk100_paged_plan(void* stream, const pk100_paged_plan_args* a) {
    if (a == nullptr) return PK100_ERR_NULL;
    if (a->requests < 0 || a->tokens < 0 || a->page_size <= 0 || a->max_pages <= 0 || a->free_capacity < 0) return PK100_ERR_SHAPE;
    if (a->requests > PK100_PLAN_MAX_REQUESTS) return PK100_ERR_LIMIT;
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
    pk100_launch_chained(paged_plan_kernel, dim3(blocks), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), *a);
    return pk100_launch_status();
}
