// Attention of many new tokens over a paged key-value cache on the tcgen05 tensor cores.
#include <type_traits>

#include "paged_attention.cuh"

namespace pk100 {
namespace chunk {

constexpr int kTile = 128;                      // (token, head) rows of an accumulator, and keys of a block
constexpr int kTileWarps = 8;                   // softmax warps of a tile: four lane quadrants, two halves of the keys
// Tiles of a block of threads.  Two, so that one's softmax runs under the other's products; of 64 features two blocks with a
// tile each fit an SM, which also covers one's beginning and end with the other's work.
template <int D> constexpr int tiles() { return D == 128 ? 2 : 1; }
template <int D> constexpr int softmax_warps() { return kTileWarps * tiles<D>(); }
template <int D> constexpr int threads() { return softmax_warps<D>() * 32 + 64; }
constexpr int kAtom = kTile * 128;              // 128 rows x 64 elements, 128-byte swizzle
constexpr int kBox = 64;                        // most keys of a TMA box
// Key blocks after which O begins again at zero.  The tensor cores cut off what falls below the last bit of the sum that they
// add to, up to 2^-23 of it for 16 keys: 1.2e-4 in 128 blocks (4e-3 over 2^19 keys in one sum).
constexpr int kFold = kFoldKeys / kTile;
// of the first time: the second tile of a pair has its turn under the first one's products
__device__ __forceinline__ constexpr int first_fold(int tile) { return kFold - tile * (kFold / 2); }
constexpr int kByFma = 5;                       // of 16 pairs of scores, whose exponentials the FMA pipe forms (two prompts: 4 426,
                                                // 5 423, 6 435 us on one card: the order of the instructions moves with it)

template <int D> constexpr int ring_slots() { return 5; }

template <int D>
struct Smem {
    static constexpr int kTiles = tiles<D>();
    uint8_t q[kTiles][D / 64][kAtom];
    uint8_t ring[ring_slots<D>()][D / 64][kAtom];          // key and value blocks in turn
    uint64_t full[ring_slots<D>()], empty[ring_slots<D>()];
    float top[kTiles][2][kTile];                           // row maxima of the halves; then sums
    uint64_t q_ready[kTiles], s_full[kTiles], p_full[kTiles], o_done[kTiles], drained;
    uint32_t tmem;
    int abort;
    unsigned shares, items;                                // of the step
    int row0[32], n[32], len[32], first[32], count[32];    // of up to 32 requests: geometry, their pairs of tiles
};

template <typename T> __host__ __device__ constexpr uint32_t type_bits() { return 0; }                                    // kind::f16 operands: fp16
template <> __host__ __device__ constexpr uint32_t type_bits<__nv_bfloat16>() { return (1u << 7) | (1u << 10); }

__device__ __forceinline__ float max_of(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// 2^x for two values at most 16: n = rint(x), a polynomial of the remainder (minimax of the relative error among those of
// degree 4 that are 1 at 0: 2.9e-6; of degree 3 the 1.01e-4 showed in the lse of rows that such a weight dominates), n into the exponent.  x below -127 counts as -127,
// where 1 less 127 in the exponent is zero to the bit: a masked score has no weight at all (and between -127 and -126 no result
// is below zero or above 2^-126).  NaN (0x7fffffff) leaves as the largest number, 0x7f7fffff, which is infinity in 16 bits.
// On the FMA pipe, where ex2.approx (16 a clock and SM) would take as long as the tensor cores' products.
__device__ __forceinline__ Pair exp2_fma(Pair x) {
    const float2 v = halves_of(x);
    x = pair_of(max_or_nan(v.x, -127.0f), max_or_nan(v.y, -127.0f));
    const Pair magic = pair_of(12582912.0f, 12582912.0f), back = pair_of(-12582912.0f, -12582912.0f);       // 1.5 * 2^23
    const Pair n = pair_add(x, magic);
    const Pair r = pair_fma(pair_add(n, back), pair_of(-1.0f, -1.0f), x);
    Pair y = pair_fma(r, pair_of(0.009582852944731712f, 0.009582852944731712f), pair_of(0.055906426161527634f, 0.055906426161527634f));
    y = pair_fma(r, y, pair_of(0.24024099111557007f, 0.24024099111557007f));
    y = pair_fma(r, y, pair_of(0.6931241750717163f, 0.6931241750717163f));
    y = pair_fma(r, y, pair_of(1.0f, 1.0f));
    const float2 whole = halves_of(n), part = halves_of(y);
    return pair_of(__uint_as_float(__float_as_uint(part.x) + (__float_as_uint(whole.x) << 23)),
                   __uint_as_float(__float_as_uint(part.y) + (__float_as_uint(whole.y) << 23)));
}

// A sum with such a number in it becomes NaN; others, below 2^45, stay as they are.
__device__ __forceinline__ float nan_if_huge(float sum) { return fmaf(sum * 1e20f, 0.0f, sum); }

// P = exp2(s * scale + shift) of 64 scores, stored as 16-bit pairs; the sum of the unrounded values.  ByFma: of 16 pairs
// of scores, how many go to the FMA pipe.
template <typename T, int ByFma>
__device__ __forceinline__ float weights_of_scores(const float (&s)[64], float scale, float shift, uint32_t p_cols) {
    const Pair scale2 = pair_of(scale, scale), shift2 = pair_of(shift, shift);
    Pair sum = pair_of(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < 64; c += 32) {
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const Pair x = pair_fma(pair_of(s[c + 2 * i], s[c + 2 * i + 1]), scale2, shift2);
            Pair e;
            if (i * ByFma % 16 + ByFma >= 16) {              // spread evenly
                e = exp2_fma(x);
            } else {
                const float2 v = halves_of(x);
                e = pair_of(exp2_approx(v.x), exp2_approx(v.y));
            }
            sum = pair_add(sum, e);
            const float2 v = halves_of(e);
            packed[i] = packed_of(v.x, v.y, T());
        }
        tmem_st_32x16(p_cols + c / 2, packed);
    }
    const float2 sums = halves_of(sum);
    return sums.x + sums.y;
}

// What a block of threads works on: 256 rows of one request and key-value head, over a share of their keys.
template <int kTiles>
struct Work {
    PagedRequest at;
    int request, head, row, rows;               // first row of the first tile inside the request; rows of both tiles that exist
    int lo, hi;                                 // keys that any of the rows sees
    int from, to;                               // key blocks of this share
    __device__ __forceinline__ Work(const PagedParams& p, const PagedRequest& at_, int request_, int head_, int pair) : at(at_), request(request_), head(head_) {
        row = pair * kTiles * kTile;
        rows = min(at.n * p.group - row, kTiles * kTile);
        const int first = row / p.group, last = (row + max(rows, 1) - 1) / p.group;
        lo = at.lo(p, first);
        hi = at.hi(p, last);
        from = lo / kTile;
        to = max((hi + kTile - 1) / kTile, from);
    }
    // key blocks of this share that a row of tile t sees
    __device__ __forceinline__ int tile_from(const PagedParams& p, int t) const {
        return max(from, at.lo(p, (row + t * kTile) / p.group) / kTile);
    }
    __device__ __forceinline__ int tile_to(const PagedParams& p, int t) const {
        const int left = min(rows - t * kTile, kTile);
        if (left <= 0) return tile_from(p, t);
        return max(tile_from(p, t), min(to, (at.hi(p, (row + t * kTile + left - 1) / p.group) + kTile - 1) / kTile));
    }
};

// The step's pairs of tiles (pairs of one tile where D is 64) and where to find one.
// Up to 32 requests: one warp orders them, the longest first, into shared memory; a request's last pairs, which see the most
// keys, come first.  Up to 256: counted from the requests, in their order.  More: numbered over the batch with gaps, request r
// from floor(first row / rows of a pair) + r on, which leaves room for its last, partial one.  Counting: 256 requests of 10 to 60 tokens
// 110 us against 125 with numbers, 200 101 against 107, 100 56.6 against 57.7; numbers: 500 197 against 210, 1000 368 against 459, 300 the same.
// (A warp orders as many as it has lanes; what ordering brings stands at the kernel, what the pass over the items costs few requests at its launch.)
constexpr int kOrdered = 32, kCounted = 256;

template <int kTiles>
__device__ __forceinline__ int pairs_of(const PagedParams& p, const PagedRequest& at) {
    constexpr int kRows = kTiles * kTile;
    const int rows = at.n * p.group;
    return rows > p.few_rows ? (rows + kRows - 1) / kRows : 0;
}

// All pairs, by a whole warp.
template <int D>
__device__ __forceinline__ int schedule(Smem<D>& sm, const PagedParams& p, int numbers) {
    const int lane = threadIdx.x % 32;
    if (p.requests > kCounted) return numbers;
    if (p.requests > kOrdered) {
        int sum = 0;
        for (int r = lane; r < p.requests; r += 32) sum += pairs_of<tiles<D>()>(p, PagedRequest(p, r));
        return __reduce_add_sync(0xffffffffu, sum);
    }
    const bool there = lane < p.requests;
    const PagedRequest at = there ? PagedRequest(p, lane) : PagedRequest(0, 0, 0, false);
    const int mine = pairs_of<tiles<D>()>(p, at), keys = there ? (p.window > 0 ? min(at.len, p.window) : at.len) : -1;
    int before = 0;
    for (int r = 0; r < p.requests; ++r) {
        const int other = __shfl_sync(0xffffffffu, keys, r), count = __shfl_sync(0xffffffffu, mine, r);
        if (other > keys || (other == keys && r < lane)) before += count;
    }
    sm.row0[lane] = at.row0;
    sm.n[lane] = at.n;
    sm.len[lane] = at.len | (at.cut ? static_cast<int>(0x80000000u) : 0);
    sm.first[lane] = before;
    sm.count[lane] = mine;
    return __reduce_add_sync(0xffffffffu, mine);
}

// The pair with this number, by a whole warp: its request (none: < 0) and place there.
struct Place { int request, pair; PagedRequest at; };
template <int D>
__device__ __forceinline__ Place place_of(const Smem<D>& sm, const PagedParams& p, int number, int numbers) {
    constexpr int kTiles = tiles<D>(), kRows = kTiles * kTile;
    const int lane = threadIdx.x % 32;
    if (p.requests <= kOrdered) {
        const int first = sm.first[lane], count = sm.count[lane];
        const uint32_t has = __ballot_sync(0xffffffffu, number >= first && number < first + count);
        const int request = has == 0 ? 0 : __ffs(has) - 1, len = sm.len[request];
        return Place{has == 0 ? -1 : request, sm.count[request] - 1 - (number - sm.first[request]),
                     PagedRequest(sm.row0[request], sm.n[request], len & 0x7fffffff, len < 0)};
    }
    if (p.requests <= kCounted) {
        int before = 0;
        for (int r0 = 0; r0 < p.requests; r0 += 32) {
            const PagedRequest at = r0 + lane < p.requests ? PagedRequest(p, r0 + lane) : PagedRequest(0, 0, 0, false);
            const int count = pairs_of<kTiles>(p, at);
            int upto = count;
#pragma unroll
            for (int off = 1; off < 32; off *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += v;
            }
            const int first = before + upto - count;
            const uint32_t has = __ballot_sync(0xffffffffu, number >= first && number < first + count);
            if (has != 0) {
                const int from = __ffs(has) - 1;
                return Place{r0 + from, __shfl_sync(0xffffffffu, count - 1 - (number - first), from),
                             PagedRequest(__shfl_sync(0xffffffffu, at.row0, from), __shfl_sync(0xffffffffu, at.n, from),
                                          __shfl_sync(0xffffffffu, at.len, from), __shfl_sync(0xffffffffu, static_cast<int>(at.cut), from) != 0)};
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        return Place{-1, 0, PagedRequest(0, 0, 0, false)};
    }
    // the last request that begins at or before the number, found 32 candidates at a time
    const int wanted = numbers - 1 - number;
    int lo = 0, hi = p.requests, begin = 0;      // begin(lo) <= wanted < begin(hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, r = lo + lane * step;
        long long b = 0x7fffffffll;
        if (r < hi) b = static_cast<long long>(max(p.starts[r], 0)) * p.group / kRows + r;
        const uint32_t before = __ballot_sync(0xffffffffu, b <= wanted);
        const int last = before == 0 ? 0 : 31 - __clz(before);
        begin = static_cast<int>(__shfl_sync(0xffffffffu, b, last));
        lo = min(lo + last * step, p.requests - 1);
        hi = min(lo + step, hi);
    }
    const PagedRequest at(p, lo);
    const int rows = at.n * p.group, pair = wanted - begin;
    return Place{pair >= 0 && pair * kRows < rows && rows > p.few_rows ? lo : -1, max(pair, 0), at};
}

#define CHUNK_WAIT(bar, parity) \
    if (!(ok = __all_sync(0xffffffffu, mbar_wait_within(&(bar), (parity), abort_flag, p.wait_ns)) != 0)) break
#define CHUNK_LOOK(bar, parity) \
    if (!(ok = __all_sync(0xffffffffu, mbar_look_within(&(bar), (parity), abort_flag, p.wait_ns)) != 0)) break

// The query heads of a key-value head are rows of one tile (row = token * group + head), so a chunk of few tokens fills
// its tiles and keys are read once for all of them.  A tile of 128 rows has eight softmax warps (half a row a thread, the
// halves' maxima meet in shared memory); a block has one TMA and one MMA warp.  Per 128-key block and tile
//   S = Q K^T  (tcgen05, both operands from shared memory, 128 TMEM columns),
//   P = exp2(scale S - m) back into the columns of S in 16 bits,
//   O += P V   (A from tensor memory, V as it lies in the cache: MN-major), D TMEM columns.
// While one tile's softmax runs, the tensor cores form the other's O and next S (heads of 64: the other block's of the
// SM).  m follows the running maximum only when that has grown by more than 2^8 (then O and l are scaled down, which is
// exact but for rounding): P stays below 2^8 (fp16: 2^14, see weight_bits), and the rescaling of O all but disappears.
// Scores, m, l and O are fp32; P is rounded to the type of V for the tensor cores, which costs what the rounding of the
// output costs (the sum l is that of the unrounded P): bf16 outputs are 2.3e-3 off instead of 1.7e-3, fp16 2.5e-4 instead of 2.0e-4,
// relative to their norm.  The rest of the rounding in a second product, as in the few-row kernel, took two prompts from 440 to 556 us.
// Bound by a tile's chain of scores, softmax and products: 3200 cycles per 128 keys of both tiles, of which the MMAs are
// 2300.  Two prompts of 7.2 k tokens, 16 / 4 heads of 128: 423 to 437 us, 1 PFLOP/s (the few-row kernel in the same place: 4.6 ms);
// 512 tokens over 32 000, 16 / 2 heads: 138 to 146 us, 0.95 PFLOP/s (764 us); 4096 over 32 000 981 us (967 with one sum of all keys).  Nine
// chunks of 5 to 561 tokens, 16 heads of 64, window 1024: 26.6 us, the latency of the longest block (6 us more in their own order).
template <typename T, int D, bool kLoop>
__global__ void __launch_bounds__(threads<D>(), 3 - tiles<D>())
paged_attention_chunk_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedParams p,
                             const int pairs, const int most_shares, const unsigned slots, int* share_count, float2* part_ml,
                             float* part_out, float2* kept_ml, float* kept_out) {
    extern __shared__ __align__(1024) uint8_t chunk_raw[];             // (the swizzled atoms need it)
    constexpr int kHalves = D / 64, kSlots = ring_slots<D>(), kSlotBytes = kHalves * kAtom, kTiles = tiles<D>(), kSoftmaxWarps = softmax_warps<D>();
    constexpr uint32_t kColumns = 256 * kTiles;                 // of tensor memory: S and O of the tiles
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>(chunk_raw);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
    volatile int* abort_flag = &sm.abort;
    if (tid == 0) {
        sm.abort = 0;
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int t = 0; t < kTiles; ++t) {
            mbar_init(&sm.q_ready[t], kTileWarps);
            mbar_init(&sm.s_full[t], 1);
            mbar_init(&sm.p_full[t], kTileWarps);
            mbar_init(&sm.o_done[t], 1);
        }
        mbar_init(&sm.drained, 1);
        fence_barrier_init();
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    if (warp == kSoftmaxWarps + 1) {
        tmem_alloc(&sm.tmem, kColumns);
        tmem_relinquish();
    }
    grid_dependency_wait();
    grid_dependents_launch();                   // (only now: the few-row kernel behind this one does not wait for what is in front of it)
    // Items of work: pair of tiles, key-value head and share of the keys, shared out where there are fewer pairs than blocks.
    if (warp == 0) {
        const int all = schedule(sm, p, pairs);
        if (lane == 0) {
            const unsigned columns = static_cast<unsigned>(all) * p.kv_heads;
            sm.shares = max(min(static_cast<unsigned>(most_shares), slots / max(columns, 1u)), 1u);
            sm.items = columns * sm.shares;
            if (blockIdx.x == 0 && most_shares > 1) *share_count = sm.shares;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sm.tmem;
    const unsigned shares = sm.shares;
    // Every role goes through the block's items: f(work, request, head, share).  One item where the grid has a block for each that
    // may exist, else the block's place in each pass over the grid, the passes forwards and backwards in turn, so that who has
    // the longest of one has the shortest of the next.
    auto one_item = [&](unsigned item, auto&& f) {
        if (item >= sm.items) return;
        // (shares of a column lie side by side: they read the same queries)
        const unsigned column = item / shares;
        const int share = static_cast<int>(item - column * shares), number = static_cast<int>(column / p.kv_heads), head = static_cast<int>(column - number * p.kv_heads);
        const Place place = place_of(sm, p, number, pairs);
        if (place.request < 0) return;
        Work<kTiles> w(p, place.at, place.request, head, place.pair);
        // a share is two blocks of keys at least
        const int blocks = w.to - w.from, parts = max(min(static_cast<int>(shares), blocks / 2), 1), from = w.from;
        if (share >= parts) w.from = w.to;
        else {
            w.from = from + static_cast<int>(static_cast<long long>(blocks) * share / parts);
            w.to = from + static_cast<int>(static_cast<long long>(blocks) * (share + 1) / parts);
        }
        f(w, place.request, head, share);
    };
    auto each_item = [&](auto&& f) {
        if constexpr (!kLoop) one_item(blockIdx.x, f);
        else {
#pragma unroll 1
            for (unsigned base = 0, back = 0; base < sm.items; base += gridDim.x, back ^= 1)
                one_item(base + (back ? gridDim.x - 1 - blockIdx.x : blockIdx.x), f);
        }
    };
    bool ok = true;
    int it = 0;                                          // ring position of the role
    if (warp == kSoftmaxWarps) {
        // ------------------------------------------------------------ TMA
        const int box = min(kBox, 1 << p.page_shift), boxes = kTile / box;         // boxes: up to 8
        bool bad = false;
        each_item([&](const Work<kTiles>& w, int request, int head, int) {
        const int* table = p.table + static_cast<long long>(request) * p.max_pages;
        int held = -32, id = 0;
        bad |= w.at.cut;
        for (int b = w.from; ok && b < w.to; ++b) {
            const int key = b * kTile + min(lane, boxes - 1) * box, page = key >> p.page_shift;
            if (((b * kTile + kTile - 1) >> p.page_shift) >= held + 32) {
                held = (b * kTile) >> p.page_shift;
                id = held + lane < p.max_pages ? table[held + lane] : -1;
            }
            int page_id = __shfl_sync(0xffffffffu, id, page - held);
            const bool need = lane < boxes && key < w.hi && key + box > w.lo;
            if (need && (page_id < 0 || page_id >= p.pages)) {
                bad = true;
                page_id = p.pages;                          // outside the tensor: zeros
            }
            const int count = __popc(__ballot_sync(0xffffffffu, need));
            const int token = key & ((1 << p.page_shift) - 1);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv, ++it) {
                const int slot = it % kSlots;
                CHUNK_LOOK(sm.empty[slot], (it / kSlots + 1) & 1);
                if (lane == 0) mbar_arrive_expect_tx(&sm.full[slot], count * box * 128 * kHalves);
                __syncwarp();
                if (need) {
#pragma unroll
                    for (int half = 0; half < kHalves; ++half)
                        tma_load_4d(sm.ring[slot][half] + lane * box * 128, kv == 0 ? &map_k : &map_v, &sm.full[slot], half * 64, token, head, page_id);
                }
                __syncwarp();
            }
        }
        });
        if (bad && p.status != nullptr) atomicOr(p.status, PK100_STATUS_PAGE);
    } else if (warp == kSoftmaxWarps + 1) {
        // ------------------------------------------------------------ MMA
        constexpr uint32_t idesc_s = make_instr_desc<KIND_F16>(kTile, kTile) | type_bits<T>();
        constexpr uint32_t idesc_o = make_instr_desc<KIND_F16>(kTile, D) | type_bits<T>() | (1u << 16);      // B is MN-major
        const uint64_t desc_q = make_smem_desc<128>(smem_u32(sm.q)), desc_ring = make_smem_desc<128>(smem_u32(sm.ring));
        // V[keys, features]: 8-key groups 1024 bytes apart, the second 64 features an atom on; 16 keys = 2048 bytes
        const uint64_t desc_v = static_cast<uint64_t>((smem_u32(sm.ring) & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kAtom >> 4) << 16) |
                                (64ull << 32) | (1ull << 46) | (2ull << 61);
        auto k_offset = [](int ks) { return static_cast<uint32_t>((ks / 4) * (kAtom / 16) + 2 * (ks % 4)); };
        const bool leader = elect_one();
        uint32_t phase[kTiles] = {};                         // parity of the tile's next block
        uint32_t q_phase[kTiles] = {};                       // of the tile's next item with blocks
        // (it: of the block's keys; its values follow)
        each_item([&](const Work<kTiles>& w, int, int, int) {
        if (!ok || w.from >= w.to) return;
        int tile_from[kTiles], tile_to[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            tile_from[t] = w.tile_from(p, t);
            tile_to[t] = w.tile_to(p, t);
        }
        auto active = [&](int t, int b) { return b >= tile_from[t] && b < tile_to[t]; };
        auto scores = [&](int t, int slot) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
                tc_mma_if<KIND_F16>(leader, tmem + t * kTile, desc_q + t * (kSlotBytes / 16) + k_offset(ks), desc_ring + slot * (kSlotBytes / 16) + k_offset(ks),
                                    idesc_s, ks > 0);
            tc_commit_if(leader, &sm.s_full[t]);
        };
        do {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                if (ok && tile_from[t] < tile_to[t]) {
                    CHUNK_LOOK(sm.q_ready[t], q_phase[t]);
                    q_phase[t] ^= 1;
                }
            if (!ok) break;
            CHUNK_WAIT(sm.full[it % kSlots], (it / kSlots) & 1);
            tc_fence_after_sync();
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                if (active(t, w.from)) scores(t, it % kSlots);
            tc_commit_if(leader, &sm.empty[it % kSlots]);
#pragma unroll 1
            for (int b = w.from; b < w.to; ++b, it += 2) {
                const int v_slot = (it + 1) % kSlots, k_slot = (it + 2) % kSlots;
                CHUNK_WAIT(sm.full[v_slot], ((it + 1) / kSlots) & 1);
                // values that no row sees may be anything: zeros
                const int k0 = b * kTile;
                if (k0 < w.lo || k0 + kTile > w.hi) {
                    for (int key = lane; key < kTile; key += 32)
                        if (k0 + key < w.lo || k0 + key >= w.hi) {
#pragma unroll
                            for (int c = 0; c < kHalves * 8; ++c)
                                *reinterpret_cast<uint4*>(sm.ring[v_slot][c / 8] + key * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
                        }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                bool next_here = false;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    if (active(t, b)) {
                        CHUNK_WAIT(sm.p_full[t], phase[t]);
                        phase[t] ^= 1;
                        tc_fence_after_sync();
#pragma unroll
                        for (int ks = 0; ks < kTile / 16; ++ks)
                            mma_from_tmem(leader, tmem + kTiles * kTile + t * D, tmem + t * kTile + ks * 8, desc_v + v_slot * (kSlotBytes / 16) + ks * 128u, idesc_o,
                                          ks > 0 || (b > tile_from[t] && (b - tile_from[t] - first_fold(t)) % kFold != 0));
                        tc_commit_if(leader, &sm.o_done[t]);
                    }
                    if (b + 1 < w.to && active(t, b + 1)) {
                        if (!next_here) {
                            CHUNK_WAIT(sm.full[k_slot], ((it + 2) / kSlots) & 1);
                            next_here = true;
                            tc_fence_after_sync();
                        }
                        scores(t, k_slot);
                    }
                }
                if (!ok) break;
                if (b + 1 < w.to && !next_here) CHUNK_WAIT(sm.full[k_slot], ((it + 2) / kSlots) & 1);     // (every block has a tile that sees it)
                tc_commit_if(leader, &sm.empty[v_slot]);
                if (b + 1 < w.to) tc_commit_if(leader, &sm.empty[k_slot]);
            }
        } while (false);
        });
        // the last arrival of the tensor cores comes before the block leaves
        if (ok && it > 0) ok = __all_sync(0xffffffffu, mbar_wait_within(&sm.empty[(it - 1) % kSlots], ((it - 1) / kSlots) & 1, abort_flag, p.wait_ns)) != 0;
    } else {
        // ------------------------------------------------------------ softmax: half a row a thread
        const int t = warp / kTileWarps, half = (warp / 4) % 2, quad = warp % 4, tile_row = quad * 32 + lane;
        // the two warps of a quadrant of a tile
        auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + t * 4 + quad) : "memory"); };
        uint32_t phase = 0;                                  // parity of the tile's next block
        each_item([&](const Work<kTiles>& w, int, int head, int share) {
        // (a tile without blocks brings no queries: its warps, which nothing holds back, would run ahead of the barrier's phases)
        if (w.tile_from(p, t) < w.tile_to(p, t)) {
            // the tile's queries, 16 bytes a thread, rows that do not exist are zeros (the scores that the ones before were
            // multiplied for have been read)
            constexpr int kChunks = D / 8, kThreads = kTileWarps * 32, kEach = kTile * kChunks / kThreads;
            const int thread = tid % kThreads;
            const uint32_t sign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;      // a negative scale turns the queries round
            uint4 v[kEach];                                  // (all requested before the first is stored)
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int r = t * kTile + (thread + j * kThreads) / kChunks, index = w.row + r, token = index / p.group;
                v[j] = r < w.rows ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.query) + (w.at.row0 + token) * p.ld_query +
                                                                    static_cast<long long>(head * p.group + index - token * p.group) * D + thread % kChunks * 8)
                                  : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int c = thread % kChunks, q_row = (thread + j * kThreads) / kChunks;
                *reinterpret_cast<uint4*>(sm.q[t][c / 8] + q_row * 128 + (((c % 8) ^ (q_row & 7)) << 4)) =
                    make_uint4(v[j].x ^ sign, v[j].y ^ sign, v[j].z ^ sign, v[j].w ^ sign);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_ready[t]);
        }
        const int index = w.row + t * kTile + tile_row, token = index / p.group;
        const bool live = t * kTile + tile_row < w.rows;
        const int row_lo = w.at.lo(p, token), row_hi = live ? w.at.hi(p, token) : 0;
        // keys that every row of the tile sees
        const int tile_rows = min(w.rows - t * kTile, kTile);
        const int all_lo = w.at.lo(p, (w.row + t * kTile + max(tile_rows, 1) - 1) / p.group), all_hi = w.at.hi(p, (w.row + t * kTile) / p.group);
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t s_cols = tmem + lanes + t * kTile + half * 64, p_cols = tmem + lanes + t * kTile + half * 32;
        const uint32_t o_cols = tmem + lanes + kTiles * kTile + t * D + half * (D / 2);
        // (-inf * 0 would be NaN; the smallest number takes any finite score to 0.  NaN stays.)
        const float scale = fabsf(p.scale_log2) < 1e-45f ? 1e-45f : fabsf(p.scale_log2);
        constexpr float kBits = weight_bits<T>(8);
        // the blocks of this tile, kFold at a time: what those before gave is kept in memory
        int b = w.tile_from(p, t);
        const int end = w.tile_to(p, t);
        bool kept = false;
#pragma unroll 1
        do {
        const int stop = min(b + (kept ? kFold : first_fold(t)), end);
        // m: reference maximum of the raw scores; l: sum over this half of the keys; limit: growth of the maximum (base 2) that m follows
        float m = -INFINITY, l = 0.0f, limit = 8.0f;
        const bool some = b < end;
        bool first = true;
        // (a wait that ran out does not end the loop: the other warp of the pair would wait at the barrier for ever)
        for (; b < stop; ++b, phase ^= 1, first = false) {
            ok &= __all_sync(0xffffffffu, mbar_wait_within(&sm.s_full[t], phase, abort_flag, p.wait_ns)) != 0;
            tc_fence_after_sync();
            float s[64];
            tmem_ld_32x32(s_cols, reinterpret_cast<uint32_t(&)[32]>(s[0]));
            tmem_ld_32x32(s_cols + 32, reinterpret_cast<uint32_t(&)[32]>(s[32]));
            tmem_ld_wait();
            const int k0 = b * kTile;
            const bool masked = k0 < all_lo || k0 + kTile > all_hi;
            if (masked) {
                const int lo = row_lo - k0 - half * 64, hi = row_hi - k0 - half * 64;
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] = i >= lo && i < hi ? s[i] : -INFINITY;
            }
            float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < 60; i += 8)
#pragma unroll
                for (int j = 0; j < 4; ++j) top[j] = max_of(top[j], s[i + 2 * j], s[i + 2 * j + 1]);
            const float own = max_of(max_of(top[0], s[60], s[61]), max_of(top[1], s[62], s[63]), fmaxf(top[2], top[3]));
            sm.top[t][half][tile_row] = own;                 // (the partner has read the last one: S of this block came after its P)
            pair_sync();                                     // (also: both halves of S have been read, P may take their place)
            const float seen = fmaxf(m, fmaxf(own, sm.top[t][half ^ 1][tile_row]));
            // (-inf - -inf is NaN: no growth; the first number that a row sees is infinitely more than none)
            if (__any_sync(0xffffffffu, (seen - m) * scale > limit)) {
                const float factor = exp2_approx((m - (seen == -INFINITY ? 0.0f : seen)) * scale);
                m = seen;
                // The exponents are s * scale - m * scale in one rounding, but m * scale has its own: of scores far from zero, where its
                // half step would take P beyond every number (from 2^27 on), m is taken off the scores first, in every block.
                limit = fabsf(m * scale) >= 16384.0f && m != -INFINITY ? -1.0f : 8.0f;
                const float off = limit < 0.0f ? m : 0.0f;
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] -= off;
                l = nan_if_huge(l) * factor;                 // (before the factor hides it)
                if (!first) {
                    ok &= __all_sync(0xffffffffu, mbar_wait_within(&sm.o_done[t], phase ^ 1, abort_flag, p.wait_ns)) != 0;
                    tc_fence_after_sync();
#pragma unroll 1
                    for (int c = 0; c < D / 2; c += 16) {
                        uint32_t o[16];
                        tmem_ld_32x16(o_cols + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                        tmem_st_32x16(o_cols + c, o);
                    }
                }
            }
            const float shift = limit < 0.0f || m == -INFINITY ? kBits : fmaf(-m, scale, kBits);
            l += weights_of_scores<T, kByFma>(s, scale, shift, p_cols);
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_full[t]);
        }
        // ------------------------------------------------------------ output: half the features a thread
        const bool last = b >= end;
        pair_sync();
        sm.top[t][half][tile_row] = l;
        pair_sync();
        l += sm.top[t][half ^ 1][tile_row];
        l = nan_if_huge(l);
        if (!last) pair_sync();                              // (the next block's scores may be there already)
        if (ok && some) {
            ok = __all_sync(0xffffffffu, mbar_wait_within(&sm.o_done[t], phase ^ 1, abort_flag, p.wait_ns)) != 0;
            tc_fence_after_sync();
        }
        if (ok && tile_rows > 0) {
            const long long row = static_cast<long long>(w.at.row0 + token) * p.heads + head * p.group + index - token * p.group;
            const long long part = static_cast<long long>(share) * p.tokens * p.heads + row;
            float* part_dst = part_out + part * D + half * (D / 2);
            // Where the 4 features from 4 * i on of this thread's half are kept: nobody else reads them, so the 32 rows of a warp put
            // theirs side by side into one row of the output's shape after the other (whose rows all exist where the tile is full).
            auto kept_at = [&](int i) {
                constexpr int kEach = D / 4, kRowsEach = 32 / kEach;                   // pieces of a row; rows that 32 of them take
                const bool full = tile_rows >= kTile;
                const int r = full ? quad * 32 + (half * (kEach / 2) + i) * kRowsEach + lane / kEach : tile_row;
                const int at = w.row + t * kTile + r, tok = at / p.group;
                const long long to = static_cast<long long>(share) * p.tokens * p.heads + static_cast<long long>(w.at.row0 + tok) * p.heads + head * p.group + at - tok * p.group;
                return reinterpret_cast<float4*>(kept_out + to * D) + (full ? lane % kEach : half * (kEach / 2) + i);
            };
            float base = fmaf(m, scale, -kBits), here = 1.0f, there = 0.0f;       // factors of O and of what is kept
            if (kept && live) {
                const float2 ml = kept_ml[2 * part + half];
                const float top = fmaxf(base, ml.x);
                here = top == -INFINITY ? 0.0f : exp2_approx(base - top);
                there = top == -INFINITY ? 0.0f : exp2_approx(ml.x - top);
                base = top;
                l = fmaf(ml.y, there, l * here);
            }
            if (kept || !last) {                             // O and what is kept, to where it is kept or back to tensor memory
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 16) {
                    uint32_t o[16];
                    tmem_ld_32x16(o_cols + c, o);
                    tmem_ld_wait();
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            float4* at = kept_at((c + i) / 4);
                            const float4 old = kept ? *at : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            const float4 v = make_float4(fmaf(old.x, there, __uint_as_float(o[i]) * here), fmaf(old.y, there, __uint_as_float(o[i + 1]) * here),
                                                         fmaf(old.z, there, __uint_as_float(o[i + 2]) * here), fmaf(old.w, there, __uint_as_float(o[i + 3]) * here));
                            if (!last) *at = v;
                            o[i] = __float_as_uint(v.x);
                            o[i + 1] = __float_as_uint(v.y);
                            o[i + 2] = __float_as_uint(v.z);
                            o[i + 3] = __float_as_uint(v.w);
                        }
                    }
                    if (last) tmem_st_32x16(o_cols + c, o);
                }
                if (last) tmem_st_wait();
                else if (live) kept_ml[2 * part + half] = make_float2(base, l);
            }
            if (last) {
                const float inverse = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
                T* dst = static_cast<T*>(p.out) + (w.at.row0 + token) * p.ld_out + static_cast<long long>(head * p.group + index - token * p.group) * D + half * (D / 2);
#pragma unroll (D == 64 ? 2 : 1)
                for (int c = 0; c < D / 2; c += 16) {
                    uint32_t o[16];
                    if (some) {
                        tmem_ld_32x16(o_cols + c, o);
                        tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = 0;
                    }
                    if (!live) continue;
                    if (shares > 1) {
                        if (some) {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(part_dst + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        }
                    } else {
                        uint32_t v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = packed_of(__uint_as_float(o[2 * i]) * inverse, __uint_as_float(o[2 * i + 1]) * inverse, T());
                        *reinterpret_cast<uint4*>(dst + c) = make_uint4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                    }
                }
                if (live && half == 0) {
                    if (shares > 1) part_ml[part] = make_float2(base, l);
                    else if (p.lse != nullptr) p.lse[row] = l > 0.0f ? (base + log2f(l)) * kLn2 : (l == 0.0f ? -INFINITY : l);
                }
            }
        }
        kept = true;
        } while (b < end);
        });
    }
    if (!ok && lane == 0 && p.status != nullptr) atomicOr(p.status, 1);
    tc_fence_before_sync();
    __syncthreads();
    // where a wait ran out, whoever's: copies and products must end before the block's memory is given away
    if (*abort_flag != 0) {
        if (warp == kSoftmaxWarps) {
            for (int i = max(it - kSlots, 0); i < it; ++i) mbar_drain(&sm.full[i % kSlots], (i / kSlots) & 1);
        } else if (warp == kSoftmaxWarps + 1) {
            tc_commit_if(elect_one(), &sm.drained);           // (the same lane every time)
            mbar_drain(&sm.drained, 0);
        }
    }
    if (warp == kSoftmaxWarps + 1) tmem_dealloc(tmem, kColumns);
}

// out of the shares of a row's keys, in their order, a warp a row.
template <typename T, int D>
__global__ void __launch_bounds__(128)
shares_join_kernel(const PagedParams p, const int* share_count, const float2* part_ml, const float* part_out) {
    grid_dependents_launch();
    grid_dependency_wait();
    const int shares = *share_count;
    if (shares == 1) return;                     // (the rows are finished)
    const int token = blockIdx.x, lane = threadIdx.x % 32;
    // the request that has the token: the last one that starts at or before it (an empty one never is)
    int lo = 0, hi = p.requests;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, r = lo + lane * step;
        const uint32_t before = __ballot_sync(0xffffffffu, r < hi && p.starts[r] <= token);
        lo = min(lo + (before == 0 ? 0 : 31 - __clz(before)) * step, p.requests - 1);
        hi = min(lo + step, hi);
    }
    const PagedRequest at(p, lo);
    if (token < at.row0 || token >= at.row0 + at.n || at.n * p.group <= p.few_rows) return;
    constexpr int kWidth = D / 32;
    for (int h = blockIdx.y * 4 + threadIdx.x / 32; h < p.heads; h += gridDim.y * 4) {
        const long long row = static_cast<long long>(token) * p.heads + h, step = static_cast<long long>(p.tokens) * p.heads;
        float top = -INFINITY, sum = 0.0f, o[kWidth] = {};
        for (int s = lane; s < shares; s += 32) {
            const float2 ml = part_ml[s * step + row];
            if (ml.y != 0.0f) top = fmaxf(top, ml.x);
        }
#pragma unroll
        for (int off = 16; off > 0; off /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
#pragma unroll 4
        for (int s = 0; s < shares; ++s) {
            const float2 ml = part_ml[s * step + row];
            if (ml.y == 0.0f) continue;                      // (a share that saw nothing left no output)
            const float weight = exp2_approx(ml.x - top);
            sum = fmaf(weight, ml.y, sum);
#pragma unroll
            for (int e = 0; e < kWidth; ++e) o[e] = fmaf(weight, part_out[(s * step + row) * D + lane * kWidth + e], o[e]);
        }
        const float inverse = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
        T* dst = static_cast<T*>(p.out) + token * p.ld_out + static_cast<long long>(h) * D + lane * kWidth;
#pragma unroll
        for (int e = 0; e < kWidth; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = packed_of(o[e] * inverse, o[e + 1] * inverse, T());
        if (p.lse != nullptr && lane == 0) p.lse[row] = sum > 0.0f ? (top + log2f(sum)) * kLn2 : (sum == 0.0f ? -INFINITY : sum);
    }
}

template <typename T, int D>
static int launch(const PagedParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, int pairs, int shares, int* share_count, float2* part_ml,
                  float* part_out, float2* kept_ml, float* kept_out, cudaStream_t stream) {
    constexpr int bytes = sizeof(Smem<D>);
    static_assert(bytes <= 227 * 1024 / (3 - tiles<D>()) - (D == 64 ? 1024 : 0), "shared memory");
    const long long slots = pk100_sm_count() * (3 - tiles<D>()), columns = static_cast<long long>(pairs) * p.kv_heads;
    // Up to 32 requests at most 32 pairs a head do not exist: a block for each that may.  With more, blocks that find nothing to
    // do would cost more than the pass over the items (200 single tokens whose max_new is not known: 207 against 167 us; the pass
    // over the items costs few requests 11 us of two prompts and 3 of nine ragged chunks).
    auto run = [&](auto loop) -> int {
        constexpr auto kernel = paged_attention_chunk_kernel<T, D, decltype(loop)::value>;
        const cudaError_t granted = pk100_grant_smem<kernel>(bytes);
        if (granted != cudaSuccess) return static_cast<int>(granted);
        const long long most = columns * shares < slots ? columns * shares : slots, blocks = decltype(loop)::value || columns < most ? most : columns;
        pk100_launch_chained(kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads<D>()), bytes, stream, map_k, map_v, p, pairs, shares,
                             static_cast<unsigned>(slots), share_count, part_ml, part_out, kept_ml, kept_out);
        return pk100_launch_status();
    };
    return p.requests <= kOrdered ? run(std::false_type()) : run(std::true_type());
}

template <typename T, int D>
static int launch_join(const PagedParams& p, const int* share_count, const float2* part_ml, const float* part_out, cudaStream_t stream) {
    pk100_launch_chained(shares_join_kernel<T, D>, dim3(p.tokens, (p.heads + 3) / 4 < 8 ? (p.heads + 3) / 4 : 8), dim3(128), 0, stream, p, share_count, part_ml,
                         part_out);
    return pk100_launch_status();
}

}  // namespace chunk

int paged_attention_chunks(int type, int head_dim, const PagedParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, int pairs, int shares,
                           int* share_count, float2* part_ml, float* part_out, float2* kept_ml, float* kept_out, cudaStream_t stream) {
    if (type == PK100_TYPE_F16)
        return head_dim == 128 ? chunk::launch<__half, 128>(p, map_k, map_v, pairs, shares, share_count, part_ml, part_out, kept_ml, kept_out, stream)
                               : chunk::launch<__half, 64>(p, map_k, map_v, pairs, shares, share_count, part_ml, part_out, kept_ml, kept_out, stream);
    return head_dim == 128 ? chunk::launch<__nv_bfloat16, 128>(p, map_k, map_v, pairs, shares, share_count, part_ml, part_out, kept_ml, kept_out, stream)
                           : chunk::launch<__nv_bfloat16, 64>(p, map_k, map_v, pairs, shares, share_count, part_ml, part_out, kept_ml, kept_out, stream);
}

int paged_attention_join(int type, int head_dim, const PagedParams& p, const int* share_count, const float2* part_ml, const float* part_out, cudaStream_t stream) {
    if (type == PK100_TYPE_F16)
        return head_dim == 128 ? chunk::launch_join<__half, 128>(p, share_count, part_ml, part_out, stream) : chunk::launch_join<__half, 64>(p, share_count, part_ml, part_out, stream);
    return head_dim == 128 ? chunk::launch_join<__nv_bfloat16, 128>(p, share_count, part_ml, part_out, stream)
                           : chunk::launch_join<__nv_bfloat16, 64>(p, share_count, part_ml, part_out, stream);
}

}  // namespace pk100
