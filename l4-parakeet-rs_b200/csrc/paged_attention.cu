// Attention of new tokens over a paged key-value cache: the copy of new keys and values into their slots, the kernel
// for requests of few rows (single tokens), and the host side.
#include "paged_attention.cuh"

namespace pk100 {

// ------------------------------------------------------------- new keys and values into the cache
struct AppendParams {
    const uint16_t* key; const uint16_t* value; long long ld_key, ld_value;
    const long long* slots;
    uint16_t* key_cache; uint16_t* value_cache;
    long long page_stride, token_stride, head_stride;
    int tokens, kv_heads, head_dim, page_shift;
    long long capacity;                                // slots of the cache
    int* counts; int n_counts;                         // of the kernel behind: zeroed
    int* status;
};

// 16 bytes of keys and of values a thread; bound by HBM: 14 500 tokens of 4 heads of 128 (59 MB) 10 us, a decode step 3 us.
__global__ void __launch_bounds__(256)
paged_append_kernel(const AppendParams p) {
    grid_dependents_launch();
    grid_dependency_wait();
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < p.n_counts; i += gridDim.x * blockDim.x) p.counts[i] = 0;
    const int chunks = p.head_dim / 8, per_token = p.kv_heads * chunks;
    const long long work = static_cast<long long>(p.tokens) * per_token;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < work; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int t = static_cast<int>(i / per_token), part = static_cast<int>(i - static_cast<long long>(t) * per_token);
        const long long slot = p.slots[t];
        if (slot < 0) continue;
        if (slot >= p.capacity) {
            if (part == 0 && p.status != nullptr) atomicOr(p.status, PK100_STATUS_PAGE);
            continue;
        }
        const uint4 k = *reinterpret_cast<const uint4*>(p.key + t * p.ld_key + part * 8);
        const uint4 v = *reinterpret_cast<const uint4*>(p.value + t * p.ld_value + part * 8);
        const long long at = (slot >> p.page_shift) * p.page_stride + (slot & ((1 << p.page_shift) - 1)) * p.token_stride +
                             (part / chunks) * p.head_stride + (part % chunks) * 8;
        *reinterpret_cast<uint4*>(p.key_cache + at) = k;
        *reinterpret_cast<uint4*>(p.value_cache + at) = v;
    }
}

// ------------------------------------------------------------- few rows
constexpr int kRows = 16;             // (token, head) rows of a tile: the M of mma.sync
constexpr int kBlock = 64;            // keys of a stage
constexpr int kRowWarps = 4;          // that compute; one more loads
constexpr int kRowThreads = kRowWarps * 32 + 32;

// What a block found out about a tile of which it had a part: row maxima (log2 scale) and sums, and the unscaled output.
struct RowsPart { float m[kRows], l[kRows]; };

template <int D> constexpr int rows_stages() { return D == 128 ? 3 : 6; }

template <int D>
struct RowsSmem {
    uint8_t k[rows_stages<D>()][D / 64][kBlock * 128];
    uint8_t v[rows_stages<D>()][D / 64][kBlock * 128];
    uint8_t p[2][2][kRows * 128];              // weights cut off, and their rests
    float top[2][kRowWarps][kRows];
    float sum[kRowWarps][kRows];
    long long scan[kRowThreads / 32];
    uint64_t full[rows_stages<D>()], empty[rows_stages<D>()];
    long long base;
    int request, abort, last;
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_rows(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_rows(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ constexpr float weight_factor() { return static_cast<float>(1 << weight_bits<T>(0)); }     // (P is 1 at most)
__device__ __forceinline__ void row_warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kRowWarps * 32) : "memory"); }

// A request's work: tiles of 16 rows per key-value head, each over the key blocks that any row of the request sees
// (one at least, so that rows without keys are written).  Zero where another kernel has the request.
struct RowsShape {
    PagedRequest at;
    int tiles, block0, blocks;
    __device__ __forceinline__ RowsShape(const PagedParams& p, int r) : at(p, r) {
        const int rows = at.n * p.group;
        tiles = rows > 0 && rows <= p.few_rows ? (rows + kRows - 1) / kRows : 0;
        block0 = at.lo(p, 0) / kBlock;
        blocks = max((at.hi(p, at.n - 1) + kBlock - 1) / kBlock - block0, 1);
    }
    __device__ __forceinline__ long long units(const PagedParams& p) const { return static_cast<long long>(tiles) * blocks * p.kv_heads; }
};

// One run over a block's units, the same for the warp that loads and those that compute:
// f(shape, request, head, tile, first unit of the tile, first and last block of this part, whole tile)
template <typename F>
__device__ __forceinline__ void rows_walk(const PagedParams& p, int request, long long base, long long unit, long long end, F&& f) {
    while (unit < end) {
        const RowsShape s(p, request);
        const long long units = s.units(p);
        if (unit >= base + units) {
            base += units;
            ++request;
            continue;
        }
        const long long tile_at = (unit - base) / s.blocks;
        const int block = static_cast<int>(unit - base - tile_at * s.blocks);
        const int count = static_cast<int>(min(static_cast<long long>(s.blocks - block), end - unit));
        f(s, request, static_cast<int>(tile_at / s.tiles), static_cast<int>(tile_at % s.tiles), base + tile_at * s.blocks, block, block + count,
          count == s.blocks);
        unit += count;
    }
}

// out of the parts that blocks [before, last] had of a row, by a warp.  (Written by other SMs: read past the L1.)
template <typename T, int D>
__device__ __forceinline__ void join_row(const PagedParams& p, const PagedRequest& at, int head, int index, int row, int before, int last,
                                         long long opening, const RowsPart* parts, const float* part_out) {
    const int lane = threadIdx.x % 32;
    auto part_of = [&](int block) { return block == before ? opening : 2ll * block; };
    float top = -INFINITY;
    for (int k = before + lane; k <= last; k += 32) top = fmaxf(top, __ldcg(&parts[part_of(k)].m[row]));
#pragma unroll
    for (int off = 16; off > 0; off /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float zero = top == -INFINITY ? 0.0f : top;
    constexpr int kWidth = D / 32;
    float o[kWidth] = {}, sum = 0.0f;
    for (int k0 = before; k0 <= last; k0 += 32) {
        const int count = min(32, last - k0 + 1);
        float weight = 0.0f;
        if (lane < count) {
            const RowsPart& q = parts[part_of(k0 + lane)];
            weight = exp2_approx(__ldcg(&q.m[row]) - zero);
            sum += weight * __ldcg(&q.l[row]);
        }
#pragma unroll 8
        for (int k = 0; k < count; ++k) {
            const float w = __shfl_sync(0xffffffffu, weight, k);
            const float* src = part_out + (part_of(k0 + k) * kRows + row) * D + lane * kWidth;
            if constexpr (kWidth == 4) {
                const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
                o[0] = fmaf(w, v.x, o[0]);
                o[1] = fmaf(w, v.y, o[1]);
                o[2] = fmaf(w, v.z, o[2]);
                o[3] = fmaf(w, v.w, o[3]);
            } else {
                const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
                o[0] = fmaf(w, v.x, o[0]);
                o[1] = fmaf(w, v.y, o[1]);
            }
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float inverse = sum > 0.0f ? 1.0f / (sum * weight_factor<T>()) : (sum == 0.0f ? 0.0f : sum);
    const int i = index / p.group;
    const long long h = head * p.group + index - i * p.group;
    T* dst = static_cast<T*>(p.out) + (at.row0 + i) * p.ld_out + h * D + lane * kWidth;
#pragma unroll
    for (int e = 0; e < kWidth; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = packed_of(o[e] * inverse, o[e + 1] * inverse, T());
    if (p.lse != nullptr && lane == 0) p.lse[static_cast<long long>(at.row0 + i) * p.heads + h] = (top + log2f(sum)) * kLn2;
}

// Single tokens are bound by reading the cache once.  All (request, head, 64-key block) units of the step lie on one
// line that the blocks share evenly, whatever the lengths: a block's part of the line is a run of blocks, with a
// tile's beginning or end wherever they fall; what a block has of a tile that others share goes to the workspace, and
// the block that comes last adds the parts up, in the order of the blocks.  The query heads of a key-value head are rows of one 16-row tile, so
// keys and values are read once for all of them.
// A warp requests 64-key stages by TMA (a page or part of one a box, 128-byte swizzle), two blocks an SM keep up to
// six of them in flight.  Q.K: each of four warps 16 keys; the row maxima are exchanged, so that all warps scale
// alike; P through shared memory; P.V: each warp a quarter of the features.
// Scores, maxima, sums and outputs are fp32; P goes to the tensor cores in two numbers of the type of V, the weight cut off and
// the rounded rest: one alone had cost what the rounding of the output costs, two cost 2 us of 128, as long as the cache's bytes
// decide.  The tensor cores cut off what falls below the last
// bit of the sum that they add to: a block's products begin at zero and are added to the row's by the FMA pipe, which rounds.
// (One sum over 2^19 keys was 4e-3 low.)  l is compensated: many small weights behind a large one are not lost in it.
// One token of 48 requests over 320 to 12 000 keys, 32 / 8 heads of 128 (712 MB): 128 to 131 us, 5.4 to 5.6 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads, 2)
paged_attention_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedParams p,
                            const bool beside, int* counts, RowsPart* parts, float* part_out) {
    extern __shared__ uint8_t rows_raw[];
    constexpr int kStages = rows_stages<D>(), kHalves = D / 64;
    RowsSmem<D>& sm = *reinterpret_cast<RowsSmem<D>*>((reinterpret_cast<uintptr_t>(rows_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    grid_dependents_launch();
    if (tid == 0) {
        sm.abort = 0;
        sm.request = 0;
        sm.base = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], kRowWarps);
        }
        fence_barrier_init();
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    // beside: the chunk kernel is in front.  It lets this one start when all that stands before it is complete, and the
    // two have nothing to do with each other: this one runs where that leaves SMs free and waits for it at its end, so
    // that what comes behind finds both complete.
    if (!beside) grid_dependency_wait();

    // this block's units: where the requests' prefix sum crosses them
    const int each = (p.requests + kRowThreads - 1) / kRowThreads, r0 = min(tid * each, p.requests), r1 = min(r0 + each, p.requests);
    long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += RowsShape(p, r).units(p);
    long long upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += v;
    }
    if (lane == 31) sm.scan[warp] = upto;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) {
        if (w < warp) upto += sm.scan[w];
        total += sm.scan[w];
    }
    const long long share = max((total + gridDim.x - 1) / gridDim.x, 1ll);
    const long long begin = min(share * blockIdx.x, total), end = min(begin + share, total);
    if (begin < end && upto - mine <= begin && begin < upto) {          // one thread
        long long base = upto - mine;
        int r = r0;
        for (long long u; base + (u = RowsShape(p, r).units(p)) <= begin; ++r) base += u;
        sm.request = r;
        sm.base = base;
    }
    __syncthreads();
    const int first_request = sm.request;
    const long long first_base = sm.base;
    volatile int* abort_flag = &sm.abort;
    int it = 0;                                          // stages of this role so far
    bool ok = true;

    if (warp == kRowWarps) {
        // ------------------------------------------------------------ loads
        const int box = min(kBlock, 1 << p.page_shift), boxes = kBlock / box;
        bool bad = false;
        rows_walk(p, first_request, first_base, begin, end, [&](const RowsShape& s, int request, int head, int tile, long long, int b0, int b1, bool) {
            const int row_first = tile * kRows / p.group, row_last = min((tile * kRows + kRows - 1) / p.group, s.at.n - 1);
            const int lo = s.at.lo(p, row_first), hi = s.at.hi(p, row_last);
            const int* table = p.table + static_cast<long long>(request) * p.max_pages;
            bad |= s.at.cut;
            const int from = max(s.block0 + b0, lo / kBlock), to = min(s.block0 + b1, (hi + kBlock - 1) / kBlock);
            int held = -32, id = 0;                         // pages [held, held + 32): one a lane
            for (int b = from; ok && b < to; ++b, ++it) {
                const int stage = it % kStages;
                ok = __all_sync(0xffffffffu, mbar_look_within(&sm.empty[stage], (it / kStages + 1) & 1, abort_flag, p.wait_ns)) != 0;
                if (!ok) break;
                const int key = b * kBlock + min(lane, boxes - 1) * box, page = key >> p.page_shift;
                const int last = (b * kBlock + kBlock - 1) >> p.page_shift;
                if (last >= held + 32) {
                    held = (b * kBlock) >> p.page_shift;
                    id = held + lane < p.max_pages ? table[held + lane] : -1;
                }
                int mine_id = __shfl_sync(0xffffffffu, id, page - held);
                const bool need = lane < boxes && key < hi && key + box > lo;
                if (need && (mine_id < 0 || mine_id >= p.pages)) {
                    bad = true;
                    mine_id = p.pages;                      // outside the tensor: zeros
                }
                const int count = __popc(__ballot_sync(0xffffffffu, need));
                if (lane == 0) mbar_arrive_expect_tx(&sm.full[stage], count * box * 128 * kHalves * 2);
                __syncwarp();
                if (need) {
                    const int token = key & ((1 << p.page_shift) - 1);
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        tma_load_4d(sm.k[stage][half] + lane * box * 128, &map_k, &sm.full[stage], half * 64, token, head, mine_id);
                        tma_load_4d(sm.v[stage][half] + lane * box * 128, &map_v, &sm.full[stage], half * 64, token, head, mine_id);
                    }
                }
                __syncwarp();
            }
        });
        if (bad && p.status != nullptr) atomicOr(p.status, PK100_STATUS_PAGE);
    } else {
        // ------------------------------------------------------------ products and softmax
        const int g = lane / 4, c = lane % 4;
        constexpr int kSteps = D / 16, kFeatureTiles = D / 32;          // k steps of Q.K; 8-feature tiles of a warp's quarter
        constexpr float kFactor = weight_factor<T>();                   // of P and so of the output, not of the sums
        rows_walk(p, first_request, first_base, begin, end,
                  [&](const RowsShape& s, int request, int head, int tile, long long tile_first, int b0, int b1, bool whole) {
            const int rows = s.at.n * p.group - tile * kRows;           // rows of the tile that exist (or more)
            const int i0 = (tile * kRows + g) / p.group, i1 = (tile * kRows + g + 8) / p.group;
            const int row_first = tile * kRows / p.group, row_last = min((tile * kRows + kRows - 1) / p.group, s.at.n - 1);
            const int lo = s.at.lo(p, row_first), hi = s.at.hi(p, row_last);
            // bounds of this thread's two rows, and those that every row of the tile keeps
            const int lo0 = s.at.lo(p, i0), lo1 = s.at.lo(p, i1), hi0 = g < rows ? s.at.hi(p, i0) : 0, hi1 = g + 8 < rows ? s.at.hi(p, i1) : 0;
            const int all_lo = s.at.lo(p, row_last), all_hi = s.at.hi(p, row_first);
            uint32_t q[kSteps][4];
            {
                const T* src0 = static_cast<const T*>(p.query) + (s.at.row0 + i0) * p.ld_query + static_cast<long long>(head * p.group + tile * kRows + g - i0 * p.group) * D;
                const T* src1 = static_cast<const T*>(p.query) + (s.at.row0 + i1) * p.ld_query + static_cast<long long>(head * p.group + tile * kRows + g + 8 - i1 * p.group) * D;
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) {
                    q[ks][0] = g < rows ? *reinterpret_cast<const uint32_t*>(src0 + ks * 16 + 2 * c) : 0;
                    q[ks][1] = g + 8 < rows ? *reinterpret_cast<const uint32_t*>(src1 + ks * 16 + 2 * c) : 0;
                    q[ks][2] = g < rows ? *reinterpret_cast<const uint32_t*>(src0 + ks * 16 + 8 + 2 * c) : 0;
                    q[ks][3] = g + 8 < rows ? *reinterpret_cast<const uint32_t*>(src1 + ks * 16 + 8 + 2 * c) : 0;
                }
            }
            float o[kFeatureTiles][4];
#pragma unroll
            for (int j = 0; j < kFeatureTiles; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, e0 = 0.0f, e1 = 0.0f;      // e: what l has too much

            const int from = max(s.block0 + b0, lo / kBlock), to = min(s.block0 + b1, (hi + kBlock - 1) / kBlock);
            for (int b = from; b < to; ++b, ++it) {
                const int stage = it % kStages, buf = it & 1;
                // (one that ran out does not end the loop: the other warps would wait at the barriers for ever)
                ok &= mbar_look_within(&sm.full[stage], (it / kStages) & 1, abort_flag, p.wait_ns);
                __syncwarp();
                float sc[2][4] = {};
                const int key_row = 16 * warp + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) {
                    uint32_t kf[4];
                    const int chunk = (ks * 2 + ((lane >> 3) & 1)) & 7;
                    ldmatrix_x4(kf, smem_u32(sm.k[stage][ks / 4]) + key_row * 128 + ((chunk ^ (key_row & 7)) << 4));
                    mma_rows(sc[0], q[ks], kf[0], kf[1], T());
                    mma_rows(sc[1], q[ks], kf[2], kf[3], T());
                }
                const int k0 = b * kBlock;
                if (k0 < all_lo || k0 + kBlock > all_hi) {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = k0 + 16 * warp + 8 * nt + 2 * c + e;
                            sc[nt][e] = key >= lo0 && key < hi0 ? sc[nt][e] * p.scale_log2 : -INFINITY;
                            sc[nt][2 + e] = key >= lo1 && key < hi1 ? sc[nt][2 + e] * p.scale_log2 : -INFINITY;
                        }
                } else {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[nt][e] *= p.scale_log2;
                }
                float t0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
                float t1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
                for (int off = 1; off < 4; off *= 2) {
                    t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, off));
                    t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, off));
                }
                if (c == 0) {
                    sm.top[buf][warp][g] = t0;
                    sm.top[buf][warp][g + 8] = t1;
                }
                row_warps_sync();
                float n0 = m0, n1 = m1;
#pragma unroll
                for (int w = 0; w < kRowWarps; ++w) {
                    n0 = fmaxf(n0, sm.top[buf][w][g]);
                    n1 = fmaxf(n1, sm.top[buf][w][g + 8]);
                }
                const float z0 = n0 == -INFINITY ? 0.0f : n0, z1 = n1 == -INFINITY ? 0.0f : n1;     // nothing seen yet: exp2(-inf) = 0
                const float a0 = exp2_approx(m0 - z0), a1 = exp2_approx(m1 - z1);
                m0 = n0;
                m1 = n1;
                float b0 = 0.0f, b1 = 0.0f;                              // sums of the block
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const float x0 = exp2_approx(sc[nt][0] - z0), x1 = exp2_approx(sc[nt][1] - z0);
                    const float y0 = exp2_approx(sc[nt][2] - z1), y1 = exp2_approx(sc[nt][3] - z1);
                    b0 += x0 + x1;
                    b1 += y0 + y1;
                    const int chunk = 2 * warp + nt;
                    auto put = [&](float u, float v, int row) {
                        // cut off, so that the rest has no other sign, and the rest of what is not zero not zero: an infinite
                        // value times the two is infinite (its last bit is set where the weight's halves, plus 0x7fff, reach the sign)
                        const uint32_t near = packed_below(u, v, T());
                        const float2 r = floats_of(near, T());
                        const int at = row * 128 + ((chunk ^ g) << 4) + 4 * c;
                        *reinterpret_cast<uint32_t*>(&sm.p[buf][0][at]) = near;
                        *reinterpret_cast<uint32_t*>(&sm.p[buf][1][at]) = packed_of(u - r.x, v - r.y, T()) | (((near + 0x7fff7fffu) >> 15) & 0x00010001u);
                    };
                    put(x0 * kFactor, x1 * kFactor, g);
                    put(y0 * kFactor, y1 * kFactor, g + 8);
                }
                add_compensated(l0, e0, a0, b0);
                add_compensated(l1, e1, a1, b1);
                float pv[kFeatureTiles][4] = {};
                row_warps_sync();
                const bool ragged = k0 < lo || k0 + kBlock > hi;         // keys that no row sees: their values may be anything
                const int p_row = (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                for (int ks = 0; ks < kBlock / 16; ++ks) {
                    uint32_t pf[4], rest[4];
                    const uint32_t p_at = smem_u32(sm.p[buf][0]) + p_row * 128 + (((ks * 2 + (lane >> 4)) ^ (p_row & 7)) << 4);
                    ldmatrix_x4(pf, p_at);
                    ldmatrix_x4(rest, p_at + kRows * 128);
                    const int v_row = ks * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                    for (int j = 0; j < kFeatureTiles / 2; ++j) {
                        uint32_t vf[4];
                        const int chunk = warp * kFeatureTiles + 2 * j + (lane >> 4);
                        ldmatrix_x4_trans(vf, smem_u32(sm.v[stage][chunk / 8]) + v_row * 128 + (((chunk & 7) ^ (v_row & 7)) << 4));
                        if (ragged) {
                            const int key = k0 + ks * 16 + 2 * c;
                            auto mask = [&](int k) { return (k >= lo && k < hi ? 0xffffu : 0u) | (k + 1 >= lo && k + 1 < hi ? 0xffff0000u : 0u); };
                            const uint32_t near = mask(key), far = mask(key + 8);
                            vf[0] &= near;
                            vf[1] &= far;
                            vf[2] &= near;
                            vf[3] &= far;
                        }
                        mma_rows(pv[2 * j], pf, vf[0], vf[1], T());
                        mma_rows(pv[2 * j + 1], pf, vf[2], vf[3], T());
                        mma_rows(pv[2 * j], rest, vf[0], vf[1], T());
                        mma_rows(pv[2 * j + 1], rest, vf[2], vf[3], T());
                    }
                }
#pragma unroll
                for (int j = 0; j < kFeatureTiles; ++j) {
                    o[j][0] = fmaf(o[j][0], a0, pv[j][0]);
                    o[j][1] = fmaf(o[j][1], a0, pv[j][1]);
                    o[j][2] = fmaf(o[j][2], a1, pv[j][2]);
                    o[j][3] = fmaf(o[j][3], a1, pv[j][3]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.empty[stage]);
            }

            // sums over the keys of all warps
#pragma unroll
            for (int off = 1; off < 4; off *= 2) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, off);
                l1 += __shfl_xor_sync(0xffffffffu, l1, off);
            }
            row_warps_sync();                                            // (sm.sum of the tile before has been read)
            if (c == 0) {
                sm.sum[warp][g] = l0;
                sm.sum[warp][g + 8] = l1;
            }
            row_warps_sync();
            l0 = l1 = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                l0 += sm.sum[w][g];
                l1 += sm.sum[w][g + 8];
            }
            if (whole) {
                const float r0i = l0 > 0.0f ? 1.0f / (l0 * kFactor) : (l0 == 0.0f ? 0.0f : l0), r1i = l1 > 0.0f ? 1.0f / (l1 * kFactor) : (l1 == 0.0f ? 0.0f : l1);
                const long long h0 = head * p.group + tile * kRows + g - i0 * p.group, h1 = head * p.group + tile * kRows + g + 8 - i1 * p.group;
                T* dst0 = static_cast<T*>(p.out) + (s.at.row0 + i0) * p.ld_out + h0 * D + warp * (D / 4) + 2 * c;
                T* dst1 = static_cast<T*>(p.out) + (s.at.row0 + i1) * p.ld_out + h1 * D + warp * (D / 4) + 2 * c;
#pragma unroll
                for (int j = 0; j < kFeatureTiles; ++j) {
                    if (g < rows) *reinterpret_cast<uint32_t*>(dst0 + 8 * j) = packed_of(o[j][0] * r0i, o[j][1] * r0i, T());
                    if (g + 8 < rows) *reinterpret_cast<uint32_t*>(dst1 + 8 * j) = packed_of(o[j][2] * r1i, o[j][3] * r1i, T());
                }
                if (p.lse != nullptr && warp == 0 && c == 0) {
                    if (g < rows) p.lse[static_cast<long long>(s.at.row0 + i0) * p.heads + h0] = (m0 + log2f(l0)) * kLn2;
                    if (g + 8 < rows) p.lse[static_cast<long long>(s.at.row0 + i1) * p.heads + h1] = (m1 + log2f(l1)) * kLn2;
                }
            } else {
                // the part that this block's run begins with is its first, the one that it ends with its second
                const long long part = 2ll * blockIdx.x + (tile_first + b0 == begin ? 0 : 1);
                float* dst = part_out + part * kRows * D + warp * (D / 4) + 2 * c;
#pragma unroll
                for (int j = 0; j < kFeatureTiles; ++j) {
                    *reinterpret_cast<float2*>(dst + g * D + 8 * j) = make_float2(o[j][0], o[j][1]);
                    *reinterpret_cast<float2*>(dst + (g + 8) * D + 8 * j) = make_float2(o[j][2], o[j][3]);
                }
                if (warp == 0 && c == 0) {
                    parts[part].m[g] = m0;
                    parts[part].m[g + 8] = m1;
                    parts[part].l[g] = l0;
                    parts[part].l[g + 8] = l1;
                }
                // the last of the tile's blocks adds the parts up
                __threadfence();
                row_warps_sync();
                const int before = static_cast<int>(tile_first / share), last = static_cast<int>((tile_first + s.blocks - 1) / share);
                if (tid == 0) sm.last = atomicAdd(&counts[before], 1) == last - before;
                row_warps_sync();
                if (sm.last) {
                    __threadfence();
                    const long long opening = 2ll * before + (tile_first == share * before ? 0 : 1);      // the others are first parts
                    for (int row = warp; row < min(rows, kRows); row += kRowWarps)
                        join_row<T, D>(p, s.at, head, tile * kRows + row, row, before, last, opening, parts, part_out);
                }
            }
        });
    }
    // A wait that ran out, the loader's or a reader's, is reported, and its warp stays until the copies have landed: the block's
    // memory is given away when all its warps have left.
    if (__any_sync(0xffffffffu, !ok)) {
        if (lane == 0 && p.status != nullptr) atomicOr(p.status, 1);
        for (int i = max(it - kStages, 0); i < it; ++i) mbar_drain(&sm.full[i % kStages], (i / kStages) & 1);
    }
    if (beside) grid_dependency_wait();
}

// ------------------------------------------------------------- host
// The tensor map of a cache: boxes of 64 features by a page or a block of keys.
static int cache_map(CUtensorMap* map, const void* base, const pk100_paged_attention_args& a) {
    const unsigned long long dims[4] = {static_cast<unsigned long long>(a.head_dim), static_cast<unsigned long long>(a.page_size),
                                        static_cast<unsigned long long>(a.kv_heads), static_cast<unsigned long long>(a.pages)};
    // (an extent of one has no distance)
    const unsigned long long strides[3] = {2ull * a.token_stride, 2ull * (a.kv_heads > 1 ? a.head_stride : a.token_stride),
                                           2ull * (a.pages > 1 ? a.page_stride : a.token_stride)};
    const unsigned box[4] = {64, static_cast<unsigned>(a.page_size < kBlock ? a.page_size : kBlock), 1, 1};
    return pk100_tensor_map_4d(map, base, dims, strides, box);
}

// Where the workspace's arrays lie.
struct PagedPlan {
    int grid;                                            // blocks of the few-row kernel
    int pairs, shares;                                   // of the other one
    long long counts, parts, part_out, share_count, share_ml, share_out, kept_ml, kept_out, bytes;
};

static long long round256(long long n) { return (n + 255) / 256 * 256; }

static PagedPlan paged_plan_of(const pk100_paged_attention_args& a) {
    PagedPlan plan{};
    const int group = a.heads / a.kv_heads;
    // no more blocks than units can exist
    const long long tiles = static_cast<long long>(a.tokens) * group / kRows + a.requests;
    const long long blocks = (static_cast<long long>(a.max_pages) * a.page_size + kBlock - 1) / kBlock;
    const long long most = 2ll * pk100_sm_count();
    plan.grid = static_cast<int>(tiles * a.kv_heads >= most || tiles * a.kv_heads * blocks >= most ? most : tiles * a.kv_heads * blocks);
    plan.counts = 0;
    plan.parts = round256(plan.grid * 4ll);
    plan.part_out = plan.parts + round256(2ll * plan.grid * static_cast<long long>(sizeof(RowsPart)));
    plan.share_count = plan.part_out + round256(2ll * plan.grid * kRows * a.head_dim * 4);
    plan.share_ml = plan.share_count + 256;
    // Keys are shared out where the pairs of tiles leave SMs idle: few new tokens over a long cache.
    const long long rows = static_cast<long long>(a.tokens) * group, each = pair_rows(a.head_dim);
    const long long items = (rows + each - 1) / each * a.kv_heads;
    plan.pairs = static_cast<int>(rows / each) + a.requests;
    const long long by_keys = blocks / 8;                // 512 keys a share at least
    long long shares = items > 0 ? pk100_sm_count() * (256 / each) / items : 1;      // (two blocks of one tile an SM)
    if (shares > by_keys) shares = by_keys;
    plan.shares = shares < 1 ? 1 : static_cast<int>(shares);
    const long long share_rows = plan.shares > 1 ? static_cast<long long>(plan.shares) * a.tokens * a.heads : 0;
    plan.share_out = plan.share_ml + round256(share_rows * 8);
    const long long kept_rows = blocks * kBlock > kFoldKeys / 2 ? static_cast<long long>(plan.shares) * a.tokens * a.heads : 0;
    plan.kept_ml = plan.share_out + round256(share_rows * a.head_dim * 4);
    plan.kept_out = plan.kept_ml + round256(kept_rows * 16);
    plan.bytes = plan.kept_out + round256(kept_rows * a.head_dim * 4);
    return plan;
}

static int paged_check(const pk100_paged_attention_args* a) {
    if (a == nullptr) return PK100_ERR_NULL;
    if (a->type != PK100_TYPE_F16 && a->type != PK100_TYPE_BF16) return PK100_ERR_UNSUPPORTED;
    if (a->tokens < 0 || a->requests < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->pages <= 0 || a->max_pages <= 0) return PK100_ERR_SHAPE;
    if (a->heads % a->kv_heads != 0) return PK100_ERR_SHAPE;
    if (a->head_dim != 64 && a->head_dim != 128) return PK100_ERR_UNSUPPORTED;
    if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64 && a->page_size != 128 && a->page_size != 256) return PK100_ERR_UNSUPPORTED;
    if (static_cast<long long>(a->max_pages) * a->page_size > (1ll << 30) || static_cast<long long>(a->tokens) * a->heads > (1ll << 30) ||
        static_cast<long long>(a->requests) * a->heads > (1ll << 30))
        return PK100_ERR_LIMIT;
    return PK100_OK;
}

template <typename T, int D>
static int launch_rows(const pk100_paged_attention_args& a, const PagedParams& p, const PagedPlan& plan, const CUtensorMap& map_k,
                       const CUtensorMap& map_v, bool beside, cudaStream_t stream) {
    constexpr auto kernel = paged_attention_rows_kernel<T, D>;
    constexpr int bytes = sizeof(RowsSmem<D>) + 1024;
    const cudaError_t granted = pk100_grant_smem<kernel>(bytes);
    if (granted != cudaSuccess) return static_cast<int>(granted);
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    RowsPart* parts = reinterpret_cast<RowsPart*>(ws + plan.parts);
    float* part_out = reinterpret_cast<float*>(ws + plan.part_out);
    pk100_launch_chained(kernel, dim3(plan.grid), dim3(kRowThreads), bytes, stream, map_k, map_v, p, beside, reinterpret_cast<int*>(ws + plan.counts),
                         parts, part_out);
    return pk100_launch_status();
}

}  // namespace pk100

using namespace pk100;

extern "C" long long pk100_paged_attention_workspace_bytes(const pk100_paged_attention_args* a) {
    return paged_check(a) == PK100_OK ? paged_plan_of(*a).bytes : 0;
}

extern "C" int pk100_paged_attention(void* stream_v, const pk100_paged_attention_args* a) {
    int rc = paged_check(a);
    if (rc != PK100_OK) return rc;
    if (a->tokens == 0 || (a->requests == 0 && a->key == nullptr)) return PK100_OK;      // (without requests new keys are written all the same)
    if (a->query == nullptr || a->key_cache == nullptr || a->value_cache == nullptr || a->out == nullptr || a->workspace == nullptr) return PK100_ERR_NULL;
    if (a->requests > 0 && (a->starts == nullptr || a->lengths == nullptr || a->block_table == nullptr)) return PK100_ERR_NULL;
    if (a->key != nullptr && (a->value == nullptr || a->slots == nullptr)) return PK100_ERR_NULL;
    const long long row = static_cast<long long>(a->heads) * a->head_dim, kv_row = static_cast<long long>(a->kv_heads) * a->head_dim;
    auto bad_ld = [&](long long ld, long long width) { return a->tokens > 1 && (ld < width || ld % 8 != 0); };     // (a single row has no distance)
    if (bad_ld(a->ld_query, row) || bad_ld(a->ld_out, row)) return PK100_ERR_SHAPE;
    if (a->key != nullptr && (bad_ld(a->ld_key, kv_row) || bad_ld(a->ld_value, kv_row))) return PK100_ERR_SHAPE;
    const long long longest = 1ll << 38;                      // (a tensor map's strides are below 2^40 bytes)
    if (a->token_stride < a->head_dim || a->token_stride % 8 != 0 || a->token_stride >= longest) return PK100_ERR_SHAPE;
    if (a->kv_heads > 1 && (a->head_stride < a->head_dim || a->head_stride % 8 != 0 || a->head_stride >= longest)) return PK100_ERR_SHAPE;
    if (a->pages > 1 && (a->page_stride < a->head_dim || a->page_stride % 8 != 0 || a->page_stride >= longest)) return PK100_ERR_SHAPE;
    auto off = [](const void* ptr, unsigned bytes) { return reinterpret_cast<uintptr_t>(ptr) % bytes != 0; };
    if (off(a->query, 16) || off(a->out, 16) || off(a->key_cache, 16) || off(a->value_cache, 16) || off(a->workspace, 256)) return PK100_ERR_ALIGN;
    if (a->key != nullptr && (off(a->key, 16) || off(a->value, 16) || off(a->slots, 8))) return PK100_ERR_ALIGN;
    if (off(a->starts, 4) || off(a->lengths, 4) || off(a->block_table, 4) || off(a->lse, 4) || off(a->status, 4)) return PK100_ERR_ALIGN;
    const PagedPlan plan = paged_plan_of(*a);
    if (a->workspace_bytes < plan.bytes) return PK100_ERR_LIMIT;
    CUtensorMap map_k, map_v;
    if ((rc = cache_map(&map_k, a->key_cache, *a)) != PK100_OK || (rc = cache_map(&map_v, a->value_cache, *a)) != PK100_OK) return rc;

    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    PagedParams p{};
    p.query = a->query; p.ld_query = a->ld_query;
    p.out = a->out; p.ld_out = a->ld_out; p.lse = a->lse;
    p.starts = a->starts; p.lengths = a->lengths; p.table = a->block_table;
    p.tokens = a->tokens; p.requests = a->requests; p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads;
    p.pages = a->pages; p.max_pages = a->max_pages;
    while ((1 << p.page_shift) < a->page_size) ++p.page_shift;
    p.causal = a->causal != 0;
    p.window = a->window <= 0 ? 0 : (a->window < (1 << 30) ? a->window : (1 << 30));
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.few_rows = kRows;
    p.status = a->status;
    p.wait_ns = pk100_wait_limit();
    // Where no request has more rows than a tile of the few-row kernel, it takes them all; the hint may be wrong, so it does then, too.
    // 16 rows by it and 17 and more by the chunk kernel: single tokens of 16 even requests with 16 heads to a key-value head 37.4 us
    // against 33.7, with 20 heads 38.2 against 33.5; of 48 ragged ones, which the few-row kernel shares out, 47.8 against 114 and 58.9 against 113.
    const int most_new = a->max_new > 0 && a->max_new < a->tokens ? a->max_new : a->tokens;
    const bool many = static_cast<long long>(most_new) * p.group > kRows;
    if (!many) p.few_rows = 0x7fffffff;
    if (a->key != nullptr) {
        AppendParams w{};
        w.key = static_cast<const uint16_t*>(a->key); w.value = static_cast<const uint16_t*>(a->value);
        w.ld_key = a->ld_key; w.ld_value = a->ld_value; w.slots = a->slots;
        w.key_cache = static_cast<uint16_t*>(a->key_cache); w.value_cache = static_cast<uint16_t*>(a->value_cache);
        w.page_stride = a->page_stride; w.token_stride = a->token_stride; w.head_stride = a->head_stride;
        w.tokens = a->tokens; w.kv_heads = a->kv_heads; w.head_dim = a->head_dim; w.page_shift = p.page_shift;
        w.capacity = static_cast<long long>(a->pages) * a->page_size;
        w.counts = reinterpret_cast<int*>(static_cast<uint8_t*>(a->workspace) + plan.counts);
        w.n_counts = plan.grid;
        w.status = a->status;
        const long long work = a->tokens * (kv_row / 8), blocks = (work + 255) / 256, most = 8ll * pk100_sm_count();
        pk100_launch_chained(paged_append_kernel, dim3(static_cast<int>(blocks < most ? blocks : most)), dim3(256), 0, stream, w);
        if ((rc = pk100_launch_status()) != PK100_OK || a->requests == 0) return rc;
    } else {
        const cudaError_t err = cudaMemsetAsync(static_cast<uint8_t*>(a->workspace) + plan.counts, 0, plan.grid * 4ull, stream);
        if (err != cudaSuccess) return static_cast<int>(err);
    }
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    int* share_count = reinterpret_cast<int*>(ws + plan.share_count);
    float2* share_ml = reinterpret_cast<float2*>(ws + plan.share_ml);
    float* share_out = reinterpret_cast<float*>(ws + plan.share_out);
    float2* kept_ml = reinterpret_cast<float2*>(ws + plan.kept_ml);
    float* kept_out = reinterpret_cast<float*>(ws + plan.kept_out);
    if (many && (rc = paged_attention_chunks(a->type, a->head_dim, p, map_k, map_v, plan.pairs, plan.shares, share_count, share_ml, share_out, kept_ml, kept_out, stream)) != PK100_OK)
        return rc;
    if (a->type == PK100_TYPE_F16)
        rc = a->head_dim == 128 ? launch_rows<__half, 128>(*a, p, plan, map_k, map_v, many, stream) : launch_rows<__half, 64>(*a, p, plan, map_k, map_v, many, stream);
    else
        rc = a->head_dim == 128 ? launch_rows<__nv_bfloat16, 128>(*a, p, plan, map_k, map_v, many, stream)
                                : launch_rows<__nv_bfloat16, 64>(*a, p, plan, map_k, map_v, many, stream);
    if (rc != PK100_OK || !many || plan.shares == 1) return rc;
    return paged_attention_join(a->type, a->head_dim, p, share_count, share_ml, share_out, stream);
}
