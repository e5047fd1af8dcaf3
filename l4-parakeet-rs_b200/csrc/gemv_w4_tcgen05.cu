// Products of a few rows with many INT4 group-128 weight rows on the tcgen05 tensor cores.
#include "gemv_w4.cuh"
#include "ptx_sm100.cuh"

namespace pk100 {
namespace wide {

constexpr int kCluster = 4;                     // blocks that share a range of weight rows, each with a part of k
constexpr int kTile = 128;                      // weight rows of an accumulator
constexpr int kTiles = 16;                      // accumulators a round: 16 TMEM columns each
constexpr int kBuffers = 4;                     // converted groups in tensor memory: 64 columns each
constexpr int kWarps = 4 * kBuffers;            // that convert: four lane quadrants a buffer
constexpr int kThreads = kWarps * 32 + 64;
constexpr int kStageBytes = kTile * kGroup;     // two groups of a tile: TMA moves a box row of 64 bytes no faster than one of 128
constexpr int kStages = 5;
constexpr int kMostGroups = 32;                 // of a block: 4 KB of activations each

struct Smem {
    uint8_t x[kMostGroups][2][16 * 128];        // activations in the codes' order, 64 k an atom, 128-byte swizzle
    uint8_t ring[kStages][kStageBytes];         // codes, 128-byte swizzle; at the end of a round the block's sums
    uint64_t full[kStages], empty[kStages], a_full[kBuffers], a_empty[kBuffers], done, x_ready, drained;
    uint32_t tmem;
    int abort;
};
static_assert(kStages * kStageBytes >= kTiles / 2 * kTile * 16 * 4, "the sums of half a round fit the ring");

#define WIDE_WAIT(bar, parity) \
    if (!(ok = __all_sync(0xffffffffu, mbar_wait_within(&(bar), (parity), abort_flag, p.wait_ns)) != 0)) break
#define WIDE_LOOK(bar, parity) \
    if (!(ok = __all_sync(0xffffffffu, mbar_look_within(&(bar), (parity), abort_flag, p.wait_ns)) != 0)) break

__device__ __forceinline__ float4 load_from_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// mma.sync costs its warp ten issue slots that nothing else can use, as much as converting the codes it multiplies.  Here
// the converted weights go to tensor memory (a row a lane: the thread that reads a row's codes writes its weights) and
// are the A operand of tcgen05.mma, 128 rows x 16 k, against up to 16 rows of activations in shared memory; the warps
// do nothing but convert.
// A cluster of four blocks owns a range of 128-row tiles, each block a quarter of k for all of them: its activations
// stay in shared memory from beginning to end, and the accumulators of 16 tiles in tensor memory.  At the end the
// blocks' sums are joined through distributed shared memory in the order of the blocks.
__global__ void __launch_bounds__(kThreads, 1)
gemv_w4g128_wide_kernel(const __grid_constant__ CUtensorMap map_codes, const GemvParams p) {
    extern __shared__ __align__(1024) uint8_t wide_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(wide_raw);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
    const int rank = static_cast<int>(cluster_ctarank()), clusters = gridDim.x / kCluster, cluster = blockIdx.x / kCluster;
    const int groups = p.k / kGroup, all = (p.n + kTile - 1) / kTile;
    // this block's pairs of groups (of the last pair there may be one)
    const int all_pairs = (groups + 1) / 2, pair0 = all_pairs * rank / kCluster, pairs = all_pairs * (rank + 1) / kCluster - pair0, g0 = 2 * pair0, count = 2 * pairs;
    const int t0 = static_cast<int>(static_cast<long long>(all) * cluster / clusters), t1 = static_cast<int>(static_cast<long long>(all) * (cluster + 1) / clusters);
    volatile int* abort_flag = &sm.abort;
    grid_dependents_launch();
    if (tid == 0) {
        sm.abort = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 8);
        }
        for (int b = 0; b < kBuffers; ++b) {
            mbar_init(&sm.a_full[b], 4);
            mbar_init(&sm.a_empty[b], 1);
        }
        mbar_init(&sm.done, 1);
        mbar_init(&sm.drained, 1);
        mbar_init(&sm.x_ready, kWarps);
        fence_barrier_init();
        prefetch_tensormap(&map_codes);
    }
    if (warp == kWarps + 1) {
        tmem_alloc(&sm.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    grid_dependency_wait();
    if (warp < kWarps) {
        // activations: 8 k a thread; pair i of a word of codes is (i, i + 4)
        for (int i = tid; i < count * 16 * 16; i += kWarps * 32) {
            const int group = i / 256, m = i / 16 % 16, word = i % 16;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (m < p.m && g0 + group < groups) x = *reinterpret_cast<const uint4*>(p.a + m * p.lda + static_cast<long long>(g0 + group) * kGroup + word * 8);
            const uint4 y = make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
            *reinterpret_cast<uint4*>(sm.x[group][word / 8] + m * 128 + (((word % 8) ^ (m & 7)) << 4)) = y;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.x_ready);
    }
    const uint32_t tmem = sm.tmem, buffers = tmem + kTiles * 16;
    bool ok = true;
    uint32_t it = 0;                             // units (128 rows x a group) of this role so far
    int rounds = 0;
#pragma unroll 1
    for (int first = t0; first < t1; first += kTiles, ++rounds) {
        const int tiles = min(t1 - first, kTiles), units = tiles * count;
        if (warp == kWarps) {
            // ------------------------------------------------------------ TMA
            const bool leader = elect_one();
            for (int t = 0; ok && t < tiles; ++t)
                for (int pair = 0; pair < pairs; ++pair, ++it) {
                    const uint32_t s = it % kStages;
                    WIDE_LOOK(sm.empty[s], (it / kStages + 1) & 1);
                    mbar_arrive_expect_tx_if(leader, &sm.full[s], kStageBytes);
                    tma_load_2d_if(leader, sm.ring[s], &map_codes, &sm.full[s], (pair0 + pair) * kGroup, (first + t) * kTile);
                }
        } else if (warp == kWarps + 1) {
            // ------------------------------------------------------------ MMA
            constexpr uint32_t idesc = make_instr_desc<KIND_F16>(kTile, 16);
            const uint64_t desc_x = make_smem_desc<128>(smem_u32(sm.x));
            const bool leader = elect_one();
            ok = ok && __all_sync(0xffffffffu, mbar_look_within(&sm.x_ready, 0, abort_flag, p.wait_ns)) != 0;
            for (int t = 0; ok && t < tiles; ++t)
                for (int group = 0; group < count; ++group, ++it) {
                    const uint32_t b = it % kBuffers;
                    WIDE_WAIT(sm.a_full[b], (it / kBuffers) & 1);
                    tc_fence_after_sync();
#pragma unroll
                    for (int ks = 0; ks < kGroup / 16; ++ks)
                        mma_from_tmem(leader, tmem + t * 16, buffers + b * 64 + ks * 8, desc_x + group * (2 * 16 * 128 / 16) + (ks / 4) * (16 * 128 / 16) + 2 * (ks % 4),
                                      idesc, group > 0 || ks > 0);
                    tc_commit_if(leader, &sm.a_empty[b]);
                }
            tc_commit_if(leader, &sm.done);
        } else {
            // ------------------------------------------------------------ conversion: a row a thread
            const uint32_t b = warp / 4, quad = warp % 4, row = quad * 32 + lane;
            const CodeMasks masks;
            // this buffer's units, every fourth one over all rounds: (tile, group) of the next
            int t = 0, group = static_cast<int>((b + kBuffers - it % kBuffers) % kBuffers);
            uint32_t unit = it + group;
            auto settle = [&] { while (group >= count && t < tiles) { group -= count; ++t; } };
            auto scale_of = [&] {
                const int n = (first + t) * kTile + static_cast<int>(row);
                return t < tiles && n < p.n && g0 + group < groups ? p.group_scales[static_cast<long long>(g0 + group) * p.n + n] : __half();
            };
            if (count > 0) settle();
            __half scale = scale_of();
            for (; count > 0 && t < tiles; unit += kBuffers) {
                const uint32_t stage = unit / 2, s = stage % kStages, half = unit % 2;          // (units come in pairs)
                const __half2 scale2 = __half2half2(scale);
                group += kBuffers;
                settle();
                scale = scale_of();
                WIDE_WAIT(sm.full[s], (stage / kStages) & 1);
                uint4 codes[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) codes[c] = *reinterpret_cast<const uint4*>(sm.ring[s] + row * 128 + (((4 * half + c) ^ (row & 7)) << 4));
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.empty[s]);
                WIDE_WAIT(sm.a_empty[b], (unit / kBuffers + 1) & 1);
                tc_fence_after_sync();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
                    const uint32_t words[4] = {codes[c].x, codes[c].y, codes[c].z, codes[c].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) weights_of(words[i], scale2, masks, reinterpret_cast<uint32_t(&)[4]>(w[4 * i]));
                    tmem_st_32x16(buffers + b * 64 + c * 16 + (quad << 21), w);
                }
                tmem_st_wait();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.a_full[b]);
            }
            it += units;
        }
        // ------------------------------------------------------------ sums of the blocks, half a round at a time
        for (int from = 0; from < tiles; from += kTiles / 2) {
            const int here = min(tiles - from, kTiles / 2);
            float* sums = reinterpret_cast<float*>(sm.ring);
            if (warp < kWarps) {
                if (from == 0 && count > 0) {
                    ok = ok && __all_sync(0xffffffffu, mbar_wait_within(&sm.done, rounds & 1, abort_flag, p.wait_ns)) != 0;
                    tc_fence_after_sync();
                }
                const int quad = warp % 4, row = quad * 32 + lane;
                for (int t = warp / 4; t < here; t += 4) {
                    uint32_t v[16];
                    if (count > 0) {
                        tmem_ld_32x16(tmem + (from + t) * 16 + (quad << 21), v);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int c = 0; c < 16; ++c) sums[(t * 16 + c) * kTile + row] = count > 0 ? __uint_as_float(v[c]) : 0.0f;
                }
                tc_fence_before_sync();
            }
            __syncwarp();
            cluster_sync_all();
            // block `rank` finishes its share of every tile's rows, four a thread
            constexpr int kShare = kTile / kCluster, kQuads = kShare / 4;
            for (int o = tid; o < here * kQuads * p.m; o += kThreads) {
                const int row = rank * kShare + o % kQuads * 4, m = o / kQuads % p.m, t = o / (kQuads * p.m), n = (first + from + t) * kTile + row;
                const uint32_t at = smem_u32(&sums[(t * 16 + m) * kTile + row]);
                float4 part[kCluster], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int r = 0; r < kCluster; ++r) part[r] = load_from_cluster(map_to_cta(at, r));
#pragma unroll
                for (int r = 0; r < kCluster; ++r) {
                    v.x += part[r].x;
                    v.y += part[r].y;
                    v.z += part[r].z;
                    v.w += part[r].w;
                }
                if (n < p.n) gemv_store(p, v.x, m, n);
                if (n + 1 < p.n) gemv_store(p, v.y, m, n + 1);
                if (n + 2 < p.n) gemv_store(p, v.z, m, n + 2);
                if (n + 3 < p.n) gemv_store(p, v.w, m, n + 3);
            }
            __syncwarp();
            fence_proxy_async_smem();            // the ring is the copies' again
            cluster_sync_all();
        }
        tc_fence_after_sync();
    }
    if (!ok && lane == 0 && p.status != nullptr) atomicOr(p.status, 1);
    tc_fence_before_sync();
    __syncthreads();
    // where a wait ran out, whoever's: copies and products must end before the block's memory is given away
    if (*abort_flag != 0) {
        if (warp == kWarps) {
            for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i) mbar_drain(&sm.full[i % kStages], (i / kStages) & 1);
        } else if (warp == kWarps + 1) {
            tc_commit_if(elect_one(), &sm.drained);           // (the same lane every time)
            mbar_drain(&sm.drained, 0);
        }
    }
    if (warp == kWarps + 1) tmem_dealloc(tmem, 512);
}

}  // namespace wide

static cudaLaunchConfig_t wide_config(int clusters, cudaStream_t stream, cudaLaunchAttribute (&attrs)[2]) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(clusters * wide::kCluster);
    cfg.blockDim = dim3(wide::kThreads);
    cfg.dynamicSmemBytes = sizeof(wide::Smem);
    cfg.stream = stream;
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = wide::kCluster;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = pk100_dependent_launch_enabled() ? 2 : 1;
    return cfg;
}

// Clusters that the current device holds at once, 0 where it holds none.
static int wide_clusters() {
    static std::atomic<int> known[kPk100Devices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    int n = dev < kPk100Devices ? known[dev].load(std::memory_order_relaxed) : 0;
    if (n != 0) return n > 0 ? n : 0;
    cudaLaunchAttribute attrs[2]{};
    cudaLaunchConfig_t cfg = wide_config(1, nullptr, attrs);
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, wide::gemv_w4g128_wide_kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    if (dev < kPk100Devices) known[dev].store(n > 0 ? n : -1, std::memory_order_relaxed);
    return n;
}

int gemv_wide_limit() { return wide::kCluster * wide::kMostGroups * kGroup; }

int launch_gemv_wide(const GemvParams& p, cudaStream_t stream) {
    const cudaError_t granted = pk100_grant_smem<wide::gemv_w4g128_wide_kernel>(sizeof(wide::Smem));
    if (granted != cudaSuccess) return static_cast<int>(granted);
    const int held = wide_clusters(), tiles = (p.n + wide::kTile - 1) / wide::kTile;
    if (held < 1) return PK100_ERR_UNSUPPORTED;
    int clusters = pk100_cta_budget() / wide::kCluster;
    if (clusters < 1) clusters = 1;                      // (not another kernel: no result depends on the cap)
    if (clusters > held) clusters = held;
    if (clusters > tiles) clusters = tiles;
    CUtensorMap map;
    const int rc = pk100_tensor_map_2d(&map, p.codes, 1, p.n, p.k / 2, p.k / 2, wide::kTile, 128);
    if (rc != PK100_OK) return rc;
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t cfg = wide_config(clusters, stream, attrs);
    cudaLaunchKernelEx(&cfg, wide::gemv_w4g128_wide_kernel, map, p);
    return pk100_launch_status();
}

}  // namespace pk100
