// Matrix product of 8-bit integers with a scale for every token's row and every channel's weights, on the 5th-generation
// tensor cores (tcgen05, kind::i8), sm_100a:
//
//   Y[t][f] = (sum_k X[t][k] W[f][k]) * xs[t] * ws[f]
//
// The sum of at most 131,071 products of two 8-bit integers is exact in 32 bits, so neither the order of the additions nor
// a cut of K changes a result.  Behind the scales (fp32): a residual is added, or the value is rounded to bfloat16, or
// a gated feed-forward's gate and up value become one.
//
// As in the bfloat16 products the weights are operand A (a feature a tensor-memory lane) and the tokens operand B (a token a
// column); a 128-byte swizzled row of shared memory holds 128 k instead of 64, an instruction takes 32 instead of 16.
//
//   weight reader up to 32 tokens: linear_rows_int8.cu
//   tile kernel   a CTA: 128 features (with a gate 128 of each half) x 32, 64 or 128 tokens over a slice of K; the slices' CTAs
//                 form a cluster and add their accumulators through distributed shared memory
//   pair kernel   CTA pairs (cta_group::2): 256 features (128 with a gate) x 256 or 128 tokens, persistent, two accumulators
//
// Measured on B200 (a copy reaches 6.57 TB/s; the bfloat16 tensor rate of 1,670 TFLOP/s twice over would be 3,340): pairs, 4096 x 8192 x
// 2048 52 us (2,650 TOPS): 128 tiles on 74 pairs are two rounds, the second with 54 pairs at work, which alone leaves 0.865 of the rate;
// gated 8192 x 2048 x 8192 232 us (2,370 TOPS), bound by what L2 hands out, 2.44 GB in all, 10 TB/s; the tensor pipe is 62 % busy.
// Tiles with slices, 64 x 8192 x 2048 10.2 us (1.6 TB/s; with the rows' launch 13.6), 333 x 1500 x 2047 with the rows' launch 10.1: the
// latency of a walk over K (0.36 us a block of 128 k), of the cluster's join and of the launches.
//
// Launched with programmatic stream serialisation: the first ring of weights is asked for while the kernel in front still
// runs.  Every wait on an mbarrier is bounded; after the limit the library's status word is raised, every role stops waiting,
// the copies in flight land, tensor memory is freed and the kernel returns.
#include "int8_product.cuh"

using namespace fwb;
using namespace fwb::tc5;
using namespace fwb::int8;

namespace {

constexpr int BK8 = 128;                 // k of a block: one 128-byte swizzle row
constexpr int K_STEPS = 4;               // instructions a block: 32 k each, 32 bytes further along the row
constexpr int A_BYTES = BM * BK8;        // 16 KiB: 128 features of a block
constexpr int SM_COUNT = 148;

struct Params : Product {
    int n_kb;                    // blocks of K
    int kb_per_split, stages;    // tile kernel
    int token_tiles, feature_tiles;      // pair kernel
};

// D: 32-bit integers; A, B: signed 8-bit integers
__host__ __device__ constexpr uint32_t make_idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// After a wait that gave up: the copies still in flight land before the block's shared memory is another's.  `asked` stages
// of the ring have been filled or are being filled; a limit of its own, as the abort flag would end mbar_wait at once.
__device__ __forceinline__ void drain(uint64_t* full_bar, int stages, int asked) {
    for (int s = 0; s < stages && s < asked; ++s) {
        const uint32_t last = (uint32_t)((asked - 1 - s) / stages) & 1;
        for (unsigned spin = 0; spin < WAIT_LIMIT && !mbar_test(&full_bar[s], last); ++spin) __nanosleep(64);
    }
}

// ------------------------------------------------------------------ tile kernel
// Stages of the ring, at most.  Measured on B200, us of the product with 2 3 4 5 6 8 stages: 64 x 8192 x 2048 in 32-token tiles and four
// slices 13.3 10.9 10.2 10.2 10.8 11.0, in one 36.1 26.3 25.8 25.8 25.6 25.6; 333 x 1500 x 2047 8.6 7.5 7.4 7.2 7.3 7.5; gated 64 x 2048 x
// 8192 15.6 13.7 13.4 13.6 13.6 13.6.  What a block of K takes is a latency that more bytes on the way do not hide.
constexpr int RING = 4;
template <int BN, int NACC>
struct Tile {
    static constexpr int EPI_WARPS = BN >= 128 ? 16 : BN >= 64 ? 8 : 4;
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr int STAGE_BYTES = NACC * A_BYTES + BN * BK8;
    static constexpr int COLS = BN * NACC;
    static constexpr int TMEM_COLS = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : 256;
    static constexpr int PARTIAL_BYTES = COLS * BM * 4;
    static constexpr int data_bytes(int stages, int splits) {
        return splits > 1 && stages * STAGE_BYTES < PARTIAL_BYTES ? PARTIAL_BYTES : stages * STAGE_BYTES;
    }
};

template <int BN, int EPI>
__global__ void __launch_bounds__((Tile<BN, EPI == EPI_GATED_BF16 ? 2 : 1>::THREADS), 1)
gemm_int8_tile_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params prm) {
    constexpr int NACC = EPI == EPI_GATED_BF16 ? 2 : 1;
    using T = Tile<BN, NACC>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int STAGES = prm.stages, splits = gridDim.z;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(tiles + T::data_bytes(STAGES, splits));
    uint64_t* empty_bar = full_bar + RING;
    uint64_t* acc_bar = empty_bar + RING;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
    float* x_scale = reinterpret_cast<float*>(tiles + T::data_bytes(STAGES, splits) + 256);     // [BN]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tok0 = blockIdx.x * BN, feat0 = blockIdx.y * BM;
    const int kb_begin = blockIdx.z * prm.kb_per_split;
    const int kb_end = kb_begin + prm.kb_per_split < prm.n_kb ? kb_begin + prm.kb_per_split : prm.n_kb;
    const int n_kb = kb_end > kb_begin ? kb_end - kb_begin : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(acc_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(tmem_holder, T::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();     // (only with tensor memory in hand: a kernel further back could hold the columns and wait for this one)
    const uint32_t tmem_base = *tmem_holder;
    int asked = 0;                                     // the producer's: stages filled so far

    if (warp == 0) {
        if (lane == 0) {
            auto load_w = [&](int s, int kb) {
                uint8_t* stage = tiles + (size_t)s * T::STAGE_BYTES;
                mbar_expect_tx(&full_bar[s], T::STAGE_BYTES);
                tma_load_2d(stage, &map_w, &full_bar[s], kb * BK8, feat0);
                if (NACC == 2) tma_load_2d(stage + A_BYTES, &map_w, &full_bar[s], kb * BK8, prm.up_row_offset + feat0);
            };
            auto load_x = [&](int s, int kb) {
                tma_load_2d(tiles + (size_t)s * T::STAGE_BYTES + NACC * A_BYTES, &map_x, &full_bar[s], kb * BK8, tok0);
            };
            // weights do not depend on the kernel in front: the first ring of them is asked for ahead of the wait for it
            const int ahead = n_kb < STAGES ? n_kb : STAGES;
            for (int i = 0; i < ahead; ++i) load_w(i, kb_begin + i);
            pdl_wait();
            for (int i = 0; i < ahead; ++i) load_x(i, kb_begin + i);
            for (asked = ahead; asked < n_kb; ++asked) {
                const int s = asked % STAGES;
                if (!mbar_wait(&empty_bar[s], (asked / STAGES - 1) & 1, abort_flag, 31, prm.status)) break;
                load_w(s, kb_begin + asked);
                load_x(s, kb_begin + asked);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = make_idesc_i8(BM, BN);
            bool ok = true;
            for (int i = 0; i < n_kb; ++i) {
                const int s = i % STAGES;
                ok = mbar_wait(&full_bar[s], (i / STAGES) & 1, abort_flag, 32, prm.status);
                if (!ok) break;
                tc_fence_after();
                const uint32_t stage = smem_u32(tiles + (size_t)s * T::STAGE_BYTES);
                const uint64_t b_desc = make_smem_desc(stage + NACC * A_BYTES);
#pragma unroll
                for (int a = 0; a < NACC; ++a) {
                    const uint64_t a_desc = make_smem_desc(stage + a * A_BYTES);
#pragma unroll
                    for (int k = 0; k < K_STEPS; ++k)
                        umma_i8(tmem_base + a * BN, a_desc + 2 * k, b_desc + 2 * k, idesc, i > 0 || k > 0 ? 1u : 0u);
                }
                umma_commit(&empty_bar[s]);
            }
            umma_commit(acc_bar);
        }
    }
    __syncwarp();

    // ---------------------------------------------------------------- epilogue
    const bool epi_warp = warp >= 2;
    constexpr int GROUPS = T::EPI_WARPS / 4;           // warps that share a quarter of the lanes: columns between them
    const int column_group = (warp - 2) >> 2, quarter = warp & 3, row = quarter * 32 + lane, f = feat0 + row;
    bool ready = true;
    float w_scale = 0.0f, up_scale = 0.0f;
    if (epi_warp) {
        if (f < prm.N) {                               // (scales of weights: as the weights themselves)
            w_scale = prm.ws[f];
            if (NACC == 2) up_scale = prm.ws[prm.up_row_offset + f];
        }
        pdl_wait();
        for (int c = (int)threadIdx.x - 64; c < BN; c += 32 * T::EPI_WARPS) x_scale[c] = tok0 + c < prm.M ? prm.xs[tok0 + c] : 0.0f;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * T::EPI_WARPS) : "memory");
        if (n_kb > 0) ready = mbar_wait(acc_bar, 0, abort_flag, 33, prm.status);
        ready = __all_sync(0xffffffffu, ready && !*abort_flag);       // tcgen05.ld needs the whole warp
        tc_fence_after();
    }
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    // the addends of several columns are asked for together and ahead of what they are added to: a store may not pass a load
    // that could be of the same memory, one by one they would cost a trip to memory each
    auto addend_of = [&](int col) {
        const int t = tok0 + col;
        return EPI == EPI_ADD_F32 && t < prm.M && f < prm.N ? prm.addend[(size_t)t * prm.N + f] : 0.0f;
    };
    auto finish = [&](int col, int v, int u, float add) {
        const int t = tok0 + col;
        if (t >= prm.M || f >= prm.N) return;
        const float xs = x_scale[col];
        store<EPI>(prm, (size_t)t * prm.N + f, scaled(v, xs, w_scale), scaled(u, xs, up_scale), add);
    };
    if (splits == 1) {
        if (epi_warp && ready) {
            constexpr int PER_GROUP = BN / GROUPS;
#pragma unroll 1
            for (int c0 = column_group * PER_GROUP; c0 < (column_group + 1) * PER_GROUP && tok0 + c0 < prm.M; c0 += 16) {
                float v[16], u[16], add[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) add[j] = addend_of(c0 + j);
                tmem_ld16(lane_addr + c0, v);
                if (NACC == 2) tmem_ld16(lane_addr + BN + c0, u);
#pragma unroll
                for (int j = 0; j < 16; ++j) finish(c0 + j, __float_as_int(v[j]), NACC == 2 ? __float_as_int(u[j]) : 0, add[j]);
            }
        }
    } else {
        // every product that read the ring has completed: the partial tile [column][row] takes its place
        int* partial = reinterpret_cast<int*>(tiles);
        const int cols = prm.M - tok0 < BN ? prm.M - tok0 : BN;       // columns that hold a token
        if (epi_warp) {
#pragma unroll 1
            for (int c0 = column_group * 16; c0 < T::COLS; c0 += 16 * GROUPS) {
                if (c0 % BN >= cols) continue;
                float v[16] = {};
                if (n_kb > 0 && ready) tmem_ld16(lane_addr + c0, v);
#pragma unroll
                for (int j = 0; j < 16; ++j) partial[(c0 + j) * BM + row] = __float_as_int(v[j]);
            }
        }
        // column c is added up and stored by rank c % splits; BATCH columns' loads are in flight together
        constexpr int BATCH = NACC == 2 ? 4 : 8;
        const uint32_t rank = cluster_rank(), base = smem_u32(partial);
        const int first = (int)rank + column_group * splits, step = GROUPS * splits;
        float add[BATCH];
        if (epi_warp)
#pragma unroll
            for (int b = 0; b < BATCH; ++b) add[b] = addend_of(first + b * step);
        tc_fence_before();
        cluster_sync_all();
        if (epi_warp) {
            for (int c0 = first; c0 < cols; c0 += BATCH * step) {
                int v[BATCH] = {}, u[BATCH] = {};
                if (c0 != first)
#pragma unroll
                    for (int b = 0; b < BATCH; ++b) add[b] = addend_of(c0 + b * step);
                for (int p = 0; p < splits; ++p)
#pragma unroll
                    for (int b = 0; b < BATCH; ++b) {
                        const int c = c0 + b * step < cols ? c0 + b * step : c0;
                        v[b] += __float_as_int(ld_dsmem_f32(base + (uint32_t)(c * BM + row) * 4, p));
                        if (NACC == 2) u[b] += __float_as_int(ld_dsmem_f32(base + (uint32_t)((BN + c) * BM + row) * 4, p));
                    }
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
                    if (c0 + b * step < cols && ready) finish(c0 + b * step, v[b], u[b], add[b]);
            }
        }
        cluster_sync_all();      // nobody leaves while a peer still reads from it
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) drain(full_bar, STAGES, asked);
    if (warp == 1) tmem_dealloc(tmem_base, T::TMEM_COLS);
}

template <int BN, int EPI>
int launch_tile(const CUtensorMap& map_w, const CUtensorMap& map_x, Params prm, int splits, cudaStream_t stream) {
    using T = Tile<BN, EPI == EPI_GATED_BF16 ? 2 : 1>;
    auto kernel = gemm_int8_tile_kernel<BN, EPI>;
    prm.kb_per_split = (prm.n_kb + splits - 1) / splits;
    prm.stages = prm.kb_per_split < RING ? prm.kb_per_split : RING;
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((prm.M + BN - 1) / BN, (prm.N + BM - 1) / BM, splits);
    config.blockDim = dim3(T::THREADS);
    config.dynamicSmemBytes = T::data_bytes(prm.stages, splits) + 1024 + 256 + BN * 4;
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = splits;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    config.attrs = attr;
    config.numAttrs = n;
    cudaError_t e = cudaLaunchKernelEx(&config, kernel, map_w, map_x, prm);
    return e == cudaSuccess ? fwb_launch_status() : (int)e;
}

// ------------------------------------------------------------------ pair kernel
constexpr int PAIR_EPI_WARPS = 16, PAIR_THREADS = 64 + 32 * PAIR_EPI_WARPS;
constexpr int TRADE_FLOATS = 8 * 32;                    // what a warp hands over of 16 columns
template <int BN>
struct PairTile {
    static constexpr int HALF_N = BN / 2;
    static constexpr int STAGE_BYTES = A_BYTES + HALF_N * BK8;
    static constexpr int STAGES = 192 * 1024 / STAGE_BYTES;
    static constexpr int TRADE_BYTES = 2 * PAIR_EPI_WARPS * TRADE_FLOATS * 4;
    // (behind 192 KiB of stages the trade buffers do not fit: a gated product's ring is one stage shorter)
    static constexpr int stages(bool gated) { return gated ? STAGES - 1 : STAGES; }
    static constexpr int smem_bytes(bool gated) { return stages(gated) * STAGE_BYTES + (gated ? TRADE_BYTES : 0) + 1024 + 512; }
};

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrive (once all products issued so far have completed) on the barrier at this offset in both CTAs.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    const uint16_t mask = 3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(smem_u32(bar)), "h"(mask)
        : "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void* ptr, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(ptr)), "r"(rank));
    return remote;
}
// A tile into this CTA's shared memory whose bytes are counted on a barrier that may live in the pair's other CTA.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(bar_cluster_addr), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar_cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}

template <int EPI, int BN>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params prm) {
    constexpr bool GATED = EPI == EPI_GATED_BF16;
    constexpr int CTA_FEATURES = GATED ? BM / 2 : BM;   // features a CTA has of a tile; with a gate its rows are 64 gate, 64 up
    using T = PairTile<BN>;
    constexpr int STAGES = T::stages(GATED), STAGE_BYTES = T::STAGE_BYTES, HALF_N = T::HALF_N;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* trade = reinterpret_cast<float*>(tiles + STAGES * STAGE_BYTES);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(tiles + STAGES * STAGE_BYTES + (GATED ? T::TRADE_BYTES : 0));
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* acc_full = empty_bar + STAGES;             // [2]: in both CTAs
    uint64_t* acc_empty = acc_full + 2;                  // [2]: the leader's, arrived on by both CTAs' epilogue warps
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();                // 0 = leader
    const int first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1, n_kb = prm.n_kb;
    const int token_tiles = prm.token_tiles, tiles_all = token_tiles * prm.feature_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * PAIR_EPI_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_holder)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();          // both CTAs' barriers exist before anybody signals across
    tc_fence_after();
    pdl_launch_dependents();     // (only with tensor memory in hand, as above)
    const uint32_t tmem_base = *tmem_holder;

    int asked = 0;                                       // the producer's: stages filled so far
    // token tiles are the fast index: pairs that run together share weight tiles in L2
    struct Place {
        int tok0, f;                                     // first token, this CTA's first feature
    };
    auto place_of = [&](int tile) {
        return Place{(tile % token_tiles) * BN, ((tile / token_tiles) * 2 + (int)rank) * CTA_FEATURES};
    };

    if (warp == 0) {
        if (lane == 0) {
            // every load of the pair reports to the leader's barrier of its stage; the leader arms it with both CTAs' bytes
            auto load_w = [&](int s, const Place& at, int kb) {
                uint8_t* stage = tiles + (size_t)s * STAGE_BYTES;
                const uint32_t bar = cluster_addr(&full_bar[s], 0);
                if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * STAGE_BYTES);
                tma_load_2d_pair(stage, &map_w, bar, kb * BK8, at.f);
                if (GATED) tma_load_2d_pair(stage + A_BYTES / 2, &map_w, bar, kb * BK8, prm.up_row_offset + at.f);
            };
            auto load_x = [&](int s, const Place& at, int kb) {
                tma_load_2d_pair(tiles + (size_t)s * STAGE_BYTES + A_BYTES, &map_x, cluster_addr(&full_bar[s], 0), kb * BK8,
                                 at.tok0 + (int)rank * HALF_N);
            };
            const int ahead = first_tile >= tiles_all ? 0 : n_kb < STAGES ? n_kb : STAGES;
            if (ahead) {
                const Place at = place_of(first_tile);
                for (int i = 0; i < ahead; ++i) load_w(i, at, i);
                pdl_wait();
                for (int i = 0; i < ahead; ++i) load_x(i, at, i);
                asked = ahead;
            }
            int s = ahead % STAGES;
            uint32_t parity = ahead == STAGES ? 0 : 1;   // of the empty barrier; the ring's first round waits for nothing
            bool ok = true;
            for (int tile = first_tile; tile < tiles_all && ok; tile += tile_step) {
                const Place at = place_of(tile);
                for (int kb = tile == first_tile ? ahead : 0; kb < n_kb; ++kb) {
                    ok = mbar_wait(&empty_bar[s], parity, abort_flag, 34, prm.status);
                    if (!ok) break;
                    load_w(s, at, kb);
                    load_x(s, at, kb);
                    ++asked;
                    if (++s == STAGES) s = 0, parity ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = make_idesc_i8(2 * BM, BN);
            bool ok = true;
            int s = 0, turn = 0;
            uint32_t parity = 0;
            for (int tile = first_tile; tile < tiles_all && ok; tile += tile_step, ++turn) {
                const int b = turn & 1;
                // both CTAs' epilogues have read what this accumulator held two tiles ago
                if (turn >= 2) ok = mbar_wait_cluster(&acc_empty[b], ((turn >> 1) - 1) & 1, abort_flag, 35, prm.status);
                if (!ok) break;
                tc_fence_after();
                for (int kb = 0; kb < n_kb; ++kb) {
                    ok = mbar_wait_cluster(&full_bar[s], parity, abort_flag, 36, prm.status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t stage = smem_u32(tiles + (size_t)s * STAGE_BYTES);
                    const uint64_t a_desc = make_smem_desc(stage), b_desc = make_smem_desc(stage + A_BYTES);
#pragma unroll
                    for (int k = 0; k < K_STEPS; ++k)
                        umma_i8_pair(tmem_base + b * BN, a_desc + 2 * k, b_desc + 2 * k, idesc, kb > 0 || k > 0 ? 1u : 0u);
                    umma_commit_pair(&empty_bar[s]);     // frees the stage in both CTAs
                    if (++s == STAGES) s = 0, parity ^= 1;
                }
                umma_commit_pair(&acc_full[b]);          // accumulator complete, in both CTAs
            }
        }
    }
    __syncwarp();

    // ---------------------------------------------------------------- epilogue (both CTAs)
    if (warp >= 2) {
        pdl_wait();
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
        constexpr int PER_GROUP = BN / (PAIR_EPI_WARPS / 4);  // the warps of a quarter of the lanes share the token columns
        int turn = 0;
        for (int tile = first_tile; tile < tiles_all; tile += tile_step, ++turn) {
            const int b = turn & 1;
            const Place at_tile = place_of(tile);
            const int tok0 = at_tile.tok0 + group * PER_GROUP;
            const bool up = GATED && quarter >= 2;
            const int f = at_tile.f + (GATED ? (quarter & 1) : quarter) * 32 + lane;
            const float w_scale = f < prm.N ? prm.ws[(up ? prm.up_row_offset : 0) + f] : 0.0f;
            bool ready = mbar_wait(&acc_full[b], (turn >> 1) & 1, abort_flag, 37, prm.status);
            // (after a wait that gave up nobody reads or stores, but everybody keeps meeting his partner's barriers)
            ready = __all_sync(0xffffffffu, ready && !*abort_flag);
            tc_fence_after();
            const uint32_t from = lane_base + b * BN + group * PER_GROUP;
#pragma unroll 1
            for (int c0 = 0; c0 < PER_GROUP; c0 += 16) {
                float v[16] = {}, add[EPI == EPI_ADD_F32 ? 16 : 1];
                float xs[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int t = tok0 + c0 + j;
                    xs[j] = t < prm.M ? prm.xs[t] : 0.0f;
                    if constexpr (EPI == EPI_ADD_F32) add[j] = t < prm.M && f < prm.N ? prm.addend[(size_t)t * prm.N + f] : 0.0f;
                }
                if (ready) tmem_ld16(from + c0, v);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = scaled(__float_as_int(v[j]), xs[j], w_scale);
                if constexpr (GATED) {
                    float* mine = trade + (size_t)(warp - 2) * TRADE_FLOATS + lane;
                    const float* theirs = trade + (size_t)((warp - 2) ^ 2) * TRADE_FLOATS + lane;
                    const int buffer = (c0 >> 4 & 1) * PAIR_EPI_WARPS * TRADE_FLOATS;
#pragma unroll
                    for (int j = 0; j < 8; ++j) mine[buffer + j * 32] = up ? v[j] : v[8 + j];
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + group * 2 + (quarter & 1)) : "memory");
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float other = theirs[buffer + j * 32];
                        const int t = tok0 + c0 + (up ? 8 : 0) + j;
                        if (ready && t < prm.M && f < prm.N)
                            store<EPI>(prm, (size_t)t * prm.N + f, up ? other : v[j], up ? v[8 + j] : other, 0.0f);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int t = tok0 + c0 + j;
                        if (ready && t < prm.M && f < prm.N)
                            store<EPI>(prm, (size_t)t * prm.N + f, v[j], 0.0f, add[EPI == EPI_ADD_F32 ? j : 0]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[b], 0));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && rank == 0 && *abort_flag) drain(full_bar, STAGES, asked);
    cluster_sync_all();          // neither CTA frees tensor memory or leaves while the other still works
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
}

template <int EPI, int BN>
int launch_pair(const CUtensorMap& map_w, const CUtensorMap& map_x, const Params& prm, long tiles, cudaStream_t stream) {
    auto kernel = gemm_int8_pair_kernel<EPI, BN>;
    constexpr int SMEM = PairTile<BN>::smem_bytes(EPI == EPI_GATED_BF16);
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * (unsigned)(tiles < SM_COUNT / 2 ? tiles : SM_COUNT / 2));
    config.blockDim = dim3(PAIR_THREADS);
    config.dynamicSmemBytes = SMEM;
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = pdl_enabled() ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&config, kernel, map_w, map_x, prm);
    return e == cudaSuccess ? fwb_launch_status() : (int)e;
}

// A [rows][K] matrix of bytes, rows `stride` bytes apart, as boxes of [box_rows][128] with 128-byte swizzle.
bool make_map_i8(CUtensorMap* map, const void* base, long rows, int K, int stride, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)((K + 15) & ~15), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)stride};
    cuuint32_t box[2] = {(cuuint32_t)BK8, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int EPI>
int launch(Params prm, int tile, int splits, cudaStream_t stream) {
    constexpr bool GATED = EPI == EPI_GATED_BF16;
    const int K = prm.K, x_stride = prm.x_stride, w_stride = prm.w_stride, w_rows = prm.w_rows;
    const void *X = prm.x, *W = prm.w;
    CUtensorMap map_w, map_x;
    if (tile < 0) {
        const int bn = -tile;
        prm.feature_tiles = (prm.N + (GATED ? BM : 2 * BM) - 1) / (GATED ? BM : 2 * BM);
        prm.token_tiles = (prm.M + bn - 1) / bn;
        const long tiles = (long)prm.token_tiles * prm.feature_tiles;
        if (tiles > 1073741823L) return FWB_TOO_LARGE;
        if (!make_map_i8(&map_w, W, w_rows, K, w_stride, GATED ? BM / 2 : BM) || !make_map_i8(&map_x, X, prm.M, K, x_stride, bn / 2))
            return FWB_UNSUPPORTED;
        return bn == 128 ? launch_pair<EPI, 128>(map_w, map_x, prm, tiles, stream) : launch_pair<EPI, 256>(map_w, map_x, prm, tiles, stream);
    }
    if (!make_map_i8(&map_w, W, w_rows, K, w_stride, BM) || !make_map_i8(&map_x, X, prm.M, K, x_stride, tile)) return FWB_UNSUPPORTED;
    switch (tile) {
        case 32: return launch_tile<32, EPI>(map_w, map_x, prm, splits, stream);
        case 64: return launch_tile<64, EPI>(map_w, map_x, prm, splits, stream);
        default: return launch_tile<128, EPI>(map_w, map_x, prm, splits, stream);
    }
}

// Which kernel takes a product: the token tile (8: the weight reader; negative: the CTA pairs') and the slices of K.
//
// Measured in chains of launches over 300 MB of weights (us).  The weight reader wins up to 16 tokens (16 x 8192 x 2048 7.9,
// tiles 9.1; gated 16 x 2048 x 8192 9.7, 10.5), and up to 32 where a CTA's activations and the matrix are small: 32 x 2048 x 2048
// 4.2 (6.0), gated 32 x 1024 x 4608 5.1 (7.1), but 32 x 8192 x 2048 11.4 (9.4), gated 32 x 2048 x 8192 15.1 (12.5).  Beyond 512 tokens
// the pairs win.  Between, a launch takes about 3 us (pairs 3 to 6) and, for every 128 k that a CTA walks, 0.36 (0.63 with a gate;
// pairs 0.29 and 0.65, a further round of tiles with a gate 0.35 to 0.45) -- a latency, or with every SM at it HBM's rate -- then its
// stores, and 1.6 us for the cluster that adds slices (3 to 6 with eight): 64 x 8192 x 2048 in 32-token tiles 27.1 16.6 10.9 11.1 with 1 2 4 8 slices, in 64-token
// tiles 27.1 17.0 11.5 12.2, pairs 22.8; 256 x 8192 x 2048 in 128-token tiles 28.8 19.0 14.3, pairs 23.6; gated 256 x 1024 x 4608 in
// 128-token tiles 10.2, pairs 9.8.  CTAs beyond what the SMs hold at once wait for a round of their own: gated 64 x 2048 x 8192 in
// 128 CTAs 14.5, in 256 22.7; clusters are not taken for that.
void choose(int M, int N, int K, bool gated, int* tile, int* splits) {
    const int n_kb = (K + BK8 - 1) / BK8, halves = gated ? 2 : 1;
    *splits = 1;
    if (M <= 16 || (M <= 32 && (long)M * K <= 65536 && (long)N * halves * K <= (16L << 20))) {
        *tile = 8;
        return;
    }
    const int pair_features = gated ? BM : 2 * BM;
    const long pair_tiles = (N + pair_features - 1) / pair_features;
    if (M > 512) {
        // 128-token tiles where 256 would leave half of the pairs without one
        *tile = pair_tiles * ((M + 255) / 256) * 2 <= SM_COUNT / 2 ? -128 : -256;
        return;
    }
    float best = 1e30f;
    auto consider = [&](int t, int s, float cost) {
        if (cost < best) best = cost, *tile = t, *splits = s;
    };
    for (int t = 32; t <= 128; t *= 2) {
        const int used = M < t ? M : t;
        for (int s = 1; s <= 8 && (s == 1 || n_kb >= 2 * s); s *= 2) {
            const long ctas = (long)((N + BM - 1) / BM) * ((M + t - 1) / t) * s;
            // CTAs the SMs hold at once, by shared memory; clusters leave SMs of a GPC over, and beyond that would wait for one another
            const int kb = (n_kb + s - 1) / s, ring = (kb < RING ? kb : RING) * (halves * A_BYTES + t * BK8), sums = s > 1 ? halves * t * BM * 4 : 0;
            const long held = (s > 1 && t == 128 ? 1 : 227 * 1024 / ((ring > sums ? ring : sums) + 2048)) * (s > 1 ? SM_COUNT * 7 / 8 : SM_COUNT);
            if (s > 1 && ctas > (held < 2 * SM_COUNT * 7 / 8 ? held : 2 * SM_COUNT * 7 / 8)) continue;
            const bool crowded = ctas > SM_COUNT && ctas <= held;
            const float walk = kb * (gated ? 0.63f : 0.36f) * (crowded ? 1.17f : 1.0f);
            const float join = s == 1 ? 0.0f : (s < 8 ? 1.6f : t == 32 ? 3.1f : 6.0f) + (crowded ? 2.0f : 0.0f);
            consider(t, s, 3.0f + ((ctas + held - 1) / held) * (walk + 0.016f * used) + join);
        }
    }
    for (int t = 128; t <= 256; t *= 2) {
        const long rounds = (pair_tiles * ((M + t - 1) / t) + SM_COUNT / 2 - 1) / (SM_COUNT / 2);
        const float start = t == 128 ? (gated ? 2.5f : 4.0f) : (gated ? 4.0f : 6.0f);
        const float walk = n_kb * (gated ? (t == 128 ? 0.64f : 0.7f) : 0.29f), more = n_kb * (gated ? (t == 128 ? 0.35f : 0.45f) : 0.29f);
        consider(-t, 1, start + walk + (rounds - 1) * more + 0.005f * M);
    }
}

}  // namespace

// X: [M][x_stride] int8 with scales xs [M]; W: [w_rows][w_stride] int8 with scales ws [w_rows]; both zero from column K on.
// Y: [M][N] fp32 (epilogues 0; 2: + addend, which may be Y) or bf16 (1; 3: gated, N features, up rows at up_row_offset,
// the gate's activation in the bits above the code, its parameter in gate_limit).  tile: 0 (the kernel's own choice), 8 (the weight
// reader, at most 32 tokens), 32, 64 or 128 tokens with `splits` (1, 2, 4, 8) slices of K, or -128 or -256 (CTA pairs).
FWB_API int fwb_gemm_int8(const void* X, const float* xs, const void* W, const float* ws, void* Y, const float* addend, int M,
                          int N, int K, int x_stride, int w_stride, int w_rows, int epilogue, int up_row_offset,
                          float gate_limit, int tile, int splits, cudaStream_t stream) {
    const int act = epilogue >> 8;
    epilogue &= 0xff;
    if (M <= 0 || N <= 0) return FWB_OK;
    if (!X || !xs || !W || !ws || !Y || K <= 0 || x_stride < K || w_stride < K) return FWB_BAD_ARGUMENT;
    if (K > MAX_K) return FWB_TOO_LARGE;
    if ((x_stride & 15) || (w_stride & 15) || (((uintptr_t)X | (uintptr_t)W) & 15)) return FWB_UNSUPPORTED;
    if (epilogue == EPI_ADD_F32 && !addend) return FWB_BAD_ARGUMENT;
    if (epilogue == EPI_GATED_BF16 ? (up_row_offset < N || w_rows < up_row_offset + N) : w_rows < N) return FWB_BAD_ARGUMENT;
    const int n_kb = (K + BK8 - 1) / BK8;
    if (tile == 0) choose(M, N, K, epilogue == EPI_GATED_BF16, &tile, &splits);
    else if ((tile != 8 && tile != 32 && tile != 64 && tile != 128 && tile != -128 && tile != -256) ||
             (splits != 1 && splits != 2 && splits != 4 && splits != 8))
        return FWB_BAD_ARGUMENT;
    Product p{(const signed char*)X, (const signed char*)W, xs, ws, Y, addend, M, N, K, x_stride, w_stride, w_rows,
              up_row_offset, act, gate_limit, status_word()};
    if (tile == 8) return few_tokens(p, epilogue, stream);
    if (tile > 0 && (N + BM - 1) / BM > 65535) tile = -256;
    Params prm{};
    static_cast<Product&>(prm) = p;
    prm.n_kb = n_kb;
    switch (epilogue) {
        case EPI_F32: return launch<EPI_F32>(prm, tile, splits, stream);
        case EPI_BF16: return launch<EPI_BF16>(prm, tile, splits, stream);
        case EPI_ADD_F32: return launch<EPI_ADD_F32>(prm, tile, splits, stream);
        case EPI_GATED_BF16: return launch<EPI_GATED_BF16>(prm, tile, splits, stream);
        default: return FWB_UNSUPPORTED;
    }
}

FWB_API int fwb_rows_int8(const void* x, int x_bf16, const float* delta, const float* norm_w, const int* rows, void* q,
                          float* scales, int R, int K, int stride, int x_rows, float eps, cudaStream_t stream);

// The same for rows that are no integers yet: x [M][K] bf16 (x_bf16) or fp32; scratch: M * stride bytes for the integers and
// 4 M behind them for the scales, stride = K rounded up to 16.  Without scratch (null): in one launch, for at most 8 tokens and 4,096
// columns, K a multiple of 8 and the rows on borders of 16 bytes.
FWB_API int fwb_linear_int8(const void* x, int x_bf16, void* scratch, const void* W, const float* ws, void* Y, const float* addend,
                            int M, int N, int K, int w_stride, int w_rows, int epilogue, int up_row_offset, float gate_limit,
                            cudaStream_t stream) {
    const int stride = (K + 15) & ~15;
    if (!scratch) {
        const int code = epilogue & 0xff;
        if (M <= 0 || N <= 0) return FWB_OK;
        if (!x || !W || !ws || !Y || K <= 0 || w_stride < K) return FWB_BAD_ARGUMENT;
        if ((w_stride & 15) || ((uintptr_t)W & 15)) return FWB_UNSUPPORTED;
        if (code == EPI_ADD_F32 && !addend) return FWB_BAD_ARGUMENT;
        if (code == EPI_GATED_BF16 ? (up_row_offset < N || w_rows < up_row_offset + N) : w_rows < N) return FWB_BAD_ARGUMENT;
        const Product p{nullptr, (const signed char*)W, nullptr, ws, Y, addend, M, N, K, stride, w_stride, w_rows,
                        up_row_offset, epilogue >> 8, gate_limit, status_word()};
        return few_raw_tokens(p, x, x_bf16 != 0, code, stream);
    }
    float* scales = reinterpret_cast<float*>(static_cast<char*>(scratch) + (size_t)M * stride);
    const int status = fwb_rows_int8(x, x_bf16, nullptr, nullptr, nullptr, scratch, scales, M, K, stride, M, 0.0f, stream);
    if (status != FWB_OK) return status;
    return fwb_gemm_int8(scratch, scales, W, ws, Y, addend, M, N, K, stride, w_stride, w_rows, epilogue, up_row_offset, gate_limit,
                         0, 1, stream);
}
