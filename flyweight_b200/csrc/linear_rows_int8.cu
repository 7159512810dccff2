// The 8-bit product of a few tokens (decode steps): a weight reader, as linear_rows.cu is for bfloat16.
//
//   Y[t][f] = (sum_k X[t][k] W[f][k]) * xs[t] * ws[f]
//
//   * A CTA owns `units` groups of eight features (with a gate eight of the gate and the eight of the up projection that go
//     with them) over all of K; its eight warps cut K between them: per step of the walk a warp takes KBLK adjacent blocks of 64 k.
//   * A ninth warp streams the weights through a ring in shared memory, row by row with bulk copies, from the kernel's first
//     moment on: nothing in the stream writes weights.  Two CTAs an SM, or four small ones.
//   * mma.sync of 16 tokens x 8 features x 32 k on 8-bit integers; a lane's 16-byte read is sixteen k of one feature, and the k
//     of a block are dealt to the fragments' slots in that order for both operands.
//   * Rows that are no integers yet (at most eight): a first pass over them finds the rows' largest magnitudes, then every block makes
//     the integers of the k that a lane feeds to its products, where int8_rows.cu would make them in a launch of its own.  The
//     same integers: a product's bits do not depend on it.
//   * The warps' sums meet in shared memory; integers, so their order is of no consequence.
//
// Bound by the weights' bytes once they are many: gated 8 x 2048 x 8192 (33.6 MB) 7.5 us, 4.5 TB/s (a copy: 6.57; bytes alone 5.1 us);
// 1 x 2048 x 2048 (4.2 MB) 2.6 us, 4.1 where the blocks make the integers too: a launch's latency and one walk.
// Every wait on an mbarrier is bounded as in the tcgen05 products.
#include "int8_product.cuh"
#include "int8_quantize.cuh"

using namespace fwb;
using namespace fwb::tc5;
using namespace fwb::int8;

namespace {

constexpr int SMEM_OF_SM = 224 * 1024;
constexpr int MAX_SLOTS = 8;
constexpr long ALL_CTAS_FROM = 2 << 20;
constexpr int EIGHT = fwb::int8::CHUNK;

struct RowsParams {
    Product p;
    int Kp;                      // bytes of a row that hold k: K rounded up to 16
    int units;                   // groups of eight features of one half per CTA
    int slots;                   // depth of the ring
    const void* raw;             // RAW: [M][K] rows that are no integers yet
};

enum Raw : int { INTEGERS = 0, RAW_BF16 = 1, RAW_F32 = 2 };

// Eight values of a raw row from column k on, zeros from K on (K and k are multiples of 8).
template <int RAW>
__device__ __forceinline__ void raw_values(const RowsParams& prm, int row, int k, float (&v)[EIGHT]);

__device__ __forceinline__ uint4 load_rows(const void* at) {     // written by the kernel before: not .nc
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at) : "memory");
    return v;
}
template <>
__device__ __forceinline__ void raw_values<RAW_BF16>(const RowsParams& prm, int row, int k, float (&v)[EIGHT]) {
    const uint4 a = k < prm.p.K ? load_rows(static_cast<const __nv_bfloat16*>(prm.raw) + (size_t)row * prm.p.K + k) : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
template <>
__device__ __forceinline__ void raw_values<RAW_F32>(const RowsParams& prm, int row, int k, float (&v)[EIGHT]) {
    const float* at = static_cast<const float*>(prm.raw) + (size_t)row * prm.p.K + k;
    const uint4 none = make_uint4(0, 0, 0, 0), a = k < prm.p.K ? load_rows(at) : none, b = k < prm.p.K ? load_rows(at + 4) : none;
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void mma_16x8x32(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// bytes between rows in shared memory: quarter-warps read two rows of 64 bytes each
__host__ __device__ constexpr int row_stride(int bytes) { return ((bytes + 127) & ~127) + 64; }

// WARPS that sum, CTAS an SM, R8 groups of eight token rows, KBLK blocks of 64 k a warp takes in a step.
template <int WARPS, int CTAS, int R8, int KBLK, int EPI, int RAW>
__global__ void __launch_bounds__(32 * (WARPS + 1), CTAS) linear_rows_int8_kernel(const RowsParams prm) {
    constexpr int NACC = EPI == EPI_GATED_BF16 ? 2 : 1, THREADS = 32 * (WARPS + 1);
    constexpr int MT = (R8 + 1) / 2;                   // 16-row tiles of the product
    constexpr int CHUNK = WARPS * KBLK * 64, W_STRIDE = row_stride(CHUNK), SLOT = 8 * W_STRIDE;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full_bar[MAX_SLOTS], empty_bar[MAX_SLOTS];
    __shared__ int abort_word;
    __shared__ unsigned tops[MAX_RAW];                 // RAW: the rows' largest magnitudes, as bits
    volatile int* abort_flag = &abort_word;
    const Product& p = prm.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int all_units = (p.N + 7) >> 3, slots = prm.slots;
    const int unit0 = blockIdx.x * prm.units;
    const int units = all_units - unit0 < prm.units ? all_units - unit0 : prm.units;
    const int groups = units * NACC, Kp = prm.Kp;
    const int chunks = (Kp + CHUNK - 1) / CHUNK, steps = chunks * groups;
    uint8_t* ring = smem;
    int* partial = reinterpret_cast<int*>(ring + slots * SLOT);                            // [warp][group][R8][32 lanes][2]

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < slots; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], WARPS);
        }
        abort_word = 0;
        for (int r = 0; r < MAX_RAW; ++r) tops[r] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    int asked = 0;                                     // the weight warp's copies into the ring so far, eight rows each
    if (warp == WARPS) {
        // ---- weights
        int slot = 0, group = 0, k = 0;
        uint32_t parity = 1;                           // of the empty barrier: the ring's first round waits for nothing
        for (; asked < steps; ++asked) {
            // (the lanes poll each for itself and go on together: a vote, or one that gave up would leave the others behind)
            if (asked >= slots && !__all_sync(0xffffffffu, mbar_wait(&empty_bar[slot], parity, abort_flag, 41, p.status)))
                break;
            const uint32_t bytes = (uint32_t)(Kp - k < CHUNK ? Kp - k : CHUNK);
            if (lane == 0) mbar_expect_tx(&full_bar[slot], 8 * bytes);
            __syncwarp();
            if (lane < 8) {
                const int feature = (unit0 + group / NACC) * 8 + lane;
                const size_t row = (feature < p.N ? feature : p.N - 1) + (size_t)(group % NACC) * p.up_row_offset;
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(smem_u32(ring + slot * SLOT + lane * W_STRIDE)), "l"(p.w + row * p.w_stride + k), "r"(bytes),
                               "r"(smem_u32(&full_bar[slot])) : "memory");
            }
            if (++group == groups) group = 0, k += CHUNK;
            if (++slot == slots) slot = 0, parity ^= 1;
        }
    }
    pdl_wait();

    if (warp < WARPS) {
        // ---- activations
        RowScale scale{};
        if constexpr (RAW != INTEGERS) {
            // as many warps a row as there are, each with a share of its eights (or several rows a warp)
            const int parts = p.M < WARPS ? WARPS / p.M : 1, part = p.M < WARPS ? warp / p.M : 0;
            for (int row = p.M < WARPS ? warp % p.M : warp; row < p.M && part < parts; row += WARPS) {
                unsigned top = 0;
#pragma unroll 4
                for (int k = (part * 32 + lane) * EIGHT; k < p.K; k += parts * 32 * EIGHT) {
                    float v[EIGHT];
                    raw_values<RAW>(prm, row, k, v);
#pragma unroll
                    for (int i = 0; i < EIGHT; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0) atomicMax(&tops[row], top);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
            scale = row_scale(tops[g < p.M ? g : 0], RAW == RAW_BF16);
        }
        uint4 x_next[KBLK][R8];
        const signed char* x_at[R8];
#pragma unroll
        for (int r = 0; r < R8; ++r) x_at[r] = g + 8 * r < p.M ? p.x + (size_t)(g + 8 * r) * p.x_stride : nullptr;
        auto fetch_rows = [&](int k) {
            if constexpr (RAW != INTEGERS) {
#pragma unroll
                for (int b = 0; b < KBLK; ++b) {
                    uint2 one = make_uint2(0, 0), two = make_uint2(0, 0);
                    if (g < p.M && k + b * 64 < p.K) {
                        float v[EIGHT];
                        raw_values<RAW>(prm, g, k + b * 64, v);
                        one = quantize(v, scale);
                        raw_values<RAW>(prm, g, k + b * 64 + EIGHT, v);
                        two = quantize(v, scale);
                    }
                    x_next[b][0] = make_uint4(one.x, one.y, two.x, two.y);
                }
            } else {
#pragma unroll
                for (int b = 0; b < KBLK; ++b)
#pragma unroll
                    for (int r = 0; r < R8; ++r)
                        x_next[b][r] = x_at[r] && k + b * 64 < Kp ? load_rows(x_at[r] + k + b * 64) : make_uint4(0, 0, 0, 0);
            }
        };
        int x_k = warp * KBLK * 64 + t * 16;
        fetch_rows(x_k);

        // ---- the walk: chunk by chunk of K, in every chunk group by group of features
        int slot = 0, w_k = 0;
        uint32_t parity = 0;
        for (int chunk = 0; chunk < chunks; ++chunk) {
            uint4 xv[KBLK][R8];
#pragma unroll
            for (int b = 0; b < KBLK; ++b)
#pragma unroll
                for (int r = 0; r < R8; ++r) xv[b][r] = x_next[b][r];
            x_k += CHUNK;
            if (chunk + 1 < chunks) fetch_rows(x_k);
            const int live = Kp - w_k - warp * KBLK * 64 - t * 16;    // this lane's k below Kp, from its first one on
            for (int group = 0; group < groups; ++group) {
                // (nothing goes by the answer: after a wait that gave up every later one ends at its first poll, the sums
                // are worth nothing and nobody stores them)
                mbar_wait(&full_bar[slot], parity, abort_flag, 42, p.status);
                const uint8_t* from = ring + slot * SLOT + g * W_STRIDE + warp * KBLK * 64 + t * 16;
                uint4 wv[KBLK];
#pragma unroll
                for (int b = 0; b < KBLK; ++b)
                    wv[b] = b * 64 < live ? *reinterpret_cast<const uint4*>(from + b * 64) : make_uint4(0, 0, 0, 0);
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[slot]);
                int acc[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][i] = 0;
#pragma unroll
                for (int b = 0; b < KBLK; ++b)
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint4 one = xv[b][2 * m];
                        const uint4 two = 2 * m + 1 < R8 ? xv[b][2 * m + 1 < R8 ? 2 * m + 1 : 0] : make_uint4(0, 0, 0, 0);
                        mma_16x8x32(acc[m], one.x, two.x, one.y, two.y, wv[b].x, wv[b].y);
                        mma_16x8x32(acc[m], one.z, two.z, one.w, two.w, wv[b].z, wv[b].w);
                    }
                int2* mine = reinterpret_cast<int2*>(partial) + (size_t)((warp * prm.units * NACC + group) * R8) * 32 + lane;
#pragma unroll
                for (int r = 0; r < R8; ++r) {
                    int2 v = make_int2(acc[r / 2][(r & 1) * 2], acc[r / 2][(r & 1) * 2 + 1]);
                    if (chunk > 0) {
                        const int2 before = mine[r * 32];
                        v.x += before.x, v.y += before.y;
                    }
                    mine[r * 32] = v;
                }
                if (++slot == slots) slot = 0, parity ^= 1;
            }
            w_k += CHUNK;
        }
    }
    __syncthreads();
    if (*abort_flag) {
        // somebody gave up: the copies still in flight land before the block's shared memory is another's.  The slot's
        // last phase, for each slot, with a limit of its own (the abort flag would end mbar_wait at once)
        if (warp == WARPS && lane < slots && asked > lane) {
            const uint32_t last = (uint32_t)((asked - 1 - lane) / slots) & 1;
            for (unsigned spin = 0; spin < WAIT_LIMIT && !mbar_test(&full_bar[lane], last); ++spin) __nanosleep(64);
        }
        return;
    }

    // ---- the warps' sums together, and what the caller wants done with them
    const int width = units * 8;
    if constexpr (RAW != INTEGERS) {
        // (the maxima become the scales)
        if (threadIdx.x < MAX_RAW) tops[threadIdx.x] = __float_as_uint(row_scale(tops[threadIdx.x], RAW == RAW_BF16).stored);
        __syncthreads();
    }
    for (int i = threadIdx.x; i < width * p.M; i += THREADS) {
        const int row = i / width, n = i - row * width, f = unit0 * 8 + n;
        if (f >= p.N) continue;
        const size_t at = (size_t)row * p.N + f;
        const float add = EPI == EPI_ADD_F32 ? p.addend[at] : 0.0f;
        float value[NACC];
#pragma unroll
        for (int a = 0; a < NACC; ++a) {
            const int* from = partial + (size_t)(((n >> 3) * NACC + a) * R8 + (row >> 3)) * 64 + ((row & 7) * 4 + ((n & 7) >> 1)) * 2 + (n & 1);
            int sum = 0;
#pragma unroll
            for (int wp = 0; wp < WARPS; ++wp) sum += from[(size_t)wp * prm.units * NACC * R8 * 64];
            value[a] = scaled(sum, RAW != INTEGERS ? __uint_as_float(tops[row]) : p.xs[row], p.ws[a * p.up_row_offset + f]);
        }
        store<EPI>(p, at, value[0], value[NACC - 1], add);
    }
}

template <int WARPS, int CTAS, int R8, int KBLK, int EPI, int RAW = INTEGERS>
int launch(RowsParams prm, cudaStream_t stream) {
    constexpr int NACC = EPI == EPI_GATED_BF16 ? 2 : 1, CHUNK = WARPS * KBLK * 64, SLOT = 8 * row_stride(CHUNK);
    constexpr int MOST = 16 / (NACC * R8) ? 16 / (NACC * R8) : 1;    // units a CTA keeps partial sums of: 32 KiB
    const Product& p = prm.p;
    const int all_units = (p.N + 7) / 8;
    // as many CTAs an SM as can be resident, or as few more as the partial sums allow, evenly filled; one for a matrix that
    // a single ring an SM nearly holds
    int rounds = (long)p.N * NACC * p.K > ALL_CTAS_FROM ? CTAS : 1;
    while ((all_units + 148 * rounds - 1) / (148 * rounds) > MOST) ++rounds;
    prm.units = (all_units + 148 * rounds - 1) / (148 * rounds);
    const int ctas = (all_units + prm.units - 1) / prm.units;
    const int fixed = WARPS * prm.units * NACC * R8 * 256;
    const int steps = prm.units * NACC * ((prm.Kp + CHUNK - 1) / CHUNK);
    int slots = (SMEM_OF_SM / CTAS - 2048 - fixed) / SLOT;
    slots = slots > MAX_SLOTS ? MAX_SLOTS : slots;
    slots = slots > steps ? steps : slots;
    prm.slots = slots < 2 ? 2 : slots;
    auto kernel = linear_rows_int8_kernel<WARPS, CTAS, R8, KBLK, EPI, RAW>;
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    fwb::pdl(kernel, ctas, 32 * (WARPS + 1), fixed + prm.slots * SLOT, stream)(prm);
    return fwb_launch_status();
}

// Measured in a chain of launches over 300 MB of weights (us): a short K fills half a step of eight warps -- 8 tokens, gated
// 1024 x 4608, 4.1 with eight warps a CTA, 3.5 with four and twice the CTAs; 16 tokens 4.5 and 3.9; at K 2048 gated 2048 x 8192
// 7.6 and 7.3, but 8192 x 2048 5.2 and 5.9, 2048 x 2048 2.9 and 3.0.
constexpr int SHORT_K = 1024;
template <int EPI>
int launch_rows(const RowsParams& prm, cudaStream_t stream) {
    const bool is_short = prm.Kp <= SHORT_K;
    if (prm.p.M > 16) return launch<8, 2, 4, 2, EPI>(prm, stream);
    if (prm.p.M > 8) return is_short ? launch<4, 4, 2, 2, EPI>(prm, stream) : launch<8, 2, 2, 4, EPI>(prm, stream);
    return is_short ? launch<4, 4, 1, 4, EPI>(prm, stream) : launch<8, 2, 1, 4, EPI>(prm, stream);
}

}  // namespace

int fwb::int8::few_tokens(const Product& p, int epilogue, cudaStream_t stream) {
    if (p.M > MAX_FEW) return FWB_TOO_LARGE;
    const RowsParams prm{p, (p.K + 15) & ~15, 0, 0, nullptr};
    switch (epilogue) {
        case EPI_F32: return launch_rows<EPI_F32>(prm, stream);
        case EPI_BF16: return launch_rows<EPI_BF16>(prm, stream);
        case EPI_ADD_F32: return launch_rows<EPI_ADD_F32>(prm, stream);
        case EPI_GATED_BF16: return launch_rows<EPI_GATED_BF16>(prm, stream);
        default: return FWB_UNSUPPORTED;
    }
}

namespace {
template <int EPI>
int launch_raw(const RowsParams& prm, bool is_bf16, cudaStream_t stream) {
    const bool is_short = prm.Kp <= SHORT_K;
    if (is_bf16) return is_short ? launch<4, 4, 1, 4, EPI, RAW_BF16>(prm, stream) : launch<8, 2, 1, 4, EPI, RAW_BF16>(prm, stream);
    return is_short ? launch<4, 4, 1, 4, EPI, RAW_F32>(prm, stream) : launch<8, 2, 1, 4, EPI, RAW_F32>(prm, stream);
}
}  // namespace

int fwb::int8::few_raw_tokens(const Product& p, const void* raw, bool is_bf16, int epilogue, cudaStream_t stream) {
    if (p.M > MAX_RAW || p.K > MAX_RAW_K) return FWB_TOO_LARGE;
    if ((p.K & 7) || ((uintptr_t)raw & 15)) return FWB_UNSUPPORTED;
    const RowsParams prm{p, (p.K + 15) & ~15, 0, 0, raw};
    switch (epilogue) {
        case EPI_F32: return launch_raw<EPI_F32>(prm, is_bf16, stream);
        case EPI_BF16: return launch_raw<EPI_BF16>(prm, is_bf16, stream);
        case EPI_ADD_F32: return launch_raw<EPI_ADD_F32>(prm, is_bf16, stream);
        case EPI_GATED_BF16: return launch_raw<EPI_GATED_BF16>(prm, is_bf16, stream);
        default: return FWB_UNSUPPORTED;
    }
}
