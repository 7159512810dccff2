// Attention of requests that share their first pages, bfloat16, head sizes up to 128, on tensor cores.
//
//   prefix kernel   a CTA: 128 rows -- (token, query head of one KV head) pairs of one group -- against one slice of the group's
//                   shared pages, in steps of 128 keys (64 at head sizes above 64): S = Q K^T by tcgen05.mma into tensor
//                   memory, a thread a row for the softmax, P as bfloat16 pairs into columns of its own, O += P V with P
//                   read from tensor memory.  The scores of a step are computed while the softmax works on those of the
//                   step before, which it holds in registers.  m follows the running maximum only when that has grown by
//                   more than 2^8.  Leaves m (in base 2), l and O, not divided, of its slice in scratch, fp32.
//   own kernel      a CTA: one token and up to 16 query heads of one KV head (the rows of mma.sync 16 x 8 x 16), in large batches
//                   as many neighbouring tokens of a request as have room there, one slice of the keys behind the shared ones;
//                   four warps take 16 keys each of every 64-key tile that TMA brings, with a running maximum and sum each.
//                   The warps' results meet in shared memory, the slices' in a cluster, the shared part's slices from scratch
//                   (or, alone, all keys are its own): m = max m_i, O = sum 2^(m_i - m) O_i, l likewise; a sink joins m and l.
//
// The shared keys are thus read once for 128 rows.  The own kernel starts as the prefix kernel's CTAs leave and waits for them
// only ahead of the join: the prefix kernel lets it start when it has itself waited for the kernel in front, so everything that the own
// kernel reads before the join was written earlier than that.
//
// Measured on B200, bf16 (us; what the bytes take at a copy's 6.57 TB/s, the products at 1,670 TFLOP/s): 64 requests of 32 heads over 8
// of 64 behind 8,192 keys, each with up to 500 of its own, 31.7 (7.8; 2.7): the prefix kernel 21.5, then 8 to 9 until the
// last own keys are walked and all is joined -- blocks' latencies from arrays to pages to products, 1.5 us a page under load;
// 256 requests behind 32,768 keys, up to 1,000 own, 175 (50.5; 41.8): 120 and 55, one behind the other.  In the prefix kernel there no
// pipe is full -- special functions 56 %, tensor 39 %, issue slots 33 %, DRAM 5 % -- the two warps a scheduler wait along the chain of
// scores, softmax and product; the own kernel reads 290 MB at 5 TB/s, four CTAs an SM.  Two prefix CTAs an SM (82 or 96 KiB each, 168
// registers a thread) hide one's softmax behind the other's products; three with the scores under P: slower.
//
// Masked keys are left out by selection; rows of V behind the last key anybody sees are cleared in shared memory, so that
// 0 * (infinity or NaN) cannot reach a result.  A page id outside the pool is fetched as zeros and masked.
// Every wait on an mbarrier is bounded: after the limit the CTA raises the library's status word, every role stops waiting, copies
// in flight land, tensor memory is freed and the CTA returns.
#include "attention_prefix.cuh"
#include "tcgen05.cuh"

using namespace fwb;
using namespace fwb::tc5;
using namespace fwb::prefix;

namespace {

constexpr int ROWS = 128;        // query rows of a prefix CTA (UMMA M)
constexpr int KEYS = PAGE;
constexpr int SOFTMAX_WARPS = 4, PREFIX_THREADS = 64 + 32 * SOFTMAX_WARPS;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.0f;   // O is rescaled when a row's maximum has grown by more than 2^8
constexpr int KV_BOX = KEYS * 128;     // 64 keys x 64 channels
constexpr int OWN_WARPS = 4, OWN_THREADS = 32 * (OWN_WARPS + 1), OWN_ROWS = 16;

struct Params {
    Batch b;
    const __nv_bfloat16* q;      // [T][nh * hd]
    __nv_bfloat16* out;          // [T][nh * hd]
    float* part_o;               // [T][nh][splits][hd]
    float* part_ml;              // [T][nh][splits][2]
    const float* sink;           // [nh] or null
    int nh, nkv, group, hd, splits, head_chunk, head_chunks;
    float scale_log2;            // softmax scale * log2(e)
    float cap_pre, cap_unit;     // capped scores: raw <- cap_unit * tanh(raw * cap_pre), cap_pre = scale / cap,
                                 // cap_unit = cap / scale, so that the scale that follows gives cap * tanh(score / cap); 0: off
    int pool_rows;               // num_pages * nkv * 64: a row from here on is fetched as zeros
    int stages;                  // own kernel: depth of the ring
    int alone;                   // own kernel: no prefix kernel in front, it walks the shared pages too
    int* status;
};

// Tensor memory of a CTA is 256 columns, so that two CTAs fit an SM: the scores of a step's keys, P (bfloat16 pairs), O.
template <int HD>
struct Layout {
    static constexpr int STEP = HD == 64 ? 128 : 64;         // keys a step
    static constexpr int PAGES = STEP / KEYS, BOXES = HD / 64;
    static constexpr int Q_BOX = ROWS * 128, Q_BYTES = BOXES * Q_BOX;
    static constexpr int KV_BYTES = PAGES * BOXES * KV_BOX;  // keys (or values) of a step
    static constexpr int SLOTS = 2;                          // of K and of V each
    static constexpr int DATA = Q_BYTES + 2 * SLOTS * KV_BYTES;
    static constexpr int SMEM = DATA + 1024 + 256;
    static constexpr int P_COL = STEP, O_COL = STEP + STEP / 2, TMEM_COLS = 256;
    static_assert(O_COL + HD <= TMEM_COLS, "tensor memory");
};

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 2^x on the special-function unit (relative error 2^-22; results below 2^-126 are 0).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two floats in a register pair, for the packed fp32 instructions.
__device__ __forceinline__ unsigned long long pair(float lo, float hi) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpair(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {         // NaN if one of them is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// The products as the issuing thread gives them out: descriptors as their two words, of which only the lower one (the address)
// changes, and the accumulate flag as a constant.  Everything it computes itself is paid once a tile between four warps' softmax.
template <bool ACCUMULATE>
__device__ __forceinline__ void umma_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "n"(ACCUMULATE ? 1 : 0)
        : "memory");
}
// A (P, bfloat16 pairs in 32-bit columns) read from tensor memory.
__device__ __forceinline__ void umma_a_tmem_lo(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// the first row of a page's tile in the pool, seen as rows of hd entries; behind the pool's end for an id that is no page
__device__ __forceinline__ int tile_row(const Params& prm, int page, int kvh) {
    return prm.b.is_page(page) ? (page * prm.nkv + kvh) * KEYS : prm.pool_rows;
}

// CAPPED: with the soft cap's code (kept out of the other form: jumping over it costs more than a tenth of a step in fetches)
template <int HD, bool CAPPED>
__global__ void __launch_bounds__(PREFIX_THREADS, 2)
prefix_tcgen05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params prm) {
    using L = Layout<HD>;
    constexpr int STEP = L::STEP, PAGES = L::PAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* q_s = base;
    uint8_t* k_s = q_s + L::Q_BYTES;
    uint8_t* v_s = k_s + L::SLOTS * L::KV_BYTES;
    uint64_t* k_full = reinterpret_cast<uint64_t*>(base + L::DATA);      // [SLOTS] each
    uint64_t* k_empty = k_full + L::SLOTS;
    uint64_t* v_full = k_empty + L::SLOTS;
    uint64_t* v_empty = v_full + L::SLOTS;
    uint64_t* q_ready = v_empty + L::SLOTS;
    uint64_t* s_ready = q_ready + 1;                       // the scores of a step are in tensor memory
    uint64_t* s_taken = s_ready + 1;                       // ... and in the softmax threads' registers
    uint64_t* p_ready = s_taken + 1;                       // P of a step is in tensor memory
    uint64_t* pv_ready = p_ready + 1;                      // ... and in O
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(pv_ready + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::SLOTS; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        mbar_init(q_ready, SOFTMAX_WARPS);
        mbar_init(s_ready, 1);
        mbar_init(s_taken, SOFTMAX_WARPS);
        mbar_init(p_ready, SOFTMAX_WARPS);
        mbar_init(pv_ready, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();                  // q, the pages and the batch's arrays come from earlier in the stream
    // Tensor memory is this CTA's before a kernel behind may start: one behind the own kernel could else take the columns and hold
    // them while it waits, by way of the own kernel, for this one.  (Not ahead of the wait: the same of the kernel in front.)
    if (warp == 1) tmem_alloc(tmem_holder, L::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    pdl_launch_dependents();     // (only now, too: the own kernel goes by everything in front of this one being done)

    // every warp finds the work by itself: the tile's tokens, its slice of the pages, how far anybody sees
    const int per_tile = ROWS / prm.head_chunk;
    const TokenTile tile = token_tile(prm.b, blockIdx.x, per_tile);
    const int pages = tile.pages, per = pages_per_slice(pages, prm.splits);
    const int page0 = blockIdx.z * per, page1 = min(pages, page0 + per);
    if (page0 >= page1) {                                  // (the whole CTA: nobody has asked for anything)
        if (warp == 1) tmem_dealloc(tmem_base, L::TMEM_COLS);
        return;
    }
    const int kvh = blockIdx.y / prm.head_chunks, head0 = (blockIdx.y % prm.head_chunks) * prm.head_chunk;
    const int heads = min(prm.head_chunk, prm.group - head0);
    const int* table = shared_row(prm.b, tile);
    int far = -1;
    for (int i = lane; i < tile.count; i += 32)
        if (prm.b.row_of(tile.first + i)) far = max(far, prm.b.last_key(prm.b.positions[tile.first + i]));
    far = min(__reduce_max_sync(0xffffffffu, far), page1 * KEYS - 1);
    const int n_pages = !table || far < page0 * KEYS ? 0 : far / KEYS + 1 - page0;
    const int n_steps = (n_pages + PAGES - 1) / PAGES;
    int asked = 0;                                         // the producer's: steps asked for so far

    if (warp == 0) {
        // a page that is none, or behind the slice's last, comes as zeros
        int ids = -1;                                      // 32 page ids, a lane each
        for (int t = 0; t < n_steps; ++t) {
            const int s = t % L::SLOTS;
            if (t * PAGES % 32 == 0) ids = t * PAGES + lane < n_pages ? table[page0 + t * PAGES + lane] : -1;
            int row[PAGES];
#pragma unroll
            for (int i = 0; i < PAGES; ++i) row[i] = tile_row(prm, __shfl_sync(0xffffffffu, ids, (t * PAGES + i) & 31), kvh);
            bool ok = true;
            if (lane == 0) {
                const uint32_t parity = ((t / L::SLOTS) - 1) & 1;
                if (t >= L::SLOTS) ok = mbar_wait(&k_empty[s], parity, abort_flag, 51, prm.status);
                if (ok) {
                    mbar_expect_tx(&k_full[s], L::KV_BYTES);
#pragma unroll
                    for (int i = 0; i < PAGES * L::BOXES; ++i)
                        tma_load_2d(k_s + (size_t)s * L::KV_BYTES + i * KV_BOX, &map_k, &k_full[s], i / PAGES * 64, row[i % PAGES]);
                    if (t >= L::SLOTS) ok = mbar_wait(&v_empty[s], parity, abort_flag, 54, prm.status);
                    if (ok) {
                        mbar_expect_tx(&v_full[s], L::KV_BYTES);
#pragma unroll
                        for (int i = 0; i < PAGES * L::BOXES; ++i)
                            tma_load_2d(v_s + (size_t)s * L::KV_BYTES + i * KV_BOX, &map_v, &v_full[s], i / PAGES * 64, row[i % PAGES]);
                    }
                    ++asked;
                }
            }
            if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
        }
    } else if (warp == 1) {
        if (lane == 0 && n_steps > 0) {
            constexpr uint32_t idesc_qk = make_idesc_mn(ROWS, STEP);
            constexpr uint32_t idesc_pv = make_idesc_mn(ROWS, HD) | IDESC_B_MN_MAJOR;
            const int k_steps = (prm.hd + UMMA_K - 1) / UMMA_K;
            const uint64_t q_desc = make_smem_desc(smem_u32(q_s)), k_desc = make_smem_desc(smem_u32(k_s));
            const uint64_t v_desc = make_smem_desc_mn_major(smem_u32(v_s), KV_BOX);
            const uint32_t q_lo = (uint32_t)q_desc, k_lo0 = (uint32_t)k_desc, v_lo0 = (uint32_t)v_desc;
            const uint32_t k_hi = (uint32_t)(k_desc >> 32), v_hi = (uint32_t)(v_desc >> 32);
            bool ok = mbar_wait(q_ready, 0, abort_flag, 52, prm.status);
            auto issue_qk = [&](int j) {
                const int s = j % L::SLOTS;
                ok = ok && mbar_wait(&k_full[s], (j / L::SLOTS) & 1, abort_flag, 53, prm.status);
                if (ok && j > 0) ok = mbar_wait(s_taken, (j - 1) & 1, abort_flag, 59, prm.status);
                if (!ok) return;
                tc_fence_after();
                const uint32_t k_lo = k_lo0 + s * (L::KV_BYTES >> 4);
#pragma unroll
                for (int kk = 0; kk < HD / UMMA_K; ++kk) {           // 16 channels: 32 bytes along the row, four to a box
                    const uint32_t qa = q_lo + (kk >> 2) * (L::Q_BOX >> 4) + 2 * (kk & 3), ka = k_lo + (kk >> 2) * (PAGES * KV_BOX >> 4) + 2 * (kk & 3);
                    if (kk == 0) umma_lo<false>(tmem_base, qa, ka, k_hi, idesc_qk);
                    else if (kk < k_steps) umma_lo<true>(tmem_base, qa, ka, k_hi, idesc_qk);
                }
                umma_commit(s_ready);
                umma_commit(&k_empty[s]);
            };
            issue_qk(0);
            for (int j = 0; j < n_steps && ok; ++j) {
                // the next scores while the softmax works on this step's, as soon as these are in its registers
                if (j + 1 < n_steps) issue_qk(j + 1);
                const int s = j % L::SLOTS;
                ok = ok && mbar_wait(&v_full[s], (j / L::SLOTS) & 1, abort_flag, 63, prm.status);
                ok = ok && mbar_wait(p_ready, j & 1, abort_flag, 55, prm.status);
                if (!ok) break;
                tc_fence_after();
                const uint32_t v_lo = v_lo0 + s * (L::KV_BYTES >> 4);
#pragma unroll
                for (int kk = 0; kk < STEP / UMMA_K; ++kk)            // 16 keys: 2048 bytes of V, 8 columns of P
                    umma_a_tmem_lo(tmem_base + L::O_COL, tmem_base + L::P_COL + kk * 8,
                                   v_lo + ((kk >> 2) * KV_BOX >> 4) + (kk & 3) * (2048 >> 4), v_hi, idesc_pv, kk > 0 ? 1u : (uint32_t)j);
                umma_commit(pv_ready);
                umma_commit(&v_empty[s]);
            }
        }
    } else {
        const int quarter = warp & 3, row = quarter * 32 + lane, swz = row & 7;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const int t_in = row / prm.head_chunk, h_in = row - t_in * prm.head_chunk;
        const bool valid = t_in < tile.count && h_in < heads;
        const int tok = tile.first + (valid ? t_in : 0), head = kvh * prm.group + head0 + (valid ? h_in : 0);
        const int hi = min(far, valid && prm.b.row_of(tok) ? prm.b.last_key(prm.b.positions[tok]) : -1);
        float m = -INFINITY, l = 0.0f;
        if (n_steps > 0) {
            const __nv_bfloat16* q_row = prm.q + ((size_t)tok * prm.nh + head) * prm.hd;
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                const uint4 v = valid && c * 8 < prm.hd ? *reinterpret_cast<const uint4*>(q_row + c * 8) : make_uint4(0u, 0u, 0u, 0u);
                *reinterpret_cast<uint4*>(q_s + (c >> 3) * L::Q_BOX + row * 128 + (((c & 7) ^ swz) << 4)) = v;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        }
        // from which key on some row of this warp does not see everything, and whether all of the slice's pages are pages
        const int whole_to = __reduce_min_sync(0xffffffffu, valid ? hi + 1 : 0x7fffffff);
        bool all_pages = true;
        for (int i = lane; i < n_pages; i += 32) all_pages &= prm.b.is_page(table[page0 + i]);
        all_pages = __all_sync(0xffffffffu, all_pages);
        const unsigned long long scale2 = pair(prm.scale_log2, prm.scale_log2);
        unsigned long long sum2 = 0;
        for (int j = 0; j < n_steps; ++j) {
            const int key0 = (page0 + j * PAGES) * KEYS;
            // (nothing goes by the answers of this loop's waits: after one that gave up every other ends at its first poll, and nobody
            // stores)
            mbar_wait(s_ready, j & 1, abort_flag, 56, prm.status);
            __syncwarp();                                  // tcgen05.ld needs the whole warp
            tc_fence_after();
            float sc[STEP];
            if constexpr (STEP == 128) tmem_ld128(lane_addr, sc);
            else tmem_ld64(lane_addr, sc);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_taken);
            if constexpr (CAPPED) {
                // a warp whose scores of this step all lie far below the cap takes the polynomial: it spares the
                // special-function unit, which the exponentials need
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < STEP; ++i) {
                    sc[i] *= prm.cap_pre;
                    top = fmaxf(top, fabsf(sc[i]));
                }
                if (__all_sync(0xffffffffu, top <= TANH_SMALL)) {
#pragma unroll
                    for (int i = 0; i < STEP; ++i) sc[i] = prm.cap_unit * tanh_small_f32(sc[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < STEP; ++i) sc[i] = prm.cap_unit * tanh_fast_f32(sc[i]);
                }
            }
            // a step every row sees whole needs no mask (rows without a token are never stored)
            const bool whole = all_pages && key0 + STEP <= whole_to;
            if (__builtin_expect(!whole, 0)) {
#pragma unroll
                for (int i = 0; i < PAGES; ++i) {
                    const int p = j * PAGES + i;
                    const int last = p < n_pages && prm.b.is_page(table[page0 + p]) ? hi : -1;
#pragma unroll
                    for (int k = 0; k < KEYS; ++k) sc[i * KEYS + k] = key0 + i * KEYS + k <= last ? sc[i * KEYS + k] : -INFINITY;
                }
            }
            // four interleaved chains for the maximum, two values a link
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < STEP; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], sc[i], sc[i + 1]);
            const float step_max = max3(mx[0], mx[1], fmaxf(mx[2], mx[3])) * prm.scale_log2;
            const bool moved = step_max > m + RESCALE_STEP;          // also: the row's first keys (m = -inf)
            float factor = 1.0f;
            if (moved) {
                factor = ex2(m - step_max);                          // 2^(-inf) = 0 for the first keys
                m = step_max;
                l *= factor;
                sum2 = fma2(sum2, pair(factor, factor), 0);
            }
            if (j > 0) {
                // PV of the step before has read its P, whose columns this one's takes, and landed in O
                mbar_wait(pv_ready, (j - 1) & 1, abort_flag, 58, prm.status);
                __syncwarp();
                tc_fence_after();
                if (__builtin_expect(__any_sync(0xffffffffu, moved), 0)) {
                    // scale this warp's rows (by exactly 1 where nothing moved)
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 16) {
                        float v[16];
                        tmem_ld16(lane_addr + L::O_COL + c0, v);
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] *= factor;
                        tmem_st16_async(lane_addr + L::O_COL + c0, v);
                    }
                    tmem_st_wait();
                }
            }
            const float zero = m == -INFINITY ? 0.0f : m;            // a row that has seen no key yet
            const unsigned long long minus = pair(-zero, -zero);
#pragma unroll
            for (int c0 = 0; c0 < STEP; c0 += 32) {
                float packed[16];
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    float p0, p1;
                    unpair(fma2(pair(sc[c0 + i], sc[c0 + i + 1]), scale2, minus), p0, p1);
                    p0 = ex2(p0), p1 = ex2(p1);                      // masked: 2^(-inf) = 0
                    sum2 = add2(sum2, pair(p0, p1));
                    packed[i >> 1] = __uint_as_float(pack2(p0, p1));
                }
                tmem_st16_async(lane_addr + L::P_COL + c0 / 2, packed);
            }
            if (!(step_max < INFINITY)) l = __int_as_float(0x7fffffff);     // an infinity or NaN among the scores
            tmem_st_wait();
            tc_fence_before();
            const int seen = far + 1 - key0;                          // keys of this step anybody may see
            if (__builtin_expect(seen < STEP, 0)) {
                // only the last step: clear the V rows behind them (whole 128-byte rows of every box)
                const int s = j % L::SLOTS;
                mbar_wait(&v_full[s], (j / L::SLOTS) & 1, abort_flag, 57, prm.status);
                uint8_t* v_tile = v_s + (size_t)s * L::KV_BYTES;
                const int chunks = (STEP - seen) * 8;
                for (int b = 0; b < L::BOXES; ++b)
                    for (int i = threadIdx.x - 64; i < chunks; i += 32 * SOFTMAX_WARPS)
                        *reinterpret_cast<uint4*>(v_tile + b * PAGES * KV_BOX + seen * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async();                                  // the cleared rows, for the tensor core
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready);
        }
        {
            float a, b;
            unpair(sum2, a, b);
            l += a + b;
        }
        bool ok = true;
        if (n_steps > 0) {
            ok = mbar_wait(pv_ready, (n_steps - 1) & 1, abort_flag, 60, prm.status);
            ok = __all_sync(0xffffffffu, ok && !*abort_flag);
        }
        if (ok) {
            tc_fence_after();
            const size_t at = ((size_t)tok * prm.nh + head) * prm.splits + blockIdx.z;
            // (a slice that a row sees nothing of is left out by its m: its O is not read)
            if (valid) *reinterpret_cast<float2*>(prm.part_ml + 2 * at) = make_float2(m, l);
            if (n_steps > 0) {
#pragma unroll
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    float v[32];
                    tmem_ld32(lane_addr + L::O_COL + c0, v);
                    if (valid) {
#pragma unroll
                        for (int c = 0; c < 32; c += 4)
                            if (c0 + c < prm.hd)
                                *reinterpret_cast<float4*>(prm.part_o + at * prm.hd + c0 + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                    }
                }
                tc_fence_before();
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag)
        for (int s = 0; s < L::SLOTS && s < asked; ++s) {            // copies still in flight land first
            const uint32_t last = (uint32_t)((asked - 1 - s) / L::SLOTS) & 1;
            for (unsigned spin = 0; spin < WAIT_LIMIT && !mbar_test(&k_full[s], last); ++spin) __nanosleep(64);
            for (unsigned spin = 0; spin < WAIT_LIMIT && !mbar_test(&v_full[s], last); ++spin) __nanosleep(64);
        }
    if (warp == 1) tmem_dealloc(tmem_base, L::TMEM_COLS);
}

// ------------------------------------------------------------------ own keys and the join
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// The tokens that a CTA takes together: at most `most` (2 to 16) neighbours of one request in one group.  Their run is cut off from its
// first token on, every `most` of them, as far as the look back of 31 - most tokens reaches, there, and from there on where the token's
// number is a multiple of `most`.
// Asked by whole warps with the request of token `t + most - 1 - lane` (anything where there is no such token).
// 0: token t is not the first of such a piece.
__device__ __forceinline__ int run_of(const Batch& b, const Token& token, int t, int most, int seg_around) {
    if (!token.table) return 1;
    const int lane = threadIdx.x & 31, seg = __shfl_sync(0xffffffffu, seg_around, most - 1);
    const int at = t + most - 1 - lane, reach = 31 - most;
    const unsigned same = __ballot_sync(0xffffffffu, at >= token.first && at < token.end && seg_around == seg);
    const int before = __ffs(~(same >> most)) - 1;         // tokens of the run in front of t, reach + 1 and more as reach + 1
    const int behind = __clz(~(same << (33 - most)));      // and behind it, at most most - 1
    // lane d: whether token t + d begins a piece (behind the run: as if)
    const int offset = before + lane;
    const bool begins = lane > behind || (offset <= reach ? offset == reach || offset % most == 0 : (t + lane) % most == 0);
    const unsigned pieces = __ballot_sync(0xffffffffu, begins);
    return pieces & 1 ? __ffs(pieces >> 1) : 0;
}
// 2^(m - of), 0 for a part that has seen nothing
__device__ __forceinline__ float part_weight(float m, float of) { return m == -INFINITY ? 0.0f : ex2(m - of); }

template <int HD>
struct OwnLayout {
    static constexpr int BOXES = HD / 64, KV_BYTES = BOXES * KV_BOX, STAGE = 2 * KV_BYTES;
    static constexpr int MERGE_FLOATS = OWN_WARPS * OWN_ROWS * (HD + 2);        // O, m and l of the warps
    static constexpr int data(int stages) { return stages * STAGE > MERGE_FLOATS * 4 ? stages * STAGE : MERGE_FLOATS * 4; }
};

template <int HD, bool TOGETHER>          // TOGETHER: a CTA takes neighbouring tokens of a request, as many as have rows (else one)
__global__ void __launch_bounds__(OWN_THREADS, HD == 64 ? 4 : 3)
own_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params prm) {
    using L = OwnLayout<HD>;
    constexpr int MAX_STAGES = 8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES];
    __shared__ int abort_word, page_ok[MAX_STAGES];
    __shared__ float joined[OWN_ROWS][2];                  // m and l of this CTA's rows, its warps together
    __shared__ float own_weight[OWN_ROWS][8], shared_weight[OWN_ROWS][MAX_SPLITS], inverse[OWN_ROWS];
    volatile int* abort_flag = &abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3, stages = prm.stages;
    const int slices = gridDim.z, slice = blockIdx.z;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], OWN_WARPS);
        }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (prm.alone) pdl_wait();
    pdl_launch_dependents();     // (the kernel behind waits for all of this one)
    const int t = blockIdx.x, chunks = (prm.group + OWN_ROWS - 1) / OWN_ROWS;
    const int kvh = blockIdx.y / chunks, head0 = kvh * prm.group + (blockIdx.y % chunks) * OWN_ROWS;
    const int heads = min(OWN_ROWS, (kvh + 1) * prm.group - head0);
    int seg_around = -1, position = -1, most = 1;
    if constexpr (TOGETHER) {
        most = OWN_ROWS / prm.group;
        const int around = t + most - 1 - lane;
        if (around >= 0 && around < prm.b.T) seg_around = prm.b.tok_seg[around];
        if (lane < most && t + lane < prm.b.T) position = prm.b.positions[t + lane];
    }
    const Token token = token_of(prm.b, t);
    const int tokens = TOGETHER ? run_of(prm.b, token, t, most, seg_around) : 1;
    if (token.pages < 0 || tokens == 0) {                  // rows of no group stay as they are; the whole cluster leaves
        pdl_wait();
        return;
    }
    // rows: token, head.  `sees`: the last key that this lane's token sees
    const int rows = tokens * heads, pages = prm.alone ? 0 : token.pages;
    int sees = token.last, last = token.last, least = token.last;
    if constexpr (TOGETHER) {
        sees = token.table ? prm.b.last_key(position) : -1;
        last = __reduce_max_sync(0xffffffffu, lane < tokens ? sees : -1);
        least = __reduce_min_sync(0xffffffffu, lane < tokens ? sees : 0x7fffffff);
    }
    const int* table = token.table;
    const int own = last >= pages * KEYS ? last / KEYS + 1 - pages : 0, per = (own + slices - 1) / slices;
    const int tile0 = pages + slice * per, tile1 = min(pages + own, tile0 + per), n_tiles = max(0, tile1 - tile0);
    __syncthreads();

    int asked = 0;
    float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    if (warp == OWN_WARPS) {
        int ids = -1;
        for (int j = 0; j < n_tiles; ++j) {
            const int s = j % stages;
            if (j % 32 == 0) ids = j + lane < n_tiles ? table[tile0 + j + lane] : -1;
            const int page = __shfl_sync(0xffffffffu, ids, j & 31);
            bool ok = true;
            if (lane == 0) {
                if (j >= stages) ok = mbar_wait(&empty[s], ((j / stages) - 1) & 1, abort_flag, 61, prm.status);
                if (ok) {
                    page_ok[s] = prm.b.is_page(page);
                    mbar_expect_tx(&full[s], L::STAGE);
                    const int row = tile_row(prm, page, kvh);
                    uint8_t* stage = ring + (size_t)s * L::STAGE;
#pragma unroll
                    for (int b = 0; b < L::BOXES; ++b) {
                        tma_load_2d(stage + b * KV_BOX, &map_k, &full[s], b * 64, row);
                        tma_load_2d(stage + L::KV_BYTES + b * KV_BOX, &map_v, &full[s], b * 64, row);
                    }
                    ++asked;
                }
            }
            if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
        }
    } else if (n_tiles > 0) {
        uint32_t qf[HD / 16][4];
        int token_of_row[2] = {0, 0}, sees_of_row[2] = {last, last};
        if constexpr (TOGETHER) {
#pragma unroll
            for (int i = 0; i < 2; ++i) token_of_row[i] = (g + 8 * i) / heads, sees_of_row[i] = __shfl_sync(0xffffffffu, sees, token_of_row[i]);
        }
        const __nv_bfloat16* q_at = prm.q + ((size_t)t * prm.nh + head0) * prm.hd;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = g + (i & 1) * 8, c = kk * 16 + (i >> 1) * 8 + t4 * 2, j = token_of_row[i & 1];
                qf[kk][i] = r < rows && c < prm.hd ? *reinterpret_cast<const uint32_t*>(q_at + ((size_t)j * prm.nh + r - j * heads) * prm.hd + c) : 0u;
            }
        const int key_k = warp * 16 + (lane >> 4) * 8 + (lane & 7), chunk_k = (lane >> 3) & 1;     // ldmatrix rows of K and V
        const int key_v = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), chunk_v = lane >> 4;
        bool ok = true;
        for (int j = 0; j < n_tiles; ++j) {
            const int s = j % stages, key0 = (tile0 + j) * KEYS + warp * 16;
            ok = mbar_wait(&full[s], (j / stages) & 1, abort_flag, 62, prm.status);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (page_ok[s] && key0 <= last) {
                const uint32_t k_at = smem_u32(ring + (size_t)s * L::STAGE), v_at = k_at + L::KV_BYTES;
                float sc[2][4] = {};
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    uint32_t b[4];
                    const int chunk = (2 * kk + chunk_k) & 7;
                    ldmatrix_x4(b, k_at + (kk >> 2) * KV_BOX + key_k * 128 + ((chunk ^ (key_k & 7)) << 4));
                    mma_bf16(sc[0], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b[0], b[1]);
                    mma_bf16(sc[1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b[2], b[3]);
                }
                if (prm.cap_pre != 0.0f) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[n][i] = prm.cap_unit * tanh_fast_f32(sc[n][i] * prm.cap_pre);
                }
                const bool whole = key0 + 15 <= least, mixed = TOGETHER && least < min(last, key0 + 15);
                if (!whole) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[n][i] = key0 + n * 8 + t4 * 2 + (i & 1) <= sees_of_row[i >> 1] ? sc[n][i] : -INFINITY;
                    // the values of keys that nobody sees, whatever they hold (the slice's last tile: nothing is copied over it)
                    for (int i = lane; i < (15 - (last - key0)) * 8 * L::BOXES; i += 32) {
                        const int r = warp * 16 + (last - key0) + 1 + (i >> 3) % (15 - (last - key0));
                        const int box = (i >> 3) / (15 - (last - key0));
                        *reinterpret_cast<uint4*>(ring + (size_t)s * L::STAGE + L::KV_BYTES + box * KV_BOX + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                float factor[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float top = quad_max(fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]))) * prm.scale_log2;
                    const float now = fmaxf(m[r], top), zero = now == -INFINITY ? 0.0f : now;
                    factor[r] = ex2(m[r] - zero);
                    m[r] = now;
                    float sum = 0.0f;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 2 * r; i < 2 * r + 2; ++i) {
                            sc[n][i] = ex2(fmaf(sc[n][i], prm.scale_log2, -zero));
                            sum += sc[n][i];
                        }
                    l[r] = l[r] * factor[r] + sum;
                }
                const uint32_t p0 = pack2(sc[0][0], sc[0][1]), p1 = pack2(sc[0][2], sc[0][3]), p2 = pack2(sc[1][0], sc[1][1]), p3 = pack2(sc[1][2], sc[1][3]);
                if (__any_sync(0xffffffffu, factor[0] != 1.0f || factor[1] != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) o[i][0] *= factor[0], o[i][1] *= factor[0], o[i][2] *= factor[1], o[i][3] *= factor[1];
                }
                auto values = [&](uint32_t (&b)[4], int n) {
                    const int chunk = (n + chunk_v) & 7;
                    ldmatrix_x4_trans(b, v_at + (n >> 3) * KV_BOX + key_v * 128 + ((chunk ^ (key_v & 7)) << 4));
                };
                if (!mixed) {
#pragma unroll
                    for (int n = 0; n < HD / 8; n += 2) {
                        uint32_t b[4];
                        values(b, n);
                        mma_bf16(o[n], p0, p1, p2, p3, b[0], b[1]);
                        mma_bf16(o[n + 1], p0, p1, p2, p3, b[2], b[3]);
                    }
                } else {
                    // some of the tokens see all of these keys: a token at a time, with the values that it sees and for its rows
#pragma unroll 1
                    for (int j = 0; j < tokens; ++j) {
                        const int seen = __shfl_sync(0xffffffffu, sees, j) - key0 - 2 * t4;
                        const uint32_t front = (seen >= 0 ? 0xffffu : 0u) | (seen >= 1 ? 0xffff0000u : 0u);
                        const uint32_t behind = (seen >= 8 ? 0xffffu : 0u) | (seen >= 9 ? 0xffff0000u : 0u);
#pragma unroll
                        for (int n = 0; n < HD / 8; n += 2) {
                            uint32_t b[4];
                            values(b, n);
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                float d[4] = {};
                                mma_bf16(d, p0, p1, p2, p3, b[2 * k] & front, b[2 * k + 1] & behind);
                                if (token_of_row[0] == j) o[n + k][0] += d[0], o[n + k][1] += d[1];
                                if (token_of_row[1] == j) o[n + k][2] += d[2], o[n + k][3] += d[3];
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
    }
    __syncthreads();
    if (*abort_flag) {
        if (warp == OWN_WARPS && lane == 0)
            for (int s = 0; s < stages && s < asked; ++s) {          // copies still in flight land first
                const uint32_t done = (uint32_t)((asked - 1 - s) / stages) & 1;
                for (unsigned spin = 0; spin < WAIT_LIMIT && !mbar_test(&full[s], done); ++spin) __nanosleep(64);
            }
        __syncthreads();
    }
    // the warps' parts into shared memory, where the ring was: o_s [warp][row][HD], ml_s [warp][row][2]
    float* o_s = reinterpret_cast<float*>(ring);
    float* ml_s = o_s + OWN_WARPS * OWN_ROWS * HD;
    if (warp < OWN_WARPS) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] = quad_sum(l[r]);
            const int row = warp * OWN_ROWS + g + 8 * r;
            if (t4 == 0) ml_s[2 * row] = m[r], ml_s[2 * row + 1] = l[r];
            if (g + 8 * r < rows) {
#pragma unroll
                for (int n = 0; n < HD / 8; ++n)
                    *reinterpret_cast<float2*>(o_s + row * HD + n * 8 + t4 * 2) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
            }
        }
    }
    __syncthreads();
    const bool cluster = slices > 1;
    if (cluster) {
        // this CTA's warps together, for its peers to read (rows stay in o_s's first quarter): every thread has channels of rows
        if (threadIdx.x < OWN_ROWS) {
            const int row = threadIdx.x;
            float top = -INFINITY, sum = 0.0f;
            for (int w = 0; w < OWN_WARPS; ++w) top = fmaxf(top, ml_s[2 * (w * OWN_ROWS + row)]);
            for (int w = 0; w < OWN_WARPS; ++w) {
                const float f = part_weight(ml_s[2 * (w * OWN_ROWS + row)], top);
                sum += f * ml_s[2 * (w * OWN_ROWS + row) + 1];
                ml_s[2 * (w * OWN_ROWS + row)] = f;        // from here on: the warp's weight
            }
            joined[row][0] = top, joined[row][1] = sum;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < rows * HD; i += OWN_THREADS) {
            const int row = i / HD;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < OWN_WARPS; ++w) {
                const float f = ml_s[2 * (w * OWN_ROWS + row)];
                if (f != 0.0f) v = fmaf(f, o_s[(w * OWN_ROWS) * HD + i], v);
            }
            o_s[i] = v;
        }
    }
    pdl_wait();                  // the shared part is there
    if (cluster) cluster_sync_all();
    // the join: of the warps' parts, or with a cluster of the CTAs', each of which has a share of the rows.  First the parts'
    // weights, a warp a row and a lane a part (all of them asked for at once), then the sums, eight parts' channels on the way
    // together
    const int shared_per = pages ? pages_per_slice(pages, prm.splits) : 0, shared = pages ? (pages + shared_per - 1) / shared_per : 0;
    const int own_parts = cluster ? slices : OWN_WARPS;
    const uint32_t o_at = smem_u32(o_s), ml_at = smem_u32(joined);
    for (int row = warp; row < rows; row += OWN_WARPS + 1) {
        const int j = TOGETHER ? row / heads : 0, head = head0 + row - j * heads;
        const size_t at = ((size_t)(t + j) * prm.nh + head) * prm.splits;
        const float sink = prm.sink ? prm.sink[head] * LOG2E : -INFINITY;
        float2 part[(MAX_SPLITS + 31) / 32], mine = make_float2(-INFINITY, 0.0f);
        if (lane < own_parts) {
            mine.x = cluster ? ld_dsmem_f32(ml_at + row * 8, lane) : ml_s[2 * (lane * OWN_ROWS + row)];
            mine.y = cluster ? ld_dsmem_f32(ml_at + row * 8 + 4, lane) : ml_s[2 * (lane * OWN_ROWS + row) + 1];
        }
        float top = fmaxf(sink, mine.x);
#pragma unroll
        for (int i = 0; i < (MAX_SPLITS + 31) / 32; ++i) {
            part[i] = lane + 32 * i < shared ? *reinterpret_cast<const float2*>(prm.part_ml + 2 * (at + lane + 32 * i)) : make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, part[i].x);
        }
        top = warp_max(top);
        const float f = part_weight(mine.x, top);
        float sum = f * mine.y + (lane == 0 ? part_weight(sink, top) : 0.0f);
        if (lane < own_parts) own_weight[row][lane] = f;
#pragma unroll
        for (int i = 0; i < (MAX_SPLITS + 31) / 32; ++i) {
            const float w = part_weight(part[i].x, top);
            if (lane + 32 * i < shared) shared_weight[row][lane + 32 * i] = w;
            sum = fmaf(w, part[i].y, sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) inverse[row] = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
    __syncthreads();
    constexpr int LANES = HD / 4;                          // threads a row, four channels each
    for (int i = threadIdx.x; i < rows * LANES; i += OWN_THREADS) {
        const int row = i / LANES, c = (i - row * LANES) * 4, j = TOGETHER ? row / heads : 0;
        if ((cluster && row % slices != slice) || c >= prm.hd) continue;
        const size_t out_row = (size_t)(t + j) * prm.nh + head0 + row - j * heads;
        const float* parts = prm.part_o + out_row * prm.splits * prm.hd + c;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](float f, const float4& x) {
            v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
        };
        // (a part that weighs nothing may hold anything: it is not read)
        for (int s0 = 0; s0 < shared; s0 += 8) {
            float4 x[8];
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                f[k] = s0 + k < shared ? shared_weight[row][s0 + k] : 0.0f;
                x[k] = f[k] != 0.0f ? *reinterpret_cast<const float4*>(parts + (size_t)(s0 + k) * prm.hd) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) add(f[k], x[k]);
        }
        for (int s = 0; s < own_parts; ++s) {
            const float f = own_weight[row][s];
            if (f == 0.0f) continue;
            add(f, cluster ? ld_dsmem_f32x4(o_at + (uint32_t)(row * HD + c) * 4, s) : *reinterpret_cast<const float4*>(o_s + (s * OWN_ROWS + row) * HD + c));
        }
        if (!*abort_flag) {
            const float inv = inverse[row];
            *reinterpret_cast<uint2*>(prm.out + out_row * prm.hd + c) = make_uint2(pack2(v.x * inv, v.y * inv), pack2(v.z * inv, v.w * inv));
        }
    }
    if (cluster) cluster_sync_all();                       // nobody leaves while a peer still reads from it
}

template <int HD>
int launch(const CUtensorMap& map_k, const CUtensorMap& map_v, Params prm, int own_slices, bool neighbours, cudaStream_t stream) {
    using L = Layout<HD>;
    auto plain = prefix_tcgen05_kernel<HD, false>;
    auto capped = prefix_tcgen05_kernel<HD, true>;
    auto own = own_kernel<HD, false>, together = own_kernel<HD, true>;
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(plain, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(capped, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(own, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(together, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    prm.alone = prm.splits == 0;
    const long tiles = most_token_tiles(prm.b.T, prm.b.n_groups, ROWS / prm.head_chunk);
    if (!prm.alone) fwb::pdl(prm.cap_pre != 0.0f ? capped : plain, dim3((unsigned)tiles, prm.nkv * prm.head_chunks, prm.splits), PREFIX_THREADS, L::SMEM, stream)(map_k, map_v, prm);
    int e = fwb_launch_status();
    if (e) return e;
    prm.stages = HD == 64 ? 3 : 2;
    const int chunks = (prm.group + OWN_ROWS - 1) / OWN_ROWS;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(prm.b.T, prm.nkv * chunks, own_slices);
    config.blockDim = dim3(OWN_THREADS);
    config.dynamicSmemBytes = OwnLayout<HD>::data(prm.stages) + 1024;
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (own_slices > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = own_slices;
    }
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    config.attrs = attr;
    config.numAttrs = n;
    cudaError_t status = cudaLaunchKernelEx(&config, neighbours ? together : own, map_k, map_v, prm);
    return status == cudaSuccess ? fwb_launch_status() : (int)status;
}

}  // namespace

namespace fwb {
namespace prefix {

bool tensor_cores_take(const void* q, const void* k_pool, const void* v_pool, const void* out, const void* part_o, const Batch& b, int nkv, int hd) {
    return hd % 8 == 0 && hd <= 128 && (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out | (uintptr_t)part_o) & 15) == 0 &&
           (long)b.num_pages * nkv * PAGE <= 2147483647L - PAGE;
}

int launch_tensor_cores(const Batch& b, const void* q, const void* k_pool, const void* v_pool, void* out, float* part_o, float* part_ml,
                        const float* sink, int nh, int nkv, int hd, int splits, int own_slices, bool neighbours, float scale, float softcap,
                        cudaStream_t stream) {
    Params prm{};
    prm.b = b;
    prm.q = static_cast<const __nv_bfloat16*>(q);
    prm.out = static_cast<__nv_bfloat16*>(out);
    prm.part_o = part_o, prm.part_ml = part_ml, prm.sink = sink;
    prm.nh = nh, prm.nkv = nkv, prm.group = nh / nkv, prm.hd = hd, prm.splits = splits;
    prm.head_chunk = prm.group < ROWS ? prm.group : ROWS;
    prm.head_chunks = (prm.group + prm.head_chunk - 1) / prm.head_chunk;
    prm.scale_log2 = scale * LOG2E;
    prm.cap_pre = softcap > 0.0f ? scale / softcap : 0.0f;
    prm.cap_unit = softcap > 0.0f ? softcap / scale : 0.0f;
    const long rows = (long)b.num_pages * nkv * PAGE;
    prm.pool_rows = (int)rows;
    prm.status = status_word();
    CUtensorMap map_k, map_v;
    if (!make_map(&map_k, k_pool, rows, hd, KEYS) || !make_map(&map_v, v_pool, rows, hd, KEYS)) return FWB_UNSUPPORTED;
    return hd <= 64 ? launch<64>(map_k, map_v, prm, own_slices, neighbours, stream)
                    : launch<128>(map_k, map_v, prm, own_slices, neighbours, stream);
}

}  // namespace prefix
}  // namespace fwb
