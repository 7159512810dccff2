// Attention of requests that share their first pages, in fp32 arithmetic (any head size up to 256, fp32 or bf16 storage).
//
//   prefix kernel   a block: 64 rows -- (token, query head of one KV head) pairs of one group -- against one slice of the
//                   group's shared pages: S = Q K^T, softmax statistics, O = P V tile by tile with the running maximum and
//                   sum; leaves m, l and O (not divided) of its slice in scratch
//   own kernel      a block: one token and the query heads of one KV head over the keys behind the shared ones, then the
//                   join of all slices: m = max m_i, O = sum e^(m_i - m) O_i, l likewise (a sink joins m and l)
//
// Masked keys are left out by selection, so neither infinities nor NaN in them reach a result; rows of V behind a request's last key
// are not read.  A row that sees no key is zero.
#include "attention_prefix.cuh"

using namespace fwb;
using namespace fwb::prefix;

namespace {

constexpr int ROWS = 64, THREADS = 256;
constexpr int OWN_HEADS = 16;            // query heads a block of the own kernel takes

struct Params {
    Batch b;
    const void* q;               // [T][nh * hd]
    const void* k;               // [num_pages][nkv][64][hd]
    const void* v;
    float* part_o;               // [T][nh][splits][hd]
    float* part_ml;              // [T][nh][splits][2]
    void* out;                   // [T][nh * hd]
    const float* sink;           // [nh] or null
    int nh, nkv, group, hd, splits, head_chunk, head_chunks;
    float scale, cap;
};

__device__ __forceinline__ float score(const Params& prm, float dot) {
    const float s = dot * prm.scale;
    return prm.cap > 0.0f ? prm.cap * tanhf(s / prm.cap) : s;
}

// a page's tile of one KV head into shared memory, rows `pitch` floats apart; rows from `rows` on become zero
template <typename T>
__device__ __forceinline__ void load_tile(float* to, const void* pool, size_t tile, int rows, int hd, int pitch) {
    const T* from = reinterpret_cast<const T*>(pool) + tile * PAGE * hd;
    for (int i = threadIdx.x; i < PAGE * hd; i += THREADS) {
        const int r = i / hd, c = i - r * hd;
        to[r * pitch + c] = r < rows ? to_f32(from[i]) : 0.0f;
    }
}

template <typename T, int COLS>          // COLS: column blocks of 64 that hold a head
__global__ void __launch_bounds__(THREADS) prefix_kernel(const Params prm) {
    extern __shared__ float smem[];
    const int hd = prm.hd, pitch = ((hd + 3) & ~3) + 4;
    float* q_s = smem;                                 // [ROWS][pitch]
    float* k_s = q_s + ROWS * pitch;                   // [PAGE][pitch]
    float* v_s = k_s + PAGE * pitch;                   // [PAGE][COLS * 64]
    float* p_s = v_s + PAGE * COLS * 64;               // [ROWS][PAGE + 4]
    pdl_wait();
    pdl_launch_dependents();
    const int per_tile = ROWS / prm.head_chunk;
    const TokenTile tile = token_tile(prm.b, blockIdx.x, per_tile);
    if (tile.count == 0) return;
    const int pages = prm.b.pages_of(tile.group), per = pages_per_slice(pages, prm.splits);
    const int page0 = blockIdx.z * per, page1 = min(pages, page0 + per);
    if (page0 >= page1) return;
    const int kvh = blockIdx.y / prm.head_chunks, head0 = (blockIdx.y % prm.head_chunks) * prm.head_chunk;
    const int heads = min(prm.head_chunk, prm.group - head0);
    const int* table = prm.b.row_of(prm.b.start_of(tile.group));
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;

    for (int i = threadIdx.x; i < ROWS * pitch; i += THREADS) {
        const int r = i / pitch, c = i - r * pitch, tok = r / prm.head_chunk, h = r % prm.head_chunk;
        const bool live = tok < tile.count && h < heads && c < hd;
        q_s[i] = live ? to_f32(reinterpret_cast<const T*>(prm.q)[((size_t)(tile.first + tok) * prm.nh + kvh * prm.group + head0 + h) * hd + c]) : 0.0f;
    }
    int last[4];                                       // the last key each of this thread's rows sees
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i, tok = r / prm.head_chunk;
        const bool live = tok < tile.count && r % prm.head_chunk < heads && prm.b.row_of(tile.first + tok);
        last[i] = live ? prm.b.positions[tile.first + tok] : -1;
    }
    float m[4], l[4], acc[4][COLS][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][c][j] = 0.0f;
    }
    for (int p = page0; p < page1; ++p) {
        const int page = table ? table[p] : -1;
        if (!prm.b.is_page(page)) continue;            // (nothing is read where no page is)
        __syncthreads();
        load_tile<T>(k_s, prm.k, (size_t)page * prm.nkv + kvh, PAGE, hd, pitch);
        load_tile<T>(v_s, prm.v, (size_t)page * prm.nkv + kvh, PAGE, hd, COLS * 64);
        __syncthreads();
        float s[4][4] = {};
        for (int d = 0; d + 3 < hd; d += 4) {
            float4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(q_s + (ty * 4 + i) * pitch + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * pitch + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[i][j] = fmaf(a[i].x, b[j].x, fmaf(a[i].y, b[j].y, fmaf(a[i].z, b[j].z, fmaf(a[i].w, b[j].w, s[i][j]))));
        }
        for (int d = hd & ~3; d < hd; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = fmaf(q_s[(ty * 4 + i) * pitch + d], k_s[(tx + 16 * j) * pitch + d], s[i][j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = p * PAGE + tx + 16 * j <= last[i] ? score(prm, s[i][j]) : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float now = fmaxf(m[i], top), base = now == -INFINITY ? 0.0f : now;
            const float factor = expf(m[i] - base);    // 0 for the first keys
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = expf(s[i][j] - base);
                p_s[(ty * 4 + i) * (PAGE + 4) + tx + 16 * j] = e;
                sum += e;
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[i] = l[i] * factor + sum;
            m[i] = now;
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][c][j] *= factor;
        }
        __syncwarp();                                  // a row's sixteen threads are one half of a warp
        for (int key = 0; key < PAGE; ++key) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = p_s[(ty * 4 + i) * (PAGE + 4) + key];
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const float4 x = *reinterpret_cast<const float4*>(v_s + key * COLS * 64 + c * 64 + tx * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // a key no row may see weighs nothing, whatever its value holds
                    acc[i][c][0] = w[i] != 0.0f ? fmaf(w[i], x.x, acc[i][c][0]) : acc[i][c][0];
                    acc[i][c][1] = w[i] != 0.0f ? fmaf(w[i], x.y, acc[i][c][1]) : acc[i][c][1];
                    acc[i][c][2] = w[i] != 0.0f ? fmaf(w[i], x.z, acc[i][c][2]) : acc[i][c][2];
                    acc[i][c][3] = w[i] != 0.0f ? fmaf(w[i], x.w, acc[i][c][3]) : acc[i][c][3];
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i, tok = r / prm.head_chunk, h = r % prm.head_chunk;
        if (tok >= tile.count || h >= heads) continue;
        const size_t at = ((size_t)(tile.first + tok) * prm.nh + kvh * prm.group + head0 + h) * prm.splits + blockIdx.z;
        if (tx == 0) {
            prm.part_ml[2 * at] = m[i];
            prm.part_ml[2 * at + 1] = l[i];
        }
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c * 64 + tx * 4 + j < hd) prm.part_o[at * hd + c * 64 + tx * 4 + j] = acc[i][c][j];
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) own_kernel(const Params prm) {
    extern __shared__ float smem[];
    const int hd = prm.hd, pitch = ((hd + 3) & ~3) + 4;
    float* q_s = smem;                                 // [OWN_HEADS][pitch]
    float* k_s = q_s + OWN_HEADS * pitch;              // [PAGE][pitch]
    float* v_s = k_s + PAGE * pitch;                   // [PAGE][hd]
    float* p_s = v_s + PAGE * hd;                      // [OWN_HEADS][PAGE]
    float* m_s = p_s + OWN_HEADS * PAGE;               // [OWN_HEADS], and the two behind it
    float* l_s = m_s + OWN_HEADS;
    float* f_s = l_s + OWN_HEADS;
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunks = (prm.group + OWN_HEADS - 1) / OWN_HEADS;
    const int kvh = blockIdx.y / chunks, head0 = kvh * prm.group + (blockIdx.y % chunks) * OWN_HEADS;
    const int heads = min(OWN_HEADS, (kvh + 1) * prm.group - head0);
    const int group = group_of(prm.b, t);
    if (group < 0) return;                             // rows of no group stay as they are
    const int pages = prm.b.pages_of(group);
    const int* table = prm.b.row_of(t);
    const int last = table ? min(prm.b.positions[t], prm.b.max_pages * PAGE - 1) : -1;
    for (int i = threadIdx.x; i < OWN_HEADS * pitch; i += THREADS) {
        const int h = i / pitch, c = i - h * pitch;
        q_s[i] = h < heads && c < hd ? to_f32(reinterpret_cast<const T*>(prm.q)[((size_t)t * prm.nh + head0 + h) * hd + c]) : 0.0f;
    }
    if (threadIdx.x < OWN_HEADS) m_s[threadIdx.x] = -INFINITY, l_s[threadIdx.x] = 0.0f;
    float acc[OWN_HEADS] = {};                         // column threadIdx.x of every head (head sizes up to 256)
    const int c = threadIdx.x;
    for (int p = pages; p * PAGE <= last; ++p) {
        const int page = table[p], seen = min(PAGE, last + 1 - p * PAGE);
        if (!prm.b.is_page(page)) continue;
        __syncthreads();
        load_tile<T>(k_s, prm.k, (size_t)page * prm.nkv + kvh, seen, hd, pitch);
        load_tile<T>(v_s, prm.v, (size_t)page * prm.nkv + kvh, seen, hd, hd);
        __syncthreads();
        for (int i = threadIdx.x; i < OWN_HEADS * PAGE; i += THREADS) {
            const int h = i / PAGE, key = i % PAGE;
            float dot = 0.0f;
            for (int d = 0; d < hd; ++d) dot = fmaf(q_s[h * pitch + d], k_s[key * pitch + d], dot);
            p_s[i] = h < heads && key < seen ? score(prm, dot) : -INFINITY;
        }
        __syncthreads();
        for (int h = warp; h < heads; h += THREADS / 32) {
            const float a = p_s[h * PAGE + lane], b = p_s[h * PAGE + 32 + lane];
            const float now = fmaxf(m_s[h], warp_max(fmaxf(a, b))), base = now == -INFINITY ? 0.0f : now;
            const float ea = expf(a - base), eb = expf(b - base), sum = warp_sum(ea + eb);
            p_s[h * PAGE + lane] = ea, p_s[h * PAGE + 32 + lane] = eb;
            __syncwarp();
            if (lane == 0) {
                f_s[h] = expf(m_s[h] - base);
                l_s[h] = l_s[h] * f_s[h] + sum;
                m_s[h] = now;
            }
        }
        __syncthreads();
        if (c < hd) {
#pragma unroll
            for (int h = 0; h < OWN_HEADS; ++h) {
                if (h >= heads) break;
                float a = acc[h] * f_s[h];
                for (int key = 0; key < seen; ++key) a = fmaf(p_s[h * PAGE + key], v_s[key * hd + c], a);
                acc[h] = a;
            }
        }
    }
    __syncthreads();
    const int per = pages_per_slice(pages, prm.splits), slices = per ? (pages + per - 1) / per : 0;
#pragma unroll
    for (int h = 0; h < OWN_HEADS; ++h) {
        if (h >= heads || c >= hd) break;
        const size_t at = ((size_t)t * prm.nh + head0 + h) * prm.splits;
        float top = fmaxf(m_s[h], prm.sink ? prm.sink[head0 + h] : -INFINITY);
        for (int s = 0; s < slices; ++s) top = fmaxf(top, prm.part_ml[2 * (at + s)]);
        const float base = top == -INFINITY ? 0.0f : top;
        float factor = expf(m_s[h] - base), o = acc[h] * factor, l = l_s[h] * factor;
        if (prm.sink) l += expf(prm.sink[head0 + h] - base);
        for (int s = 0; s < slices; ++s) {
            factor = expf(prm.part_ml[2 * (at + s)] - base);
            o = fmaf(factor, prm.part_o[(at + s) * hd + c], o);
            l = fmaf(factor, prm.part_ml[2 * (at + s) + 1], l);
        }
        reinterpret_cast<T*>(prm.out)[((size_t)t * prm.nh + head0 + h) * hd + c] = from_f32<T>(l == 0.0f ? 0.0f : o / l);
    }
}

template <typename Kernel>
int configure(Kernel kernel, size_t smem) {
    return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
}

template <typename T, int COLS>
int launch_prefix(const Params& prm, cudaStream_t stream) {
    const int pitch = ((prm.hd + 3) & ~3) + 4;
    const size_t smem = (size_t)(ROWS * pitch + PAGE * pitch + PAGE * COLS * 64 + ROWS * (PAGE + 4)) * 4;
    const int e = configure(prefix_kernel<T, COLS>, smem);
    if (e) return e;
    const long tiles = most_token_tiles(prm.b.T, prm.b.n_groups, ROWS / prm.head_chunk);
    fwb::pdl(prefix_kernel<T, COLS>, dim3((unsigned)tiles, prm.nkv * prm.head_chunks, prm.splits), THREADS, smem, stream)(prm);
    return fwb_launch_status();
}

template <typename T>
int launch(const Params& prm, cudaStream_t stream) {
    int e = prm.hd <= 64 ? launch_prefix<T, 1>(prm, stream) : prm.hd <= 128 ? launch_prefix<T, 2>(prm, stream)
            : launch_prefix<T, 4>(prm, stream);
    if (e) return e;
    const int pitch = ((prm.hd + 3) & ~3) + 4, chunks = (prm.group + OWN_HEADS - 1) / OWN_HEADS;
    const size_t smem = (size_t)(OWN_HEADS * pitch + PAGE * pitch + PAGE * prm.hd + OWN_HEADS * PAGE + 3 * OWN_HEADS) * 4;
    e = configure(own_kernel<T>, smem);
    if (e) return e;
    fwb::pdl(own_kernel<T>, dim3(prm.b.T, prm.nkv * chunks), THREADS, smem, stream)(prm);
    return fwb_launch_status();
}

}  // namespace

// q, out: [T][nh * hd]; pools [num_pages][nkv][64][hd]; all bf16 or all fp32.  positions, tok_seg: [T]; block_table:
// [n_segments][max_pages]; group_start: [n_groups + 1], group_pages: [n_groups]; part_o: fp32 [T][nh][splits][hd], part_ml: fp32
// [T][nh][splits][2], scratch.  sink: [nh] or null; softcap 0: off.  own_slices (1, 2, 4, 8): how many CTAs share a token's own keys
// on the tensor cores.
FWB_API int fwb_attention_prefix(const void* q, const void* k_pool, const void* v_pool, int is_bf16, const int* positions,
                                 const int* tok_seg, const int* block_table, int n_segments, int max_pages, int num_pages,
                                 const int* group_start, const int* group_pages, int n_groups, float* part_o, float* part_ml,
                                 void* out, int T, int nh, int nkv, int hd, int splits, int own_slices, float scale,
                                 const float* sink, float softcap, cudaStream_t stream) {
    if (T <= 0 || n_groups <= 0) return FWB_OK;
    if (!q || !k_pool || !v_pool || !positions || !tok_seg || !block_table || !group_start || !group_pages || !part_o ||
        !part_ml || !out || n_segments <= 0 || max_pages <= 0 || num_pages <= 0 || splits < 1 || !(softcap >= 0.0f) ||
        (own_slices != 1 && own_slices != 2 && own_slices != 4 && own_slices != 8))
        return FWB_BAD_ARGUMENT;
    if (nkv <= 0 || nh <= 0 || nh % nkv || hd < 1 || hd > 256) return FWB_UNSUPPORTED;
    if (nkv > 4095 || max_pages > 33554431 || splits > 65535) return FWB_TOO_LARGE;
    if (softcap > 0.0f && scale == 0.0f) return FWB_UNSUPPORTED;
    Params prm{};
    prm.b = Batch{positions, tok_seg, block_table, group_start, group_pages, T, n_segments, n_groups, max_pages, num_pages};
    if (is_bf16 && tensor_cores_take(q, k_pool, v_pool, out, part_o, prm.b, nkv, hd))
        return launch_tensor_cores(prm.b, q, k_pool, v_pool, out, part_o, part_ml, sink, nh, nkv, hd, splits, own_slices, scale, softcap, stream);
    prm.q = q, prm.k = k_pool, prm.v = v_pool, prm.part_o = part_o, prm.part_ml = part_ml, prm.out = out, prm.sink = sink;
    prm.nh = nh, prm.nkv = nkv, prm.group = nh / nkv, prm.hd = hd, prm.splits = splits;
    prm.head_chunk = prm.group < ROWS ? prm.group : ROWS;
    prm.head_chunks = (prm.group + prm.head_chunk - 1) / prm.head_chunk;
    prm.scale = scale, prm.cap = softcap;
    return is_bf16 ? launch<__nv_bfloat16>(prm, stream) : launch<float>(prm, stream);
}
