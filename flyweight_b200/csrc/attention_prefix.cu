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
//
// Two groups of ten requests behind 1,024 keys, 10 heads over 5 of 80, capped scores, fp32: 25 us on B200, 8 MB (0.3 TB/s).  Neither memory
// nor the multiply-adds bound it.  64 rows a block, four by four scores a thread, a warp whose eight rows nobody has only fetches:
// ten tokens of two heads are 20 rows, so three of eight warps compute.  The own kernel is 100 blocks, which take their pages one
// after the other, copies, scores, softmax and values each behind a barrier with nothing of the next page on the way.
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
    int vector;                  // rows of four channels start on borders of four elements
    float scale, cap;
};

__device__ __forceinline__ float score(const Params& prm, float dot) {
    const float s = dot * prm.scale;
    return prm.cap > 0.0f ? prm.cap * tanhf(s / prm.cap) : s;
}

__device__ __forceinline__ float4 load4(const float* at) { return *reinterpret_cast<const float4*>(at); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* at) {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
// A page's tiles of one KV head, keys and values, into shared memory: rows `pitch` and `v_pitch` floats apart, channels from hd
// up to the next multiple of four and rows from `rows` on zero.
template <typename T>
__device__ __forceinline__ void load_tiles(const Params& prm, float* k_s, int pitch, float* v_s, int v_pitch, size_t tile, int rows) {
    const int hd = prm.hd, quads = (hd + 3) >> 2;
    const T *k = reinterpret_cast<const T*>(prm.k) + tile * PAGE * hd, *v = reinterpret_cast<const T*>(prm.v) + tile * PAGE * hd;
    const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (prm.vector) {
#pragma unroll 4
        for (int i = threadIdx.x; i < PAGE * quads; i += THREADS) {
            const int r = i / quads, c = (i - r * quads) * 4;
            const float4 a = r < rows ? load4(k + i * 4) : none, b = r < rows ? load4(v + i * 4) : none;
            *reinterpret_cast<float4*>(k_s + r * pitch + c) = a;
            *reinterpret_cast<float4*>(v_s + r * v_pitch + c) = b;
        }
    } else {
        for (int i = threadIdx.x; i < PAGE * quads * 4; i += THREADS) {
            const int r = i / (quads * 4), c = i - r * quads * 4;
            const bool live = r < rows && c < hd;
            k_s[r * pitch + c] = live ? to_f32(k[r * hd + c]) : 0.0f;
            v_s[r * v_pitch + c] = live ? to_f32(v[r * hd + c]) : 0.0f;
        }
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
    const int pages = tile.pages, per = pages_per_slice(pages, prm.splits);
    const int page0 = blockIdx.z * per, page1 = min(pages, page0 + per);
    if (page0 >= page1) return;
    const int kvh = blockIdx.y / prm.head_chunks, head0 = (blockIdx.y % prm.head_chunks) * prm.head_chunk;
    const int heads = min(prm.head_chunk, prm.group - head0);
    const int* table = shared_row(prm.b, tile);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, rows = tile.count * prm.head_chunk;
    const bool works = (threadIdx.x >> 5) * 8 < rows;  // a warp has eight rows; those without any only fetch

    for (int i = threadIdx.x; i < rows * pitch; i += THREADS) {
        const int r = i / pitch, c = i - r * pitch, tok = r / prm.head_chunk, h = r % prm.head_chunk;
        const bool live = h < heads && c < hd;
        q_s[i] = live ? to_f32(reinterpret_cast<const T*>(prm.q)[((size_t)(tile.first + tok) * prm.nh + kvh * prm.group + head0 + h) * hd + c]) : 0.0f;
    }
    int last[4], whole_to = 0x7fffffff;                // the last key each of this thread's rows sees; the least of them
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i, tok = r / prm.head_chunk;
        const bool is_row = tok < tile.count && r % prm.head_chunk < heads;
        last[i] = is_row && prm.b.row_of(tile.first + tok) ? prm.b.last_key(prm.b.positions[tile.first + tok]) : -1;
        if (is_row) whole_to = min(whole_to, last[i]);
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
        load_tiles<T>(prm, k_s, pitch, v_s, COLS * 64, (size_t)page * prm.nkv + kvh, PAGE);
        __syncthreads();
        if (!works) continue;
        float s[4][4] = {};
#pragma unroll 2
        for (int d = 0; d < hd; d += 4) {               // (channels behind the last are zero in both)
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
        // a key that a row does not see weighs nothing, whatever its value holds; where all four rows see all keys nobody asks
        const bool whole = __all_sync(0xffffffffu, p * PAGE + PAGE - 1 <= whole_to);
#pragma unroll 4
        for (int key = 0; key < PAGE; ++key) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = p_s[(ty * 4 + i) * (PAGE + 4) + key];
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const float4 x = *reinterpret_cast<const float4*>(v_s + key * COLS * 64 + c * 64 + tx * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!whole && w[i] == 0.0f) continue;
                    acc[i][c][0] = fmaf(w[i], x.x, acc[i][c][0]), acc[i][c][1] = fmaf(w[i], x.y, acc[i][c][1]);
                    acc[i][c][2] = fmaf(w[i], x.z, acc[i][c][2]), acc[i][c][3] = fmaf(w[i], x.w, acc[i][c][3]);
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

// (threads as (part of the keys, head, four channels) for O: items of head and channels, `parts` threads an item)
template <typename T>
__global__ void __launch_bounds__(THREADS) own_kernel(const Params prm) {
    extern __shared__ float smem[];
    const int hd = prm.hd, quads = (hd + 3) >> 2, pitch = quads * 4 + 4;
    float* q_s = smem;                                 // [OWN_HEADS][pitch]
    float* k_s = q_s + OWN_HEADS * pitch;              // [PAGE][pitch]
    float* v_s = k_s + PAGE * pitch;                   // [PAGE][quads * 4]
    float* p_s = v_s + PAGE * quads * 4;               // [OWN_HEADS][PAGE]
    float* m_s = p_s + OWN_HEADS * PAGE;               // [OWN_HEADS], and the two behind it
    float* l_s = m_s + OWN_HEADS;
    float* f_s = l_s + OWN_HEADS;
    __shared__ float shared_weight[OWN_HEADS][MAX_SPLITS], own_weight[OWN_HEADS], inverse[OWN_HEADS];
    // (the prefix kernel has waited for what lies in front of it before it let this one start: only its own results are missing)
    pdl_launch_dependents();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunks = (prm.group + OWN_HEADS - 1) / OWN_HEADS;
    const int kvh = blockIdx.y / chunks, head0 = kvh * prm.group + (blockIdx.y % chunks) * OWN_HEADS;
    const int heads = min(OWN_HEADS, (kvh + 1) * prm.group - head0);
    const Token token = token_of(prm.b, t);
    if (token.pages < 0) {                             // rows of no group stay as they are
        pdl_wait();
        return;
    }
    const int pages = token.pages, last = token.last;
    for (int i = threadIdx.x; i < heads * pitch; i += THREADS) {
        const int h = i / pitch, c = i - h * pitch;
        q_s[i] = c < hd ? to_f32(reinterpret_cast<const T*>(prm.q)[((size_t)t * prm.nh + head0 + h) * hd + c]) : 0.0f;
    }
    if (threadIdx.x < OWN_HEADS) m_s[threadIdx.x] = -INFINITY, l_s[threadIdx.x] = 0.0f;
    const int items = heads * quads, parts = items >= THREADS ? 1 : THREADS / items < PAGE ? THREADS / items : PAGE;
    constexpr int MOST = OWN_HEADS * 64 / THREADS;     // items a thread has at most (head sizes up to 256)
    float4 acc[MOST];
#pragma unroll
    for (int n = 0; n < MOST; ++n) acc[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int part = parts > 1 ? threadIdx.x / items : 0, item0 = parts > 1 ? threadIdx.x - part * items : threadIdx.x;
    const bool works = part < parts;
    for (int p = pages; p * PAGE <= last; ++p) {
        const int page = token.table[p], seen = min(PAGE, last + 1 - p * PAGE);
        if (!prm.b.is_page(page)) continue;
        __syncthreads();
        load_tiles<T>(prm, k_s, pitch, v_s, quads * 4, (size_t)page * prm.nkv + kvh, seen);
        __syncthreads();
        {
            const int key = threadIdx.x & 63;
            for (int h = threadIdx.x >> 6; h < heads; h += THREADS / 64) {
                float d0 = 0.0f, d1 = 0.0f;
#pragma unroll 4
                for (int d = 0; d < quads; ++d) {
                    const float4 a = *reinterpret_cast<const float4*>(q_s + h * pitch + 4 * d), b = *reinterpret_cast<const float4*>(k_s + key * pitch + 4 * d);
                    d0 = fmaf(a.x, b.x, fmaf(a.y, b.y, d0));
                    d1 = fmaf(a.z, b.z, fmaf(a.w, b.w, d1));
                }
                p_s[h * PAGE + key] = key < seen ? score(prm, d0 + d1) : -INFINITY;
            }
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
#pragma unroll
        for (int n = 0; n < MOST; ++n) {
            const int item = item0 + n * THREADS, h = item / quads, c = (item - h * quads) * 4;
            if (!works || item >= items) break;
            const float f = f_s[h];
            float4 a = acc[n];
            a.x *= f, a.y *= f, a.z *= f, a.w *= f;
            for (int key = part; key < seen; key += parts) {
                const float w = p_s[h * PAGE + key];
                const float4 x = *reinterpret_cast<const float4*>(v_s + key * quads * 4 + c);
                a.x = fmaf(w, x.x, a.x), a.y = fmaf(w, x.y, a.y), a.z = fmaf(w, x.z, a.z), a.w = fmaf(w, x.w, a.w);
            }
            acc[n] = a;
        }
    }
    pdl_wait();                                        // the shared part is there
    __syncthreads();
    // the parts' sums where K was; the weights of the slices, a warp a head and a lane a slice
    float4* sums = reinterpret_cast<float4*>(k_s);     // [parts][items]
#pragma unroll
    for (int n = 0; n < MOST; ++n)
        if (works && item0 + n * THREADS < items) sums[part * items + item0 + n * THREADS] = acc[n];
    const int per = pages_per_slice(pages, prm.splits), slices = per ? (pages + per - 1) / per : 0;
    for (int h = warp; h < heads; h += THREADS / 32) {
        const size_t at = ((size_t)t * prm.nh + head0 + h) * prm.splits;
        const float sink = prm.sink ? prm.sink[head0 + h] : -INFINITY;
        float2 of[(MAX_SPLITS + 31) / 32];
        float top = fmaxf(m_s[h], sink);
#pragma unroll
        for (int i = 0; i < (MAX_SPLITS + 31) / 32; ++i) {
            of[i] = lane + 32 * i < slices ? *reinterpret_cast<const float2*>(prm.part_ml + 2 * (at + lane + 32 * i)) : make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, of[i].x);
        }
        top = warp_max(top);
        const float base = top == -INFINITY ? 0.0f : top, mine = expf(m_s[h] - base);
        float sum = lane == 0 ? l_s[h] * mine + expf(sink - base) : 0.0f;
#pragma unroll
        for (int i = 0; i < (MAX_SPLITS + 31) / 32; ++i) {
            const float w = expf(of[i].x - base);
            if (lane + 32 * i < slices) shared_weight[h][lane + 32 * i] = w;
            sum = fmaf(w, of[i].y, sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) own_weight[h] = mine, inverse[h] = sum;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += THREADS) {
        const int h = i / quads, c = (i - h * quads) * 4;
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int n = 0; n < parts; ++n) {
            const float4 x = sums[n * items + i];
            o[0] += x.x, o[1] += x.y, o[2] += x.z, o[3] += x.w;
        }
        const float* from = prm.part_o + ((size_t)t * prm.nh + head0 + h) * prm.splits * hd + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (c + j >= hd) break;
            o[j] *= own_weight[h];
            // (a slice that weighs nothing may hold anything: it is not read)
#pragma unroll 4
            for (int s = 0; s < slices; ++s) {
                const float w = shared_weight[h][s];
                o[j] = fmaf(w, w != 0.0f ? from[(size_t)s * hd + j] : 0.0f, o[j]);
            }
            const float total = inverse[h];
            reinterpret_cast<T*>(prm.out)[((size_t)t * prm.nh + head0 + h) * hd + c + j] = from_f32<T>(total == 0.0f ? 0.0f : o[j] / total);
        }
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
    const size_t smem = (size_t)(OWN_HEADS * pitch + PAGE * pitch + PAGE * (pitch - 4) + OWN_HEADS * PAGE + 3 * OWN_HEADS) * 4;
    e = configure(own_kernel<T>, smem);
    if (e) return e;
    fwb::pdl(own_kernel<T>, dim3(prm.b.T, prm.nkv * chunks), THREADS, smem, stream)(prm);
    return fwb_launch_status();
}

}  // namespace

// q, out: [T][nh * hd]; pools [num_pages][nkv][64][hd]; all bf16 or all fp32.  positions, tok_seg: [T]; block_table:
// [n_segments][max_pages]; group_start: [n_groups + 1], group_pages: [n_groups]; part_o: fp32 [T][nh][splits][hd], part_ml: fp32
// [T][nh][splits][2], scratch.  sink: [nh] or null; softcap 0: off.  own_slices (1, 2, 4, 8): how many CTAs share a token's own keys
// on the tensor cores.  neighbours: there, neighbouring tokens of a request are taken together where two have at most sixteen query
// heads of a KV head.  splits 0 (on the tensor cores): without the prefix kernel and its scratch, every
// token walks the shared pages by itself.
FWB_API int fwb_attention_prefix(const void* q, const void* k_pool, const void* v_pool, int is_bf16, const int* positions,
                                 const int* tok_seg, const int* block_table, int n_segments, int max_pages, int num_pages,
                                 const int* group_start, const int* group_pages, int n_groups, float* part_o, float* part_ml,
                                 void* out, int T, int nh, int nkv, int hd, int splits, int own_slices, int neighbours, float scale,
                                 const float* sink, float softcap, cudaStream_t stream) {
    if (T <= 0 || n_groups <= 0) return FWB_OK;
    if (!q || !k_pool || !v_pool || !positions || !tok_seg || !block_table || !group_start || !group_pages || (splits && (!part_o || !part_ml)) ||
        !out || n_segments <= 0 || max_pages <= 0 || num_pages <= 0 || splits < 0 || !(scale > 0.0f && scale < INFINITY) ||
        !(softcap >= 0.0f && softcap < INFINITY) || !(softcap / scale < INFINITY) ||
        (own_slices != 1 && own_slices != 2 && own_slices != 4 && own_slices != 8))
        return FWB_BAD_ARGUMENT;
    if (nkv <= 0 || nh <= 0 || nh % nkv || hd < 1 || hd > 256) return FWB_UNSUPPORTED;
    if (nkv > 4095 || max_pages > 33554431 || splits > MAX_SPLITS) return FWB_TOO_LARGE;
    Params prm{};
    prm.b = Batch{positions, tok_seg, block_table, group_start, group_pages, T, n_segments, n_groups, max_pages, num_pages};
    if (is_bf16 && tensor_cores_take(q, k_pool, v_pool, out, part_o, prm.b, nkv, hd))
        return launch_tensor_cores(prm.b, q, k_pool, v_pool, out, part_o, part_ml, sink, nh, nkv, hd, splits, own_slices,
                                   neighbours && 2 * (nh / nkv) <= 16, scale, softcap, stream);
    if (splits == 0) return FWB_UNSUPPORTED;
    prm.q = q, prm.k = k_pool, prm.v = v_pool, prm.part_o = part_o, prm.part_ml = part_ml, prm.out = out, prm.sink = sink;
    prm.nh = nh, prm.nkv = nkv, prm.group = nh / nkv, prm.hd = hd, prm.splits = splits;
    prm.head_chunk = prm.group < ROWS ? prm.group : ROWS;
    prm.head_chunks = (prm.group + prm.head_chunk - 1) / prm.head_chunk;
    prm.vector = hd % 4 == 0 && (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0;
    prm.scale = scale, prm.cap = softcap;
    return is_bf16 ? launch<__nv_bfloat16>(prm, stream) : launch<float>(prm, stream);
}
