// Rows of integers with a scale each, the operands of the 8-bit products:
//
//   s_r = max_k |y_rk| / 127      q_rk = round(y_rk / s_r), ties to even
//
// with y the rows themselves or their RMS norm, y = (x r) w, r = 1 / sqrt(mean(x^2) + eps), behind a residual sum
// x += delta where there is one (int8_quantize.cuh: the rounding, rows of zeros, infinities).
//
// Rows of integers lie `stride` bytes apart, a multiple of 16 (what TMA asks of a row), and are zero behind column K.
//
// Bound by memory.  A row is read once and held in registers between its passes (rows of more than 16,384 are read again).
// Many rows: a warp has up to 2,048 columns of one, so that as much as possible is on the way at once and nobody waits at
// a barrier; few: a block has a row, a thread eight columns, for the shortest way through.  Rounding by adding 1.5 * 2^23, whose
// low byte is the integer: the conversion instructions have a quarter of the adders' rate.
//
// Measured on B200: 4,096 rows of 8,192 in bf16 19.0 us (100 MB: 5.3 TB/s, of 6.57 that a copy reaches; issue slots half busy),
// 8,192 of 2,048 in fp32 15.8 (5.3 TB/s), with the norm and eight pieces a thread 21.5 (3.9 TB/s: the registers of a warp that holds
// a whole row leave 28 % of the warps).
#include "int8_quantize.cuh"

using namespace fwb;
using namespace fwb::int8;

namespace {

constexpr int WARP_ROWS = 4;             // warps of a block whose warps have a row each

struct RowsInt8Params {
    const void* x;               // [.][K] bf16 or fp32
    const float* delta;          // [.][K] or null: added into x first (fp32 rows)
    const float* norm_w;         // [K] or null: no norm
    const int* rows;             // row indices or null
    signed char* q;              // [R][stride]
    float* scales;               // [R]
    int R, K, stride, x_rows;    // x_rows: rows that x has, for the indices
    float eps;
    int vector;                  // rows start on 16-byte borders and K is a multiple of 8
};

// Eight elements of a row as they lie in memory, zeros behind its end.
template <typename T> struct Raw;
template <> struct Raw<float> { float4 a, b; };
template <> struct Raw<__nv_bfloat16> { uint4 a; };
__device__ __forceinline__ void load(Raw<float>& to, const float* row, int k, int K, int vector) {
    if (vector) {
        to.a = *reinterpret_cast<const float4*>(row + k), to.b = *reinterpret_cast<const float4*>(row + k + 4);
    } else {
        float v[CHUNK];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) v[i] = k + i < K ? row[k + i] : 0.0f;
        to.a = make_float4(v[0], v[1], v[2], v[3]), to.b = make_float4(v[4], v[5], v[6], v[7]);
    }
}
__device__ __forceinline__ void load(Raw<__nv_bfloat16>& to, const __nv_bfloat16* row, int k, int K, int vector) {
    if (vector) to.a = *reinterpret_cast<const uint4*>(row + k);
    else {
        uint32_t v[CHUNK];
        const unsigned short* at = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) v[i] = k + i < K ? at[k + i] : 0;
        to.a = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
}
__device__ __forceinline__ void values(const Raw<float>& r, float (&v)[CHUNK]) {
    v[0] = r.a.x, v[1] = r.a.y, v[2] = r.a.z, v[3] = r.a.w, v[4] = r.b.x, v[5] = r.b.y, v[6] = r.b.z, v[7] = r.b.w;
}
__device__ __forceinline__ void values(const Raw<__nv_bfloat16>& r, float (&v)[CHUNK]) {
    const uint32_t p[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(p[i] << 16);
        v[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u);
    }
}

// What the threads of a row hold, put together; every one of them gets the result.
template <bool WARP>
__device__ __forceinline__ unsigned row_max(unsigned v, unsigned* scratch) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, scratch[lane < warps ? lane : 0]);
}
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    v = warp_sum(v);
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    return warp_sum(lane < warps ? scratch[lane] : 0.0f);
}

enum Form : int { PLAIN = 0, NORM = 1, NORM_DELTA = 2 };

__device__ __forceinline__ void keep(Raw<float>& r, const float (&v)[CHUNK]) {
    r.a = make_float4(v[0], v[1], v[2], v[3]), r.b = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void keep(Raw<__nv_bfloat16>&, const float (&)[CHUNK]) {}

// WARP: a warp has a row (else the block).  CHUNKS: eight-element pieces a thread holds; 0: rows of any length, read again in
// every pass.
template <typename T, int FORM, bool WARP, int CHUNKS>
__global__ void __launch_bounds__(WARP ? 32 * WARP_ROWS : CHUNKS == 8 ? 256 : 1024) rows_int8_kernel(const RowsInt8Params prm) {
    constexpr int HELD = CHUNKS ? CHUNKS : 1;
    __shared__ float sums[32];
    __shared__ unsigned tops[32];
    const int K = prm.K, step = (WARP ? 32 : blockDim.x) * CHUNK, k0 = (WARP ? threadIdx.x & 31 : threadIdx.x) * CHUNK;
    pdl_entry();
    const int r = WARP ? blockIdx.x * WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && r >= prm.R) return;
    const int from = FORM == NORM && prm.rows ? prm.rows[r] : r;
    if (FORM == NORM && (from < 0 || from >= prm.x_rows)) {            // no such row: zeros
        for (int k = k0; k < prm.stride; k += step) *reinterpret_cast<uint2*>(prm.q + (size_t)r * prm.stride + k) = make_uint2(0, 0);
        if (k0 == 0) prm.scales[r] = 0.0f;
        return;
    }
    const T* row = reinterpret_cast<const T*>(prm.x) + (size_t)from * K;
    Raw<T> raw[HELD];
    if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int c = 0; c < HELD; ++c)
            if (k0 + c * step < K) load(raw[c], row, k0 + c * step, K, prm.vector);
    }
    // visit(k, values): every chunk of this thread's; what it leaves in the values stays (fp32 rows that are held)
    auto each = [&](auto&& visit) {
        float v[CHUNK];
        if constexpr (CHUNKS > 0) {
#pragma unroll
            for (int c = 0; c < HELD; ++c)
                if (k0 + c * step < K) {
                    values(raw[c], v);
                    visit(k0 + c * step, v);
                    if (FORM != PLAIN) keep(raw[c], v);
                }
        } else {
            for (int k = k0; k < K; k += step) {
                load(raw[0], row, k, K, prm.vector);
                values(raw[0], v);
                visit(k, v);
            }
        }
    };
    float inv_rms = 1.0f;
    if constexpr (FORM != PLAIN) {
        float square = 0.0f;
        each([&](int k, float (&v)[CHUNK]) {
            if constexpr (FORM == NORM_DELTA) {
                Raw<float> more;
                float d[CHUNK];
                load(more, prm.delta + (size_t)r * K, k, K, prm.vector);
                values(more, d);
                float* at = const_cast<float*>(reinterpret_cast<const float*>(row)) + k;       // the residual sum, in place
#pragma unroll
                for (int i = 0; i < CHUNK; ++i) v[i] += d[i];
                if (prm.vector) {
                    *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(at + 4) = make_float4(v[4], v[5], v[6], v[7]);
                } else {
#pragma unroll
                    for (int i = 0; i < CHUNK; ++i)
                        if (k + i < K) at[i] = v[i];
                }
            }
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) square = fmaf(v[i], v[i], square);
        });
        inv_rms = 1.0f / sqrtf(row_sum<WARP>(square, sums) / (float)K + prm.eps);
    }
    auto finish_norm = [&](int k, float (&v)[CHUNK]) {
        Raw<float> more;
        float gain[CHUNK];
        load(more, prm.norm_w, k, K, prm.vector);
        values(more, gain);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) v[i] = (v[i] * inv_rms) * gain[i];
    };
    // magnitudes as bits: in their order infinity lies above every number and NaN above infinity
    unsigned top = 0;
    each([&](int k, float (&v)[CHUNK]) {
        if (FORM != PLAIN) finish_norm(k, v);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i)
            if (FORM == PLAIN || prm.vector || k + i < K) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    });
    top = row_max<WARP>(top, tops);
    const RowScale scale = row_scale(top, sizeof(T) == 2);
    if (k0 == 0) prm.scales[r] = scale.stored;
    signed char* out = prm.q + (size_t)r * prm.stride;
    each([&](int k, float (&v)[CHUNK]) {
        if (FORM != PLAIN && CHUNKS == 0) finish_norm(k, v);
        uint2 packed = quantize(v, scale);
        if (FORM != PLAIN && !prm.vector && k + CHUNK > K) {           // what a norm made of columns that are none
            const unsigned long long mask = ~0ull >> (8 * (k + CHUNK - K));
            packed.x &= (uint32_t)mask, packed.y &= (uint32_t)(mask >> 32);
        }
        *reinterpret_cast<uint2*>(out + k) = packed;
    });
    // from the last chunk to the stride: at most one piece of eight
    if (k0 == 0 && ((K + 7) & ~7) < prm.stride) *reinterpret_cast<uint2*>(out + ((K + 7) & ~7)) = make_uint2(0, 0);
}

template <typename T, int FORM, bool WARP, int CHUNKS>
void launch(const RowsInt8Params& prm, int threads, cudaStream_t stream) {
    fwb::pdl(rows_int8_kernel<T, FORM, WARP, CHUNKS>, WARP ? (prm.R + WARP_ROWS - 1) / WARP_ROWS : prm.R, threads, 0, stream)(prm);
}

// Measured on B200 (us, by blocks and by warps; 1,000 2,368 4,000 6,000 8,192 rows): 1,024 columns of bf16 2.2 2.7, 3.4 3.0, 4.5 4.4, 6.6 4.9,
// 9.1 5.7, of fp32 2.6 3.1, 3.7 4.5, 5.0 5.3, 6.8 6.1, 9.2 7.2; 2,048 of bf16 2.7 4.5, 4.7 4.8, 6.8 6.9, 9.5 8.6, 12.2 10.4, of fp32 3.3 4.6,
// 5.4 6.5, 7.9 9.9, 11.2 12.8, 15.2 15.8, behind a norm 4.8 6.8, 8.5 8.6, 12.5 13.8, 17.9 17.6, 23.4 22.3.  The two change places between
// 2,368 rows (where a warp a row fills the SMs) and 6,000; in between this border costs up to 2 us.
constexpr int MANY_ROWS = 148 * 16;
template <typename T, int FORM>
void launch(const RowsInt8Params& prm, cudaStream_t stream) {
    const int pieces = (prm.K + CHUNK - 1) / CHUNK;
    const bool many = prm.R >= MANY_ROWS;
    if (pieces <= 32) launch<T, FORM, true, 1>(prm, 32 * WARP_ROWS, stream);
    else if (many && pieces <= 128) launch<T, FORM, true, 4>(prm, 32 * WARP_ROWS, stream);
    else if (many && pieces <= 256) launch<T, FORM, true, 8>(prm, 32 * WARP_ROWS, stream);
    else if (many && pieces <= 2048) launch<T, FORM, false, 8>(prm, pieces <= 512 ? 64 : pieces <= 1024 ? 128 : 256, stream);
    else if (pieces <= 1024) launch<T, FORM, false, 1>(prm, (pieces + 31) / 32 * 32, stream);
    else if (pieces <= 2048) launch<T, FORM, false, 2>(prm, 1024, stream);
    else launch<T, FORM, false, 0>(prm, 1024, stream);
}

}  // namespace

// x: [.][K] (row r, or rows[r]) in bf16 (x_bf16) or fp32; q: [R][stride] int8, stride >= K a multiple of 16; scales: [R].
// norm_w: [K] or null; with it x is fp32, has x_rows rows (an index beyond them gives zeros), and delta [.][K] (or null) is added into
// x in place first.
FWB_API int fwb_rows_int8(const void* x, int x_bf16, const float* delta, const float* norm_w, const int* rows, void* q,
                          float* scales, int R, int K, int stride, int x_rows, float eps, cudaStream_t stream) {
    if (R <= 0) return FWB_OK;
    if (!x || !q || !scales || K <= 0 || stride < K || (stride & 15) || ((uintptr_t)q & 15)) return FWB_BAD_ARGUMENT;
    if ((delta && !norm_w) || (norm_w && x_bf16) || (rows && (delta || !norm_w))) return FWB_UNSUPPORTED;
    if (!rows && R > x_rows) return FWB_BAD_ARGUMENT;
    RowsInt8Params prm{x, delta, norm_w, rows, (signed char*)q, scales, R, K, stride, x_rows, eps, 0};
    const uintptr_t bits = (uintptr_t)x | (uintptr_t)delta | (uintptr_t)norm_w;
    prm.vector = (K & 7) == 0 && (bits & 15) == 0;
    if (delta) launch<float, NORM_DELTA>(prm, stream);
    else if (norm_w) launch<float, NORM>(prm, stream);
    else if (x_bf16) launch<__nv_bfloat16, PLAIN>(prm, stream);
    else launch<float, PLAIN>(prm, stream);
    return fwb_launch_status();
}
