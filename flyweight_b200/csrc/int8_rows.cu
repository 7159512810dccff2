// Rows of integers with a scale each, the operands of the 8-bit products:
//
//   s_r = max_k |y_rk| / 127      q_rk = round(y_rk / s_r), ties to even
//
// with y the rows themselves or their RMS norm, y = (x r) w, r = 1 / sqrt(mean(x^2) + eps), behind a residual sum
// x += delta where there is one.  The quotient's rounding is the exact one: a product with 1 / s decides all but the values
// next to a half, and there the sign of x - (n +- 1/2) s, which one fused multiply-add gives without an error, decides.
// A row of zeros has the scale 0.  A row that holds an infinity or a NaN has the scale NaN (and integers 0): whatever is
// made of it is NaN.
//
// Rows of integers lie `stride` bytes apart, a multiple of 16 (what TMA asks of a row), and are zero behind column K.
#include "common.cuh"

using namespace fwb;

namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 8;                 // elements a thread takes at once

struct RowsInt8Params {
    const void* x;               // [.][K] bf16 or fp32
    const float* delta;          // [.][K] or null: added into x first (fp32 rows)
    const float* norm_w;         // [K] or null: no norm
    const int* rows;             // row indices or null
    signed char* q;              // [R][stride]
    float* scales;               // [R]
    int R, K, stride;
    float eps;
    int vector;                  // rows start on 16-byte borders and K is a multiple of 8
};

template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int k, int K, int vector, float (&v)[CHUNK]) {
    if (vector) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(row + k), b = *reinterpret_cast<const float4*>(row + k + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(row + k);
            const uint32_t p[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(p[i] << 16);
                v[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.0f;
    }
}

__device__ __forceinline__ int quantize(float x, float s, float inv) {
    const float t = x * inv;
    float n = rintf(t);
    if (fabsf(fabsf(t - n) - 0.5f) < 1e-4f) {          // next to a half: 127 * 2^-23 is far less than this
        const float up = fmaf(-(n + 0.5f), s, x), down = fmaf(-(n - 0.5f), s, x);
        const bool odd = ((int)n) & 1;
        if (up > 0.0f || (up == 0.0f && odd)) n += 1.0f;
        else if (down < 0.0f || (down == 0.0f && odd)) n -= 1.0f;
    }
    return (int)fminf(fmaxf(n, -127.0f), 127.0f);      // (a NaN comes out as a number)
}

__device__ __forceinline__ float block_max(float v, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_max(v);
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    v = scratch[lane < (int)(blockDim.x >> 5) ? lane : 0];
    return warp_max(v);
}

// A block a row; every pass reads the row again (it lies in L1 or L2 by then).
template <typename T, bool NORM>
__global__ void __launch_bounds__(THREADS) rows_int8_kernel(const RowsInt8Params prm) {
    __shared__ float scratch[33];
    pdl_entry();
    const int r = blockIdx.x, K = prm.K;
    const size_t source = prm.rows ? (size_t)prm.rows[r] : (size_t)r;
    const T* row = reinterpret_cast<const T*>(prm.x) + source * K;
    float inv_rms = 1.0f;
    if constexpr (NORM) {
        float square = 0.0f;
        for (int k = threadIdx.x * CHUNK; k < K; k += THREADS * CHUNK) {
            float v[CHUNK];
            load_chunk(row, k, K, prm.vector, v);
            if (prm.delta) {
                float d[CHUNK];
                load_chunk(prm.delta + source * K, k, K, prm.vector, d);
                float* at = const_cast<float*>(reinterpret_cast<const float*>(row));
#pragma unroll
                for (int i = 0; i < CHUNK; ++i) {
                    v[i] += d[i];
                    if (k + i < K) at[k + i] = v[i];
                }
            }
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) square = fmaf(v[i], v[i], square);
        }
        inv_rms = 1.0f / sqrtf(block_sum(square, scratch) / (float)K + prm.eps);
    }
    auto value = [&](int k, float (&v)[CHUNK]) {
        load_chunk(row, k, K, prm.vector, v);
        if constexpr (NORM) {
            float w[CHUNK];
            load_chunk(prm.norm_w, k, K, prm.vector, w);
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) v[i] = (v[i] * inv_rms) * w[i];
        }
    };
    float most = 0.0f, bad = 0.0f;
    for (int k = threadIdx.x * CHUNK; k < K; k += THREADS * CHUNK) {
        float v[CHUNK];
        value(k, v);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            most = fmaxf(most, fabsf(v[i]));
            bad += v[i] * 0.0f;                        // NaN where v is none or no finite number
        }
    }
    most = block_max(bad != bad ? INFINITY : most, scratch);
    const float s = most / 127.0f, inv = most < 1e-30f || most > 3e38f ? 0.0f : 1.0f / s;
    if (threadIdx.x == 0) prm.scales[r] = most > 3.402823466e38f ? __int_as_float(0x7fffffff) : (most < 1e-30f ? 0.0f : s);
    for (int k = threadIdx.x * CHUNK; k < prm.stride; k += THREADS * CHUNK) {
        float v[CHUNK] = {};
        if (k < K) value(k, v);
        uint32_t word[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < CHUNK; ++i)
            if (k + i < K) word[i >> 2] |= (uint32_t)(quantize(v[i], s, inv) & 0xff) << (8 * (i & 3));
        *reinterpret_cast<uint2*>(prm.q + (size_t)r * prm.stride + k) = make_uint2(word[0], word[1]);
    }
}

}  // namespace

// x: [.][K] (row r, or rows[r]) in bf16 (x_bf16) or fp32; q: [R][stride] int8, stride >= K a multiple of 16; scales: [R].
// norm_w: [K] or null; with it x is fp32, and delta [.][K] (or null) is added into x in place first.
FWB_API int fwb_rows_int8(const void* x, int x_bf16, const float* delta, const float* norm_w, const int* rows, void* q,
                          float* scales, int R, int K, int stride, float eps, cudaStream_t stream) {
    if (R <= 0) return FWB_OK;
    if (!x || !q || !scales || K <= 0 || stride < K || (stride & 15) || ((uintptr_t)q & 15)) return FWB_BAD_ARGUMENT;
    if ((delta && !norm_w) || (norm_w && x_bf16) || (delta && rows)) return FWB_UNSUPPORTED;
    RowsInt8Params prm{x, delta, norm_w, rows, (signed char*)q, scales, R, K, stride, eps, 0};
    const uintptr_t bits = (uintptr_t)x | (uintptr_t)delta | (uintptr_t)norm_w;
    prm.vector = (K & 7) == 0 && (bits & 15) == 0;
    if (norm_w) fwb::pdl(rows_int8_kernel<float, true>, R, THREADS, 0, stream)(prm);
    else if (x_bf16) fwb::pdl(rows_int8_kernel<__nv_bfloat16, false>, R, THREADS, 0, stream)(prm);
    else fwb::pdl(rows_int8_kernel<float, false>, R, THREADS, 0, stream)(prm);
    return fwb_launch_status();
}
