// What the kernels of the 8-bit products have in common: the arguments and what becomes of a sum.
#pragma once

#include "tcgen05.cuh"

namespace fwb {
namespace int8 {

enum Epilogue : int { EPI_F32 = 0, EPI_BF16 = 1, EPI_ADD_F32 = 2, EPI_GATED_BF16 = 3 };

constexpr int MAX_K = 131071;            // 128 * 128 * K < 2^31

struct Product {
    const signed char* x;        // [M][x_stride], zero from column K on
    const signed char* w;        // [w_rows][w_stride], likewise
    const float* xs;             // [M]
    const float* ws;             // [w_rows]
    void* y;                     // [M][N]
    const float* addend;         // [M][N]
    int M, N, K, x_stride, w_stride, w_rows;
    int up_row_offset, act;      // with a gate: the up projection's first row, the gate's activation
    float limit;
    int* status;
};

// A sum behind its scales: rounded after every step in every kernel (no multiply-add takes two of them together), so that a
// result has the same bits whichever kernel makes it.
__device__ __forceinline__ float scaled(int sum, float xs, float ws) { return __fmul_rn(__fmul_rn((float)sum, xs), ws); }

// What becomes of one value (with a gate: of two).
template <int EPI>
__device__ __forceinline__ void store(const Product& p, size_t at, float v, float u, float add) {
    if (EPI == EPI_F32) reinterpret_cast<float*>(p.y)[at] = v;
    else if (EPI == EPI_BF16) reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
    else if (EPI == EPI_ADD_F32) reinterpret_cast<float*>(p.y)[at] = __fadd_rn(v, add);
    else {
        float y = tc5::gated_fast(p.act, p.limit, v, u);
        // a row or feature of the scale NaN: these two cut off by minima and maxima, which take the number beside a NaN
        if ((p.act == tc5::GATE_SWISH_CLAMPED || p.act == tc5::GATE_RELU) && (v != v || u != u)) y = __int_as_float(0x7fffffff);
        reinterpret_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(y);
    }
}

// The product of a few tokens (host function, linear_rows_int8.cu); at most MAX_FEW of them.
constexpr int MAX_FEW = 32;
int few_tokens(const Product& p, int epilogue, cudaStream_t stream);
// The same on rows that are no integers yet (raw: [M][K], rows on borders of 16 bytes), which every block brings to integers by
// itself: for at most MAX_RAW tokens and MAX_RAW_K columns, K a multiple of 8.
constexpr int MAX_RAW = 8, MAX_RAW_K = 4096;
int few_raw_tokens(const Product& p, const void* raw, bool is_bf16, int epilogue, cudaStream_t stream);

}  // namespace int8
}  // namespace fwb
