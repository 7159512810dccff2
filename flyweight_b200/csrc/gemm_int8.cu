// Matrix product of 8-bit integers with a scale for every token's row and every channel's weights:
//
//   Y[t][f] = (sum_k X[t][k] W[f][k]) * xs[t] * ws[f]
//
// The sum of at most 131,071 products of two 8-bit integers is exact in 32 bits, so neither the order of the additions nor
// a cut of K changes a result.  Behind the scales (fp32): a residual is added, or the value is rounded to bfloat16, or
// a gated feed-forward's gate and up value become one.
#include "tcgen05.cuh"

using namespace fwb;
using namespace fwb::tc5;

namespace {

enum Epilogue : int { EPI_F32 = 0, EPI_BF16 = 1, EPI_ADD_F32 = 2, EPI_GATED_BF16 = 3 };

struct Params {
    const signed char* x;        // [M][x_stride]
    const signed char* w;        // [rows][w_stride]
    const float* xs;             // [M]
    const float* ws;             // [rows]
    void* y;                     // [M][N]
    const float* addend;         // [M][N]
    int M, N, K, x_stride, w_stride;
    int up_row_offset, act;
    float limit;
};

// A block makes 64 tokens x 64 features: a thread 4 x 4 (twice with a gate), four k at a time by dot products of four bytes.
template <int EPI>
__global__ void __launch_bounds__(256) gemm_int8_simple_kernel(const Params prm) {
    constexpr int NACC = EPI == EPI_GATED_BF16 ? 2 : 1;
    __shared__ int xt[64][17], wt[NACC][64][17];
    pdl_entry();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int t0 = blockIdx.y * 64, f0 = blockIdx.x * 64;
    int acc[NACC][4][4] = {};
    for (int k0 = 0; k0 < prm.K; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = i >> 4, k = k0 + (i & 15) * 4;
            xt[r][i & 15] = t0 + r < prm.M && k < prm.x_stride ? *reinterpret_cast<const int*>(prm.x + (size_t)(t0 + r) * prm.x_stride + k) : 0;
            for (int a = 0; a < NACC; ++a)
                wt[a][r][i & 15] = f0 + r < prm.N && k < prm.w_stride
                    ? *reinterpret_cast<const int*>(prm.w + ((size_t)a * prm.up_row_offset + f0 + r) * prm.w_stride + k) : 0;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int a = 0; a < NACC; ++a) acc[a][i][j] = __dp4a(xt[ty * 4 + i][k], wt[a][tx + 16 * j][k], acc[a][i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int t = t0 + ty * 4 + i, f = f0 + tx + 16 * j;
            if (t >= prm.M || f >= prm.N) continue;
            const size_t at = (size_t)t * prm.N + f;
            const float v = (float)acc[0][i][j] * prm.xs[t] * prm.ws[f];
            if (EPI == EPI_F32) reinterpret_cast<float*>(prm.y)[at] = v;
            else if (EPI == EPI_BF16) reinterpret_cast<__nv_bfloat16*>(prm.y)[at] = __float2bfloat16_rn(v);
            else if (EPI == EPI_ADD_F32) reinterpret_cast<float*>(prm.y)[at] = v + prm.addend[at];
            else {
                const float u = (float)acc[NACC - 1][i][j] * prm.xs[t] * prm.ws[prm.up_row_offset + f];
                reinterpret_cast<__nv_bfloat16*>(prm.y)[at] = __float2bfloat16_rn(gated_fast(prm.act, prm.limit, v, u));
            }
        }
}

constexpr int MAX_K = 131071;            // 128 * 128 * K < 2^31

}  // namespace

// X: [M][x_stride] int8 with scales xs [M]; W: [w_rows][w_stride] int8 with scales ws [w_rows]; both zero from column K on.
// Y: [M][N] fp32 (epilogues 0; 2: + addend, which may be Y) or bf16 (1; 3: gated, N features, up rows at up_row_offset,
// the gate's activation in the bits above the code, its parameter in gate_limit).
FWB_API int fwb_gemm_int8(const void* X, const float* xs, const void* W, const float* ws, void* Y, const float* addend, int M,
                          int N, int K, int x_stride, int w_stride, int w_rows, int epilogue, int up_row_offset,
                          float gate_limit, cudaStream_t stream) {
    const int act = epilogue >> 8;
    epilogue &= 0xff;
    if (M <= 0 || N <= 0) return FWB_OK;
    if (!X || !xs || !W || !ws || !Y || K <= 0 || x_stride < K || w_stride < K) return FWB_BAD_ARGUMENT;
    if (K > MAX_K) return FWB_TOO_LARGE;
    if ((x_stride & 15) || (w_stride & 15) || (((uintptr_t)X | (uintptr_t)W) & 15)) return FWB_UNSUPPORTED;
    if (epilogue == EPI_ADD_F32 && !addend) return FWB_BAD_ARGUMENT;
    if (epilogue == EPI_GATED_BF16 ? (up_row_offset < N || w_rows < up_row_offset + N) : w_rows < N) return FWB_BAD_ARGUMENT;
    const Params prm{(const signed char*)X, (const signed char*)W, xs, ws, Y, addend, M, N, K, x_stride, w_stride,
                     up_row_offset, act, gate_limit};
    const dim3 grid((N + 63) / 64, (M + 63) / 64);
    if (grid.y > 65535u) return FWB_TOO_LARGE;
    switch (epilogue) {
        case EPI_F32: fwb::pdl(gemm_int8_simple_kernel<EPI_F32>, grid, 256, 0, stream)(prm); break;
        case EPI_BF16: fwb::pdl(gemm_int8_simple_kernel<EPI_BF16>, grid, 256, 0, stream)(prm); break;
        case EPI_ADD_F32: fwb::pdl(gemm_int8_simple_kernel<EPI_ADD_F32>, grid, 256, 0, stream)(prm); break;
        case EPI_GATED_BF16: fwb::pdl(gemm_int8_simple_kernel<EPI_GATED_BF16>, grid, 256, 0, stream)(prm); break;
        default: return FWB_UNSUPPORTED;
    }
    return fwb_launch_status();
}
