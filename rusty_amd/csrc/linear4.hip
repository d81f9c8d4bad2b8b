// Linears with 4-bit affine weights (RQ_Q_AFFINE_U4):
//   Y[m, n] = sum_k X[m, k] W[n, k],  W[n, k] = u[n, k] s[n, k/G] + b[n, k/G],
// u in 0..15, two codes a byte (the even k in the low nibble), an f32 scale and
// bias per G consecutive k of a row.
#include <algorithm>

#include "common.hpp"

namespace rq {
namespace {

constexpr int TH = 256;

__global__ __launch_bounds__(TH) void k_dequantize4(const uint8_t *__restrict__ codes, const float *__restrict__ scales,
                                                    const float *__restrict__ biases, float *__restrict__ out,
                                                    int64_t pairs, int64_t group) {
    for (int64_t i = (int64_t)blockIdx.x * TH + threadIdx.x; i < pairs; i += (int64_t)gridDim.x * TH) {
#pragma clang fp contract(off)
        const uint32_t c = codes[i];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int64_t g = (2 * i + e) / group;
            const float p = (float)(e ? c >> 4 : c & 15u) * scales[g];
            out[2 * i + e] = p + (biases ? biases[g] : 0.0f);
        }
    }
}

// Any shape, alignment and dtype: one block per output feature, its threads
// stride over the code bytes of the row, once per token.
__global__ __launch_bounds__(TH) void k_linear4_generic(const uint8_t *__restrict__ codes,
                                                        const float *__restrict__ scales,
                                                        const float *__restrict__ biases, int64_t group,
                                                        const void *__restrict__ X, int x_f16, void *__restrict__ Y,
                                                        int y_f16, int64_t M, int64_t N, int64_t K) {
    __shared__ float red[TH / 64];
    const int64_t n = blockIdx.x, gk = K / group;
    const int t = threadIdx.x;
    const uint8_t *row = codes + n * (K / 2);
    for (int64_t m = 0; m < M; ++m) {
        float acc = 0.0f;
        for (int64_t i = t; i < K / 2; i += TH) {
            const uint32_t c = row[i];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int64_t k = 2 * i + e, g = n * gk + k / group;
                const float x = x_f16 ? (float)static_cast<const _Float16 *>(X)[m * K + k]
                                      : static_cast<const float *>(X)[m * K + k];
                const float w = __builtin_fmaf((float)(e ? c >> 4 : c & 15u), scales[g], biases ? biases[g] : 0.0f);
                acc = __builtin_fmaf(w, x, acc);
            }
        }
        for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
        if (t % 64 == 0) red[t / 64] = acc;
        __syncthreads();
        if (t == 0) {
            float v = 0.0f;
            for (int i = 0; i < TH / 64; ++i) v += red[i];
            if (y_f16) static_cast<_Float16 *>(Y)[m * N + n] = (_Float16)v;
            else static_cast<float *>(Y)[m * N + n] = v;
        }
        __syncthreads();
    }
}

}  // namespace

int launch_dequantize4(const rq_qweight &w, float *out, hipStream_t s) {
    const int64_t pairs = w.n_out * w.k_in / 2;
    if (pairs == 0) return RQ_OK;
    const int64_t blocks = std::min<int64_t>(cdiv(pairs, TH), 65536);
    hipLaunchKernelGGL(k_dequantize4, dim3((unsigned)blocks), dim3(TH), 0, s, (const uint8_t *)w.codes, w.scales,
                       w.biases, out, pairs, (int64_t)w.group);
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

int launch_linear4(const rq_qweight &w, const void *x, rq_dtype xt, void *y, rq_dtype yt, int64_t m, hipStream_t s) {
    if (!grid_ok(w.n_out, TH)) return fail(RQ_ERR_SHAPE, "n_out too large for the generic kernel");
    hipLaunchKernelGGL(k_linear4_generic, dim3((unsigned)w.n_out), dim3(TH), 0, s, (const uint8_t *)w.codes, w.scales,
                       w.biases, (int64_t)w.group, x, xt == RQ_F16 ? 1 : 0, y, yt == RQ_F16 ? 1 : 0, m, w.n_out, w.k_in);
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

}  // namespace rq
