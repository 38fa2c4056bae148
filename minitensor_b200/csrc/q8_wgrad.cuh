// q8_wgrad.cuh -- Linear's weight gradient from an 8-bit checkpoint of its input.
//
//   dW[k][n] = sum over rows m of xhat[m][k] * dY[m][n],  xhat = code * 2^(b - 127)
//
// Simple form: 64 x 64 tiles of dW, 16 rows of the sum per step, float FMA.
#pragma once

#include "lowbit_common.cuh"

namespace mt {
namespace wgrad8 {

using lowbit::Mat;
using lowbit::Q8;

constexpr int T = 64, KT = 16;

__global__ void __launch_bounds__(256) simple_kernel(Q8 q, Mat dy, Mat dw, int64_t rows, int64_t K, int64_t N) {
    __shared__ float a[KT][T], b[KT][T];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t k0 = (int64_t)blockIdx.y * T, n0 = (int64_t)blockIdx.x * T;
    float acc[4][4] = {};
    for (int64_t m0 = 0; m0 < rows; m0 += KT) {
        for (int i = threadIdx.x; i < KT * T; i += 256) {
            const int64_t m = m0 + i / T, k = k0 + i % T, n = n0 + i % T;
            a[i / T][i % T] = m < rows && k < K ? lowbit::code_value(q.codes[m * q.cp + k], q.fmt) *
                                                      lowbit::scale_value(q.scales[m * q.sp + k / lowbit::kBlock])
                                                : 0.f;
            b[i / T][i % T] = m < rows && n < N ? dy.p[m * dy.rs + n * dy.cs] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[m][ty + 16 * i], b[m][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t k = k0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (k < K && n < N) dw.p[k * dw.rs + n * dw.cs] = acc[i][j];
        }
}

}  // namespace wgrad8
}  // namespace mt
