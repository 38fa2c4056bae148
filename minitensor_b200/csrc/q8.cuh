// q8.cuh -- a float tensor saved in 8-bit blocks and read back (lowbit_common.cuh has the
// form). Both directions are one pass over memory: at 8192 x 4096 to int8 31 us (169 MB,
// 5.4 TB/s), to bfloat16 20.5 us (101 MB, 4.9 TB/s).
#pragma once

#include "lowbit_common.cuh"

namespace mt {
namespace q8 {

using lowbit::Mat;
using lowbit::Q8;

constexpr int kWarps = 8;
constexpr int kRows = 4;   // rows in flight per warp
constexpr int kDequantWidth = 8 * 256;   // features per CTA of the scalar dequantisation

// A warp takes a chunk of 32 * VEC features of kRows rows at a time (VEC = 4: 16-byte loads).
template <int VEC>
__global__ void __launch_bounds__(32 * kWarps) quantize_kernel(Mat x, Q8 q, int64_t rows, int64_t K) {
    const int lane = threadIdx.x & 31;
    const int64_t first = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * 32 * VEC;
    if (first >= K) return;   // the whole warp
    const int f = (int)first + lane * VEC;
    const bool in = f < K;
    for (int64_t r0 = (int64_t)blockIdx.y * kRows; r0 < rows; r0 += (int64_t)gridDim.y * kRows) {
        float v[kRows][VEC];
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            if (in && r0 + j < rows) {
                if (VEC == 4) lowbit::load_row<VEC>(v[j], x.p + (r0 + j) * x.rs, f);
                else v[j][0] = x.p[(r0 + j) * x.rs + f * x.cs];
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[j][i] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < kRows; ++j)
            if (r0 + j < rows) lowbit::store_q8<VEC>(v[j], q.codes + (r0 + j) * q.cp, q.scales + (r0 + j) * q.sp, q.fmt, f, in);
    }
}

__device__ __forceinline__ void put(float* o, float v) { *o = v; }
__device__ __forceinline__ void put(__nv_bfloat16* o, float v) { *o = __float2bfloat16_rn(v); }

// N = 16: 16 codes (half a block) per thread, 16-byte accesses. N = 1: any pitch and length, 8 codes
// of a thread in flight, 256 apart.
template <typename T, int N>
__global__ void __launch_bounds__(256) dequantize_kernel(Q8 q, T* out, int64_t pitch, int64_t rows, int64_t K) {
    if (N == 16) {
        const int64_t f = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
        if (f >= K) return;
        for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
            const float s = lowbit::scale_value(q.scales[row * q.sp + f / lowbit::kBlock]);
            const uint4 w = *reinterpret_cast<const uint4*>(q.codes + row * q.cp + f);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
            alignas(16) T t[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) put(&t[i], lowbit::code_value((u[i / 4] >> (8 * (i % 4))) & 0xFFu, q.fmt) * s);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i)
                reinterpret_cast<uint4*>(out + row * pitch + f)[i] = reinterpret_cast<const uint4*>(t)[i];
        }
    } else {
        const int64_t f0 = (int64_t)blockIdx.x * kDequantWidth + threadIdx.x;
        const int left = (int)min(K - f0, (int64_t)kDequantWidth);   // columns from this thread's first on
        for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
            const uint8_t* cr = q.codes + row * q.cp + f0;
            const uint8_t* sr = q.scales + row * q.sp + f0 / lowbit::kBlock;
            T* o = out + row * pitch + f0;
            uint8_t c[8], b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool in = i * 256 < left;
                c[i] = in ? cr[i * 256] : 0;
                b[i] = in ? sr[i * 256 / lowbit::kBlock] : 0;
            }
            if (q.fmt == lowbit::kInt8) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i * 256 < left) put(o + i * 256, lowbit::code_value(c[i], lowbit::kInt8) * lowbit::scale_value(b[i]));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i * 256 < left) put(o + i * 256, lowbit::code_value(c[i], lowbit::kE4M3) * lowbit::scale_value(b[i]));
            }
        }
    }
}

}  // namespace q8
}  // namespace mt
