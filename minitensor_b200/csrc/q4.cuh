// q4.cuh -- Linear weights in 4 bits with group scales.
//
// Column n of a weight W [in, out] is row n of the codes: W[k][n] ~ (c - 8) * s[n][k / group],
// c = 0..15, s bfloat16 (group 32, 64 or 128). A row is padded with code 8 (value 0) to spans
// of 128 codes, 64 bytes each. The 32-bit word 4 t + b of a span holds the codes
// 32 b + 8 t + (0..7) of the span: code 2 i in bits 4 i .. 4 i + 3, code 2 i + 1 in bits
// 4 i + 16 .. 4 i + 19. So one 16-byte piece (fixed t) has 8 codes of each of the four
// 32-code blocks, and the two codes of a pair sit at the same place of the word's halves.
#pragma once

#include "lowbit_common.cuh"

namespace mt {
namespace q4 {

using lowbit::Mat;

constexpr int kSpan = 128;        // codes per 64-byte span
constexpr int kSpanWords = 16;

struct Weight {
    uint32_t* codes;              // row pitch cp words
    __nv_bfloat16* scales;        // row pitch sp elements
    int64_t cp, sp;
    int64_t K, N;                 // in, out
    int group;
};

// First code of word w of a row.
__host__ __device__ __forceinline__ int64_t word_k(int64_t w) {
    return w / kSpanWords * kSpan + (w % 4) * 32 + (w % kSpanWords) / 4 * 8;
}
// Bit position of code j (0..7) of a word.
__host__ __device__ __forceinline__ int code_shift(int j) { return 4 * (j >> 1) + 16 * (j & 1); }

// One thread per column n and span of 128 inputs: s = bf16(amax / 7), c = round(w / s) + 8. A group with
// an infinity or a NaN gets the scale NaN.
__global__ void __launch_bounds__(128) quantize_kernel(Mat w, Weight q, int64_t spans) {
    const int64_t n = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (n >= q.N) return;
    for (int64_t sp = blockIdx.y; sp < spans; sp += gridDim.y) {
        float inv_of[4];   // scale of each 32-code block of the span
        for (int g0 = 0; g0 < kSpan; g0 += q.group) {
            uint32_t a = 0;
            for (int j = 0; j < q.group; ++j) {
                const int64_t k = sp * kSpan + g0 + j;
                if (k < q.K) a = max(a, lowbit::abs_bits(w.p[k * w.rs + n * w.cs]));
            }
            const float amax = a >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(a);
            const __nv_bfloat16 s = __float2bfloat16_rn(__fdiv_rn(amax, 7.f));
            const int64_t g = (sp * kSpan + g0) / q.group;
            if (sp * kSpan + g0 < q.K) q.scales[n * q.sp + g] = s;
            for (int j = 0; j < q.group; j += 32) inv_of[(g0 + j) / 32] = __bfloat162float(s);
        }
        for (int i = 0; i < kSpanWords; ++i) {
            const int64_t k0 = word_k(sp * kSpanWords + i);
            const float s = inv_of[i % 4];
            uint32_t word = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                int c = 8;
                if (k0 + j < q.K && s > 0.f)
                    c = 8 + max(-8, min(7, __float2int_rn(__fdiv_rn(w.p[(k0 + j) * w.rs + n * w.cs], s))));
                word |= (uint32_t)c << code_shift(j);
            }
            q.codes[n * q.cp + sp * kSpanWords + i] = word;
        }
    }
}

__global__ void __launch_bounds__(128) dequantize_kernel(Weight q, Mat w) {
    const int64_t n = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (n >= q.N) return;
    for (int64_t k0 = (int64_t)blockIdx.y * 8; k0 < q.K; k0 += (int64_t)gridDim.y * 8) {
        const int64_t in = k0 % kSpan;
        const uint32_t word = q.codes[n * q.cp + k0 / kSpan * kSpanWords + in % 32 / 8 * 4 + in / 32];
        const float s = __bfloat162float(q.scales[n * q.sp + k0 / q.group]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k0 + j < q.K) w.p[(k0 + j) * w.rs + n * w.cs] = (float)((int)((word >> code_shift(j)) & 15u) - 8) * s;
    }
}

}  // namespace q4
}  // namespace mt
