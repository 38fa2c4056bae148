// lowbit_common.cuh -- the 8-bit block form, the exact three-part bfloat16 form of a float
// and the small reductions shared by the low-bit kernels.
//
// 8-bit blocks. A row is cut into blocks of 32 features (the last one shorter); a block has
// one scale byte b, and a code c stands for c * 2^(b - 127). b is the smallest byte for
// which amax <= top * 2^(b - 127), top = 127 (int8) or 448 (e4m3), so no code is clipped.
// A scale that is a power of two costs up to one bit against amax / top in float, and buys
// that every value has at most 8 significant bits: it is a bfloat16, exactly, and the weight
// gradient can feed it to bfloat16 MMAs without a second rounding. A block that holds an
// infinity or a NaN has b = 255 and stands for NaN everywhere.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "mt_common.cuh"

namespace mt {
namespace lowbit {

enum : int { kInt8 = 0, kE4M3 = 1 };
constexpr int kBlock = 32;   // features per 8-bit block

// A 2-D float view: element (r, c) at p + r * rs + c * cs.
struct Mat {
    float* p;
    int64_t rs, cs;
};

// An 8-bit tensor: unit column stride, byte pitches.
struct Q8 {
    uint8_t* codes;
    uint8_t* scales;
    int64_t cp, sp;
    int fmt;
};

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Scale byte of a block whose largest magnitude has the bits `a`: with amax = (1 + m) 2^(E-127)
// and top = (1 + t) 2^s, amax <= top 2^(b-127) first holds at b = E - s + (m > t).
__device__ __forceinline__ uint32_t scale_byte(uint32_t a, int fmt) {
    if (a >= 0x7F800000u) return 255u;
    const int s = fmt == kInt8 ? 6 : 8;
    const uint32_t t = fmt == kInt8 ? 0x7E0000u : 0x600000u;
    const int b = (int)(a >> 23) - s + ((a & 0x7FFFFFu) > t ? 1 : 0);
    return b < 0 ? 0u : (uint32_t)b;
}
// 2^(127 - b) for b <= 254; 0 for the byte of a non-finite block (its codes are then 0).
__device__ __forceinline__ float inv_scale(uint32_t b) { return b == 255u ? 0.f : __uint_as_float((254u - b) << 23); }
// 2^(b - 127); NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t b) {
    return b == 0 ? __uint_as_float(0x00400000u) : b == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(b << 23);
}

// Code of one value: round to nearest even of v * 2^(127 - b). The product is exact unless it
// is far below half a step, and no code is clipped (see scale_byte). A NaN times the 0 of a
// non-finite block must not reach the conversion.
__device__ __forceinline__ uint32_t encode8(float v, float inv, int fmt) {
    if (inv == 0.f) return 0u;
    const float u = v * inv;
    if (fmt == kInt8) return (uint32_t)__float2int_rn(u) & 0xFFu;
    return (uint32_t)__nv_cvt_float_to_fp8(u, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float code_value(uint32_t c, int fmt) {
    if (fmt == kInt8) return (float)(int)(int8_t)c;
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
    return __half2float(__half(h));
}

// Sum over the lanes of a warp, the same value in every lane.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the WPR warps that share a row. One __syncthreads: `buf` alternates between two
// halves of `red`, so the next row's writes cannot meet this row's reads.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[WPR], int& buf) {
    v = warp_sum(v);
    if (WPR == 1) return v;
    float* r = red[buf];
    buf ^= 1;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) r[w] = v;
    __syncthreads();
    float s = lane < WPR ? r[lane] : 0.f;
    return warp_sum(s);
}

// VEC features of a row of unit stride that begins at `row`.
template <int VEC>
__device__ __forceinline__ void load_row(float (&v)[VEC], const float* row, int f) {
    if (VEC == 4) {
        const float4 x = *reinterpret_cast<const float4*>(row + f);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        v[0] = row[f];
    }
}
template <int VEC>
__device__ __forceinline__ void store_row(const float (&v)[VEC], float* row, int f) {
    if (VEC == 4) *reinterpret_cast<float4*>(row + f) = make_float4(v[0], v[1], v[2], v[3]);
    else row[f] = v[0];
}

// Quantises VEC values per lane, the first of feature f, into a row of codes and its scales;
// 32 / VEC lanes share a block. Lanes behind the row's end pass zeros and in = false. All 32
// lanes call it.
template <int VEC>
__device__ __forceinline__ void store_q8(const float (&v)[VEC], uint8_t* codes, uint8_t* scales, int fmt, int f, bool in) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) a = max(a, abs_bits(v[i]));
    if (VEC == 1) {
        a = __reduce_max_sync(0xffffffffu, a);
    } else {
#pragma unroll
        for (int o = 16 / VEC; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    }
    const uint32_t b = scale_byte(a, fmt);
    const float inv = inv_scale(b);
    if (!in) return;
    if (VEC == 4) {
        uint32_t w = 0;
        if (fmt == kInt8) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) w |= encode8(v[i], inv, kInt8) << (8 * i);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) w |= encode8(v[i], inv, kE4M3) << (8 * i);
        }
        *reinterpret_cast<uint32_t*>(codes + f) = w;
    } else {
        codes[f] = (uint8_t)(fmt == kInt8 ? encode8(v[0], inv, kInt8) : encode8(v[0], inv, kE4M3));
    }
    if ((f & (kBlock - 1)) == 0) scales[(uint32_t)f / kBlock] = (uint8_t)b;
}

}  // namespace lowbit
}  // namespace mt
