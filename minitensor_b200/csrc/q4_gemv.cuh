// q4_gemv.cuh -- y = x W + b with 4-bit weights for few rows of x, in integer arithmetic.
//
// One row of x is bound by reading W once; 6.5 TB/s are 13 T weights a second, 45 a cycle of an
// SM, so a weight can cost only a fraction of an instruction. Unpacking to half precision and
// mma.sync on it took 450 and later 110 instructions for the 128 x 16 weights of a warp's
// step; integers take 60.
//
// Mathematics. Per span of 128 features x becomes a fixed-point number of 30 bits and a sign,
// X = rn(x * 2^(29 - e)) with 2^e <= max |x| < 2^(e + 1), off by 2^-30 of the span's largest at
// most, and X four signed digits of 8 bits, X = sum d_j 256^j. The codes 0..15 of a word are
// unsigned bytes after a mask (three instructions for 8 weights), so the tensor core's u8 x s8
// product (mma.sync m16n8k32, 1,950 multiply-adds a cycle measured) gives sum c d_j exactly.
// Its accumulator begins at -8 sum d_j, which takes the codes' offset off exactly, too:
//   y = sum over groups of scale * 2^(e - 29) * sum_j 256^j * sum (c - 8) d_j,
// float only from the group's scale on. The four digits of a row are four columns of the
// product, a tile of 8 columns holds two rows of x.
//
// A span that holds an infinity or a NaN has no fixed point; a CTA that meets one computes its
// tiles by float FMA.
//
// Work. A CTA of 16 warps keeps its rows of x in shared memory and walks over tiles of 16 weight
// rows; kp warps share a tile, each taking a part of its spans. Four spans of codes and
// scales are in flight per warp, across tiles. The warps' sums meet in shared memory and are
// added in order. blockIdx.y takes up to 16 rows of x each.
#pragma once

#include "q4.cuh"

namespace mt {
namespace q4 {

constexpr int kGemvWarps = 16;
constexpr int kGemvThreads = 32 * kGemvWarps;
constexpr int kGemvDepth = 4;          // spans in flight per warp
constexpr int kGemvMaxTiles = 8;       // 8-column tiles: 16 rows of x

struct Gemv {
    Mat x;
    Weight w;
    const float* bias;
    Mat y;
    int64_t M;
    int rows;                          // of x per blockIdx.y, at most 2 NT
    int relu;
    int span0, spans;                  // this launch's part of K, in spans
    int accumulate, finish;            // y holds the sum over earlier spans; bias and ReLU are due
    int kp;                            // warps per tile: 1, 2, 4, 8 or 16
    int tiles;                         // of 16 weight rows
    int xvec;                          // rows of x on 16-byte boundaries, unit stride
};

// Shared memory: digits [8 NT columns][spans * 128 + 16] (the 16 put neighbouring columns on other
// banks), accumulator starts [2 NT rows][2][spans * segments] of two ints, powers of two
// [2 NT rows][2][spans], sums [warps][16][2 NT].
__host__ __device__ constexpr size_t gemv_smem(int nt, int group, int spans) {
    return (size_t)8 * nt * (spans * kSpan + 16) + (size_t)4 * nt * spans * (kSpan / group) * 8 +
           (size_t)4 * nt * spans * 4 + (size_t)kGemvWarps * 16 * 2 * nt * 4;
}

__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Puts this CTA's rows and spans of x into shared memory; returns whether all of it is finite.
// A warp takes a span, a lane 4 of its features. A word's bytes are masked out as codes
// 0 4 1 5 and 2 6 3 7 of its 8, the digits go in that order.
template <int NT, int G>
__device__ __forceinline__ bool gemv_stage_x(const Gemv& p, uint8_t* xs, int2* zi, float* fs) {
    constexpr int SEG = kSpan / G;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col_bytes = p.spans * kSpan + 16;
    const int64_t m0 = (int64_t)blockIdx.y * p.rows;
    int bad = 0;
    for (int i = warp; i < 2 * NT * p.spans; i += kGemvWarps) {
        const int r = i / p.spans, s = i - r * p.spans;
        const int64_t m = m0 + r, k = (int64_t)(p.span0 + s) * kSpan + lane * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < p.rows && m < p.M) {
            if (p.xvec && k + 4 <= p.w.K) {
                const float4 q = *reinterpret_cast<const float4*>(p.x.p + m * p.x.rs + k);
                v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k + j < p.w.K) v[j] = p.x.p[m * p.x.rs + (k + j) * p.x.cs];
            }
        }
        uint32_t a = max(max(lowbit::abs_bits(v[0]), lowbit::abs_bits(v[1])),
                         max(lowbit::abs_bits(v[2]), lowbit::abs_bits(v[3])));
        a = __reduce_max_sync(0xffffffffu, a);
        bad |= a >= 0x7F800000u;
        const int e = max((int)(a >> 23), 30);   // biased exponent
        const float up = __uint_as_float((uint32_t)(283 - e) << 23);
        uint32_t d[4] = {0, 0, 0, 0};            // digit j of the lane's four values
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            int X = __float2int_rn(v[c] * up);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int dj = (int)(int8_t)X;
                d[j] |= (uint32_t)(dj & 0xFF) << (8 * c);
                X = (X - dj) >> 8;
            }
        }
        uint8_t* o = xs + (size_t)(4 * r) * col_bytes + s * kSpan + (lane % 8) / 2 * 32 + lane / 8 * 8 + (lane & 1) * 4;
        int sum[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // Even lanes hold codes 0..3, odd lanes 4..7 of an octet.
            const uint32_t other = __shfl_xor_sync(0xffffffffu, d[j], 1);
            const uint32_t word = lane & 1 ? __byte_perm(other, d[j], 0x7362) : __byte_perm(d[j], other, 0x5140);
            *reinterpret_cast<uint32_t*>(o + (size_t)j * col_bytes) = word;
            sum[j] = __dp4a((int)d[j], 0x01010101, 0);
#pragma unroll
            for (int w = 1; w < G / 4; w <<= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], w);
        }
        if (lane % (G / 4) == 0) {
            const int at = s * SEG + lane / (G / 4);
            zi[(2 * r) * p.spans * SEG + at] = make_int2(-8 * sum[0], -8 * sum[1]);
            zi[(2 * r + 1) * p.spans * SEG + at] = make_int2(-8 * sum[2], -8 * sum[3]);
        }
        if (lane == 0) {
            const float f = __uint_as_float((uint32_t)(e - 29) << 23);
            fs[(2 * r) * p.spans + s] = f;
            fs[(2 * r + 1) * p.spans + s] = f * 65536.f;
        }
    }
    return __syncthreads_or(bad) == 0;
}

// The sums of one tile by float FMA, for x that is not finite.
template <int NT>
__device__ __noinline__ void gemv_tile_float(const Gemv& p, int64_t tile, int s0, int s1, float* red) {
    const int lane = threadIdx.x & 31;
    const int64_t m0 = (int64_t)blockIdx.y * p.rows;
    for (int r = 0; r < 16; ++r) {
        const int64_t n = min(tile * 16 + r, p.w.N - 1);
        for (int m = 0; m < p.rows && m0 + m < p.M; ++m) {
            float acc = 0.f;
            for (int64_t w = (int64_t)(p.span0 + s0) * kSpanWords + lane; w < (int64_t)(p.span0 + s1) * kSpanWords; w += 32) {
                const int64_t k0 = word_k(w);
                if (k0 >= p.w.K) continue;
                const uint32_t word = p.w.codes[n * p.w.cp + w];
                const float s = __bfloat162float(p.w.scales[n * p.w.sp + k0 / p.w.group]);
                for (int j = 0; j < 8 && k0 + j < p.w.K; ++j)
                    acc = fmaf(p.x.p[(m0 + m) * p.x.rs + (k0 + j) * p.x.cs],
                               (float)((int)((word >> code_shift(j)) & 15u) - 8) * s, acc);
            }
            acc = lowbit::warp_sum(acc);
            if (lane == 0) red[r * 2 * NT + m] = acc;
        }
    }
}

// All warps of the CTA, from different places of their loops.
__device__ __forceinline__ void gemv_barrier() { asm volatile("barrier.sync 1, %0;" ::"n"(kGemvThreads) : "memory"); }

template <int NT, int G>
__global__ void __launch_bounds__(kGemvThreads, 1) gemv_kernel(const Gemv p) {
    constexpr int SEG = kSpan / G;
    extern __shared__ __align__(16) uint8_t gemv_smem_raw[];
    const int col_bytes = p.spans * kSpan + 16;
    uint8_t* xs = gemv_smem_raw;
    int2* zi = reinterpret_cast<int2*>(xs + (size_t)8 * NT * col_bytes);
    float* fs = reinterpret_cast<float*>(zi + (size_t)4 * NT * p.spans * SEG);
    float* red = fs + (size_t)4 * NT * p.spans;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int part = warp % p.kp, sub = warp / p.kp, per_cta = kGemvWarps / p.kp;
    const int s0 = p.spans * part / p.kp, ns = p.spans * (part + 1) / p.kp - s0;
    const int stride = (int)gridDim.x * per_cta;
    const int first = (int)blockIdx.x * per_cta;
    const int rounds = p.tiles > first ? (p.tiles - first + stride - 1) / stride : 0;   // the same for all warps

    uint4 wa[kGemvDepth], wb[kGemvDepth];
    uint16_t sa[kGemvDepth][SEG], sb[kGemvDepth][SEG];
    // Load cursor: rows g and g + 8 of a round's tile, from this warp's first span on.
    const uint4 *la = nullptr, *lb = nullptr;
    const uint16_t *ga = nullptr, *gb = nullptr;
    int l_round = -1, l_s = ns;
    // Groups of the last span that K reaches; those behind it have no scale.
    const int groups = (int)((p.w.K + G - 1) / G) - (p.span0 + s0) * SEG;
    auto fetch = [&](int d) {
        if (l_s == ns) {
            l_s = 0;
            if (++l_round < rounds) {
                const int64_t n = ((int64_t)first + sub + (int64_t)l_round * stride) * 16 + g;
                const int64_t na = min(n, p.w.N - 1), nb = min(n + 8, p.w.N - 1);
                const int64_t at = (int64_t)(p.span0 + s0) * 4 + t;
                la = reinterpret_cast<const uint4*>(p.w.codes + na * p.w.cp) + at;
                lb = reinterpret_cast<const uint4*>(p.w.codes + nb * p.w.cp) + at;
                const uint16_t* s = reinterpret_cast<const uint16_t*>(p.w.scales) + (int64_t)(p.span0 + s0) * SEG;
                ga = s + na * p.w.sp;
                gb = s + nb * p.w.sp;
            }
        }
        if (l_round >= rounds) return;
        wa[d] = __ldcs(la + l_s * 4);
        wb[d] = __ldcs(lb + l_s * 4);
#pragma unroll
        for (int i = 0; i < SEG; ++i) {
            const int at = l_s * SEG + i;
            sa[d][i] = at < groups ? __ldg(ga + at) : (uint16_t)0;
            sb[d][i] = at < groups ? __ldg(gb + at) : (uint16_t)0;
        }
        ++l_s;
    };
    if (ns > 0) {
#pragma unroll
        for (int d = 0; d < kGemvDepth; ++d) fetch(d);
    }
    const bool fast = gemv_stage_x<NT, G>(p, xs, zi, fs);   // ends with a __syncthreads

    float tot[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) tot[i][0] = tot[i][1] = 0.f;
    int round = 0;

    // One round is over for this warp: its sums to shared memory, then the CTA adds them up.
    auto flush = [&]() {
        float* mine = red + warp * 16 * 2 * NT;
        if (fast) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                // Lanes t and t ^ 1 hold the low and the high digits of a row.
                const float a = tot[i][0] + __shfl_xor_sync(0xffffffffu, tot[i][0], 1);
                const float b = tot[i][1] + __shfl_xor_sync(0xffffffffu, tot[i][1], 1);
                if ((t & 1) == 0) {
                    mine[g * 2 * NT + i * 2 + t / 2] = a;
                    mine[(g + 8) * 2 * NT + i * 2 + t / 2] = b;
                }
                tot[i][0] = tot[i][1] = 0.f;
            }
        } else {
            gemv_tile_float<NT>(p, (int64_t)first + sub + (int64_t)round * stride, s0, s0 + ns, mine);
        }
        gemv_barrier();
        const int64_t m0 = (int64_t)blockIdx.y * p.rows;
        for (int o = threadIdx.x; o < per_cta * 16 * p.rows; o += kGemvThreads) {
            const int row = o % 16, m = o / 16 % p.rows, ct = o / (16 * p.rows);
            const float* r = red + (ct * p.kp * 16 + row) * 2 * NT + m;
            float v = r[0];
            for (int i = 1; i < p.kp; ++i) v += r[i * 16 * 2 * NT];
            const int64_t n = ((int64_t)first + ct + (int64_t)round * stride) * 16 + row;
            if (n < p.w.N && m0 + m < p.M) {
                float* y = p.y.p + (m0 + m) * p.y.rs + n * p.y.cs;
                if (p.accumulate) v += *y;
                if (p.finish) {
                    if (p.bias) v += p.bias[n];
                    if (p.relu) v = v > 0.f ? v : 0.f;
                }
                *y = v;
            }
        }
        gemv_barrier();
        ++round;
    };

    if (ns == 0 || !fast) {
        while (round < rounds) flush();
        return;
    }
    const uint8_t* xl = xs + (size_t)g * col_bytes + s0 * kSpan + t * 32;
    const int2* zl = zi + (t * p.spans + s0) * SEG;   // row t / 2 of the tile, digits' half t & 1
    const float* fl = fs + t * p.spans + s0;
    const int items = rounds * ns;
    int c_s = 0;
    for (int i0 = 0; i0 < items; i0 += kGemvDepth) {
#pragma unroll
        for (int d = 0; d < kGemvDepth; ++d) {
            if (i0 + d < items) {
                const uint32_t A[4] = {wa[d].x, wa[d].y, wa[d].z, wa[d].w};
                const uint32_t B[4] = {wb[d].x, wb[d].y, wb[d].z, wb[d].w};
                float fa[SEG], fb[SEG];
#pragma unroll
                for (int i = 0; i < SEG; ++i) {
                    fa[i] = __uint_as_float((uint32_t)sa[d][i] << 16);
                    fb[i] = __uint_as_float((uint32_t)sb[d][i] << 16);
                }
                fetch(d);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint8_t* x = xl + (size_t)nt * 8 * col_bytes + c_s * kSpan;
                    const uint4 x0 = *reinterpret_cast<const uint4*>(x), x1 = *reinterpret_cast<const uint4*>(x + 16);
                    const uint32_t X[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
                    const float f = fl[nt * 4 * p.spans + c_s];
#pragma unroll
                    for (int i = 0; i < SEG; ++i) {
                        const int2 z = zl[nt * 4 * p.spans * SEG + c_s * SEG + i];
                        int acc[4] = {z.x, z.y, z.x, z.y};
#pragma unroll
                        for (int b = i * 4 / SEG; b < (i + 1) * 4 / SEG; ++b)
                            mma_u8s8(acc, A[b] & 0x0F0F0F0Fu, B[b] & 0x0F0F0F0Fu, (A[b] >> 4) & 0x0F0F0F0Fu,
                                     (B[b] >> 4) & 0x0F0F0F0Fu, X[2 * b], X[2 * b + 1]);
                        tot[nt][0] = fmaf(f, fa[i] * (float)(acc[0] + 256 * acc[1]), tot[nt][0]);
                        tot[nt][1] = fmaf(f, fb[i] * (float)(acc[2] + 256 * acc[3]), tot[nt][1]);
                    }
                }
                if (++c_s == ns) { c_s = 0; flush(); }
            }
        }
    }
}

}  // namespace q4
}  // namespace mt
