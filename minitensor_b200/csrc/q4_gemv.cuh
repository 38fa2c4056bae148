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
// Work. A CTA of 16 warps keeps its rows of x in shared memory and has a run of tiles of 16
// weight rows, whose spans, taken tile after tile, are cut into 16 equal parts: one barrier,
// then a tile's partial sums are added in order. A warp's codes come GROUP spans (4 or
// 2 KB) at a time by cp.async, two groups in flight: each lane copies the pieces that it will read, so
// nothing but its own wait stands between. The scales of a group are spread over the four
// lanes of a row. blockIdx.y takes up to 16 rows of x each.
#pragma once

#include "q4.cuh"

namespace mt {
namespace q4 {

constexpr int kGemvWarps = 16;
constexpr int kGemvThreads = 32 * kGemvWarps;
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
    int tiles_each, tiles_more;        // tiles of 16 weight rows per blockIdx.x, and CTAs that have one more
    int xvec;                          // rows of x on 16-byte boundaries, unit stride
};

// Spans per copy group; more columns leave less room and need less of it.
__host__ __device__ constexpr int gemv_group(int nt) { return nt == 1 ? 4 : 2; }
// Bytes of a warp's two groups.
__host__ __device__ constexpr int gemv_ring(int nt) { return 2 * gemv_group(nt) * 1024; }
// Spans in shared memory: whole groups, zeros behind the last span.
__host__ __device__ constexpr int gemv_pad(int nt, int spans) {
    return (spans + gemv_group(nt) - 1) / gemv_group(nt) * gemv_group(nt);
}
// Tiles of a CTA between two barriers; with its warps they make the partial sums.
__host__ __device__ constexpr int gemv_run(int nt) { return 192 / nt - (kGemvWarps - 1); }

// Shared memory: digits [8 NT columns][spans * 128 + 16] (the 16 put neighbouring columns on other
// banks), accumulator starts and powers of two [2 NT rows][2][spans * segments + 1] of 16 bytes,
// partial sums [run + 15][16][2 NT], codes [warps][2][group][rows g, g + 8][lanes] of 16 bytes.
__host__ __device__ constexpr size_t gemv_smem(int nt, int group, int spans) {
    return (size_t)8 * nt * (gemv_pad(nt, spans) * kSpan + 16) + (size_t)4 * nt * (gemv_pad(nt, spans) * (kSpan / group) + 1) * 16 +
           (size_t)(gemv_run(nt) + kGemvWarps - 1) * 16 * 2 * nt * 4 + (size_t)kGemvWarps * gemv_ring(nt);
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
__device__ __forceinline__ bool gemv_stage_x(const Gemv& p, uint8_t* xs, int4* zs) {
    constexpr int SEG = kSpan / G, WARPS = kGemvWarps;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int spans = gemv_pad(NT, p.spans), col_bytes = spans * kSpan + 16;
    const int64_t m0 = (int64_t)blockIdx.y * p.rows;
    int bad = 0;
    constexpr int BATCH = 4;   // spans whose loads are in flight together
    for (int i0 = warp; i0 < 2 * NT * spans; i0 += BATCH * WARPS) {
    float vs[BATCH][4];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        const int i = i0 + u * WARPS, r = i / spans, s = i - r * spans;
        const int64_t m = m0 + r, k = (int64_t)(p.span0 + s) * kSpan + lane * 4;
        vs[u][0] = vs[u][1] = vs[u][2] = vs[u][3] = 0.f;
        if (r < p.rows && m < p.M && s < p.spans) {
            if (p.xvec && k + 4 <= p.w.K) {
                const float4 q = *reinterpret_cast<const float4*>(p.x.p + m * p.x.rs + k);
                vs[u][0] = q.x; vs[u][1] = q.y; vs[u][2] = q.z; vs[u][3] = q.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k + j < p.w.K) vs[u][j] = p.x.p[m * p.x.rs + (k + j) * p.x.cs];
            }
        }
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        const int i = i0 + u * WARPS, r = i / spans, s = i - r * spans;
        if (r >= 2 * NT) break;
        if (r >= p.rows) {   // no row of x: zeros
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint32_t*>(xs + (size_t)(4 * r + j) * col_bytes + s * kSpan + lane * 4) = 0;
            if (lane < 2 * SEG) zs[(2 * r + lane / SEG) * (spans * SEG + 1) + s * SEG + lane % SEG] = make_int4(0, 0, 0, 0);
            continue;
        }
        const float (&v)[4] = vs[u];
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
            const int at = 2 * r * (spans * SEG + 1) + s * SEG + lane / (G / 4);
            const float f = __uint_as_float((uint32_t)(e - 29) << 23);
            zs[at] = make_int4(-8 * sum[0], -8 * sum[1], __float_as_int(f), 0);
            zs[at + spans * SEG + 1] = make_int4(-8 * sum[2], -8 * sum[3], __float_as_int(f * 65536.f), 0);
        }
    }
    }
    return __syncthreads_or(bad) == 0;
}

// A warp's part of one tile, spans [s0, s1), by float FMA: for x that is not finite.
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

template <int NT, int G>
__global__ void __launch_bounds__(kGemvThreads, 1) gemv_kernel(const Gemv p) {
    constexpr int SEG = kSpan / G, GROUP = gemv_group(NT), WARPS = kGemvWarps;
    extern __shared__ __align__(16) uint8_t gemv_smem_raw[];
    const int spans = gemv_pad(NT, p.spans), col_bytes = spans * kSpan + 16;
    uint8_t* xs = gemv_smem_raw;
    int4* zs = reinterpret_cast<int4*>(xs + (size_t)8 * NT * col_bytes);
    float* red = reinterpret_cast<float*>(zs + (size_t)4 * NT * (spans * SEG + 1));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    uint4* ring = reinterpret_cast<uint4*>(red + (gemv_run(NT) + WARPS - 1) * 16 * 2 * NT) +
                  warp * (gemv_ring(NT) / 16) + lane;

    // This CTA's tiles, in runs whose partial sums fit.
    const int gpt = spans / GROUP;   // groups per tile
    const int cta0 = (int)blockIdx.x * p.tiles_each + min((int)blockIdx.x, p.tiles_more);
    const int cta1 = cta0 + p.tiles_each + ((int)blockIdx.x < p.tiles_more ? 1 : 0);
    const int scales = (int)((p.w.K + G - 1) / G) - p.span0 * SEG;   // of a row, from this launch's first span on
    // Groups that begin before this span have all their spans and scales.
    const int whole = min(p.spans, scales / SEG) / GROUP * GROUP;
    const int64_t m0 = (int64_t)blockIdx.y * p.rows;
    bool fast = true;

    for (int tile0 = cta0; tile0 < cta1; tile0 += gemv_run(NT)) {
        const int tiles = min(gemv_run(NT), cta1 - tile0);
        const int total = tiles * gpt;
        const int lo = (int)((int64_t)total * warp / WARPS), hi = (int)((int64_t)total * (warp + 1) / WARPS);

        // Copy cursor: rows g and g + 8 of a tile, at a group's first span.
        const uint4 *la = nullptr, *lb = nullptr;
        const uint16_t *ga = nullptr, *gb = nullptr;
        int l_i = lo, l_tile = gpt ? lo / gpt : 0, l_s = (lo - l_tile * gpt) * GROUP;
        const uint32_t ring32 = smem_u32(ring);
        uint32_t to = ring32;
        uint16_t sa[SEG], sb[SEG];   // scales of span t of the group fetched last
        auto place = [&]() {
            const int64_t n = (int64_t)(tile0 + l_tile) * 16 + g;
            const int64_t na = min(n, p.w.N - 1), nb = min(n + 8, p.w.N - 1);
            const int64_t at = (int64_t)(p.span0 + l_s) * 4 + t;
            la = reinterpret_cast<const uint4*>(p.w.codes + na * p.w.cp) + at;
            lb = reinterpret_cast<const uint4*>(p.w.codes + nb * p.w.cp) + at;
            const uint16_t* s = reinterpret_cast<const uint16_t*>(p.w.scales) + (int64_t)(p.span0 + l_s + t) * SEG;
            ga = s + na * p.w.sp;
            gb = s + nb * p.w.sp;
        };
        if (lo < hi) place();
        auto fetch = [&]() {
            if (l_i < hi) {
                if (l_s < whole) {
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) {
                        cp_async16(to + j * 1024, la + j * 4);
                        cp_async16(to + j * 1024 + 512, lb + j * 4);
                    }
                    if (GROUP == 4 || t < GROUP) {
#pragma unroll
                        for (int i = 0; i < SEG; ++i) {
                            sa[i] = __ldg(ga + i);
                            sb[i] = __ldg(gb + i);
                        }
                    }
                    la += GROUP * 4;
                    lb += GROUP * 4;
                    ga += GROUP * SEG;
                    gb += GROUP * SEG;
                } else {   // the row ends in this group
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) {
                        if (l_s + j < p.spans) {
                            cp_async16(to + j * 1024, la + j * 4);
                            cp_async16(to + j * 1024 + 512, lb + j * 4);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < SEG; ++i) {
                        const bool in = t < GROUP && l_s + t < p.spans && (l_s + t) * SEG + i < scales;
                        sa[i] = in ? __ldg(ga + i) : (uint16_t)0;
                        sb[i] = in ? __ldg(gb + i) : (uint16_t)0;
                    }
                }
                ++l_i;
                to = to == ring32 ? ring32 + GROUP * 1024 : ring32;
                l_s += GROUP;
                if (l_s >= spans && l_i < hi) { l_s = 0; ++l_tile; place(); }
            }
            cp_async_commit();
        };
        fetch();
        if (tile0 == cta0) fast = gemv_stage_x<NT, G>(p, xs, zs);   // ends with a __syncthreads

        int tile = gpt ? lo / gpt : 0, c_s = (lo - tile * gpt) * GROUP;
        if (fast) {
            float tot[NT][2];
#pragma unroll
            for (int i = 0; i < NT; ++i) tot[i][0] = tot[i][1] = 0.f;
            const uint8_t* xl = xs + (size_t)g * col_bytes + t * 32;
            const int4* zl = zs + t * (spans * SEG + 1);   // row t / 2 of an 8-column tile, its low or high digits
            const uint4* w = ring;
#pragma unroll 1
            for (int i = lo; i < hi; ++i) {
                uint16_t ca[SEG], cb[SEG];
#pragma unroll
                for (int k = 0; k < SEG; ++k) { ca[k] = sa[k]; cb[k] = sb[k]; }
                fetch();
                cp_async_wait<1>();
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    const uint4 wa = w[j * 64], wb = w[j * 64 + 32];
                    const uint32_t A[4] = {wa.x, wa.y, wa.z, wa.w};
                    const uint32_t B[4] = {wb.x, wb.y, wb.z, wb.w};
                    float fa[SEG], fb[SEG];
#pragma unroll
                    for (int k = 0; k < SEG; ++k) {
                        fa[k] = __uint_as_float(__shfl_sync(0xffffffffu, (uint32_t)ca[k], (lane & 28) + j) << 16);
                        fb[k] = __uint_as_float(__shfl_sync(0xffffffffu, (uint32_t)cb[k], (lane & 28) + j) << 16);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint8_t* x = xl + nt * 8 * col_bytes + (c_s + j) * kSpan;
                        const uint4 x0 = *reinterpret_cast<const uint4*>(x), x1 = *reinterpret_cast<const uint4*>(x + 16);
                        const uint32_t X[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                        for (int k = 0; k < SEG; ++k) {
                            const int4 z = zl[nt * 4 * (spans * SEG + 1) + (c_s + j) * SEG + k];
                            const float f = __int_as_float(z.z);
                            int acc[4] = {z.x, z.y, z.x, z.y};
#pragma unroll
                            for (int b = k * 4 / SEG; b < (k + 1) * 4 / SEG; ++b)
                                mma_u8s8(acc, A[b] & 0x0F0F0F0Fu, B[b] & 0x0F0F0F0Fu, (A[b] >> 4) & 0x0F0F0F0Fu,
                                         (B[b] >> 4) & 0x0F0F0F0Fu, X[2 * b], X[2 * b + 1]);
                            tot[nt][0] = fmaf(f, fa[k] * (float)(acc[0] + 256 * acc[1]), tot[nt][0]);
                            tot[nt][1] = fmaf(f, fb[k] * (float)(acc[2] + 256 * acc[3]), tot[nt][1]);
                        }
                    }
                }
                w = w == ring ? ring + GROUP * 64 : ring;
                c_s += GROUP;
                if (c_s == spans || i == hi - 1) {
                    // This warp's part of the tile; parts in order have slots in order.
                    float* mine = red + (tile + warp) * 16 * 2 * NT;
#pragma unroll
                    for (int k = 0; k < NT; ++k) {
                        // Lanes t and t ^ 1 hold the low and the high digits of a row.
                        const float a = tot[k][0] + __shfl_xor_sync(0xffffffffu, tot[k][0], 1);
                        const float b = tot[k][1] + __shfl_xor_sync(0xffffffffu, tot[k][1], 1);
                        if ((t & 1) == 0) {
                            mine[g * 2 * NT + k * 2 + t / 2] = a;
                            mine[(g + 8) * 2 * NT + k * 2 + t / 2] = b;
                        }
                        tot[k][0] = tot[k][1] = 0.f;
                    }
                    c_s = 0;
                    ++tile;
                }
            }
        } else {
            for (int i = lo; i < hi;) {
                const int n = min(hi - i, gpt - (i - tile * gpt));
                const int s = (i - tile * gpt) * GROUP;
                gemv_tile_float<NT>(p, tile0 + tile, min(s, p.spans), min(s + n * GROUP, p.spans),
                                    red + (tile + warp) * 16 * 2 * NT);
                i += n;
                ++tile;
            }
        }
        cp_async_wait_all();
        __syncthreads();
        for (int o = threadIdx.x; o < tiles * 16 * p.rows; o += kGemvThreads) {
            const int row = o % 16, m = o / 16 % p.rows, tl = o / (16 * p.rows);
            float v = 0.f;
            if (gpt) {
                // Warps whose parts meet the tile: the last w with total * w / warps <= its first
                // and its last group.
                const int w0 = ((tl * gpt + 1) * WARPS - 1) / total, w1 = ((tl + 1) * gpt * WARPS - 1) / total;
                const float* r = red + ((tl + w0) * 16 + row) * 2 * NT + m;
                v = r[0];
                for (int w = w0 + 1; w <= w1; ++w)
                    if ((int)((int64_t)total * w / WARPS) < (int)((int64_t)total * (w + 1) / WARPS))
                        v += r[(w - w0) * 16 * 2 * NT];
            }
            const int64_t n = (int64_t)(tile0 + tl) * 16 + row;
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
        __syncthreads();
    }
}

}  // namespace q4
}  // namespace mt
