// q4_gemv.cuh -- y = x W + b with 4-bit weights for few rows of x, in integer arithmetic.
//
// One row of x is bound by reading W once; 6.5 TB/s are 13 T weights a second, 45 a cycle of an
// SM, so a weight can cost only a fraction of an instruction. Unpacking to half precision and
// mma.sync on it took 110 instructions for the 128 x 16 weights of a warp's step.
//
// Mathematics. Per span of 128 features x becomes fixed-point numbers of 30 bits and a sign:
// X_0 = rn(x * 2^(29 - e)) with 2^e <= max |x| < 2^(e + 1), X_1 = rn(2^31 times the remainder), and
// so on. A remainder is exact in float, and two numbers hold every entry from 2^(e - 37) on with
// all its bits; for a smaller one the product is gone through again with X_2 and X_3, until
// nothing is left of x. A number for itself, off by up to 2^(e - 30), would lose the small entries of a
// span whose large ones meet weights of 0. X is four signed digits of 8 bits, X = sum d_j 256^j,
// the bytes of (X + 0x808080) ^ 0x808080: the addition carries what makes the lower bytes, less
// 128, signed.
// A code c in a byte's upper half with that half's top bit turned is the signed byte 16 (c - 8),
// so eight codes are unpacked by three instructions, and the tensor core's s8 x s8 product
// (mma.sync m16n8k32, 1,950 multiply-adds a cycle measured) gives sum 16 (c - 8) d_j exactly:
//   y = sum over groups of scale * 2^(e - 33) * sum_j 256^j * sum 16 (c - 8) d_j,
// and the same of the second number times 2^-31, float only from the group's scale on. The eight
// digits of a row are the eight columns of a tile of the product.
//
// A span that holds an infinity or a NaN has no fixed point; a CTA that meets one computes its
// tiles by float FMA.
//
// Work. A CTA of 16 warps keeps its rows of x in shared memory and has a run of tiles of 16
// weight rows, whose spans, taken tile after tile, are cut into 16 equal parts: one barrier,
// then a tile's partial sums are added in order. A warp's codes come GROUP spans (4 or
// 2 KB) at a time by cp.async, two groups in flight: each lane copies the pieces that it will read, so
// nothing but its own wait stands between. The scales of a group are spread over the four
// lanes of a row. blockIdx.y takes up to 4 rows of x each.
//
// Measured: one row on 8192 -> 32768 (group 128) 33 us for 139 MB; longer weights add 5.8 TB/s, the
// rest is start and end (launch, first loads while x is staged, the sums). One row on 4096 ->
// 4096 9 us. More rows are bound by the digits' products and scales (with cold caches, by events,
// 4096 -> 16384: 1 row 18, 2 rows 20, 4 rows 27 us; with one number a span, which lost small
// entries, 4 rows 23). A second pass, for spans that reach over 2^37: 8192 -> 32768 42 -> 68 us.
#pragma once

#include "q4.cuh"

namespace mt {
namespace q4 {

constexpr int kGemvWarps = 16;
constexpr int kGemvThreads = 32 * kGemvWarps;
constexpr int kGemvMaxRows = 4;        // rows of x per CTA, a tile of 8 columns each

struct Gemv {
    Mat x;
    Weight w;
    const float* bias;
    Mat y;
    int64_t M;
    int rows;                          // of x per blockIdx.y, at most NT
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
// banks), powers of two [NT rows][spans + 1], partial sums [run + 15][16][NT], codes
// [warps][2][group][rows g, g + 8][lanes] of 16 bytes.
// Whole lines: cp.async into 16-byte pieces that straddle 32-byte sectors took 20 % longer.
__host__ __device__ constexpr int round128(int n) { return (n + 127) & ~127; }
__host__ __device__ constexpr size_t gemv_smem(int nt, int spans) {
    return (size_t)8 * nt * (gemv_pad(nt, spans) * kSpan + 16) + round128(nt * (gemv_pad(nt, spans) + 1) * 4) +
           (size_t)(gemv_run(nt) + kGemvWarps - 1) * 16 * nt * 4 + (size_t)kGemvWarps * gemv_ring(nt);
}

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The even and the odd nibbles of a word as signed bytes 16 (c - 8): codes 0 4 1 5 and 2 6 3 7.
__device__ __forceinline__ uint32_t even_codes(uint32_t w) { return ((w << 4) & 0xF0F0F0F0u) ^ 0x80808080u; }
__device__ __forceinline__ uint32_t odd_codes(uint32_t w) { return (w & 0xF0F0F0F0u) ^ 0x80808080u; }

// The least biased exponent taken for a span: two numbers then reach down to 2^-149.
constexpr int kGemvMinExp = 38;

enum : int { kStageDone = 0, kStageMore = 1, kStageNotFinite = 2 };

// Puts the numbers 2 pass and 2 pass + 1 of this CTA's rows and spans of x into shared memory; returns
// whether that is all, another pass has to follow, or x is not finite. A warp takes a span, a lane the four
// features that meet one unpacked word: of octet lane / 2 of the span 0 4 1 5 or 2 6 3 7.
// Loads of four spans are in flight together.
template <int NT>
__device__ __forceinline__ int gemv_stage_x(const Gemv& p, uint8_t* xs, float* fs, int pass) {
    constexpr int BATCH = 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int spans = gemv_pad(NT, p.spans), col_bytes = spans * kSpan + 16;
    const int64_t m0 = (int64_t)blockIdx.y * p.rows;
    const int octet = lane >> 1, first = octet * 8 + (lane & 1) * 2;   // features first, first + 1, first + 4, first + 5
    uint8_t* to = xs + octet % 4 * 32 + octet / 4 * 8 + (lane & 1) * 4;
    int bad = 0, more = 0;
#pragma unroll 1
    for (int r = 0; r < NT; ++r) {
        const bool row = r < p.rows && m0 + r < p.M;
        const float* x = p.x.p + (m0 + r) * p.x.rs;
#pragma unroll 1
        for (int sb = warp; sb < spans; sb += BATCH * kGemvWarps) {
            float v[BATCH][4];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int s = sb + u * kGemvWarps;
                const int64_t k = (int64_t)(p.span0 + s) * kSpan + first;
                v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.f;
                if (row && s < p.spans) {
                    if (p.xvec && k + 6 <= p.w.K) {
                        const float2 a = *reinterpret_cast<const float2*>(x + k), b = *reinterpret_cast<const float2*>(x + k + 4);
                        v[u][0] = a.x; v[u][1] = a.y; v[u][2] = b.x; v[u][3] = b.y;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int64_t kj = k + j + (j & 2);
                            if (kj < p.w.K) v[u][j] = x[kj * p.x.cs];
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int s = sb + u * kGemvWarps;
                if (s >= spans) break;
                uint32_t a = max(max(lowbit::abs_bits(v[u][0]), lowbit::abs_bits(v[u][1])),
                                 max(lowbit::abs_bits(v[u][2]), lowbit::abs_bits(v[u][3])));
                a = __reduce_max_sync(0xffffffffu, a);
                bad |= a >= 0x7F800000u;
                const int e = max((int)(a >> 23), kGemvMinExp);   // biased exponent
                // Entries below this exponent have bits behind this pass's numbers.
                const int least = e - 37 - 62 * pass;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t b = lowbit::abs_bits(v[u][j]);
                    more |= b != 0 && max((int)(b >> 23), 1) < least;
                }
                if (pass == 0) {
                    const float up = __uint_as_float((uint32_t)(283 - e) << 23);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u][j] *= up;
                } else if (e > kGemvMinExp + 62 * (pass - 1)) {
                    // 2^31 times what number 2 pass - 1, of step 2^(2 - 62 pass) in units of 2^e, leaves. Of
                    // values from 2^24 of its steps on (or beyond a float's range) that is nothing. Two
                    // factors: one might be beyond that range itself.
                    const int n = 125 - e + 62 * pass, h = n / 2;
                    const float up0 = __uint_as_float((uint32_t)(127 + h) << 23), up1 = __uint_as_float((uint32_t)(127 + n - h) << 23);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float w = v[u][j] * up0 * up1;
                        v[u][j] = fabsf(w) < 16777216.f ? (w - rintf(w)) * 2147483648.f : 0.f;
                    }
                } else {   // the passes before had all of the span
                    v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.f;
                }
                uint8_t* o = to + (size_t)(8 * r) * col_bytes + s * kSpan;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t d[4];   // the four digits of a value
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int X = __float2int_rn(v[u][j]);
                        d[j] = (uint32_t)(X + 0x808080) ^ 0x808080u;
                        v[u][j] = (v[u][j] - (float)X) * 2147483648.f;
                    }
                    // Values in the order 0 4 1 5 (d[0], d[2], d[1], d[3]); one digit of each to a word.
                    const uint32_t l0 = __byte_perm(d[0], d[2], 0x5140), l1 = __byte_perm(d[1], d[3], 0x5140);
                    const uint32_t h0 = __byte_perm(d[0], d[2], 0x7362), h1 = __byte_perm(d[1], d[3], 0x7362);
                    *reinterpret_cast<uint32_t*>(o) = __byte_perm(l0, l1, 0x5410);
                    *reinterpret_cast<uint32_t*>(o + col_bytes) = __byte_perm(l0, l1, 0x7632);
                    *reinterpret_cast<uint32_t*>(o + 2 * (size_t)col_bytes) = __byte_perm(h0, h1, 0x5410);
                    *reinterpret_cast<uint32_t*>(o + 3 * (size_t)col_bytes) = __byte_perm(h0, h1, 0x7632);
                    o += 4 * (size_t)col_bytes;
                }
                // 2^30 times the span's unit. 2^16 of it come off the scales, whose products with the sums
                // of digits would overflow from 2^98 on (2^-16 of the least bfloat16 is a float still). With
                // the rest, sums do not fall below a float's normal numbers where y does not; with 2^16
                // for 2^14 the low digits' could overflow first.
                if (lane == 0) fs[r * (spans + 1) + s] = __uint_as_float((uint32_t)max(e - 3 - 62 * max(pass - 1, 0), 1) << 23);
            }
        }
    }
    if (!__syncthreads_or(bad | more)) return kStageDone;
    return __syncthreads_or(bad) ? kStageNotFinite : kStageMore;
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
            if (lane == 0) red[r * NT + m] = acc;
        }
    }
}

template <int NT, int G>
__global__ void __launch_bounds__(kGemvThreads, 1) gemv_kernel(const Gemv p) {
    constexpr int SEG = kSpan / G, GROUP = gemv_group(NT), WARPS = kGemvWarps;
    extern __shared__ __align__(128) uint8_t gemv_smem_raw[];
    const int spans = gemv_pad(NT, p.spans), col_bytes = spans * kSpan + 16;
    uint8_t* xs = gemv_smem_raw;
    float* fs = reinterpret_cast<float*>(xs + (size_t)8 * NT * col_bytes);
    float* red = fs + round128(NT * (spans + 1) * 4) / 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    uint4* ring = reinterpret_cast<uint4*>(red + (gemv_run(NT) + WARPS - 1) * 16 * NT) +
                  warp * (gemv_ring(NT) / 16) + lane;

    // This CTA's tiles, in runs whose partial sums fit.
    const int gpt = spans / GROUP;   // groups per tile
    const int cta0 = (int)blockIdx.x * p.tiles_each + min((int)blockIdx.x, p.tiles_more);
    const int cta1 = cta0 + p.tiles_each + ((int)blockIdx.x < p.tiles_more ? 1 : 0);
    const int scales = (int)((p.w.K + G - 1) / G) - p.span0 * SEG;   // of a row, from this launch's first span on
    // Groups that begin before this span have all their spans and scales.
    const int whole = min(p.spans, scales / SEG) / GROUP * GROUP;
    const int64_t m0 = (int64_t)blockIdx.y * p.rows;
    int state = kStageDone;

    for (int pass = 0;; ++pass) {
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
            if (tile0 == cta0) state = gemv_stage_x<NT>(p, xs, fs, pass);   // ends with a __syncthreads

            int tile = gpt ? lo / gpt : 0, c_s = (lo - tile * gpt) * GROUP;
            if (state != kStageNotFinite) {
                float tot[NT][2];
#pragma unroll
                for (int i = 0; i < NT; ++i) tot[i][0] = tot[i][1] = 0.f;
                const uint8_t* xl = xs + (size_t)g * col_bytes + t * 32;
                const uint4* w = ring;
                // A lane's digits: 2^16 for the high ones, 2^-31 for the second number, 2^-62 for later passes;
                // and 2^-14 for what the spans' powers of two still have too much.
                const float weight = (t & 1 ? 4.f : 0x1p-14f) * (t & 2 ? 0x1p-31f : 1.f) * (pass ? 0x1p-62f : 1.f);
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
                            fa[k] = __uint_as_float(__shfl_sync(0xffffffffu, (uint32_t)ca[k], (lane & 28) + j) << 16) * 0x1p-16f;
                            fb[k] = __uint_as_float(__shfl_sync(0xffffffffu, (uint32_t)cb[k], (lane & 28) + j) << 16) * 0x1p-16f;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint8_t* x = xl + nt * 8 * col_bytes + (c_s + j) * kSpan;
                            const uint4 x0 = *reinterpret_cast<const uint4*>(x), x1 = *reinterpret_cast<const uint4*>(x + 16);
                            const uint32_t X[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
                            const float f = fs[nt * (spans + 1) + c_s + j];
#pragma unroll
                            for (int k = 0; k < SEG; ++k) {
                                int acc[4] = {0, 0, 0, 0};
#pragma unroll
                                for (int b = k * 4 / SEG; b < (k + 1) * 4 / SEG; ++b)
                                    mma_s8(acc, even_codes(A[b]), even_codes(B[b]), odd_codes(A[b]), odd_codes(B[b]), X[2 * b], X[2 * b + 1]);
                                tot[nt][0] = fmaf(f, fa[k] * (float)(acc[0] + 256 * acc[1]), tot[nt][0]);
                                tot[nt][1] = fmaf(f, fb[k] * (float)(acc[2] + 256 * acc[3]), tot[nt][1]);
                            }
                        }
                    }
                    w = w == ring ? ring + GROUP * 64 : ring;
                    c_s += GROUP;
                    if (c_s == spans || i == hi - 1) {
                        // This warp's part of the tile; parts in order have slots in order.
                        float* mine = red + (tile + warp) * 16 * NT;
#pragma unroll
                        for (int k = 0; k < NT; ++k) {
                            // Lanes t = 0..3 hold the low and the high digits of the first and of the
                            // second number.
                            float a = tot[k][0] * weight, b = tot[k][1] * weight;
                            a += __shfl_xor_sync(0xffffffffu, a, 2);
                            b += __shfl_xor_sync(0xffffffffu, b, 2);
                            a += __shfl_xor_sync(0xffffffffu, a, 1);
                            b += __shfl_xor_sync(0xffffffffu, b, 1);
                            if (t == 0) {
                                mine[g * NT + k] = a;
                                mine[(g + 8) * NT + k] = b;
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
                                        red + (tile + warp) * 16 * NT);
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
                    const float* r = red + ((tl + w0) * 16 + row) * NT + m;
                    v = r[0];
                    for (int w = w0 + 1; w <= w1; ++w)
                        if ((int)((int64_t)total * w / WARPS) < (int)((int64_t)total * (w + 1) / WARPS))
                            v += r[(w - w0) * 16 * NT];
                }
                const int64_t n = (int64_t)(tile0 + tl) * 16 + row;
                if (n < p.w.N && m0 + m < p.M) {
                    float* y = p.y.p + (m0 + m) * p.y.rs + n * p.y.cs;
                    if (p.accumulate || pass) v += *y;
                    if (p.finish && state != kStageMore) {
                        if (p.bias) v += p.bias[n];
                        if (p.relu) v = v > 0.f ? v : 0.f;
                    }
                    *y = v;
                }
            }
            __syncthreads();
        }
        if (state != kStageMore) break;
    }
}

}  // namespace q4
}  // namespace mt
