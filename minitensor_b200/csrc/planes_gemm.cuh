// planes_gemm.cuh -- a float-accurate tensor-core product for a left operand that bfloat16
// holds exactly (8-bit checkpoints, 4-bit weight codes).
//
//   D[r][c] = sum_k A[r][k] * B[c][k],  A bfloat16, B float
//
// Mathematics. A float is the exact sum of three bfloat16 numbers: truncating it to its top
// 8 significand bits leaves a remainder of 16 bits, truncating that leaves 8 (split3; below
// 2^-110 the last part runs out of exponents, off by at most 2^-133). So
// A * B is the sum of three products of 8-bit by 8-bit significands, each exact in the
// float accumulator: three kind::f16 MMAs per k-step instead of the three of 3xTF32 at half
// their rate, twice as fast, and no bits of the operands are lost.
//
// Accumulation. The tensor core adds into its accumulator by truncation, so a long sum
// drifts towards zero by about one part in 2^24 per step; over thousands of rows that
// exceeds a float sum's error. The accumulator is therefore drained every SPC k-steps
// (32 to 128 values of k) into registers that add with rounding, while the next chunk goes
// into the other half of TMEM. The 4-bit product multiplies by the group's scale there, once
// per group instead of once per weight.
//
// Work. A pair of CTAs shares a 256 x 256 tile (tcgen05 cta_group::2, as umma_gemm2.cuh): each
// holds its 128 rows of A and its 128 columns of the three planes of B, 64 KB per 64-deep
// stage, 3 stages. Warp 0 loads by TMA, warp 1 of the even CTA issues the MMAs, warps 2-9
// drain: lane quarter = warp & 3, 128 columns each, 128 accumulators per thread. Products that
// do not fill the GPU with such tiles take 256 x 128 ones, five stages and four accumulators
// (777 x 1001 x 1303: 25.6 -> 18 us; large ones stay, since 64 values of k of such a tile, bound
// by reads of shared memory, take about 1,000 cycles, and of a 256 x 256 tile 1,600). The tiles of
// a last round that would leave clusters idle are split over k between them; their parts go to
// scratch and a second kernel adds them in order.
// Waits: what follows a wait here are copies and MMAs, or reads of tensor memory behind a
// tcgen05 fence, and no thread's ordinary stores, so none needs an acquire at cluster scope, which
// seems to cost the L1 with the scales in it at every chunk: groups of 32, 2048 x 4096 x 8192 379
// against 337 us, 2048 x 5376 x 1536 168 against 128 us.
// Bound: tensor pipe, 3 * 2 R C K operations: 8192^3 in 1956 us, 1686 TFLOP/s of bfloat16 work,
// 1.01 of the measured cuBLAS rate (one launch at full clock; a few after one another 2075 us, in a
// row 2.25 to 2.4 ms, under the power cap).
// Three 64-deep stages, because 64 KB a stage leave room for no fourth; 256 x 256 tiles, because
// a CTA alone on 128 x 256 would move 112 KB through shared memory in the time that bandwidth
// has for 190 KB of reads and writes, of which the MMAs' reads alone are 144 KB.
#pragma once

#include "lowbit_common.cuh"
#include "q4.cuh"

namespace mt {
namespace planes {

using lowbit::Mat;

constexpr int BM = 256;                 // rows of a pair tile
constexpr int BK = 64;                  // k per stage: 128-byte rows
constexpr uint32_t A_BYTES = 128 * BK * 2;
constexpr float kCodeUnit = 2048.f;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);
constexpr uint32_t EPI_BYTES = EPI_WARPS * 32 * 20 * 4;

// By the columns of a pair tile, 256 or 128.
template <int BN>
struct Cfg {
    static constexpr int STAGES = BN == 256 ? 3 : 5;
    static constexpr int ACCS = 512 / BN;                      // accumulators, all of tensor memory
    static constexpr uint32_t B_BYTES = BN / 2 * BK * 2;       // one plane of a CTA's columns
    static constexpr uint32_t STAGE_BYTES = A_BYTES + 3 * B_BYTES;
    static constexpr uint32_t RING_BYTES = STAGE_BYTES * STAGES;
    static constexpr uint32_t SMEM_BYTES = 1024 + RING_BYTES + EPI_BYTES + 8 * (2 * STAGES + 2 * ACCS) + 16;
    static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
};

struct Params {
    int R, C;                    // rows of A, rows of B
    int kblocks;                 // 64-deep blocks of k
    int tiles_r, tiles_c;
    int whole, splits;           // tiles [0, whole) are done at once, the others in `splits` parts of k
    int units;                   // whole + splits * (tiles - whole)
    float* out;                  // D[r][c] at out + r * os_r + c * os_c
    int64_t os_r, os_c;
    float* part;                 // part s of tile t at ((t - whole) * splits + s) * 256 * BN
    const __nv_bfloat16* scales; // SCALED: scale of row r, chunk j at r * sp + j
    int64_t sp;
    int groups;                  // scales per row; chunks behind them have no codes
    const float* bias;           // per row r, may be null (SCALED)
    int relu;
    // Not SCALED, db_tiles > 0: db[c] at db + c * db_cs = the sum over t of col_sums[t * C + c].
    const float* col_sums;
    int db_tiles;
    float* db;
    int64_t db_cs;
};

// Tile t -> blocks of rows and columns. Row blocks go in groups of 8, so that clusters at work
// share rows of A and B in L2.
__device__ __forceinline__ void tile_of(const Params& p, int t, int& rb, int& cb) {
    const int per = 8 * p.tiles_c;
    const int g = t / per, in = t - g * per;
    const int rows = min(8, p.tiles_r - g * 8);
    cb = in / rows;
    rb = g * 8 + in - cb * rows;
}
// Unit u -> tile, part and the k-blocks [kb0, kb1) of the part, which begins on a chunk. sp < 0: whole.
template <int SPC>
__device__ __forceinline__ int unit_of(const Params& p, int u, int& sp, int& kb0, int& kb1) {
    if (u < p.whole) {
        sp = -1;
        kb0 = 0;
        kb1 = p.kblocks;
        return u;
    }
    const int t = (u - p.whole) / p.splits;
    sp = u - p.whole - t * p.splits;
    constexpr int cpb = SPC == 8 ? 2 : 1;                      // k-blocks per chunk boundary
    const int nb = (p.kblocks + cpb - 1) / cpb;
    kb0 = (int)((long long)nb * sp / p.splits) * cpb;
    kb1 = min(p.kblocks, (int)((long long)nb * (sp + 1) / p.splits) * cpb);
    return p.whole + t;
}

// kind::f16 instruction descriptor: bfloat16 operands, K-major, float accumulate.
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_bf16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
}

// SPC: k16-steps per chunk, 2, 4 or 8.
template <bool SCALED, int SPC, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
    using G = Cfg<BN>;
    constexpr int STAGES = G::STAGES, ACCS = G::ACCS, HALF = BN / 2;
    constexpr uint32_t B_BYTES = G::B_BYTES, STAGE_BYTES = G::STAGE_BYTES, RING_BYTES = G::RING_BYTES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = smem;
    float* epi = reinterpret_cast<float*>(smem + RING_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + RING_BYTES + EPI_BYTES);
    uint64_t* full = bars;
    uint64_t* empty = bars + STAGES;
    uint64_t* acc_full = bars + 2 * STAGES;
    uint64_t* acc_empty = acc_full + ACCS;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(acc_empty + ACCS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(acc_empty + ACCS) + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int a = 0; a < ACCS; ++a) {
            mbar_init(smem_u32(&acc_full[a]), 1);
            mbar_init(smem_u32(&acc_empty[a]), 2 * EPI_WARPS);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32((const void*)tmem_slot), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    int rb, cb, sp, kb0, kb1;
    pdl_start();   // the kernel that joins split tiles
    if (warp == 0) {
        if (lane == 0) {
            pdl_wait();
            int s = 0;
            uint32_t ph = 0;
            for (int u = first; u < p.units; u += step) {
                tile_of(p, unit_of<SPC>(p, u, sp, kb0, kb1), rb, cb);
                const int r0 = rb * BM + (int)rank * 128, c0 = cb * BN + (int)rank * HALF;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait_short(smem_u32(&empty[s]), ph ^ 1, abort_flag, kDevTimeoutEmpty)) goto done;
                    const uint32_t sa = smem_u32(ring + s * STAGE_BYTES);
                    if (leader) mbar_arrive_expect_tx(smem_u32(&full[s]), 2 * STAGE_BYTES);
                    const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
                    tma_load_3d_pair(sa, &tmA, bar, kb * BK, r0, 0);
                    tma_load_3d_pair(sa + A_BYTES, &tmB, bar, kb * BK, c0, 0);
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
            // The last releases of the stages: they are committed behind the accumulator that ends the
            // drains' work, and those of the odd CTA come from its peer. None may arrive in shared
            // memory that the CTA has left.
            for (int i = 0; i < STAGES; ++i) {
                if (!mbar_wait_short(smem_u32(&empty[s]), ph ^ 1, abort_flag, kDevTimeoutEmpty)) goto done;
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (leader && elect_one()) {
            constexpr uint32_t idesc = idesc_bf16(BM, BN);
            constexpr int STEPS = SPC == 2 ? 2 : 4;    // of a chunk in one stage
            const uint64_t a0 = umma_desc(smem_u32(ring), 16, 1024, kLayoutSw128);
            const uint32_t peer = 1;
            int s = 0, n = 0;          // stage, chunks begun
            uint32_t ph = 0;
            bool ok = true;
            for (int u = first; u < p.units && ok; u += step) {
                unit_of<SPC>(p, u, sp, kb0, kb1);
                int in_chunk = 0;
                for (int kb = kb0; kb < kb1; ++kb) {
                    ok = mbar_wait_short(smem_u32(&full[s]), ph, abort_flag, kDevTimeoutFull);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t sa = a0 + s * (STAGE_BYTES >> 4);
#pragma unroll
                    for (int sub = 0; sub < 4; sub += STEPS) {
                        const int a = n % ACCS;
                        if (in_chunk == 0) {
                            ok = mbar_wait_short(smem_u32(&acc_empty[a]), ((n / ACCS) & 1) ^ 1, abort_flag, kDevTimeoutAccEmpty);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        const uint32_t more = in_chunk > 0 ? 1u : 0u;
                        // Smallest plane first: its sums meet a small accumulator.
#pragma unroll
                        for (int pl = 2; pl >= 0; --pl)
#pragma unroll
                            for (int k = sub; k < sub + STEPS; ++k)
                                umma_bf16_pair(tmem_base + a * BN, sa + k * 2, sa + ((A_BYTES + pl * B_BYTES) >> 4) + k * 2, idesc,
                                               pl < 2 || k > sub ? 1u : more);
                        in_chunk += STEPS;
                        if (in_chunk == SPC || (kb == kb1 - 1 && sub + STEPS == 4)) {
                            umma_commit_pair(smem_u32(&acc_full[a]));
                            umma_commit_pair(mapa_shared(smem_u32(&acc_full[a]), peer));
                            ++n;
                            in_chunk = 0;
                        }
                    }
                    if (!ok) break;
                    umma_commit_pair(smem_u32(&empty[s]));
                    umma_commit_pair(mapa_shared(smem_u32(&empty[s]), peer));
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
            }
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        float* buf = epi + (warp - 2) * 32 * 20;
        const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + half * HALF;
        const uint32_t empty_bar = mapa_shared(smem_u32(acc_empty), 0);
        int n = 0;
        if (!SCALED && p.db_tiles > 0) {
            pdl_wait();
            // The bias gradient, while the first tiles load: 4 columns per warp, 8 lanes each, which
            // take every eighth partial sum.
            const int sub = lane & 7;
            for (int64_t c0 = ((int64_t)blockIdx.x * EPI_WARPS + warp - 2) * 4; c0 < p.C; c0 += (int64_t)gridDim.x * EPI_WARPS * 4) {
                const int64_t c = c0 + (lane >> 3);
                float s = 0.f;
                if (c < p.C) {
#pragma unroll 8
                    for (int t = sub; t < p.db_tiles; t += 8) s += p.col_sums[(int64_t)t * p.C + c];
                }
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (sub == 0 && c < p.C) p.db[c * p.db_cs] = s;
            }
        }
        for (int u = first; u < p.units; u += step) {
            const int tile = unit_of<SPC>(p, u, sp, kb0, kb1);
            tile_of(p, tile, rb, cb);
            const int row0 = rb * BM + (int)rank * 128 + q * 32;
            const int col0 = cb * BN + half * HALF;
            const int chunks = ((kb1 - kb0) * 4 + SPC - 1) / SPC;
            const __nv_bfloat16* sc = nullptr;
            const int g0 = kb0 * 4 / SPC;
            if (SCALED) sc = p.scales + (int64_t)min(row0 + lane, p.R - 1) * p.sp;
            float acc[HALF];
#pragma unroll
            for (int j = 0; j < HALF; ++j) acc[j] = 0.f;
#pragma unroll 1
            for (int ch = 0; ch < chunks; ++ch, ++n) {
                const int a = n % ACCS;
                float scale = 1.f;
                if (SCALED) scale = g0 + ch < p.groups ? __bfloat162float(sc[g0 + ch]) : 0.f;
                if (!mbar_wait_short(smem_u32(&acc_full[a]), (n / ACCS) & 1, abort_flag, kDevTimeoutAccFull)) goto done;
                __syncwarp();
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < HALF / 16; ++c) {
                    uint32_t r[16];
                    tmem_ld_32x32b_x16(taddr + a * BN + c * 16, r);
                    tmem_ld_wait();
                    if (c == HALF / 16 - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(empty_bar + a * 8);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        acc[c * 16 + j] = SCALED ? fmaf(__uint_as_float(r[j]), scale, acc[c * 16 + j])
                                                 : acc[c * 16 + j] + __uint_as_float(r[j]);
                }
            }
            const bool whole = sp < 0;
            // The parts of a tile are stored as whole tiles, along r or c as D is.
            const bool along_r = p.os_r == 1;
            const int pr = (int)rank * 128 + q * 32, pc = half * HALF;
            float* out = whole ? p.out + (int64_t)row0 * p.os_r + (int64_t)col0 * p.os_c
                               : p.part + ((int64_t)(tile - p.whole) * p.splits + sp) * (BM * BN) + (along_r ? pc * BM + pr : pr * BN + pc);
            const int64_t os_r = whole ? p.os_r : along_r ? 1 : BN, os_c = whole ? p.os_c : along_r ? BM : 1;
            const int rows = whole ? min(32, p.R - row0) : 32, cols = whole ? min(HALF, p.C - col0) : HALF;
            if (SCALED) {
                const int row = row0 + lane;
                const float b = whole && p.bias && row < p.R ? p.bias[row] : 0.f;
#pragma unroll
                for (int j = 0; j < HALF; ++j) {
                    acc[j] = fmaf(acc[j], kCodeUnit, b);
                    if (whole && p.relu) acc[j] = acc[j] > 0.f ? acc[j] : 0.f;
                }
            }
            if (os_r == 1) {
                // Lanes are neighbours in memory: one 128-byte line per column.
                if (lane < rows) {
                    float* o = out + lane;
#pragma unroll
                    for (int j = 0; j < HALF; ++j) {
                        if (j < cols) *o = acc[j];
                        o += os_c;
                    }
                }
            } else {
                // 32 x 16 blocks turned in shared memory (rows of 20 floats: 16-byte accesses of
                // 8 lanes fall on different banks), then 4 lanes along c and 8 rows at a time.
                const bool vec = os_c == 1 && os_r % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
                for (int c = 0; c < HALF; c += 16) {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        *reinterpret_cast<float4*>(buf + lane * 20 + j) = make_float4(acc[c + j], acc[c + j + 1], acc[c + j + 2], acc[c + j + 3]);
                    __syncwarp();
                    if (vec && c + 16 <= cols) {
                        const int r = lane >> 2, j = (lane & 3) * 4;
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            if (i + r < rows)
                                *reinterpret_cast<float4*>(out + (i + r) * os_r + c + j) = *reinterpret_cast<const float4*>(buf + (i + r) * 20 + j);
                    } else {
                        const int r = lane >> 4, j = lane & 15;
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            if (i + r < rows && c + j < cols) out[(i + r) * os_r + (c + j) * os_c] = buf[(i + r) * 20 + j];
                    }
                }
            }
        }
    }

done:
    if (warp == 0 && lane == 0 && *abort_flag) {
        // Give copies already issued time to land before the CTA leaves.
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// The tiles that were done in parts: the sum of the parts in order (+ bias per row, ReLU). A thread
// has 8 elements.
template <int BN>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
    const int t = blockIdx.x;
    pdl_wait();
    int rb, cb;
    tile_of(p, p.whole + t, rb, cb);
    const bool along_r = p.os_r == 1;
    const float* part = p.part + (int64_t)t * p.splits * (BM * BN);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // 256 neighbours along r or c per step, whichever is D's unit stride.
        const int e = (blockIdx.y * 8 + i) * 256 + threadIdx.x;
        const int r = along_r ? e % BM : e / BN, c = along_r ? e / BM : e % BN;
        const float* at = part + (along_r ? c * BM + r : r * BN + c);
        float v = *at;
        for (int s = 1; s < p.splits; ++s) v += at[s * (BM * BN)];
        const int64_t row = (int64_t)rb * BM + r, col = (int64_t)cb * BN + c;
        if (row < p.R && col < p.C) {
            if (p.bias) v += p.bias[row];
            if (p.relu) v = v > 0.f ? v : 0.f;
            p.out[row * p.os_r + col * p.os_c] = v;
        }
    }
}

// x = h + m + l exactly, each part a bfloat16 (truncations: 8 + 8 + 8 significand bits). An
// infinity or NaN is its own first part.
__device__ __forceinline__ void split3(float x, uint16_t (&o)[3]) {
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7F800000u) == 0x7F800000u) {
        o[0] = (uint16_t)(b >> 16) | ((b & 0x7FFFFFu) ? 0x40u : 0u);   // a NaN stays one
        o[1] = o[2] = 0;
        return;
    }
    const uint32_t h = b & 0xFFFF0000u;
    const float r = x - __uint_as_float(h);
    const uint32_t m = __float_as_uint(r) & 0xFFFF0000u;
    const float l = r - __uint_as_float(m);
    o[0] = (uint16_t)(h >> 16);
    o[1] = (uint16_t)(m >> 16);
    o[2] = (uint16_t)(__float_as_uint(l) >> 16);
}

// Planes of B for a sum over rows of x [M, N]: out[plane][n][m], m padded with zeros to `pitch`.
// 64 x 64 tiles turned in shared memory. col_sums, if not null: sums of each tile's columns
// at [tile][N], for the bias gradient.
__device__ __forceinline__ void split_rows(const Mat& x, __nv_bfloat16* out, int64_t M, int64_t N, int64_t pitch,
                                           float* col_sums, int block, float (*s)[65], float (*cs)[64]) {
    const int64_t n0 = (int64_t)block * 64;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t mt = blockIdx.y; mt * 64 < pitch; mt += gridDim.y) {
        const int64_t m0 = mt * 64;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int64_t m = m0 + ty + 4 * i;
            const float v = m < M && n0 + tx < N ? x.p[m * x.rs + (n0 + tx) * x.cs] : 0.f;
            s[ty + 4 * i][tx] = v;
            sum += v;
        }
        cs[ty][tx] = sum;
        __syncthreads();
        if (col_sums && ty == 0 && n0 + tx < N) {
            col_sums[mt * N + n0 + tx] = cs[0][tx] + cs[1][tx] + cs[2][tx] + cs[3][tx];
        }
        const int64_t m = m0 + 2 * lane;
        if (m < pitch) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t n = n0 + warp * 8 + i;
                if (n >= N) break;
                uint16_t a[3], b[3];
                split3(s[2 * lane][warp * 8 + i], a);
                split3(s[2 * lane + 1][warp * 8 + i], b);
#pragma unroll
                for (int pl = 0; pl < 3; ++pl)
                    *reinterpret_cast<uint32_t*>(out + (pl * N + n) * pitch + m) = a[pl] | ((uint32_t)b[pl] << 16);
            }
        }
        __syncthreads();
    }
}

// Planes of B for a sum over columns of x [M, K]: out[plane][m][k], planes of plane_rows rows, k
// padded with zeros to `pitch` (a multiple of 4).
__device__ __forceinline__ void split_cols(const Mat& x, bool vec, __nv_bfloat16* out, int64_t M, int64_t K, int64_t pitch, int block,
                                           int64_t plane_rows) {
    const int64_t k = ((int64_t)block * 256 + threadIdx.x) * 4;
    if (k >= pitch) return;
#pragma unroll 4
    for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
        uint16_t o[4][3];
        if (vec && k + 4 <= K) {
            const float4 v = *reinterpret_cast<const float4*>(x.p + m * x.rs + k);
            split3(v.x, o[0]);
            split3(v.y, o[1]);
            split3(v.z, o[2]);
            split3(v.w, o[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) split3(k + i < K ? x.p[m * x.rs + (k + i) * x.cs] : 0.f, o[i]);
        }
#pragma unroll
        for (int pl = 0; pl < 3; ++pl)
            *reinterpret_cast<uint2*>(out + (pl * plane_rows + m) * pitch + k) =
                make_uint2(o[0][pl] | ((uint32_t)o[1][pl] << 16), o[2][pl] | ((uint32_t)o[3][pl] << 16));
    }
}

// A for the 4-bit product: out[n][k] = (code - 8) / kCodeUnit, k up to `pitch` (whole spans). A
// thread takes a word: 128 + c is a bfloat16 with c in its low bits, and 136 comes off exactly.
// The unit keeps the sum over a group, at most 128 * 8 times the largest x, within x's range
// until the group's scale meets it; the tile is multiplied by it when it is done.
__device__ __forceinline__ void expand_q4(const q4::Weight& q, __nv_bfloat16* out, int64_t pitch, int block) {
    const int64_t k = ((int64_t)block * 256 + threadIdx.x) * 8;
    if (k >= pitch) return;
    const int64_t in = k % q4::kSpan;
    const int64_t w = k / q4::kSpan * q4::kSpanWords + in % 32 / 8 * 4 + in / 32;
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.f, 136.f);
    const __nv_bfloat162 unit = __floats2bfloat162_rn(1.f / kCodeUnit, 1.f / kCodeUnit);
#pragma unroll 4
    for (int64_t n = blockIdx.y; n < q.N; n += gridDim.y) {
        const uint32_t word = q.codes[n * q.cp + w];
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = ((word >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
            const __nv_bfloat162 d = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off), unit);
            o[i] = *reinterpret_cast<const uint32_t*>(&d);
        }
        *reinterpret_cast<uint4*>(out + n * pitch + k) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// A for the weight gradient: out[k][m] = value of (m, k), m padded with zeros to `pitch`. A thread
// takes 16 features of a row (VEC: one 16-byte load; rows of codes on 16-byte boundaries).
template <bool VEC>
__device__ __forceinline__ void expand_q8(const lowbit::Q8& q, __nv_bfloat16* out, int64_t M, int64_t K, int64_t pitch,
                                          int block, uint16_t (*s)[66]) {
    const int64_t k0 = (int64_t)block * 64;
    const int row = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t mt = blockIdx.y; mt * 64 < pitch; mt += gridDim.y) {
        const int64_t m0 = mt * 64, k = k0 + part * 16;
        uint32_t w[4] = {0, 0, 0, 0};
        float scale = 0.f;
        if (m0 + row < M && k < K) {
            const uint8_t* c = q.codes + (m0 + row) * q.cp + k;
            scale = lowbit::scale_value(q.scales[(m0 + row) * q.sp + k / lowbit::kBlock]);
            if (VEC && k + 16 <= K) {
                const uint4 v = *reinterpret_cast<const uint4*>(c);
                w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k + i < K) w[i / 4] |= (uint32_t)c[i] << (8 * (i % 4));
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float v = lowbit::code_value((w[i / 4] >> (8 * (i % 4))) & 0xFFu, q.fmt) * scale;
            s[part * 16 + i][row] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
        }
        __syncthreads();
        const int64_t m = m0 + 2 * lane;
        if (m < pitch) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t ko = k0 + warp * 8 + i;
                if (ko >= K) break;
                *reinterpret_cast<uint32_t*>(out + ko * pitch + m) = *reinterpret_cast<const uint32_t*>(&s[warp * 8 + i][2 * lane]);
            }
        }
        __syncthreads();
    }
}

// Both operands of the weight gradient in one launch: blocks [0, blocks_b) of x do dY, the others
// the checkpoint.
template <bool VEC>
__global__ void __launch_bounds__(256) prepare_q8_kernel(lowbit::Q8 q, __nv_bfloat16* a, int64_t K, Mat dy, __nv_bfloat16* b,
                                                         int64_t N, float* col_sums, int64_t M, int64_t pitch, int blocks_b) {
    __shared__ union {
        struct { float s[64][65], cs[4][64]; } rows;
        uint16_t codes[64][66];
    } sm;
    pdl_start();
    if ((int)blockIdx.x < blocks_b) split_rows(dy, b, M, N, pitch, col_sums, blockIdx.x, sm.rows.s, sm.rows.cs);
    else expand_q8<VEC>(q, a, M, K, pitch, blockIdx.x - blocks_b, sm.codes);
}
// Both operands of the 4-bit product in one launch: blocks [0, blocks_b) of x do x.
__global__ void __launch_bounds__(256) prepare_q4_kernel(q4::Weight q, __nv_bfloat16* a, Mat x, bool vec, __nv_bfloat16* b, int64_t M,
                                                         int64_t pitch, int blocks_b) {
    pdl_start();
    if ((int)blockIdx.x < blocks_b) split_cols(x, vec, b, M, q.K, pitch, blockIdx.x, M);
    else expand_q4(q, a, pitch, blockIdx.x - blocks_b);
}

}  // namespace planes
}  // namespace mt
