// q4_batch.cuh -- y = x W + b with 4-bit weights for batches of rows: tcgen05 with the unpacked
// weights in tensor memory.
//
// Mathematics: x = h + m + l exactly, three bfloat16 parts (split3), as in planes_gemm.cuh. The
// parts of up to 64 rows stand side by side as the columns of one MMA tile,
//   D[n][part, row] = sum over a group of (c[n][k] - 8) / kCodeUnit * part[row][k],
// and y gathers scale[n] * (h + m + l) group by group in registers, added with rounding.
//
// Why this shape. Up to some hundred rows the weights' bytes bound the product (0.5 byte per
// weight at 6.5 TB/s: 8192 weights of a 128 x 64 step in 182 cycles of an SM). Unpacked to
// bfloat16 in shared memory, a weight would cost 2 bytes written and 2 read for every MMA on it,
// 128 bytes a cycle being all there is. So a thread unpacks its row of the step into 32
// registers (11 instructions per 8 weights) and stores them to tensor memory, from where the
// MMA takes them; shared memory carries only the packed codes and the parts of x.
//
// Work. The spans of 128 k of all tiles of 128 weight rows, taken tile after tile, are cut into
// one run per CTA, so that all SMs end together; a tile inside one run is written at once, the
// parts of a cut one go to scratch and a second kernel adds them in order. Warp 0 loads by
// TMA (codes and x parts of a span per stage). The two 64-deep halves of a span go
// their own ways: warps 1 and 2 issue their MMAs, warps 4-7 and 8-11 unpack (lane quarter =
// warp & 3), each with its own accumulators and unpacked steps in tensor memory. Warps 12-19
// drain the accumulators, half of the rows of x each. What bounds a step is the roles'
// instructions and hand-overs (a half is 182 cycles of memory, an MMA 24 cycles at 16 rows of
// x), hence two issuers and waits in few instructions. Up to 64 rows of x at a time ("pass").
//
// Measured on 4096 -> 16384 (group 64): 16 rows 25 us, 64 rows 36 us, 192 rows 98 us; one issuer
// took 35 us for 16 rows, and unpacked steps and accumulators in half of tensor memory with two
// CTAs per SM no less.
#pragma once

#include "planes_gemm.cuh"

namespace mt {
namespace q4b {

using lowbit::Mat;

constexpr int kRows = 64;                 // rows of x of a pass, at most
constexpr int THREADS = 32 * 20;
constexpr int EPI_WARPS = 8;
constexpr uint32_t CODE_BYTES = 128 * 64; // a span of 128 weight rows

// Sizes by NB, the blocks of 8 rows of x per drain warp: 16 NB rows of x at most.
template <int NB>
struct Cfg {
    static constexpr int ROWS = 16 * NB;
    static constexpr int COLS = 48 * NB;                       // columns of the MMA tile at most
    static constexpr int ACC = NB == 1 ? 3 : NB == 2 ? 2 : 1;       // accumulators of a half
    static constexpr int A_STAGES = NB <= 1 ? 3 : NB == 2 ? 2 : 3 - (NB == 4);   // unpacked steps of a half, 32 columns each
    static constexpr int STAGES = NB <= 2 ? 6 : NB == 3 ? 4 : 3;
    static_assert(2 * ACC * COLS + 64 * A_STAGES <= 512, "tensor memory");
};

struct Params {
    int64_t N;                   // weight rows (outputs)
    int64_t M;
    int rows;                    // of x per pass
    int cols;                    // MMA tile width: 3 rows, rounded up to 16
    int spans, groups;
    int tiles;                   // of weight rows; tile t of pass s is number s * tiles + t
    int each, more;              // spans of a CTA's run, and how many CTAs have one more
    float* part;                 // [CTA][first or last tile of its run][row of x][128]
    const __nv_bfloat16* scales;
    int64_t sp;
    const float* bias;
    Mat y;
    int relu;
    uint32_t stage_bytes;
};

__host__ __device__ constexpr uint32_t stage_bytes(int cols) { return CODE_BYTES + 2u * cols * 128u; }
template <int NB>
__host__ __device__ constexpr uint32_t smem_bytes(int cols) {
    return 1024 + Cfg<NB>::STAGES * stage_bytes(cols) + 8 * (2 * Cfg<NB>::STAGES + 4 * Cfg<NB>::A_STAGES + 4 * Cfg<NB>::ACC) + 16;
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
// D (+)= A[tmem] * B[smem]^T, bfloat16, one CTA.
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accum)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
// The first span of CTA c's run, counted over all tiles.
__host__ __device__ __forceinline__ int run_begin(const Params& p, int c) { return c * p.each + (c < p.more ? c : p.more); }

// (c - 8) / kCodeUnit of a word's 8 codes, in order, as four pairs: 128 + c is a bfloat16 with c
// in its low bits, and one multiply-add takes 128 + 8 off and scales, exactly.
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t* o) {
    const __nv_bfloat162 unit = __floats2bfloat162_rn(1.f / planes::kCodeUnit, 1.f / planes::kCodeUnit);
    const __nv_bfloat162 off = __floats2bfloat162_rn(-136.f / planes::kCodeUnit, -136.f / planes::kCodeUnit);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
        const __nv_bfloat162 d = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), unit, off);
        o[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

template <int NB, int G>
__global__ void __launch_bounds__(THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const Params p) {
    using C = Cfg<NB>;
    constexpr int SPC = G == 32 ? 2 : 4;      // k16-steps per accumulator: a group, or half of one
    constexpr int CHUNKS = 4 / SPC;           // accumulators per half of a span
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::STAGES * p.stage_bytes);
    uint64_t* full = bars;
    uint64_t* empty = full + C::STAGES;
    uint64_t* a_full = empty + C::STAGES;
    uint64_t* a_empty = a_full + 2 * C::A_STAGES;          // [half][step]
    uint64_t* acc_full = a_empty + 2 * C::A_STAGES;
    uint64_t* acc_empty = acc_full + 2 * C::ACC;           // [half][accumulator]
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(acc_empty + 2 * C::ACC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(acc_empty + 2 * C::ACC) + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int begin = run_begin(p, blockIdx.x), count = run_begin(p, blockIdx.x + 1) - begin;
    const int t_first = begin / p.spans, s_first = begin - t_first * p.spans;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 10);           // eight unpacking warps, two issuers
        }
        for (int s = 0; s < 2 * C::A_STAGES; ++s) {
            mbar_init(smem_u32(&a_full[s]), 4);
            mbar_init(smem_u32(&a_empty[s]), 1);
        }
        for (int a = 0; a < 2 * C::ACC; ++a) {
            mbar_init(smem_u32(&acc_full[a]), 1);
            mbar_init(smem_u32(&acc_empty[a]), EPI_WARPS);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32((const void*)tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_start();   // the kernel that joins cut tiles
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const uint32_t tmem_a = tmem_base + 2 * C::ACC * C::COLS;

    float acc[8 * NB];   // of the draining warps
    if (warp == 0) {
        if (lane == 0) {
            // The codes of the first spans are on their way before x is split.
            // A position in the run: tile of the pass, span, the pass's first row of x parts.
            struct Cursor { int tile, s, row; };
            Cursor code{t_first % p.tiles, s_first, t_first / p.tiles * 3 * p.rows}, x = code;
            auto step = [&](Cursor& c) {
                if (++c.s < p.spans) return;
                c.s = 0;
                if (++c.tile == p.tiles) { c.tile = 0; c.row += 3 * p.rows; }
            };
            auto load_codes = [&](int s) {
                mbar_arrive_expect_tx(smem_u32(&full[s]), p.stage_bytes);
                tma_load_2d(smem_u32(smem + s * p.stage_bytes) + 2 * p.cols * 128, &tmW, smem_u32(&full[s]), code.s * 64,
                            code.tile * 128);
                step(code);
            };
            for (int i = 0; i < min(count, C::STAGES); ++i) load_codes(i);
            pdl_wait();
            int s = 0;
            uint32_t ph = 0;
            for (int i = 0; i < count; ++i) {
                if (i >= C::STAGES) {
                    if (!mbar_wait_short(smem_u32(&empty[s]), ph ^ 1, abort_flag, kDevTimeoutEmpty)) break;
                    load_codes(s);
                }
                const uint32_t to = smem_u32(smem + s * p.stage_bytes), bar = smem_u32(&full[s]);
                tma_load_2d(to, &tmX, bar, x.s * 128, x.row);
                tma_load_2d(to + p.cols * 128, &tmX, bar, x.s * 128 + 64, x.row);
                step(x);
                if (++s == C::STAGES) { s = 0; ph ^= 1; }
            }
            // The last releases of the stages are committed behind the accumulators that end the drains'
            // work, and must not arrive in shared memory that the CTA has left.
            for (int i = 0; i < C::STAGES; ++i) {
                if (!mbar_wait_short(smem_u32(&empty[s]), ph ^ 1, abort_flag, kDevTimeoutEmpty)) break;
                if (++s == C::STAGES) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp <= 2) {
        const int half = __shfl_sync(0xffffffffu, warp, 0) - 1;
        if (elect_one()) {
            const uint32_t idesc = planes::idesc_bf16(128, p.cols);
            uint64_t b = umma_desc(smem_u32(smem) + half * p.cols * 128, 16, 1024, kLayoutSw128);
            const uint32_t acc0 = tmem_base + half * C::ACC * C::COLS, a0 = tmem_a + half * C::A_STAGES * 32;
            const uint32_t a_bar = smem_u32(a_full + half * C::A_STAGES), acc_bar = smem_u32(acc_full + half * C::ACC);
            int s = 0, ab = 0, n = 0;
            uint32_t ph = 0, aph = 0, nph = 0;
            for (int i = 0; i < count; ++i) {
                if (!mbar_wait_short(smem_u32(&full[s]), ph, abort_flag, kDevTimeoutFull)) break;
                if (!mbar_wait_short(a_bar + ab * 8, aph, abort_flag, kDevTimeoutMisc)) break;
                bool ok = true;
#pragma unroll
                for (int step = 0; step < 4; ++step) {
                    if (step % SPC == 0) {
                        ok = mbar_wait_short(acc_bar + (2 * C::ACC + n) * 8, nph ^ 1, abort_flag, kDevTimeoutAccEmpty);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    umma_bf16_ts(acc0 + n * C::COLS, a0 + ab * 32 + step * 8, b + step * 2, idesc, step % SPC ? 1u : 0u);
                    if (step % SPC == SPC - 1) {
                        umma_commit(acc_bar + n * 8);
                        if (++n == C::ACC) { n = 0; nph ^= 1; }
                    }
                }
                if (!ok) break;
                umma_commit(a_bar + (2 * C::A_STAGES + ab) * 8);
                umma_commit(smem_u32(&empty[s]));
                if (++ab == C::A_STAGES) { ab = 0; aph ^= 1; }
                b += p.stage_bytes >> 4;
                if (++s == C::STAGES) { s = 0; ph ^= 1; b -= C::STAGES * (p.stage_bytes >> 4); }
            }
        }
    } else if (warp >= 4 && warp < 12) {
        // Row `row` of the weight tile, one half of each span. TMA puts 16-byte piece t of a row
        // at piece t ^ (row / 2 % 4).
        const int q = warp & 3, row = q * 32 + lane, half = (warp - 4) >> 2;
        const uint32_t a_bar = smem_u32(a_full + half * C::A_STAGES);
        const uint32_t a0 = tmem_a + ((uint32_t)(q * 32) << 16) + half * C::A_STAGES * 32;
        int s = 0, ab = 0;
        uint32_t ph = 0, aph = 0;
        for (int i = 0; i < count; ++i) {
            if (!mbar_wait_short(smem_u32(&full[s]), ph, abort_flag, kDevTimeoutFull)) break;
            const uint8_t* codes = smem + s * p.stage_bytes + 2 * p.cols * 128 + row * 64 + half * 8;
            uint2 w[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) w[t] = *reinterpret_cast<const uint2*>(codes + ((t ^ ((row >> 1) & 3)) << 4));
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty[s]));
            if (++s == C::STAGES) { s = 0; ph ^= 1; }
            uint32_t r[32];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                unpack8(w[t].x, r + t * 4);
                unpack8(w[t].y, r + 16 + t * 4);
            }
            if (!mbar_wait_short(a_bar + (2 * C::A_STAGES + ab) * 8, aph ^ 1, abort_flag, kDevTimeoutEmpty)) break;
            tc_fence_after();
            tmem_st_32x32b_x32(a0 + ab * 32, r);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(a_bar + ab * 8);
            if (++ab == C::A_STAGES) { ab = 0; aph ^= 1; }
        }
        for (int i = 0; i < C::A_STAGES; ++i) {   // as for the stages, those of the unpacked steps
            if (!mbar_wait_short(a_bar + (2 * C::A_STAGES + ab) * 8, aph ^ 1, abort_flag, kDevTimeoutEmpty)) break;
            if (++ab == C::A_STAGES) { ab = 0; aph ^= 1; }
        }
    } else if (warp >= 12) {
        const int q = warp & 3, half = (warp - 12) >> 2;   // here of the rows of x
        const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + half * (8 * NB);
        const uint32_t acc_bar = smem_u32(acc_full);
#pragma unroll
        for (int j = 0; j < 8 * NB; ++j) acc[j] = 0.f;
        // The scales of a span are loaded while the one before it is at work.
        constexpr int GROUPS = 128 / G;
        uint16_t next[GROUPS];
        int tile = t_first % p.tiles, s = s_first, from = s_first;   // `from`: the first span of the run in the tile
        int64_t m0 = (int64_t)(t_first / p.tiles) * p.rows;
        bool first = true;                                           // the run's first tile
        const uint16_t* sc = nullptr;
        auto scales_of = [&](int tile) {
            sc = reinterpret_cast<const uint16_t*>(p.scales) + min((int64_t)tile * 128 + q * 32 + lane, p.N - 1) * p.sp;
        };
        auto load_scales = [&](int s) {
#pragma unroll
            for (int k = 0; k < GROUPS; ++k) next[k] = s * GROUPS + k < p.groups ? __ldg(sc + s * GROUPS + k) : (uint16_t)0;
        };
        scales_of(tile);
        load_scales(s);
        bool ok = true;
        int n = 0;
        uint32_t nph = 0;
#pragma unroll 1
        for (int i = 0; i < count && ok; ++i) {
            float scale[GROUPS];
#pragma unroll
            for (int k = 0; k < GROUPS; ++k) scale[k] = __uint_as_float((uint32_t)next[k] << 16);
            if (s + 1 < p.spans) {
                load_scales(s + 1);
            } else if (i + 1 < count) {
                scales_of(tile + 1 == p.tiles ? 0 : tile + 1);
                load_scales(0);
            }
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int at = h * C::ACC + n;
                    const float sca = scale[(h * CHUNKS + c) * GROUPS / (2 * CHUNKS)];
                    ok = ok && mbar_wait_short(acc_bar + at * 8, nph, abort_flag, kDevTimeoutAccFull);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t t0 = taddr + at * C::COLS;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint32_t hi[8], mi[8], lo[8];
                        tmem_ld_32x32b_x8(t0 + b * 8, hi);
                        tmem_ld_32x32b_x8(t0 + p.rows + b * 8, mi);
                        tmem_ld_32x32b_x8(t0 + 2 * p.rows + b * 8, lo);
                        tmem_ld_wait();
                        if (b == NB - 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(acc_bar + (2 * C::ACC + at) * 8);
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            acc[b * 8 + j] = fmaf(sca, __uint_as_float(hi[j]) + (__uint_as_float(mi[j]) + __uint_as_float(lo[j])), acc[b * 8 + j]);
                    }
                }
                if (++n == C::ACC) { n = 0; nph ^= 1; }
            }
            if (++s == p.spans || i == count - 1) {
                // One store per row of x, by pointers that step from row to row.
                const int64_t row = (int64_t)tile * 128 + q * 32 + lane;
                const bool whole = from == 0 && s == p.spans;
                const int rows = min(p.rows, whole ? (int)min(p.M - m0, (int64_t)kRows) : kRows) - half * (8 * NB);
                float* to = whole ? p.y.p + (m0 + half * (8 * NB)) * p.y.rs + row * p.y.cs
                                  : p.part + (((int64_t)blockIdx.x * 2 + (first ? 0 : 1)) * p.rows + half * (8 * NB)) * 128 + q * 32 + lane;
                const int64_t step = whole ? p.y.rs : 128;
                const float bias = whole && p.bias && row < p.N ? p.bias[row] : 0.f;
                const float unit = whole ? planes::kCodeUnit : 1.f;
                const bool mine = !whole || row < p.N, relu = whole && p.relu;
#pragma unroll
                for (int j = 0; j < 8 * NB; ++j) {
                    float v = fmaf(acc[j], unit, bias);
                    if (relu) v = v > 0.f ? v : 0.f;
                    if (mine && j < rows) *to = v;
                    to += step;
                    acc[j] = 0.f;
                }
                from = s = 0;
                first = false;
                if (++tile == p.tiles) { tile = 0; m0 += p.rows; }
            }
        }
    }
    if (warp == 0 && lane == 0 && *abort_flag) {
        // Give copies already issued time to land before the CTA leaves.
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// Tiles that several runs share: the sum of their parts in order (+ bias, ReLU). blockIdx.x: tile,
// blockIdx.y: two rows of x.
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
    const int t = blockIdx.x, first = t * p.spans, last = first + p.spans - 1;
    const int wide = p.more * (p.each + 1);   // spans of the runs that have one more
    auto owner = [&](int x) { return x < wide ? x / (p.each + 1) : p.more + (x - wide) / p.each; };
    const int c0 = owner(first), c1 = owner(last);
    const int m = blockIdx.y * 2 + (threadIdx.x >> 7), r = threadIdx.x & 127;
    const int64_t row = (int64_t)(t % p.tiles) * 128 + r, mm = (int64_t)(t / p.tiles) * p.rows + m;
    pdl_wait();
    if (c0 == c1 || m >= p.rows || row >= p.N || mm >= p.M) return;
    float v = 0.f;
    for (int c = c0; c <= c1; ++c) {
        const int slot = run_begin(p, c) / p.spans == t ? 0 : 1;
        v += p.part[(((int64_t)c * 2 + slot) * p.rows + m) * 128 + r];
    }
    v = fmaf(v, planes::kCodeUnit, p.bias ? p.bias[row] : 0.f);
    if (p.relu) v = v > 0.f ? v : 0.f;
    p.y.p[mm * p.y.rs + row * p.y.cs] = v;
}

// The parts of x for q4b::gemm_kernel: out[pass][part][row of the pass][k].
__global__ void __launch_bounds__(256) split_passes_kernel(Mat x, bool vec, __nv_bfloat16* out, int64_t M, int64_t K, int64_t pitch, int rows) {
    pdl_start();
    const int64_t m0 = (int64_t)blockIdx.z * rows;
    const Mat part{x.p + m0 * x.rs, x.rs, x.cs};
    planes::split_cols(part, vec, out + (int64_t)blockIdx.z * 3 * rows * pitch, min((int64_t)rows, M - m0), K, pitch, blockIdx.x, rows);
}

}  // namespace q4b
}  // namespace mt
