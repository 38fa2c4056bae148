// rms_norm.cuh -- root-mean-square norm with the residual's addition, its output in float
// and/or in 8-bit blocks, and its backward pass.
//
//   h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * gamma
//   dx = rstd * (g - xhat * mean(g * xhat)) + dh,  g = dy * gamma,  xhat = h * rstd
//   dgamma = sum over rows of dy * xhat
//
// Both directions are bound by memory: a row is read once and held in registers between its
// reduction and its use. WPR warps share a row; each lane holds V pieces of VEC features
// (VEC = 4: 16-byte accesses, for rows on 16-byte boundaries; VEC = 1 otherwise). Rows
// longer than the largest variant and rows whose features are not neighbours go through the
// *_long kernels, which read them twice (1202 x 15597: forward 195 us there, 112 in registers;
// backward 136 and 103). Statistics and sums are float; the sum over rows for dgamma is one
// partial per row group in a fixed order, added in order by a second kernel, so results do not
// depend on timing.
//
// Measured at 8192 x 4096 with a residual: forward with float and int8 outputs 85 us (571 MB,
// 6.7 TB/s), backward 79 us (537 MB, 6.8 TB/s) and 5 us for dgamma's sum. The backward launch
// has as many CTAs as are resident at once, each with all loads of a row in flight; 4 CTAs of 8
// warps per SM, of which two were resident, with dh loaded behind the reduction, took 130 us.
// Rows off the 16-byte grid are bound by instructions: 1027 x 5001 with e4m3 output 24 us.
#pragma once

#include "lowbit_common.cuh"

namespace mt {
namespace rms {

using lowbit::Mat;
using lowbit::Q8;

struct Fwd {
    Mat x, r, gamma, h, y;     // r.p, h.p, y.p may be null; gamma and rstd: row 0, stride cs
    Mat rstd;                  // may be null
    Q8 q;                      // codes may be null
    int64_t rows;
    int64_t K;
    float eps;
};

struct Bwd {
    Mat dy, h, gamma, rstd, dh, dx;   // dh.p may be null
    float* part;                      // [row groups][K] partials of dgamma, null if not wanted
    int64_t rows;
    int64_t K;
};

// CTAs per SM that the registers have to allow: x and the residual are in flight together.
constexpr int fwd_ctas(int floats, int threads) { return threads > 512 ? 1 : threads > 256 ? 2 : floats <= 16 ? 4 : floats <= 32 ? 3 : 2; }

template <int VEC, int V, int WPR, int RPC>
__global__ void __launch_bounds__(32 * WPR * RPC, fwd_ctas(VEC * V, 32 * WPR * RPC)) fwd_kernel(const Fwd p) {
    static_assert(WPR == 1 || RPC == 1, "rows that share a CTA have one warp each");
    __shared__ float red[2][WPR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int w = RPC > 1 ? 0 : warp;
    int buf = 0;
    for (int64_t row = (int64_t)blockIdx.x * RPC + (RPC > 1 ? warp : 0); row < p.rows; row += (int64_t)gridDim.x * RPC) {
        float v[V][VEC];
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int f = ((c * WPR + w) * 32 + lane) * VEC;
            if (f < p.K) {
                lowbit::load_row<VEC>(v[c], p.x.p + row * p.x.rs, f);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[c][i] = 0.f;
            }
        }
        if (p.r.p) {
            float r[V][VEC];
#pragma unroll
            for (int c = 0; c < V; ++c) {
                const int f = ((c * WPR + w) * 32 + lane) * VEC;
                if (f < p.K) lowbit::load_row<VEC>(r[c], p.r.p + row * p.r.rs, f);
            }
#pragma unroll
            for (int c = 0; c < V; ++c) {
                const int f = ((c * WPR + w) * 32 + lane) * VEC;
                if (f < p.K) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[c][i] += r[c][i];
                    if (p.h.p) lowbit::store_row<VEC>(v[c], p.h.p + row * p.h.rs, f);
                }
            }
        } else if (p.h.p) {
#pragma unroll
            for (int c = 0; c < V; ++c) {
                const int f = ((c * WPR + w) * 32 + lane) * VEC;
                if (f < p.K) lowbit::store_row<VEC>(v[c], p.h.p + row * p.h.rs, f);
            }
        }
#pragma unroll
        for (int c = 0; c < V; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss = fmaf(v[c][i], v[c][i], ss);
        ss = lowbit::row_sum<WPR>(ss, red, buf);
        const float rstd = 1.f / sqrtf(ss / (float)p.K + p.eps);
        if (p.rstd.p && lane == 0 && w == 0) p.rstd.p[row * p.rstd.cs] = rstd;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int f = ((c * WPR + w) * 32 + lane) * VEC;
            const bool in = f < p.K;
            if (f - lane * VEC >= p.K) break;   // the whole warp
            if (in) {
                float g[VEC];
                lowbit::load_row<VEC>(g, p.gamma.p, f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[c][i] = v[c][i] * rstd * g[i];
                if (p.y.p) lowbit::store_row<VEC>(v[c], p.y.p + row * p.y.rs, f);
            }
            if (p.q.codes) lowbit::store_q8<VEC>(v[c], p.q.codes + row * p.q.cp, p.q.scales + row * p.q.sp, p.q.fmt, f, in);
        }
    }
}

// Rows of any length: the row is read again for the output (from h where h is stored, since h
// may be x or r itself; each element is read and written by the same thread).
constexpr int kLongWarps = 32;
__global__ void __launch_bounds__(32 * kLongWarps) fwd_long_kernel(const Fwd p) {
    __shared__ float red[2][kLongWarps];
    int buf = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        float ss = 0.f;
        for (int64_t f = threadIdx.x; f < p.K; f += blockDim.x) {
            float v = p.x.p[row * p.x.rs + f * p.x.cs];
            if (p.r.p) v += p.r.p[row * p.r.rs + f * p.r.cs];
            if (p.h.p) p.h.p[row * p.h.rs + f * p.h.cs] = v;
            ss = fmaf(v, v, ss);
        }
        ss = lowbit::row_sum<kLongWarps>(ss, red, buf);
        const float rstd = 1.f / sqrtf(ss / (float)p.K + p.eps);
        if (p.rstd.p && threadIdx.x == 0) p.rstd.p[row * p.rstd.cs] = rstd;
        for (int64_t f0 = threadIdx.x & ~31; f0 < p.K; f0 += blockDim.x) {
            const int64_t f = f0 + (threadIdx.x & 31);
            const bool in = f < p.K;
            float v[1] = {0.f};
            if (in) {
                if (p.h.p) {
                    v[0] = p.h.p[row * p.h.rs + f * p.h.cs];
                } else {
                    v[0] = p.x.p[row * p.x.rs + f * p.x.cs];
                    if (p.r.p) v[0] += p.r.p[row * p.r.rs + f * p.r.cs];
                }
                v[0] = v[0] * rstd * p.gamma.p[f * p.gamma.cs];
                if (p.y.p) p.y.p[row * p.y.rs + f * p.y.cs] = v[0];
            }
            if (p.q.codes) lowbit::store_q8<1>(v, p.q.codes + row * p.q.cp, p.q.scales + row * p.q.sp, p.q.fmt, (int)f, in);
        }
    }
}

// dx of a row and this row group's share of dgamma, whose terms stay in registers over all
// rows of the group.
template <int VEC, int V, int WPR, int RPC>
__global__ void __launch_bounds__(32 * WPR * RPC) bwd_kernel(const Bwd p) {
    static_assert(WPR == 1 || RPC == 1, "rows that share a CTA have one warp each");
    __shared__ float red[2][WPR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int w = RPC > 1 ? 0 : warp;
    const int64_t group = (int64_t)blockIdx.x * RPC + (RPC > 1 ? warp : 0);
    int buf = 0;
    float dg[V][VEC];
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) dg[c][i] = 0.f;
    for (int64_t row = group; row < p.rows; row += (int64_t)gridDim.x * RPC) {
        float dy[V][VEC], xh[V][VEC], dh[V][VEC];
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int f = ((c * WPR + w) * 32 + lane) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) dy[c][i] = xh[c][i] = dh[c][i] = 0.f;
            if (f < p.K) {
                lowbit::load_row<VEC>(dy[c], p.dy.p + row * p.dy.rs, f);
                lowbit::load_row<VEC>(xh[c], p.h.p + row * p.h.rs, f);
                if (p.dh.p) lowbit::load_row<VEC>(dh[c], p.dh.p + row * p.dh.rs, f);
            }
        }
        const float rstd = p.rstd.p[row * p.rstd.cs];
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int f = ((c * WPR + w) * 32 + lane) * VEC;
            if (f < p.K) {
                float g[VEC];
                lowbit::load_row<VEC>(g, p.gamma.p, f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    xh[c][i] *= rstd;
                    dg[c][i] = fmaf(dy[c][i], xh[c][i], dg[c][i]);
                    dy[c][i] *= g[i];
                    dot = fmaf(dy[c][i], xh[c][i], dot);
                }
            }
        }
        dot = lowbit::row_sum<WPR>(dot, red, buf) / (float)p.K;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int f = ((c * WPR + w) * 32 + lane) * VEC;
            if (f < p.K) {
                float d[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) d[i] = fmaf(rstd, fmaf(-xh[c][i], dot, dy[c][i]), dh[c][i]);
                lowbit::store_row<VEC>(d, p.dx.p + row * p.dx.rs, f);
            }
        }
    }
    if (p.part) {
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int f = ((c * WPR + w) * 32 + lane) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (f + i < p.K) p.part[group * p.K + f + i] = dg[c][i];
        }
    }
}

__global__ void __launch_bounds__(32 * kLongWarps) bwd_long_kernel(const Bwd p) {
    __shared__ float red[2][kLongWarps];
    int buf = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const float rstd = p.rstd.p[row * p.rstd.cs];
        float dot = 0.f;
        for (int64_t f = threadIdx.x; f < p.K; f += blockDim.x)
            dot = fmaf(p.dy.p[row * p.dy.rs + f * p.dy.cs] * p.gamma.p[f * p.gamma.cs],
                       p.h.p[row * p.h.rs + f * p.h.cs] * rstd, dot);
        dot = lowbit::row_sum<kLongWarps>(dot, red, buf) / (float)p.K;
        for (int64_t f = threadIdx.x; f < p.K; f += blockDim.x) {
            const float g = p.dy.p[row * p.dy.rs + f * p.dy.cs] * p.gamma.p[f * p.gamma.cs];
            float d = rstd * fmaf(-(p.h.p[row * p.h.rs + f * p.h.cs] * rstd), dot, g);
            if (p.dh.p) d += p.dh.p[row * p.dh.rs + f * p.dh.cs];
            p.dx.p[row * p.dx.rs + f * p.dx.cs] = d;
        }
    }
}

// dgamma partials for rows of any length: thread = feature, blockIdx.y = row group (rows y,
// y + groups, ... ascending). Runs before bwd_long_kernel, whose dx may be dy itself.
__global__ void __launch_bounds__(256) dgamma_long_kernel(const Bwd p) {
    const int64_t f = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (f >= p.K) return;
    float s = 0.f;
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y)
        s = fmaf(p.dy.p[row * p.dy.rs + f * p.dy.cs], p.h.p[row * p.h.rs + f * p.h.cs] * p.rstd.p[row * p.rstd.cs], s);
    p.part[(int64_t)blockIdx.y * p.K + f] = s;
}

// out[f] = sum over g of part[g][f]: 32 sums over g = i (mod 32), each ascending, added in order.
__global__ void __launch_bounds__(1024) sum_parts_kernel(const float* part, int64_t groups, int64_t K, Mat out) {
    __shared__ float s[32][33];
    const int64_t f = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float a = 0.f;
    if (f < K) {
#pragma unroll 4
        for (int64_t g = threadIdx.y; g < groups; g += 32) a += part[g * K + f];
    }
    s[threadIdx.y][threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.y == 0 && f < K) {
#pragma unroll
        for (int i = 1; i < 32; ++i) a += s[i][threadIdx.x];
        out.p[f * out.cs] = a;
    }
}

}  // namespace rms
}  // namespace mt
