// mt_lowbit.cu -- C entries of the low-bit operators (declared in include/mtgemm.h): argument
// checks, choice of kernel and launches.
#include <algorithm>
#include <atomic>
#include <cstdio>

#include "mtgemm.h"
#include "mt_host.h"
#include "lowbit_common.cuh"
#include "planes_gemm.cuh"
#include "q4.cuh"
#include "q4_batch.cuh"
#include "q4_gemv.cuh"
#include "q8.cuh"
#include "rms_norm.cuh"

namespace {

using mt::host::fail;
using mt::host::launched;
using mt::lowbit::Mat;
using mt::lowbit::Q8;

constexpr int64_t kMaxExtent = INT32_MAX - 4096;   // rows or features of one operand

// A checked 2-D view, or a vector as one row.
struct View2 {
    Mat m{nullptr, 0, 0};
    int64_t rows = 0, cols = 0;
    bool given = false;
};

int to_mat(const mt_tensor* t, const char* who, const char* name, View2& v) {
    if (!t) return fail(MT_EINVAL, "%s: %s is null", who, name);
    if (t->ndim != 2) return fail(MT_EINVAL, "%s: %s must be 2-D, got %u-D", who, name, t->ndim);
    if (t->shape[0] > (uint64_t)kMaxExtent || t->shape[1] > (uint64_t)kMaxExtent)
        return fail(MT_EUNSUPPORTED, "%s: %s has an extent beyond 2^31 - 4097", who, name);
    v.rows = (int64_t)t->shape[0];
    v.cols = (int64_t)t->shape[1];
    if (v.rows * v.cols > 0 && !t->data) return fail(MT_EINVAL, "%s: %s has a null data pointer", who, name);
    v.m = Mat{t->data ? t->data + t->offset : nullptr, (int64_t)t->strides[0], (int64_t)t->strides[1]};
    v.given = true;
    return MT_OK;
}

// A vector of n elements: [n], [1, n] or [n, 1].
int to_vec(const mt_tensor* t, int64_t n, const char* who, const char* name, View2& v) {
    if (!t) return fail(MT_EINVAL, "%s: %s is null", who, name);
    uint64_t total = 1;
    int64_t stride = 1;
    int longer = 0;
    for (uint32_t i = 0; i < t->ndim && i < MT_MAX_DIMS; ++i) {
        total *= t->shape[i];
        if (t->shape[i] != 1) { stride = (int64_t)t->strides[i]; ++longer; }
    }
    if (t->ndim < 1 || t->ndim > 2 || longer > 1 || (int64_t)total != n)
        return fail(MT_EINVAL, "%s: %s must hold %lld elements in one dimension", who, name, (long long)n);
    if (n > 0 && !t->data) return fail(MT_EINVAL, "%s: %s has a null data pointer", who, name);
    v.m = Mat{t->data ? t->data + t->offset : nullptr, 0, stride};
    v.rows = 1;
    v.cols = n;
    v.given = true;
    return MT_OK;
}

// Byte ranges for the overlap check.
struct Span {
    uintptr_t lo, hi;   // [lo, hi)
    int64_t pitch;      // bytes between rows of unit-stride columns, 0 if not of that form
    int64_t width;      // bytes of such a row
};
Span span_of(const View2& v) {
    Span s{0, 0, 0, 0};
    if (!v.given || v.rows * v.cols == 0) return s;
    s.lo = reinterpret_cast<uintptr_t>(v.m.p);
    s.hi = s.lo + 4 * (uintptr_t)((v.rows - 1) * v.m.rs + (v.cols - 1) * v.m.cs + 1);
    if (v.m.cs == 1 || v.cols == 1) { s.pitch = 4 * v.m.rs; s.width = 4 * v.cols; }
    return s;
}
Span span_of_rows(const void* p, int64_t rows, int64_t pitch, int64_t width) {
    Span s{0, 0, 0, 0};
    if (!p || rows == 0 || width == 0) return s;
    s.lo = reinterpret_cast<uintptr_t>(p);
    s.hi = s.lo + (uintptr_t)((rows - 1) * pitch + width);
    s.pitch = pitch;
    s.width = width;
    return s;
}
// Conservative: ranges that meet overlap, except disjoint column windows of one row pitch.
bool overlap(const Span& a, const Span& b) {
    if (a.lo >= a.hi || b.lo >= b.hi || a.hi <= b.lo || b.hi <= a.lo) return false;
    if (a.pitch > 0 && a.pitch == b.pitch) {
        const int64_t diff = (int64_t)(b.lo - a.lo);
        const int64_t d = ((diff % a.pitch) + a.pitch) % a.pitch;
        if (d >= a.width && d + b.width <= a.pitch) return false;
    }
    return true;
}
bool same_view(const View2& a, const View2& b) {
    return a.given && b.given && a.m.p == b.m.p && a.rows == b.rows && a.cols == b.cols &&
           (a.rows <= 1 || a.m.rs == b.m.rs) && (a.cols <= 1 || a.m.cs == b.m.cs);
}
// An output whose elements are all different memory.
int check_distinct(const View2& v, const char* who, const char* name) {
    if (!v.given || v.rows * v.cols <= 1) return MT_OK;
    const int64_t rs = v.rows > 1 ? v.m.rs : INT64_MAX / 2, cs = v.cols > 1 ? v.m.cs : INT64_MAX / 2;
    const bool by_row = v.rows <= 1 || (cs > 0 && (v.cols <= 1 || rs > (v.cols - 1) * cs));
    const bool by_col = v.cols <= 1 || (rs > 0 && (v.rows <= 1 || cs > (v.rows - 1) * rs));
    if (rs <= 0 || cs <= 0 || !(by_row || by_col))
        return fail(MT_EINVAL, "%s: %s is an output with overlapping or broadcast elements", who, name);
    return MT_OK;
}
int check_apart(const Span& out, const char* out_name, const Span& in, const char* in_name, const char* who) {
    if (overlap(out, in)) return fail(MT_EINVAL, "%s: %s and %s share memory", who, out_name, in_name);
    return MT_OK;
}

int64_t blocks_of(int64_t cols) { return (cols + mt::lowbit::kBlock - 1) / mt::lowbit::kBlock; }

int to_q8(const mt_q8* q, const char* who, Q8& o, int64_t& rows, int64_t& cols) {
    if (!q) return fail(MT_EINVAL, "%s: the 8-bit tensor is null", who);
    if (q->format != MT_Q8_INT8 && q->format != MT_Q8_E4M3) return fail(MT_EINVAL, "%s: bad 8-bit format %d", who, q->format);
    if (q->rows > (uint64_t)kMaxExtent || q->cols > (uint64_t)kMaxExtent)
        return fail(MT_EUNSUPPORTED, "%s: the 8-bit tensor has an extent beyond 2^31 - 4097", who);
    rows = (int64_t)q->rows;
    cols = (int64_t)q->cols;
    if (rows * cols > 0 && (!q->codes || !q->scales)) return fail(MT_EINVAL, "%s: the 8-bit tensor has a null pointer", who);
    if (rows > 1 && (q->code_pitch < q->cols || q->scale_pitch < (uint64_t)blocks_of(cols)))
        return fail(MT_EINVAL, "%s: the 8-bit tensor's pitch is smaller than a row", who);
    if (q->code_pitch > (1ull << 40) || q->scale_pitch > (1ull << 40))
        return fail(MT_EINVAL, "%s: the 8-bit tensor's pitch is out of range", who);
    o = Q8{static_cast<uint8_t*>(q->codes), q->scales, (int64_t)q->code_pitch, (int64_t)q->scale_pitch, q->format};
    return MT_OK;
}
Span code_span(const Q8& q, int64_t rows, int64_t cols) { return span_of_rows(q.codes, rows, q.cp, cols); }
Span scale_span(const Q8& q, int64_t rows, int64_t cols) { return span_of_rows(q.scales, rows, q.sp, blocks_of(cols)); }

int to_q4(const mt_q4* q, const char* who, mt::q4::Weight& o) {
    if (!q) return fail(MT_EINVAL, "%s: the 4-bit weight is null", who);
    if (q->group != 32 && q->group != 64 && q->group != 128)
        return fail(MT_EINVAL, "%s: group must be 32, 64 or 128, got %llu", who, (unsigned long long)q->group);
    if (q->in > (uint64_t)kMaxExtent || q->out > (uint64_t)kMaxExtent)
        return fail(MT_EUNSUPPORTED, "%s: the 4-bit weight has an extent beyond 2^31 - 4097", who);
    const uint64_t spans = (q->in + 127) / 128, groups = (q->in + q->group - 1) / q->group;
    if (q->in * q->out > 0) {
        if (!q->codes || !q->scales) return fail(MT_EINVAL, "%s: the 4-bit weight has a null pointer", who);
        if ((reinterpret_cast<uintptr_t>(q->codes) & 15) || q->code_pitch % 16)
            return fail(MT_EINVAL, "%s: rows of 4-bit codes must start on 16-byte boundaries", who);
        if (reinterpret_cast<uintptr_t>(q->scales) & 1) return fail(MT_EINVAL, "%s: misaligned 4-bit scales", who);
        if (q->code_pitch < 64 * spans || q->scale_pitch < groups)
            return fail(MT_EINVAL, "%s: the 4-bit weight's pitch is smaller than a row", who);
        if (q->code_pitch > (1ull << 40) || q->scale_pitch > (1ull << 40))
            return fail(MT_EINVAL, "%s: the 4-bit weight's pitch is out of range", who);
    }
    o = mt::q4::Weight{static_cast<uint32_t*>(q->codes), static_cast<__nv_bfloat16*>(q->scales),
                       (int64_t)q->code_pitch / 4, (int64_t)q->scale_pitch, (int64_t)q->in, (int64_t)q->out,
                       (int)q->group};
    return MT_OK;
}
Span q4_code_span(const mt::q4::Weight& q) { return span_of_rows(q.codes, q.K ? q.N : 0, 4 * q.cp, (q.K + 127) / 128 * 64); }
Span q4_scale_span(const mt::q4::Weight& q) {
    return span_of_rows(q.scales, q.K ? q.N : 0, 2 * q.sp, 2 * ((q.K + q.group - 1) / q.group));
}

bool unit_cols(const View2& v) { return !v.given || v.cols <= 1 || v.m.cs == 1; }

// Rows of unit stride that start on 16-byte boundaries.
bool vec4(const View2& v) {
    if (!v.given) return true;
    return v.m.cs == 1 && (reinterpret_cast<uintptr_t>(v.m.p) & 15) == 0 && (v.rows <= 1 || v.m.rs % 4 == 0);
}

unsigned grid_of(int64_t n, int64_t most) { return (unsigned)std::max<int64_t>(1, std::min(n, most)); }

#define MT_TRY(expr)                  \
    do {                              \
        const int rc_ = (expr);       \
        if (rc_ != MT_OK) return rc_; \
    } while (0)

// ------------------------------------- RMS norm ---------------------------------------

// Pieces of 32 lanes x VEC features in the largest row held in registers.
constexpr int64_t fwd_pieces(bool vec) { return vec ? 32 * 8 : 32 * 16; }
constexpr int64_t bwd_pieces(bool vec) { return vec ? 32 * 4 : 32 * 16; }

template <int VEC, int V, int WPR, int RPC>
int launch_fwd(const mt::rms::Fwd& p, cudaStream_t st) {
    const int64_t ctas = (p.rows + RPC - 1) / RPC;
    mt::rms::fwd_kernel<VEC, V, WPR, RPC><<<grid_of(ctas, INT32_MAX), 32 * WPR * RPC, 0, st>>>(p);
    return launched("rms_norm launch");
}

// Warps per row and pieces per lane by the row's length: 8 warps, as many as keep a CTA's
// share of the registers small, until a lane would hold more than 32 floats. Rows that are
// too few to fill the GPU take 32 warps each.
template <int VEC>
int run_fwd(const mt::rms::Fwd& p, cudaStream_t st) {
    const int64_t pieces = (p.K + 32 * VEC - 1) / (32 * VEC);
    const bool few = p.rows <= 2 * mt::host::sm_count();
    if (pieces <= 4) return launch_fwd<VEC, 4, 1, 4>(p, st);
    if (few && pieces <= 32) return launch_fwd<VEC, 1, 32, 1>(p, st);
    if (pieces <= 32) return launch_fwd<VEC, 4, 8, 1>(p, st);
    if (!few && pieces <= 64) return launch_fwd<VEC, 8, 8, 1>(p, st);
    if constexpr (VEC == 1) {
        if (pieces > 256) return launch_fwd<1, 16, 32, 1>(p, st);
        if (!few) return pieces <= 128 ? launch_fwd<1, 8, 16, 1>(p, st) : launch_fwd<1, 16, 16, 1>(p, st);
    }
    if (pieces <= 128) return launch_fwd<VEC, 4, 32, 1>(p, st);
    return launch_fwd<VEC, 8, 32, 1>(p, st);
}

// Row groups whose dgamma partials are kept; the launch has one per CTA (or warp, RPC > 1).
template <int VEC, int V, int WPR, int RPC>
int64_t bwd_groups(int64_t rows) {
    // As many CTAs as are resident at once, asked once per device.
    static std::atomic<int> resident[64];
    int dev = 0;
    cudaGetDevice(&dev);
    int per_sm = resident[dev & 63].load();
    if (per_sm == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, mt::rms::bwd_kernel<VEC, V, WPR, RPC>, 32 * WPR * RPC, 0) ==
                cudaSuccess && per_sm > 0) {
            resident[dev & 63].store(per_sm);
        } else {
            cudaGetLastError();
            per_sm = 1;
        }
    }
    const int64_t ctas = std::min<int64_t>((rows + RPC - 1) / RPC, (int64_t)mt::host::sm_count() * per_sm);
    return ctas * RPC;
}
template <int VEC, int V, int WPR, int RPC>
int launch_bwd(const mt::rms::Bwd& p, int64_t groups, cudaStream_t st) {
    mt::rms::bwd_kernel<VEC, V, WPR, RPC><<<(unsigned)(groups / RPC), 32 * WPR * RPC, 0, st>>>(p);
    return launched("rms_norm_backward launch");
}

// Calls f with the variant for the row length as template arguments.
template <int VEC, typename F>
int with_bwd_variant(int64_t K, F&& f) {
    const int64_t pieces = (K + 32 * VEC - 1) / (32 * VEC);
    if (pieces <= 4) return f.template run<VEC, 4, 1, 4>();
    if (pieces <= 32) return f.template run<VEC, 2, 16, 1>();
    if (pieces <= 64) return f.template run<VEC, 4, 16, 1>();
    if constexpr (VEC == 4) return f.template run<4, 4, 32, 1>();
    else if (pieces <= 128) return f.template run<1, 8, 16, 1>();
    else return pieces <= 256 ? f.template run<1, 8, 32, 1>() : f.template run<1, 16, 32, 1>();
}
struct GroupsOf {
    int64_t rows, *out;
    template <int VEC, int V, int WPR, int RPC> int run() { *out = bwd_groups<VEC, V, WPR, RPC>(rows); return MT_OK; }
};
struct LaunchBwd {
    const mt::rms::Bwd& p;
    int64_t groups;
    cudaStream_t st;
    template <int VEC, int V, int WPR, int RPC> int run() { return launch_bwd<VEC, V, WPR, RPC>(p, groups, st); }
};

// ------------------------- exact-by-float tensor-core product -------------------------

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Scratch of one call, given back on every way out (stream order makes that safe).
struct Scratch {
    void* p = nullptr;
    size_t bytes = 0;
    cudaStream_t st;
    explicit Scratch(cudaStream_t s) : st(s) {}
    Scratch(const Scratch&) = delete;
    ~Scratch() { mt::host::scratch_free(p, bytes, st); }
    int take(size_t n, const char* who) {
        bytes = n;
        return mt::host::scratch_alloc(&p, n, st, who);
    }
};

// How a product is cut: columns of a tile, tiles done at once, and in how many parts of k the
// others. A full round of clusters takes whole tiles; the tiles of a last round that would leave
// clusters idle are split between them. Cycles: a 64-deep block of a 256 x 256 tile takes about
// 1,600, of a 256 x 128 tile (bound by shared memory) 1,000; a tile's end 6,000 or 3,500; a split
// another kernel, 4,000, and its parts' way through memory at 5,000 bytes a cycle.
double plan_tiles(mt::planes::Params& p, int bn, int64_t chunk_blocks, int64_t clusters) {
    const double block = bn == 256 ? 1600. : 1000., end = bn == 256 ? 6000. : 3500.;
    p.tiles_c = (p.C + bn - 1) / bn;
    const int64_t tiles = (int64_t)p.tiles_r * p.tiles_c, rest = tiles % clusters;
    const int64_t nb = (p.kblocks + chunk_blocks - 1) / chunk_blocks;
    p.whole = (int)tiles;
    p.splits = 1;
    const double round = (double)nb * chunk_blocks * block + end;
    double last = rest ? round : 0.;   // the last round as it is
    const int64_t most = rest ? std::min<int64_t>(64, std::min(nb, clusters / rest)) : 1;
    for (int64_t s = 2; s <= most; ++s) {
        const double cost = (double)((nb + s - 1) / s * chunk_blocks) * block + end +
                            (double)(2 * s + 1) * rest * (mt::planes::BM * bn * 4) / 5000. + 4000.;
        if (cost < last) {
            last = cost;
            p.splits = (int)s;
            p.whole = (int)(tiles - rest);
        }
    }
    return (double)(tiles / clusters) * round + last;
}

// Launches a kernel that calls pdl_wait before it reads what the kernel before it wrote.
template <typename... Args>
int launch_after(void (*kern)(Args...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const char* who, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return mt::host::cuda_fail(e, who);
    }
    return launched(who);
}

// Tiles and splits of a product over `kpitch` padded values of k; *bn columns of a tile and
// *part_bytes of scratch for the parts of split tiles.
template <int SPC>
int plan_planes(mt::planes::Params& p, int64_t kpitch, int* bn, size_t* part_bytes, const char* who) {
    using namespace mt::planes;
    p.kblocks = (int)((kpitch + BK - 1) / BK);
    p.tiles_r = (p.R + BM - 1) / BM;
    if ((int64_t)p.tiles_r * ((p.C + 127) / 128) > INT32_MAX / 64) return fail(MT_EUNSUPPORTED, "%s: too many output tiles", who);
    const int64_t clusters = std::max(1, mt::host::sm_count() / 2), chunk = SPC == 8 ? 2 : 1;
    Params narrow = p;
    *bn = 256;
    if (plan_tiles(narrow, 128, chunk, clusters) < plan_tiles(p, 256, chunk, clusters)) {
        p = narrow;
        *bn = 128;
    }
    const int64_t in_parts = (int64_t)p.tiles_r * p.tiles_c - p.whole;
    p.units = (int)(p.whole + in_parts * p.splits);
    *part_bytes = (size_t)in_parts * p.splits * BM * *bn * sizeof(float);
    return MT_OK;
}

// D = A * B^T: a [R][kpitch], b [3][C][kpitch], both bfloat16. p is planned and carries the output,
// the scales (SCALED), the bias and the scratch for parts. The kernel before it on the stream
// made a and b.
template <bool SCALED, int SPC, int BN>
int run_planes(const mt::planes::Params& p, const __nv_bfloat16* a, const __nv_bfloat16* b, int64_t kpitch, cudaStream_t st,
               const char* who) {
    using namespace mt::planes;
    CUtensorMap ta, tb;
    const uint64_t da[3] = {(uint64_t)kpitch, (uint64_t)p.R, 1}, db[3] = {(uint64_t)kpitch, (uint64_t)p.C, 3};
    const uint64_t sa[2] = {(uint64_t)kpitch * 2, (uint64_t)kpitch * 2 * p.R}, sb[2] = {(uint64_t)kpitch * 2, (uint64_t)kpitch * 2 * p.C};
    const uint32_t ba[3] = {BK, 128, 1}, bb[3] = {BK, BN / 2, 3};
    if (!mt::host::encode_bf16(&ta, a, 3, da, sa, ba) || !mt::host::encode_bf16(&tb, b, 3, db, sb, bb))
        return fail(MT_ECUDA, "%s: tensor map encoding failed", who);
    static std::atomic<uint64_t> smem_set{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(smem_set.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(gemm_kernel<SCALED, SPC, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<BN>::SMEM_BYTES);
        if (e != cudaSuccess) return mt::host::cuda_fail(e, who);
        smem_set.fetch_or(bit);
    }
    const unsigned grid = 2 * (unsigned)std::min(p.units, std::max(1, mt::host::sm_count() / 2));
    const int in_parts = p.tiles_r * p.tiles_c - p.whole;
    MT_TRY(launch_after(gemm_kernel<SCALED, SPC, BN>, dim3(grid), dim3(THREADS), Cfg<BN>::SMEM_BYTES, st, who, ta, tb, p));
    if (in_parts) MT_TRY(launch_after(join_kernel<BN>, dim3((unsigned)in_parts, BM * BN / 2048), dim3(256), 0, st, who, p));
    char path[96];
    snprintf(path, sizeof path, "%s planes bn=%d whole=%d splits=%d", who, BN, p.whole, p.splits);
    mt::host::set_path(path);
    return MT_OK;
}

int wgrad_planes(const Q8& q, const Mat& dy, const Mat& dw, const Mat& db, int64_t M, int64_t K, int64_t N,
                 cudaStream_t st, const char* who) {
    const int64_t pitch = std::max<int64_t>(8, round_up(M, 8));
    const size_t a_bytes = round_up(K * pitch * 2, 256), b_bytes = round_up(3 * N * pitch * 2, 256);
    const int64_t tiles_m = (pitch + 63) / 64;
    const size_t s_bytes = db.p ? round_up(tiles_m * N * sizeof(float), 256) : 0;
    mt::planes::Params p{};
    p.R = (int)K;
    p.C = (int)N;
    int bn = 0;
    size_t part_bytes = 0;
    MT_TRY(plan_planes<8>(p, pitch, &bn, &part_bytes, who));
    Scratch ws(st);
    MT_TRY(ws.take(a_bytes + b_bytes + s_bytes + part_bytes, who));
    __nv_bfloat16* a = static_cast<__nv_bfloat16*>(ws.p);
    __nv_bfloat16* b = a + a_bytes / 2;
    float* sums = db.p ? reinterpret_cast<float*>(b + b_bytes / 2) : nullptr;
    p.part = reinterpret_cast<float*>(static_cast<char*>(ws.p) + a_bytes + b_bytes + s_bytes);
    const bool vec = (reinterpret_cast<uintptr_t>(q.codes) & 15) == 0 && (M == 1 || q.cp % 16 == 0);
    const int64_t blocks_a = (K + 63) / 64, blocks_b = (N + 63) / 64;
    const dim3 grid((unsigned)(blocks_a + blocks_b), grid_of(tiles_m, 65535));
    if (vec) mt::planes::prepare_q8_kernel<true><<<grid, 256, 0, st>>>(q, a, K, dy, b, N, sums, M, pitch, (int)blocks_b);
    else mt::planes::prepare_q8_kernel<false><<<grid, 256, 0, st>>>(q, a, K, dy, b, N, sums, M, pitch, (int)blocks_b);
    MT_TRY(launched(who));
    if (K == 0) {   // the bias gradient alone
        if (!db.p) return MT_OK;
        mt::rms::sum_parts_kernel<<<(unsigned)((N + 31) / 32), dim3(32, 32), 0, st>>>(sums, tiles_m, N, db);
        return launched(who);
    }
    p.out = dw.p;
    p.os_r = dw.rs;
    p.os_c = dw.cs;
    p.col_sums = sums;
    p.db_tiles = db.p ? (int)tiles_m : 0;
    p.db = db.p;
    p.db_cs = db.cs;
    return bn == 256 ? run_planes<false, 8, 256>(p, a, b, pitch, st, who) : run_planes<false, 8, 128>(p, a, b, pitch, st, who);
}

template <int SPC>
int linear_q4_planes(const View2& x, const mt::q4::Weight& w, const float* bias, const Mat& y, int64_t M, int relu,
                     cudaStream_t st, const char* who) {
    const int64_t pitch = round_up(w.K, mt::q4::kSpan);
    const size_t a_bytes = round_up(w.N * pitch * 2, 256), b_bytes = round_up(3 * M * pitch * 2, 256);
    mt::planes::Params p{};
    p.R = (int)w.N;
    p.C = (int)M;
    int bn = 0;
    size_t part_bytes = 0;
    MT_TRY(plan_planes<SPC>(p, pitch, &bn, &part_bytes, who));
    Scratch ws(st);
    MT_TRY(ws.take(a_bytes + b_bytes + part_bytes, who));
    __nv_bfloat16* a = static_cast<__nv_bfloat16*>(ws.p);
    __nv_bfloat16* b = a + a_bytes / 2;
    p.part = reinterpret_cast<float*>(static_cast<char*>(ws.p) + a_bytes + b_bytes);
    const int64_t blocks_a = (pitch / 8 + 255) / 256, blocks_b = (pitch / 4 + 255) / 256;
    mt::planes::prepare_q4_kernel<<<dim3((unsigned)(blocks_a + blocks_b), grid_of((std::max(w.N, M) + 7) / 8, 65535)), 256, 0, st>>>(
        w, a, x.m, vec4(x), b, M, pitch, (int)blocks_b);
    MT_TRY(launched(who));
    p.out = y.p;
    p.os_r = y.cs;
    p.os_c = y.rs;
    p.scales = w.scales;
    p.sp = w.sp;
    p.groups = (int)((w.K + w.group - 1) / w.group);
    p.bias = bias;
    p.relu = relu;
    return bn == 256 ? run_planes<true, SPC, 256>(p, a, b, pitch, st, who) : run_planes<true, SPC, 128>(p, a, b, pitch, st, who);
}

// ------------------------------ 4 bits, batches ---------------------------------------

template <int NB, int G>
int launch_q4b(const mt::q4b::Params& p, const CUtensorMap& tw, const CUtensorMap& tx, int64_t ctas, cudaStream_t st, const char* who) {
    using namespace mt::q4b;
    static std::atomic<uint64_t> smem_set{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(smem_set.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(gemm_kernel<NB, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<NB>(Cfg<NB>::COLS));
        if (e != cudaSuccess) return mt::host::cuda_fail(e, who);
        smem_set.fetch_or(bit);
    }
    return launch_after(gemm_kernel<NB, G>, dim3((unsigned)ctas), dim3(THREADS), smem_bytes<NB>(p.cols), st, who, tw, tx, p);
}
template <int NB>
int launch_q4b(int group, const mt::q4b::Params& p, const CUtensorMap& tw, const CUtensorMap& tx, int64_t ctas, cudaStream_t st,
               const char* who) {
    switch (group) {
        case 32: return launch_q4b<NB, 32>(p, tw, tx, ctas, st, who);
        case 64: return launch_q4b<NB, 64>(p, tw, tx, ctas, st, who);
        default: return launch_q4b<NB, 128>(p, tw, tx, ctas, st, who);
    }
}

int linear_q4_batch(const View2& x, const mt::q4::Weight& w, const float* bias, const Mat& y, int64_t M, int relu,
                    cudaStream_t st, const char* who) {
    using namespace mt::q4b;
    const int64_t passes = (M + kRows - 1) / kRows, rows = (M + passes - 1) / passes;
    const int64_t pitch = round_up(w.K, mt::q4::kSpan), tiles = (w.N + 127) / 128;
    const int64_t all = passes * tiles * (pitch / mt::q4::kSpan);   // spans of all tiles
    if (passes > 65535 || all > INT32_MAX / 2) return fail(MT_EUNSUPPORTED, "%s: too many tiles", who);
    // Runs: either one per SM, or tiles in s equal parts, which walk along k side by side and share
    // the parts of x in L2 while they are hot. By spans: a run's start and end take about ten, the
    // join of cut tiles three; runs at different places of k take longer, the more rows of x the
    // longer. 64 rows on 4096 x 16384: 148 runs 53 us, 128 whole tiles 39 us; 128 rows on
    // 4001 x 11003: 148 runs 91 us, 172 whole tiles 108 us.
    const int64_t sms = mt::host::sm_count(), spans = pitch / mt::q4::kSpan, nb = (rows + 15) / 16;
    int64_t ctas = std::max<int64_t>(1, std::min(sms, all / 2));
    double least = (double)((all + ctas - 1) / ctas) * (nb == 1 ? 1. : nb == 2 ? 1.2 : 1.5) + 13.;
    for (int64_t s = 1; s <= 8 && spans % s == 0; s *= 2) {
        const double cost = (double)((passes * tiles * s + sms - 1) / sms) * (double)(spans / s + 10) + (s > 1 ? 3. : 0.);
        if (cost < least) { least = cost; ctas = passes * tiles * s; }
    }
    const bool cut = (all / ctas) % spans || all % ctas;
    const size_t x_bytes = round_up(passes * 3 * rows * pitch * 2, 256);
    const size_t part_bytes = cut ? (size_t)ctas * 2 * rows * 128 * sizeof(float) : 0;
    Scratch ws(st);
    MT_TRY(ws.take(x_bytes + part_bytes, who));
    __nv_bfloat16* parts = static_cast<__nv_bfloat16*>(ws.p);
    split_passes_kernel<<<dim3((unsigned)((pitch / 4 + 255) / 256), (unsigned)rows, (unsigned)passes), 256, 0, st>>>(
        x.m, vec4(x), parts, M, w.K, pitch, (int)rows);
    MT_TRY(launched(who));
    Params p{};
    p.N = w.N;
    p.M = M;
    p.rows = (int)rows;
    p.cols = (int)round_up(3 * rows, 16);
    p.spans = (int)(pitch / mt::q4::kSpan);
    p.groups = (int)((w.K + w.group - 1) / w.group);
    p.scales = w.scales;
    p.sp = w.sp;
    p.bias = bias;
    p.y = y;
    p.relu = relu;
    p.stage_bytes = stage_bytes(p.cols);
    p.tiles = (int)tiles;
    p.each = (int)(all / ctas);
    p.more = (int)(all % ctas);
    p.part = cut ? reinterpret_cast<float*>(static_cast<char*>(ws.p) + x_bytes) : nullptr;
    CUtensorMap tw, tx;
    const uint64_t dw[2] = {(uint64_t)p.spans * 64, (uint64_t)w.N}, dx[2] = {(uint64_t)pitch, (uint64_t)(passes * 3 * rows)};
    const uint64_t sx[1] = {(uint64_t)pitch * 2};
    const uint32_t bw[2] = {64, 128}, bx[2] = {64, (uint32_t)p.cols};
    if (!mt::host::encode_u8(&tw, w.codes, dw, (uint64_t)w.cp * 4, bw) || !mt::host::encode_bf16(&tx, parts, 2, dx, sx, bx))
        return fail(MT_ECUDA, "%s: tensor map encoding failed", who);
    switch (nb) {
        case 1: MT_TRY(launch_q4b<1>(w.group, p, tw, tx, ctas, st, who)); break;
        case 2: MT_TRY(launch_q4b<2>(w.group, p, tw, tx, ctas, st, who)); break;
        case 3: MT_TRY(launch_q4b<3>(w.group, p, tw, tx, ctas, st, who)); break;
        default: MT_TRY(launch_q4b<4>(w.group, p, tw, tx, ctas, st, who)); break;
    }
    if (cut)
        MT_TRY(launch_after(join_kernel, dim3((unsigned)(passes * tiles), (unsigned)(rows + 1) / 2), dim3(256), 0, st, who, p));
    char path[96];
    snprintf(path, sizeof path, "%s batch rows=%d x %d ctas=%d", who, p.rows, (int)passes, (int)ctas);
    mt::host::set_path(path);
    return MT_OK;
}

// ------------------------------- 4 bits, few rows -------------------------------------

constexpr size_t kMaxSmem = 232448;

template <int NT, int G>
int launch_gemv(const mt::q4::Gemv& p, dim3 grid, cudaStream_t st, const char* who) {
    static std::atomic<uint64_t> smem_set{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(smem_set.load() & bit)) {
        cudaError_t e = cudaFuncSetAttribute(mt::q4::gemv_kernel<NT, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
        if (e != cudaSuccess) return mt::host::cuda_fail(e, who);
        smem_set.fetch_or(bit);
    }
    mt::q4::gemv_kernel<NT, G><<<grid, mt::q4::kGemvThreads, mt::q4::gemv_smem(NT, p.spans), st>>>(p);
    return launched(who);
}
template <int NT>
int launch_gemv(const mt::q4::Gemv& p, dim3 grid, cudaStream_t st, const char* who) {
    switch (p.w.group) {
        case 32: return launch_gemv<NT, 32>(p, grid, st, who);
        case 64: return launch_gemv<NT, 64>(p, grid, st, who);
        default: return launch_gemv<NT, 128>(p, grid, st, who);
    }
}

// Rows per CTA: as many as 4, but rather 2 (their CTAs read the weights again, from L2) than K in
// several launches of at most `most` spans.
struct GemvPlan {
    int64_t chunks, rows, most, launches;
};
GemvPlan plan_gemv(int64_t M, int64_t spans) {
    using namespace mt::q4;
    GemvPlan g;
    g.chunks = (M + kGemvMaxRows - 1) / kGemvMaxRows;
    g.rows = (M + g.chunks - 1) / g.chunks;
    while (g.rows > 2 && gemv_smem((int)g.rows, (int)spans) > kMaxSmem) {
        ++g.chunks;
        g.rows = (M + g.chunks - 1) / g.chunks;
    }
    g.most = std::max<int64_t>(1, spans);
    while (g.most > 1 && gemv_smem((int)g.rows, (int)g.most) > kMaxSmem) g.most = (g.most + 1) / 2;
    g.launches = spans ? (spans + g.most - 1) / g.most : 1;   // no inputs: the bias alone
    return g;
}

int linear_q4_gemv(const View2& x, const mt::q4::Weight& w, const float* bias, const Mat& y, int64_t M, int relu,
                   cudaStream_t st, const char* who) {
    using namespace mt::q4;
    const int64_t spans = (w.K + kSpan - 1) / kSpan;
    const auto [chunks, rows, most, launches] = plan_gemv(M, spans);
    const int sms = mt::host::sm_count();
    const int64_t ctas = std::max<int64_t>(1, sms / chunks);
    Gemv p{};
    p.w = w;
    p.bias = bias;
    p.rows = (int)rows;
    p.relu = relu;
    const int64_t tiles = (w.N + 15) / 16;
    dim3 grid(grid_of(tiles, ctas));
    p.tiles_each = (int)(tiles / grid.x);
    p.tiles_more = (int)(tiles % grid.x);
    p.xvec = vec4(x);
    // Without inputs there may be more rows than a grid has chunks.
    for (int64_t c0 = 0; c0 < chunks; c0 += 65535) {
        const int64_t m0 = c0 * rows;
        grid.y = (unsigned)std::min<int64_t>(65535, chunks - c0);
        p.x = Mat{x.m.p + m0 * x.m.rs, x.m.rs, x.m.cs};
        p.y = Mat{y.p + m0 * y.rs, y.rs, y.cs};
        p.M = M - m0;
        for (int64_t i = 0; i < launches; ++i) {
            const int64_t s0 = i * most;
            p.span0 = (int)s0;
            p.spans = (int)std::min(most, spans - s0);
            p.accumulate = i > 0;
            p.finish = i == launches - 1;
            switch (rows) {
                case 1: MT_TRY(launch_gemv<1>(p, grid, st, who)); break;
                case 2: MT_TRY(launch_gemv<2>(p, grid, st, who)); break;
                case 3: MT_TRY(launch_gemv<3>(p, grid, st, who)); break;
                default: MT_TRY(launch_gemv<4>(p, grid, st, who)); break;
            }
        }
    }
    char path[96];
    snprintf(path, sizeof path, "%s gemv rows=%d x %d", who, (int)rows, (int)chunks);
    mt::host::set_path(path);
    return MT_OK;
}

}  // namespace

extern "C" {

MT_API int mt_rms_norm(const mt_tensor* x, const mt_tensor* residual, const mt_tensor* gamma, const mt_tensor* h,
                       const mt_tensor* y, const mt_tensor* rstd, const mt_q8* q8, float eps, void* stream) {
    const char* who = "rms_norm";
    View2 vx, vr, vg, vh, vy, vs;
    Q8 q{nullptr, nullptr, 0, 0, 0};
    MT_TRY(to_mat(x, who, "x", vx));
    const int64_t M = vx.rows, K = vx.cols;
    if (K == 0) return fail(MT_EINVAL, "%s: rows of no features have no mean", who);
    MT_TRY(to_vec(gamma, K, who, "gamma", vg));
    if (residual) MT_TRY(to_mat(residual, who, "residual", vr));
    if (h) MT_TRY(to_mat(h, who, "h", vh));
    if (y) MT_TRY(to_mat(y, who, "y", vy));
    if (rstd) MT_TRY(to_vec(rstd, M, who, "rstd", vs));
    for (const View2* v : {&vr, &vh, &vy})
        if (v->given && (v->rows != M || v->cols != K))
            return fail(MT_EINVAL, "%s: residual, h and y must have x's shape [%lld, %lld]", who, (long long)M, (long long)K);
    if (!(eps >= 0.f)) return fail(MT_EINVAL, "%s: eps must not be negative", who);
    Span sq{0, 0, 0, 0}, ss{0, 0, 0, 0};
    if (q8) {
        int64_t qr, qc;
        MT_TRY(to_q8(q8, who, q, qr, qc));
        if (qr != M || qc != K) return fail(MT_EINVAL, "%s: the 8-bit output must have x's shape", who);
        sq = code_span(q, M, K);
        ss = scale_span(q, M, K);
    }
    if (!h && !y && !rstd && !q8) return fail(MT_EINVAL, "%s: no output is wanted", who);
    MT_TRY(check_distinct(vh, who, "h"));
    MT_TRY(check_distinct(vy, who, "y"));
    MT_TRY(check_distinct(vs, who, "rstd"));
    const Span in[] = {span_of(vx), span_of(vr), span_of(vg)};
    const Span out[] = {span_of(vh), span_of(vy), span_of(vs), sq, ss};
    const View2 *vin[] = {&vx, &vr, &vg}, *vout[] = {&vh, &vy, nullptr, nullptr, nullptr};
    for (int o = 0; o < 5; ++o) {
        for (int i = 0; i < 3; ++i)
            if (!(i < 2 && vout[o] && same_view(*vout[o], *vin[i])) && overlap(out[o], in[i]))
                return fail(MT_EINVAL, "%s: an output shares memory with an input", who);
        for (int p = 0; p < o; ++p)
            if (overlap(out[o], out[p])) return fail(MT_EINVAL, "%s: two outputs share memory", who);
    }
    if (M == 0) return MT_OK;
    mt::rms::Fwd p{vx.m, vr.m, vg.m, vh.m, vy.m, vs.m, q, M, K, eps};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool vec = K % 4 == 0 && vec4(vx) && vec4(vr) && vec4(vg) && vec4(vh) && vec4(vy) &&
                     (!q8 || ((reinterpret_cast<uintptr_t>(q.codes) & 3) == 0 && (M == 1 || q.cp % 4 == 0)));
    int rc;
    const bool unit = unit_cols(vx) && unit_cols(vr) && unit_cols(vg) && unit_cols(vh) && unit_cols(vy);
    if (!unit || (K + 32 * (vec ? 4 : 1) - 1) / (32 * (vec ? 4 : 1)) > fwd_pieces(vec)) {
        mt::rms::fwd_long_kernel<<<grid_of(M, INT32_MAX), 32 * mt::rms::kLongWarps, 0, st>>>(p);
        rc = launched("rms_norm launch");
        if (rc == MT_OK) mt::host::set_path("rms_norm long rows");
        return rc;
    }
    rc = vec ? run_fwd<4>(p, st) : run_fwd<1>(p, st);
    if (rc == MT_OK) mt::host::set_path(vec ? "rms_norm vec=4" : "rms_norm vec=1");
    return rc;
}

MT_API int mt_rms_norm_backward(const mt_tensor* dy, const mt_tensor* h, const mt_tensor* gamma,
                                const mt_tensor* rstd, const mt_tensor* dh, const mt_tensor* dx,
                                const mt_tensor* dgamma, void* stream) {
    const char* who = "rms_norm_backward";
    View2 vdy, vh, vg, vs, vdh, vdx, vdg;
    MT_TRY(to_mat(dy, who, "dy", vdy));
    const int64_t M = vdy.rows, K = vdy.cols;
    if (K == 0) return fail(MT_EINVAL, "%s: rows of no features have no mean", who);
    MT_TRY(to_mat(h, who, "h", vh));
    MT_TRY(to_vec(gamma, K, who, "gamma", vg));
    MT_TRY(to_vec(rstd, M, who, "rstd", vs));
    if (dh) MT_TRY(to_mat(dh, who, "dh", vdh));
    MT_TRY(to_mat(dx, who, "dx", vdx));
    if (dgamma) MT_TRY(to_vec(dgamma, K, who, "dgamma", vdg));
    for (const View2* v : {&vh, &vdh, &vdx})
        if (v->given && (v->rows != M || v->cols != K))
            return fail(MT_EINVAL, "%s: h, dh and dx must have dy's shape [%lld, %lld]", who, (long long)M, (long long)K);
    MT_TRY(check_distinct(vdx, who, "dx"));
    MT_TRY(check_distinct(vdg, who, "dgamma"));
    const View2* in[] = {&vdy, &vdh, &vh, &vg, &vs};
    for (int i = 0; i < 5; ++i) {
        if (!(i < 2 && same_view(vdx, *in[i])) && overlap(span_of(vdx), span_of(*in[i])))
            return fail(MT_EINVAL, "%s: dx shares memory with an input", who);
        if (overlap(span_of(vdg), span_of(*in[i]))) return fail(MT_EINVAL, "%s: dgamma shares memory with an input", who);
    }
    MT_TRY(check_apart(span_of(vdx), "dx", span_of(vdg), "dgamma", who));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    mt::rms::Bwd p{vdy.m, vh.m, vg.m, vs.m, vdh.m, vdx.m, nullptr, M, K};
    const bool vec = K % 4 == 0 && vec4(vdy) && vec4(vh) && vec4(vg) && vec4(vdh) && vec4(vdx);
    const bool unit = unit_cols(vdy) && unit_cols(vh) && unit_cols(vg) && unit_cols(vdh) && unit_cols(vdx);
    const bool is_long = !unit || (K + 32 * (vec ? 4 : 1) - 1) / (32 * (vec ? 4 : 1)) > bwd_pieces(vec);
    int64_t groups = 0;
    if (is_long) {
        // blockIdx.y of the partial sums' kernel, of which a grid has 65,535.
        groups = std::min<int64_t>({M, 65535, std::max<int64_t>(1, 8LL * mt::host::sm_count() * 256 / K)});
    } else {
        MT_TRY(vec ? with_bwd_variant<4>(K, GroupsOf{M, &groups}) : with_bwd_variant<1>(K, GroupsOf{M, &groups}));
    }
    void* ws = nullptr;
    const size_t bytes = dgamma ? (size_t)groups * K * sizeof(float) : 0;
    MT_TRY(mt::host::scratch_alloc(&ws, bytes, st, who));
    p.part = static_cast<float*>(ws);
    int rc = MT_OK;
    if (M > 0) {
        if (is_long) {
            if (p.part) {
                mt::rms::dgamma_long_kernel<<<dim3((unsigned)((K + 255) / 256), (unsigned)groups), 256, 0, st>>>(p);
                rc = launched("rms_norm_backward dgamma launch");
            }
            if (rc == MT_OK) {
                mt::rms::bwd_long_kernel<<<grid_of(M, INT32_MAX), 32 * mt::rms::kLongWarps, 0, st>>>(p);
                rc = launched("rms_norm_backward launch");
            }
        } else {
            rc = vec ? with_bwd_variant<4>(K, LaunchBwd{p, groups, st}) : with_bwd_variant<1>(K, LaunchBwd{p, groups, st});
        }
    }
    if (rc == MT_OK && dgamma) {
        mt::rms::sum_parts_kernel<<<(unsigned)((K + 31) / 32), dim3(32, 32), 0, st>>>(p.part, groups, K, vdg.m);
        rc = launched("rms_norm_backward dgamma sum launch");
    }
    mt::host::scratch_free(ws, bytes, st);
    if (rc == MT_OK)
        mt::host::set_path(is_long ? "rms_norm_backward long rows" : vec ? "rms_norm_backward vec=4" : "rms_norm_backward vec=1");
    return rc;
}

MT_API int mt_quantize_q8(const mt_tensor* x, const mt_q8* q, void* stream) {
    const char* who = "quantize_q8";
    View2 vx;
    Q8 o;
    int64_t M, K;
    MT_TRY(to_mat(x, who, "x", vx));
    MT_TRY(to_q8(q, who, o, M, K));
    if (vx.rows != M || vx.cols != K) return fail(MT_EINVAL, "%s: the 8-bit tensor must have x's shape", who);
    MT_TRY(check_apart(code_span(o, M, K), "the codes", span_of(vx), "x", who));
    MT_TRY(check_apart(scale_span(o, M, K), "the scales", span_of(vx), "x", who));
    MT_TRY(check_apart(code_span(o, M, K), "the codes", scale_span(o, M, K), "the scales", who));
    if (M * K == 0) return MT_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool vec = K % 4 == 0 && vec4(vx) && (reinterpret_cast<uintptr_t>(o.codes) & 3) == 0 && (M == 1 || o.cp % 4 == 0);
    const int64_t width = 32 * (vec ? 4 : 1) * mt::q8::kWarps;
    const dim3 grid((unsigned)((K + width - 1) / width), grid_of((M + mt::q8::kRows - 1) / mt::q8::kRows, 65535));
    if (vec) mt::q8::quantize_kernel<4><<<grid, 32 * mt::q8::kWarps, 0, st>>>(vx.m, o, M, K);
    else mt::q8::quantize_kernel<1><<<grid, 32 * mt::q8::kWarps, 0, st>>>(vx.m, o, M, K);
    MT_TRY(launched("quantize_q8 launch"));
    mt::host::set_path(vec ? "quantize_q8 vec=4" : "quantize_q8 vec=1");
    return MT_OK;
}

MT_API int mt_dequantize_q8(const mt_q8* q, void* out, int type, uint64_t pitch, void* stream) {
    const char* who = "dequantize_q8";
    Q8 o;
    int64_t M, K;
    MT_TRY(to_q8(q, who, o, M, K));
    if (type != MT_F32 && type != MT_BF16) return fail(MT_EINVAL, "%s: bad output type %d", who, type);
    if (M * K == 0) return MT_OK;
    if (!out) return fail(MT_EINVAL, "%s: null output", who);
    const int es = type == MT_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % es) return fail(MT_EINVAL, "%s: misaligned output", who);
    if ((M > 1 && pitch < (uint64_t)K) || pitch > (1ull << 40)) return fail(MT_EINVAL, "%s: the output's pitch is smaller than a row or out of range", who);
    const Span so = span_of_rows(out, M, (int64_t)pitch * es, K * es);
    MT_TRY(check_apart(so, "the output", code_span(o, M, K), "the codes", who));
    MT_TRY(check_apart(so, "the output", scale_span(o, M, K), "the scales", who));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto al16 = [](const void* p, int64_t pitch_bytes, int64_t rows) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || pitch_bytes % 16 == 0);
    };
    const bool vec = K % 16 == 0 && al16(o.codes, o.cp, M) && al16(out, (int64_t)pitch * es, M);
    const int64_t width = vec ? 256 * 16 : mt::q8::kDequantWidth;
    const dim3 grid((unsigned)((K + width - 1) / width), grid_of(M, 65535));
    if (type == MT_F32) {
        float* f = static_cast<float*>(out);
        if (vec) mt::q8::dequantize_kernel<float, 16><<<grid, 256, 0, st>>>(o, f, (int64_t)pitch, M, K);
        else mt::q8::dequantize_kernel<float, 1><<<grid, 256, 0, st>>>(o, f, (int64_t)pitch, M, K);
    } else {
        __nv_bfloat16* f = static_cast<__nv_bfloat16*>(out);
        if (vec) mt::q8::dequantize_kernel<__nv_bfloat16, 16><<<grid, 256, 0, st>>>(o, f, (int64_t)pitch, M, K);
        else mt::q8::dequantize_kernel<__nv_bfloat16, 1><<<grid, 256, 0, st>>>(o, f, (int64_t)pitch, M, K);
    }
    MT_TRY(launched("dequantize_q8 launch"));
    mt::host::set_path(vec ? "dequantize_q8 vec=16" : "dequantize_q8 vec=1");
    return MT_OK;
}

MT_API int mt_linear_wgrad_q8(const mt_q8* x, const mt_tensor* dY, const mt_tensor* dW, const mt_tensor* db,
                              void* stream) {
    const char* who = "linear_wgrad_q8";
    Q8 q;
    int64_t M, K;
    View2 vdy, vdw, vdb;
    MT_TRY(to_q8(x, who, q, M, K));
    MT_TRY(to_mat(dY, who, "dY", vdy));
    MT_TRY(to_mat(dW, who, "dW", vdw));
    const int64_t N = vdy.cols;
    if (vdy.rows != M)
        return fail(MT_EINVAL, "%s: dY has %lld rows, the 8-bit input %lld", who, (long long)vdy.rows, (long long)M);
    if (vdw.rows != K || vdw.cols != N)
        return fail(MT_EINVAL, "%s: dW must be [%lld, %lld]", who, (long long)K, (long long)N);
    if (db) MT_TRY(to_vec(db, N, who, "db", vdb));
    MT_TRY(check_distinct(vdw, who, "dW"));
    MT_TRY(check_distinct(vdb, who, "db"));
    for (const View2* o : {&vdw, &vdb}) {
        MT_TRY(check_apart(span_of(*o), "an output", span_of(vdy), "dY", who));
        MT_TRY(check_apart(span_of(*o), "an output", code_span(q, M, K), "the codes", who));
        MT_TRY(check_apart(span_of(*o), "an output", scale_span(q, M, K), "the scales", who));
    }
    MT_TRY(check_apart(span_of(vdw), "dW", span_of(vdb), "db", who));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (N == 0) return MT_OK;
    return wgrad_planes(q, vdy.m, vdw.m, vdb.m, M, K, N, st, who);
}

MT_API int mt_quantize_q4(const mt_tensor* W, const mt_q4* q, void* stream) {
    const char* who = "quantize_q4";
    View2 vw;
    mt::q4::Weight o;
    MT_TRY(to_mat(W, who, "W", vw));
    MT_TRY(to_q4(q, who, o));
    if (vw.rows != o.K || vw.cols != o.N) return fail(MT_EINVAL, "%s: W must be [%lld, %lld]", who, (long long)o.K, (long long)o.N);
    MT_TRY(check_apart(q4_code_span(o), "the codes", span_of(vw), "W", who));
    MT_TRY(check_apart(q4_scale_span(o), "the scales", span_of(vw), "W", who));
    MT_TRY(check_apart(q4_code_span(o), "the codes", q4_scale_span(o), "the scales", who));
    if (o.K * o.N == 0) return MT_OK;
    const int64_t spans = (o.K + mt::q4::kSpan - 1) / mt::q4::kSpan;
    mt::q4::quantize_kernel<<<dim3((unsigned)((o.N + 127) / 128), grid_of(spans, 65535)), 128, 0,
                              static_cast<cudaStream_t>(stream)>>>(vw.m, o, spans);
    MT_TRY(launched("quantize_q4 launch"));
    mt::host::set_path("quantize_q4");
    return MT_OK;
}

MT_API int mt_dequantize_q4(const mt_q4* q, const mt_tensor* W, void* stream) {
    const char* who = "dequantize_q4";
    View2 vw;
    mt::q4::Weight o;
    MT_TRY(to_q4(q, who, o));
    MT_TRY(to_mat(W, who, "W", vw));
    if (vw.rows != o.K || vw.cols != o.N) return fail(MT_EINVAL, "%s: W must be [%lld, %lld]", who, (long long)o.K, (long long)o.N);
    MT_TRY(check_distinct(vw, who, "W"));
    MT_TRY(check_apart(span_of(vw), "W", q4_code_span(o), "the codes", who));
    MT_TRY(check_apart(span_of(vw), "W", q4_scale_span(o), "the scales", who));
    if (o.K * o.N == 0) return MT_OK;
    mt::q4::dequantize_kernel<<<dim3((unsigned)((o.N + 127) / 128), grid_of((o.K + 7) / 8, 65535)), 128, 0,
                                static_cast<cudaStream_t>(stream)>>>(o, vw.m);
    MT_TRY(launched("dequantize_q4 launch"));
    mt::host::set_path("dequantize_q4");
    return MT_OK;
}

MT_API int mt_linear_fwd_q4(const mt_tensor* X, const mt_q4* W, const mt_tensor* bias, const mt_tensor* Y, int relu,
                            void* stream) {
    const char* who = "linear_fwd_q4";
    View2 vx, vb, vy;
    mt::q4::Weight w;
    MT_TRY(to_mat(X, who, "X", vx));
    MT_TRY(to_q4(W, who, w));
    MT_TRY(to_mat(Y, who, "Y", vy));
    if (vx.cols != w.K)
        return fail(MT_EINVAL, "%s: x features (%lld) != weight in (%lld)", who, (long long)vx.cols, (long long)w.K);
    if (vy.rows != vx.rows || vy.cols != w.N) return fail(MT_EINVAL, "%s: Y shape mismatch", who);
    if (bias) {
        MT_TRY(to_vec(bias, w.N, who, "bias", vb));
        if (w.N > 1 && vb.m.cs != 1) return fail(MT_EINVAL, "%s: bias must be contiguous", who);
    }
    MT_TRY(check_distinct(vy, who, "Y"));
    const Span in[] = {span_of(vx), span_of(vb), q4_code_span(w), q4_scale_span(w)};
    const char* names[] = {"X", "bias", "the codes", "the scales"};
    for (int i = 0; i < 4; ++i) MT_TRY(check_apart(span_of(vy), "Y", in[i], names[i], who));
    const int64_t M = vx.rows;
    if (M * w.N == 0) return MT_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Few rows in integers, batches with the weights in tensor memory, prompts as a product of
    // unpacked operands. Microseconds, either side: 192 rows on weights of 4096 x 16384 (group 64) 96
    // and 109, 256 rows 138 and 109; 4 rows there 27 and 31, 5 rows 35 and 31. 5 to 8 rows take the
    // weights twice, which on small ones costs less than a batch's further launches: 8 rows in a row of
    // calls on 4096 x 4096 16.5 and 18.4, on 4096 x 6000 17.0 and 18.2, on 4096 x 11008 24.7 and 21.2.
    // In two launches: 1 row on 20000 x 16384 63 and 86, 2 rows on 16384 x 4096 36 and 31, but 56 and
    // 101 on 12000 x 16384 in groups of 32, which cost a batch twice the drains. In three: 1 row on
    // 30000 x 4096 58 and 45.
    if (M > 192 && w.K > 0) {
        switch (w.group) {   // k16-steps per group
            case 32: return linear_q4_planes<2>(vx, w, vb.m.p, vy.m, M, relu, st, who);
            case 64: return linear_q4_planes<4>(vx, w, vb.m.p, vy.m, M, relu, st, who);
            default: return linear_q4_planes<8>(vx, w, vb.m.p, vy.m, M, relu, st, who);
        }
    }
    const int64_t few = w.K * w.N <= 24 << 20 ? 2 * mt::q4::kGemvMaxRows : mt::q4::kGemvMaxRows;
    const int64_t spans = (w.K + mt::q4::kSpan - 1) / mt::q4::kSpan;
    if (w.K > 0 && (M > few || plan_gemv(M, spans).launches > (M == 1 || w.group == 32 ? 2 : 1)))
        return linear_q4_batch(vx, w, vb.m.p, vy.m, M, relu, st, who);
    return linear_q4_gemv(vx, w, vb.m.p, vy.m, M, relu, st, who);
}

}  // extern "C"

namespace mt {
namespace host {

int lowbit_device_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_dev_status, sizeof(int)) != cudaSuccess) return -MT_ECUDA;
    if (reset) {
        const int z = 0;
        cudaMemcpyToSymbol(g_dev_status, &z, sizeof(int));
    }
    return v;
}

}  // namespace host
}  // namespace mt
