"""The low-bit operators on the GPU against their plain 64-bit forms (tests/lowbit_ref.py)."""
import pytest
import torch

import lowbit_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mt(eng):
    import minitensor_b200
    return minitensor_b200


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g) * scale


def host(t):
    return t.detach().cpu()


def strided(t, how):
    """The same values on the GPU in another layout."""
    rows, cols = t.shape
    if how == "dense":
        return t.cuda()
    if how == "transposed":
        return t.t().contiguous().cuda().t()
    if how == "window":        # a column window of a wider buffer, off the 16-byte grid
        base = torch.full((rows, cols + 7), float("nan"), device="cuda")
        base[:, 3:3 + cols] = t.cuda()
        return base[:, 3:3 + cols]
    if how == "every second":
        base = torch.full((2 * rows, 2 * cols), float("nan"), device="cuda")
        base[::2, ::2] = t.cuda()
        return base[::2, ::2]
    if how == "pitched":       # 16-byte rows with a pitch
        base = torch.full((rows, cols + 8), float("nan"), device="cuda")
        base[:, :cols] = t.cuda()
        return base[:, :cols]
    raise AssertionError(how)


LAYOUTS = ["dense", "transposed", "window", "every second", "pitched"]

# ---- RMS norm ---------------------------------------------------------------------------
# y = h * rstd * gamma. With s terms per lane and ten shuffle or shared-memory levels, the sum
# of squares is off by at most (s + 10) u, half of which reaches rstd; squares, the division by
# K, the addition of eps, the square root, the division and two products add at most 6 u, and
# h's own rounding, where a residual is added, u of itself and u of the row's root mean
# square. s <= 32 in registers, K / 1024 in rows longer than that.

def norm_bound(K):
    return 0.5 * (max(32, K / 1024) + 10) + 10


SHAPES = [(1, 1), (1, 4096), (3, 5), (5, 32), (2, 33), (7, 100), (9, 128), (300, 127), (4, 512), (130, 516), (3, 1000),
          (3, 1024), (2, 1025), (5, 4100), (320, 1028), (2, 4097), (2, 8191), (3, 16384), (2, 20000), (1, 32768), (2, 8193),
          (320, 12289), (2, 16383), (2, 16385), (2, 40004), (1, 70001)]


@pytest.mark.parametrize("rows,K", SHAPES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_rms_norm(mt, rows, K, with_residual):
    g = gen(rows * 100003 + K)
    x, gamma = rand(g, rows, K), 1 + rand(g, K, scale=0.1)
    r = rand(g, rows, K, scale=3.0) if with_residual else None
    out = mt.rms_norm(x.cuda(), gamma.cuda(), residual=r.cuda() if with_residual else None, eps=1e-6)
    h, rstd, y = R.rms_norm(x, r, gamma, 1e-6)
    if with_residual:
        assert torch.equal(host(out.h), x + r)
    assert out.q8 is None
    b = norm_bound(K)
    assert R.worst(host(out.rstd) - rstd, rstd) <= b
    # the rounding of h is relative to h itself
    assert R.worst(host(out.y) - y, y) <= b + 1


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("rows,K", [(6, 96), (5, 1028), (3, 130)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_rms_norm_layouts(mt, layout, rows, K, fmt):
    g = gen(K)
    x, r, gamma = rand(g, rows, K), rand(g, rows, K), 1 + rand(g, K, scale=0.1)
    dense = mt.rms_norm(x.cuda(), gamma.cuda(), residual=r.cuda(), q8=fmt)
    out = mt.rms_norm(strided(x, layout), gamma.cuda(), residual=strided(r, layout), q8=fmt)
    h, rstd, y = R.rms_norm(x, r, gamma, 1e-6)
    assert R.worst(host(out.y) - y, y) <= norm_bound(K) + 1
    assert torch.equal(out.h, dense.h)
    # the 8-bit output is exactly the 8-bit form of the float output
    q = mt.quantize_q8(out.y, fmt)
    assert torch.equal(q.codes.view(torch.uint8), out.q8.codes.view(torch.uint8))
    assert torch.equal(q.scales, out.q8.scales)


@pytest.mark.parametrize("K", [64, 100, 4096, 40004])
def test_rms_norm_in_place_and_8_bit_output_alone(mt, K):
    g = gen(K)
    x, r, gamma = rand(g, 5, K), rand(g, 5, K), 1 + rand(g, K, scale=0.1)
    ref = mt.rms_norm(x.cuda(), gamma.cuda(), residual=r.cuda(), q8="int8")
    xd = x.cuda()
    out = mt.rms_norm(xd, gamma.cuda(), residual=r.cuda(), q8="int8", want_y=False, inplace=True)
    assert out.y is None and out.h is xd
    assert torch.equal(xd, ref.h) and torch.equal(out.q8.codes, ref.q8.codes) and torch.equal(out.rstd, ref.rstd)


def test_rms_norm_special_rows(mt):
    K = 200
    x = torch.ones(5, K)
    x[0] = 0                      # all zeros: eps alone
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3] = 1e-30                  # squares underflow: eps alone
    gamma = torch.ones(K)
    out = mt.rms_norm(x.cuda(), gamma.cuda(), eps=1e-6, q8="int8")
    y = host(out.y)
    assert torch.equal(y[0], torch.zeros(K))
    assert torch.isnan(y[1]).all()
    assert torch.isnan(y[2, 9]) and torch.equal(y[2, :9], torch.zeros(9))
    assert R.worst(y[3] - 1e-27, torch.full((K,), 1e-27)) <= 40
    assert R.worst(y[4] - 1 / (1 + 1e-6) ** 0.5, torch.ones(K)) <= norm_bound(K)
    v = host(mt.dequantize_q8(out.q8))
    assert torch.isnan(v[1]).all() and torch.isnan(v[2, :32]).all() and not torch.isnan(v[2, 32:]).any()
    assert torch.equal(v[0], torch.zeros(K))


def test_rms_norm_empty_and_strided_gamma(mt):
    out = mt.rms_norm(torch.empty(0, 8, device="cuda"), torch.ones(8, device="cuda"), q8="int8")
    assert out.y.shape == (0, 8) and out.q8.codes.shape == (0, 8)
    g = gen(3)
    x, gamma = rand(g, 4, 36), rand(g, 36)
    wide = torch.zeros(36, 2, device="cuda")
    wide[:, 1] = gamma.cuda()
    a = mt.rms_norm(x.cuda(), wide[:, 1]).y
    assert torch.allclose(a, mt.rms_norm(x.cuda(), gamma.cuda()).y, rtol=1e-5, atol=0)


# dx is off, relative to its terms' magnitudes, by the sum over the row (as above) and at
# most 8 roundings; dgamma by the sum over the rows in any order and 3 roundings.
@pytest.mark.parametrize("rows,K", SHAPES + [(2000, 64), (1200, 260)])
@pytest.mark.parametrize("with_dh", [False, True])
def test_rms_norm_backward(mt, rows, K, with_dh):
    g = gen(rows * 7 + K)
    h, gamma, dy = rand(g, rows, K, scale=2.0), 1 + rand(g, K, scale=0.1), rand(g, rows, K)
    dh = rand(g, rows, K) if with_dh else None
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(1) + 1e-6)).float()
    dx, dgamma = mt.rms_norm_backward(dy.cuda(), h.cuda(), gamma.cuda(), rstd.cuda(), dh=dh.cuda() if with_dh else None)
    want, mag, want_g, mag_g = R.rms_norm_backward(dy, h, gamma, rstd, dh)
    assert R.worst(host(dx) - want, mag) <= max(32, K / 1024) + 10 + 8
    assert R.worst(host(dgamma) - want_g, mag_g) <= rows + 3


@pytest.mark.parametrize("layout", LAYOUTS)
def test_rms_norm_backward_layouts(mt, layout):
    g = gen(5)
    h, gamma, dy, dh = rand(g, 9, 132), rand(g, 132), rand(g, 9, 132), rand(g, 9, 132)
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(1) + 1e-6)).float()
    dx, dgamma = mt.rms_norm_backward(strided(dy, layout), strided(h, layout), gamma.cuda(), rstd.cuda(),
                                      dh=strided(dh, layout))
    want, mag, want_g, mag_g = R.rms_norm_backward(dy, h, gamma, rstd, dh)
    assert R.worst(host(dx) - want, mag) <= 50 and R.worst(host(dgamma) - want_g, mag_g) <= 12


def test_rms_norm_gradient_matches_differences(mt):
    # f(x, gamma) = sum(y * c) in 64 bits of the formula; central differences of step 1e-4
    # are off by O(step^2) ~ 1e-8 of f's third derivatives and 1e-12 of f by rounding.
    g = gen(11)
    x, gamma, c = rand(g, 3, 20).double(), (1 + rand(g, 20, scale=0.1)).double(), rand(g, 3, 20).double()

    def f(x, gamma):
        return (R.rms_norm(x, None, gamma, 1e-6)[2] * c).sum()

    rstd = R.rms_norm(x, None, gamma, 1e-6)[1].float()
    dx, dgamma = mt.rms_norm_backward(c.float().cuda(), x.float().cuda(), gamma.float().cuda(), rstd.cuda())
    e = 1e-4
    for i, j in ((0, 0), (1, 7), (2, 19)):
        d = torch.zeros_like(x)
        d[i, j] = e
        assert abs(float((f(x + d, gamma) - f(x - d, gamma)) / (2 * e)) - float(dx[i, j])) < 1e-5
    d = torch.zeros_like(gamma)
    d[4] = e
    assert abs(float((f(x, gamma + d) - f(x, gamma - d)) / (2 * e)) - float(dgamma[4])) < 1e-5


def test_rms_norm_backward_empty(mt):
    dx, dg = mt.rms_norm_backward(torch.empty(0, 8, device="cuda"), torch.empty(0, 8, device="cuda"),
                                  torch.ones(8, device="cuda"), torch.empty(0, device="cuda"))
    assert dx.shape == (0, 8) and torch.equal(host(dg), torch.zeros(8))


# ---- 8 bits -----------------------------------------------------------------------------

def q8_input(g, rows, cols):
    """Magnitudes from 2^-140 to 2^120, block by block, zeros and exact powers of two among
    them, and values next to a scale's border."""
    x = rand(g, rows, cols)
    e = torch.randint(-140, 120, (rows, -(-cols // 32)), generator=g).repeat_interleave(32, 1)[:, :cols]
    x = torch.ldexp(x, e)
    x[:, ::37] = 0
    if rows > 2 and cols >= 32:
        x[0, :32] = 0
        x[1, :32] = torch.linspace(-127, 127, 32)
        x[2, :32] = torch.nextafter(torch.tensor(127.0), torch.tensor(200.0))
    return x


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (4, 33), (6, 128), (3, 1000), (9, 1024), (2, 4099), (7, 160)])
@pytest.mark.parametrize("layout", ["dense", "transposed", "window", "pitched"])
def test_quantize_q8_is_exact(mt, fmt, rows, cols, layout):
    x = q8_input(gen(rows + cols), rows, cols)
    q = mt.quantize_q8(strided(x, layout), fmt)
    b = R.q8_scale_bytes(x, fmt)
    assert torch.equal(host(q.scales).long(), b)
    assert torch.equal(host(q.codes).view(torch.uint8) & 0x7F if fmt == "e4m3" else host(q.codes),
                       R.q8_codes(x, b, fmt).view(torch.uint8) & 0x7F if fmt == "e4m3" else R.q8_codes(x, b, fmt))
    v = R.q8_values(host(q.codes).float(), host(q.scales))
    assert torch.equal(host(mt.dequantize_q8(q)).double(), v)
    assert torch.equal(host(mt.dequantize_q8(q, dtype=torch.bfloat16)), v.float().to(torch.bfloat16))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_quantize_q8_non_finite_blocks(mt, fmt):
    x = torch.ones(3, 100)
    x[0, 40] = float("inf")
    x[1, 99] = float("nan")
    q = mt.quantize_q8(x.cuda(), fmt)
    v = host(mt.dequantize_q8(q))
    bad = torch.zeros(3, 100, dtype=torch.bool)
    bad[0, 32:64] = True
    bad[1, 96:] = True
    assert torch.equal(torch.isnan(v), bad) and torch.equal(v[~bad], x[~bad])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_dequantize_q8_of_a_pitched_view(mt, fmt):
    x = q8_input(gen(1), 6, 96)
    q = mt.quantize_q8(x.cuda(), fmt)
    wide = torch.zeros(6, 130, dtype=torch.int8, device="cuda")
    wide[:, 1:97] = q.codes.view(torch.int8)
    view = mt.Q8Tensor(wide[:, 1:97].view(q.codes.dtype), q.scales)
    assert torch.equal(mt.dequantize_q8(view), mt.dequantize_q8(q))


WGRAD_SHAPES = [(1, 1, 1), (2, 3, 5), (16, 64, 64), (17, 65, 63), (100, 130, 257), (128, 128, 128), (129, 256, 300),
                (300, 33, 700), (1000, 520, 136), (64, 600, 1100)]


def wgrad_input(g, M, K, N, fmt, mt):
    q = mt.quantize_q8(rand(g, M, K).cuda(), fmt)
    return q, rand(g, M, N) * torch.exp(rand(g, M, 1))


def check_wgrad(q, dy, dW, db):
    xv = R.q8_values(host(q.codes).float(), host(q.scales))
    M = dy.shape[0]
    want, mag = xv.t() @ dy.double(), xv.abs().t() @ dy.double().abs()
    assert R.worst(host(dW) - want, mag) <= M + 8
    assert R.worst(host(db) - dy.double().sum(0, keepdim=True), dy.double().abs().sum(0, keepdim=True)) <= M


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("M,K,N", WGRAD_SHAPES)
def test_linear_weight_grad_q8(mt, fmt, M, K, N):
    q, dy = wgrad_input(gen(M * K + N), M, K, N, fmt, mt)
    dW, db = mt.linear_weight_grad_q8(q, dy.cuda())
    check_wgrad(q, dy, dW, db)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_linear_weight_grad_q8_layouts(mt, layout):
    q, dy = wgrad_input(gen(2), 70, 96, 132, "int8", mt)
    check_wgrad(q, dy, *mt.linear_weight_grad_q8(q, strided(dy, layout)))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_linear_weight_grad_q8_keeps_every_bit(mt, fmt):
    """One row: dW[k][n] = xhat[k] * dy[n] needs one rounding, so it is the float product."""
    g = gen(4)
    x = rand(g, 1, 96)
    dy = rand(g, 1, 200) * torch.exp(5 * rand(g, 1, 200))
    q = mt.quantize_q8(x.cuda(), fmt)
    dW, db = mt.linear_weight_grad_q8(q, dy.cuda())
    want = host(mt.dequantize_q8(q)).double().t() @ dy.double()
    assert R.worst(host(dW) - want, want) <= 3     # three exact parts, added in float
    assert torch.equal(host(db), dy)


def test_linear_weight_grad_q8_split_over_the_rows(mt):
    """One tile of dW from many rows, whose sum is cut into parts."""
    q, dy = wgrad_input(gen(9), 5000, 40, 70, "int8", mt)
    got = mt.linear_weight_grad_q8(q, dy.cuda())
    assert "splits=1" not in mt.engine.last_path()
    check_wgrad(q, dy, *got)


def test_linear_weight_grad_q8_small_gradients(mt):
    """Gradients down to 2^-125: the third part of the smallest is off by at most 2^-133, which x,
    a power of two here, carries into dW."""
    g = gen(10)
    x = torch.ones(1, 64)
    dy = torch.ldexp(torch.rand(1, 130, generator=g) + 1, torch.randint(-125, -90, (1, 130), generator=g))
    dW, db = mt.linear_weight_grad_q8(mt.quantize_q8(x.cuda()), dy.cuda())
    err = (host(dW).double() - dy.double()).abs()
    assert (err <= 2.0 ** -133 + 3 * R.U * dy.double()).all()
    assert torch.equal(host(db), dy)


def test_linear_weight_grad_q8_empty(mt):
    q = mt.quantize_q8(torch.empty(0, 64, device="cuda"))
    dW, db = mt.linear_weight_grad_q8(q, torch.empty(0, 40, device="cuda"))
    assert torch.equal(host(dW), torch.zeros(64, 40)) and torch.equal(host(db), torch.zeros(1, 40))


def test_linear_weight_grad_q8_non_finite(mt):
    """A NaN block of the checkpoint reaches its 32 rows of dW, an infinite gradient its column,
    and nothing else."""
    x, dy = torch.ones(40, 96), torch.ones(40, 70)
    x[3, 40] = float("nan")
    dy[5, 9] = float("inf")
    dy[6, 11] = float("nan")
    dW, db = mt.linear_weight_grad_q8(mt.quantize_q8(x.cuda()), dy.cuda())
    dW, db = host(dW), host(db)
    assert torch.isnan(dW[32:64]).all()
    rest = torch.cat([dW[:32], dW[64:]])
    assert torch.isinf(rest[:, 9]).all() and torch.isnan(rest[:, 11]).all()
    keep = [n for n in range(70) if n not in (9, 11)]
    assert torch.equal(rest[:, keep], torch.full((64, 68), 40.0))
    assert torch.isinf(db[0, 9]) and torch.isnan(db[0, 11]) and torch.equal(db[0, keep], torch.full((68,), 40.0))


def test_training_step_through_a_checkpoint(mt):
    """norm -> Linear -> its backward -> the norm's, as a training step calls them."""
    g = gen(8)
    M, K, N = 96, 256, 160
    x, r, gamma = rand(g, M, K).cuda(), rand(g, M, K).cuda(), (1 + rand(g, K, scale=0.1)).cuda()
    W, b, dY, dh = rand(g, K, N, scale=0.1).cuda(), rand(g, 1, N).cuda(), rand(g, M, N).cuda(), rand(g, M, K).cuda()
    n = mt.rms_norm(x, gamma, residual=r, q8="int8")
    Y, saved = mt.linear_forward_q8(n.y, W, b)
    assert torch.equal(saved.codes, n.q8.codes) and torch.equal(saved.scales, n.q8.scales)
    assert torch.equal(Y, mt.linear_forward(n.y, W, b))
    dX, dW, db = mt.linear_backward_q8(saved, W, dY)
    check_wgrad(saved, host(dY), dW, db)
    eX, _, eb = mt.linear_backward(n.y, W, dY)
    assert torch.equal(dX, eX)
    dx, dgamma = mt.rms_norm_backward(dX, n.h, gamma, n.rstd, dh=dh)
    want, mag, want_g, mag_g = R.rms_norm_backward(host(dX), host(n.h), host(gamma), host(n.rstd), host(dh))
    assert R.worst(host(dx) - want, mag) <= 50 and R.worst(host(dgamma) - want_g, mag_g) <= M + 3


# ---- 4 bits -----------------------------------------------------------------------------

Q4_SHAPES = [(1, 1), (5, 3), (64, 16), (127, 40), (128, 64), (129, 17), (300, 130), (1000, 33), (1024, 256)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N", Q4_SHAPES)
def test_quantize_q4_is_exact(mt, group, K, N):
    W = rand(gen(K + N), K, N)
    W[:, N // 2] = 0
    q = mt.quantize_q4(W.cuda(), group)
    codes, s = R.q4_quantize(W, group)
    assert torch.equal(host(q.scales), s)
    assert torch.equal(host(q.codes), R.q4_pack(codes, K))
    assert torch.equal(host(mt.dequantize_q4(q)).double(), R.q4_weight(codes, s, group))
    qt = mt.quantize_q4(W.t().contiguous().cuda().t(), group)
    assert torch.equal(qt.codes, q.codes) and torch.equal(qt.scales, q.scales)


# Sizes that are cut in every way: tiles of 128 or 256 columns, at once, in parts, or the last
# round in parts.
@pytest.mark.parametrize("M,K,N,cut", [(130, 260, 200, "bn=128 whole=4 splits=1"), (1100, 70, 90, "bn=128 whole=0 splits=9"),
                                       (300, 5000, 4100, "bn=256 whole=340 splits=1"), (700, 2100, 2300, "bn=256 whole=74 splits=6")])
def test_linear_weight_grad_q8_cuts(mt, M, K, N, cut):
    q, dy = wgrad_input(gen(M + K + N), M, K, N, "int8", mt)
    got = mt.linear_weight_grad_q8(q, dy.cuda())
    assert mt.engine.last_path().endswith(cut)
    check_wgrad(q, dy, *got)


def q4_case(g, M, K, N, group):
    codes = torch.randint(0, 16, (N, K), generator=g)
    s = (0.01 * torch.exp(rand(g, N, -(-K // group)))).to(torch.bfloat16)
    x = rand(g, M, K) * torch.exp(rand(g, 1, K))
    return x, codes, s


def check_q4(y, x, codes, s, group, bias, relu):
    """Many rows: y is the sum over groups of s * sum (c - 8) x; a tensor-core step aligns 17
    terms to the largest and may drop 2 u of it from each (34 u), 24 steps meet in one
    accumulator at 2 u each, the groups are added as a float sum of at most K terms, and the
    scale's product and the bias add 2 u. Few rows: the products and sums are exact integers
    after x is rounded to 2^-30 of the largest of its span of 128 (2^-6 u); two conversions, two
    products and the bias add 5 u, the spans a float sum. Either way fewer than K + 90."""
    K = x.shape[1]
    W = R.q4_weight(codes, s, group)
    full = s.double().repeat_interleave(group, 1)[:, :K].t()
    spans = torch.nn.functional.pad(x.double().abs(), (0, -K % 128)).view(x.shape[0], -1, 128)
    top = spans.amax(2, keepdim=True).expand_as(spans).reshape(x.shape[0], -1)[:, :K]
    want, mag = x.double() @ W, x.double().abs() @ (W.abs() + 8 * full) + 2.0 ** -6 * (top @ W.abs())
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    err = host(y).double() - (want.clamp_min(0) if relu else want)
    assert R.worst(err, mag) <= K + 90


Q4_ROWS = [1, 2, 3, 5, 8, 9, 16, 21, 40, 130, 300]


@pytest.mark.parametrize("M", Q4_ROWS)
@pytest.mark.parametrize("K,N,group", [(1, 1, 32), (31, 5, 32), (128, 16, 64), (300, 130, 32), (1000, 77, 128),
                                       (2048, 264, 64), (1111, 401, 128)])
def test_linear_forward_q4(mt, M, K, N, group):
    g = gen(M * 1000003 + K * 1009 + N)
    x, codes, s = q4_case(g, M, K, N, group)
    bias = rand(g, N) if N % 2 else None
    relu = M % 2 == 0
    w = mt.Q4Weight(R.q4_pack(codes, K).cuda(), s.cuda(), K, group)
    y = mt.linear_forward_q4(x.cuda(), w, bias=bias.cuda() if bias is not None else None, relu=relu)
    check_q4(y, x, codes, s, group, bias, relu)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N,cut", [(200, 300, 300, "bn=128 whole=4 splits=1"), (500, 1300, 4800, "bn=128 whole=74 splits=11"),
                                       (1030, 700, 2600, "bn=256 whole=55 splits=1"), (200, 4000, 4097, "bn=256 whole=0 splits=4")])
def test_linear_forward_q4_cuts(mt, M, K, N, cut, group):
    g = gen(M + K + N + group)
    x, codes, s = q4_case(g, M, K, N, group)
    bias = rand(g, N)
    w = mt.Q4Weight(R.q4_pack(codes, K).cuda(), s.cuda(), K, group)
    y = mt.linear_forward_q4(x.cuda(), w, bias=bias.cuda(), relu=True)
    assert mt.engine.last_path().endswith(cut)
    check_q4(y, x, codes, s, group, bias, True)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("M", [1, 4, 50])
def test_linear_forward_q4_layouts(mt, layout, M):
    g = gen(M)
    x, codes, s = q4_case(g, M, 260, 50, 64)
    w = mt.Q4Weight(R.q4_pack(codes, 260).cuda(), s.cuda(), 260, 64)
    check_q4(mt.linear_forward_q4(strided(x, layout), w), x, codes, s, 64, None, False)


@pytest.mark.parametrize("M", Q4_ROWS)
@pytest.mark.parametrize("offset", [0, 37, 150])
def test_linear_forward_q4_finds_every_position(mt, M, offset):
    """Rows of x with a single value: y is s * (c - 8) * x. x's parts and digits are exact; at most
    three products and sums round, the tensor core's by truncation (2 u). A lost part of x
    (2^-8 or 2^-16 of it) is far off."""
    K, N, group = 288, 80, 32
    g = gen(M)
    at = (torch.arange(M) * 11 + offset) % K
    x = torch.zeros(M, K)
    x[torch.arange(M), at] = rand(g, M) * torch.exp(5 * rand(g, M))
    codes = torch.randint(0, 16, (N, K), generator=g)
    s = torch.exp(rand(g, N, K // group)).to(torch.bfloat16)
    w = mt.Q4Weight(R.q4_pack(codes, K).cuda(), s.cuda(), K, group)
    want = x.double() @ R.q4_weight(codes, s, group)
    assert R.worst(host(mt.linear_forward_q4(x.cuda(), w)) - want, want) <= 7


def test_linear_forward_q4_range_of_x(mt):
    """Blocks of x from 2^-120 to 2^125 in one call."""
    K, N = 512, 48
    g = gen(5)
    for M in (1, 6, 20, 200):
        for top in (125, 100):
            x, codes, s = q4_case(g, M, K, N, 64)
            e = torch.randint(-120, top, (M, K // 32), generator=g).repeat_interleave(32, 1)
            x = torch.ldexp(torch.rand(M, K, generator=g) + 0.5, e)
            x[0, :32] = 1.5 * 2.0 ** top
            s = (s.float() * 1e-6).to(torch.bfloat16)
            w = mt.Q4Weight(R.q4_pack(codes, K).cuda(), s.cuda(), K, 64)
            check_q4(mt.linear_forward_q4(x.cuda(), w), x, codes, s, 64, None, False)


@pytest.mark.parametrize("M,K", [(16, 12800), (5, 24000), (1, 60000)])
def test_linear_forward_q4_long_rows(mt, M, K):
    """Rows of x that do not fit shared memory at once."""
    g = gen(K)
    x, codes, s = q4_case(g, M, K, 33, 128)
    w = mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, 128)
    bias = rand(g, 33)
    check_q4(mt.linear_forward_q4(x.cuda(), w, bias=bias.cuda(), relu=True), x, codes, s, 128, bias, True)


def pack_fast(codes, K):
    """R.q4_pack for long rows: spans of 128 codes are packed alike."""
    N = codes.shape[0]
    spans = -(-K // 128)
    full = torch.full((N, spans * 128), 8, dtype=torch.int64)
    full[:, :K] = codes
    return R.q4_pack(full.view(N * spans, 128), 128).view(N, spans * 64)


def test_linear_forward_q4_non_finite(mt):
    """A NaN or an infinity in one row of x stays in that row; a NaN scale in its column."""
    K, N = 256, 48
    codes = torch.full((N, K), 9, dtype=torch.int64)
    s = torch.ones(N, 4, dtype=torch.bfloat16)
    s[7, 2] = float("nan")
    for M in (3, 40, 200):
        x = torch.ones(M, K)
        x[0, 5], x[1, 200] = float("nan"), float("inf")
        w = mt.Q4Weight(R.q4_pack(codes, K).cuda(), s.cuda(), K, 64)
        y = host(mt.linear_forward_q4(x.cuda(), w))
        assert torch.isnan(y[0]).all() and torch.isnan(y[:, 7]).all()
        keep = [n for n in range(N) if n != 7]
        assert torch.equal(y[1, keep], torch.full((N - 1,), float("inf")))
        assert torch.equal(y[2:, keep], torch.full((M - 2, N - 1), 256.0))


def test_linear_forward_q4_empty(mt):
    w = mt.quantize_q4(torch.randn(64, 32).cuda())
    assert mt.linear_forward_q4(torch.empty(0, 64, device="cuda"), w).shape == (0, 32)
    none = mt.quantize_q4(torch.empty(0, 32, device="cuda"))
    bias = torch.randn(32, device="cuda")
    y = mt.linear_forward_q4(torch.empty(3, 0, device="cuda"), none, bias=bias)
    assert torch.equal(y, bias.expand(3, 32))


def test_decoding_step(mt):
    """norm -> 4-bit Linear -> residual -> norm, as one decoded token goes through."""
    g = gen(21)
    K, N = 256, 256
    x, r, gamma, W = rand(g, 1, K), rand(g, 1, K), 1 + rand(g, K, scale=0.1), rand(g, K, N, scale=0.06)
    w = mt.quantize_q4(W.cuda(), 64)
    n = mt.rms_norm(x.cuda(), gamma.cuda(), residual=r.cuda())
    y = mt.linear_forward_q4(n.y, w)
    check_q4(y, host(n.y), *R.q4_quantize(W, 64), 64, None, False)
    n2 = mt.rms_norm(y, gamma.cuda(), residual=n.h, inplace=True)
    h, rstd, want = R.rms_norm(host(n2.h), None, gamma, 1e-6)
    assert R.worst(host(n2.y) - want, want) <= norm_bound(K) + 1


# ---- how calls are made: graphs, streams, memory shared on purpose, far offsets ------------

def calls(mt, g):
    """name -> (inputs, call) for every operator; the call reads its inputs afresh."""
    M, K, N = 40, 160, 132
    x, r, dh, dy = (rand(g, M, K).cuda() for _ in range(4))
    gamma = (1 + rand(g, K, scale=0.1)).cuda()
    rstd = torch.rand(M, generator=g).cuda() + 0.5
    dY = rand(g, M, N).cuda()
    W = rand(g, K, N, scale=0.1).cuda()
    q = mt.quantize_q8(x, "int8")
    w = mt.quantize_q4(W, 32)
    wide = rand(g, 300, K).cuda()
    long_q, long_dy = mt.quantize_q8(rand(g, 4096, 96).cuda()), rand(g, 4096, 70).cuda()
    long_x, long_w = rand(g, 260, 8192).cuda(), mt.quantize_q4(rand(g, 8192, 64).cuda(), 64)

    def flat(v):
        if isinstance(v, torch.Tensor):
            return [v]
        if isinstance(v, mt.Q8Tensor):
            return [v.codes.view(torch.uint8), v.scales]
        if isinstance(v, mt.Q4Weight):
            return [v.codes, v.scales.view(torch.int16)]
        return [t for e in v if e is not None for t in flat(e)]

    return {
        "norm": ([x, r, gamma], lambda **k: flat(mt.rms_norm(x, gamma, residual=r, q8="e4m3", **k))),
        "norm backward": ([dy, x, gamma, rstd, dh], lambda **k: flat(mt.rms_norm_backward(dy, x, gamma, rstd, dh=dh, **k))),
        "quantize": ([x], lambda **k: flat(mt.quantize_q8(x, **k))),
        "dequantize": ([q.codes], lambda **k: flat(mt.dequantize_q8(q, dtype=torch.bfloat16, **k))),
        "weight grad": ([q.codes, dY], lambda **k: flat(mt.linear_weight_grad_q8(q, dY, **k))),
        "forward and checkpoint": ([x, W], lambda **k: flat(mt.linear_forward_q8(x, W, **k))),
        "backward": ([q.codes, W, dY], lambda **k: flat(mt.linear_backward_q8(q, W, dY, **k))),
        "quantize 4": ([W], lambda **k: flat(mt.quantize_q4(W, 32, **k))),
        "dequantize 4": ([w.codes], lambda **k: flat(mt.dequantize_q4(w, **k))),
        "4 bits, one row": ([x], lambda **k: flat(mt.linear_forward_q4(x[:1], w, **k))),
        "4 bits, batch": ([x], lambda **k: flat(mt.linear_forward_q4(x, w, **k))),
        "weight grad, split": ([long_q.codes, long_dy], lambda **k: flat(mt.linear_weight_grad_q8(long_q, long_dy, **k))),
        "4 bits, prompt, split": ([long_x], lambda **k: flat(mt.linear_forward_q4(long_x, long_w, **k))),
        "4 bits, prompt": ([wide], lambda **k: flat(mt.linear_forward_q4(wide, w, **k))),
    }


NAMES = ["norm", "norm backward", "quantize", "dequantize", "weight grad", "forward and checkpoint", "backward", "quantize 4",
         "dequantize 4", "4 bits, one row", "4 bits, batch", "4 bits, prompt", "weight grad, split", "4 bits, prompt, split"]


def change(inputs):
    for t in inputs:
        if t.dtype == torch.float32:
            t.mul_(1.5)
        else:
            t.copy_(t.flip(0))


@pytest.mark.parametrize("name", NAMES)
def test_captured_call_reads_its_inputs_at_replay(mt, name):
    inputs, call = calls(mt, gen(1))[name]
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(2):
        change(inputs)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("name", ["norm backward", "weight grad", "weight grad, split", "4 bits, batch", "4 bits, prompt",
                                  "4 bits, prompt, split"])
def test_two_graphs_at_once_have_scratch_of_their_own(mt, name):
    sides = []
    for seed in (2, 3):
        _, call = calls(mt, gen(seed))[name]
        want = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [call() for _ in range(3)]
        sides.append((graph, out, want, torch.cuda.Stream(), call))   # call holds the graph's inputs
    for _ in range(5):
        for graph, _, _, stream, _ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in sides:
        for o in out:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.parametrize("name", NAMES)
def test_stream_argument_and_repeated_calls(mt, name):
    _, call = calls(mt, gen(4))[name]
    want = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    a = call(stream=stream)
    b = call(stream=stream.cuda_stream)
    stream.synchronize()
    for o in (a, b):
        assert all(torch.equal(x, y) for x, y in zip(o, want))
    assert mt.engine.device_status() == 0


def test_norm_gradient_in_place_of_its_inputs(mt):
    """dx over dy, and over dh, through the C entry; a residual without h."""
    import ctypes
    from minitensor_b200 import engine, lowbit
    L = lowbit._lowbit_lib()
    g = gen(6)
    v, b = engine.view, ctypes.byref
    for M, K in ((9, 260), (3, 33), (2, 40004)):
        h, gamma, dy, dh = rand(g, M, K).cuda(), rand(g, K).cuda(), rand(g, M, K).cuda(), rand(g, M, K).cuda()
        rstd = torch.rand(M, generator=g).cuda() + 0.5
        want, want_g = mt.rms_norm_backward(dy, h, gamma, rstd, dh=dh)
        for over in ("dy", "dh"):
            a, c = dy.clone(), dh.clone()
            dx = a if over == "dy" else c
            dgamma = torch.empty(K, device="cuda")
            assert L.mt_rms_norm_backward(b(v(a)), b(v(h)), b(v(gamma)), b(v(rstd)), b(v(c)), b(v(dx)), b(v(dgamma)), None) == 0
            torch.cuda.synchronize()
            assert torch.equal(dx, want) and torch.equal(dgamma, want_g)
        r = rand(g, M, K).cuda()
        y = torch.empty(M, K, device="cuda")
        assert L.mt_rms_norm(b(v(h)), b(v(r)), b(v(gamma)), None, b(v(y)), None, None, 1e-6, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(y, mt.rms_norm(h, gamma, residual=r).y)


def test_broadcast_inputs(mt):
    g = gen(7)
    row = rand(g, 1, 96)
    x = row.cuda().expand(5, 96)
    gamma = torch.tensor([1.25], device="cuda").expand(96)
    out = mt.rms_norm(x, gamma, q8="int8")
    h, rstd, y = R.rms_norm(row.expand(5, 96), None, torch.full((96,), 1.25), 1e-6)
    assert R.worst(host(out.y) - y, y) <= norm_bound(96) + 1
    q = mt.quantize_q8(x)
    assert torch.equal(mt.dequantize_q8(q)[3], mt.dequantize_q8(mt.quantize_q8(row.cuda()))[0])
    dY = torch.tensor([[2.0]], device="cuda").expand(5, 70)
    check_wgrad(q, host(dY).contiguous(), *mt.linear_weight_grad_q8(q, dY))
    W = rand(g, 96, 40)
    w = mt.quantize_q4(W.cuda(), 32)
    codes, s = R.q4_quantize(W, 32)
    check_q4(mt.linear_forward_q4(x, w), row.expand(5, 96), codes, s, 32, None, False)


def test_offsets_beyond_32_bits(mt):
    """Rows 2^30 floats (and codes 2^31 bytes) apart."""
    g = gen(8)
    M, K, N = 3, 256, 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    base = torch.empty((M - 1) * 2 ** 30 + K, device="cuda")
    far = base.as_strided((M, K), (2 ** 30, 1))
    x, dY = rand(g, M, K), rand(g, M, N)
    far.copy_(x.cuda())
    gamma = torch.ones(K, device="cuda")
    near = mt.rms_norm(x.cuda(), gamma, q8="int8")
    got = mt.rms_norm(far, gamma, q8="int8")
    assert torch.equal(got.y, near.y) and torch.equal(got.q8.codes, near.q8.codes)
    rstd = near.rstd
    assert torch.equal(mt.rms_norm_backward(far, far, gamma, rstd)[0], mt.rms_norm_backward(x.cuda(), x.cuda(), gamma, rstd)[0])
    w = mt.quantize_q4(rand(g, K, N).cuda(), 64)
    for rows in (1, 3):
        assert torch.equal(mt.linear_forward_q4(far[3 - rows:], w), mt.linear_forward_q4(x[3 - rows:].cuda(), w))
    q = mt.quantize_q8(far)
    assert torch.equal(q.codes, mt.quantize_q8(x.cuda()).codes)
    store = torch.empty((M - 1) * 2 ** 31 + K, dtype=torch.int8, device="cuda")
    codes = store.as_strided((M, K), (2 ** 31, 1))
    codes.copy_(q.codes)
    far_q = mt.Q8Tensor(codes, q.scales)
    assert torch.equal(mt.dequantize_q8(far_q), mt.dequantize_q8(q))
    a, b = mt.linear_weight_grad_q8(far_q, dY.cuda()), mt.linear_weight_grad_q8(q, dY.cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- kernels that end with releases on their way -----------------------------------------

def test_weight_grad_one_call_behind_the_other(mt):
    """Whole tiles, split tiles and short sums in turn, each kernel's shared memory taken over by the
    next: equal bits every time and no wait that ran out. (The stages' last releases are waited for
    before a CTA leaves; one that arrived later would write to the next kernel's shared memory.)"""
    g = gen(31)
    cases = [wgrad_input(g, M, K, N, "int8", mt) for M, K, N in ((16, 64, 64), (300, 1300, 2300), (5000, 40, 70), (65, 520, 600))]
    cases = [(q, dy.cuda()) for q, dy in cases]
    want = [mt.linear_weight_grad_q8(q, dy) for q, dy in cases]
    got = [[mt.linear_weight_grad_q8(q, dy) for q, dy in cases] for _ in range(30)]
    for turn in got:
        assert all(torch.equal(a, c) and torch.equal(b, d) for (a, b), (c, d) in zip(turn, want))
    assert mt.engine.device_status() == 0


def test_batches_of_4_bit_products_one_call_behind_the_other(mt):
    """The same for batches: runs over cut tiles, whole tiles, and runs shorter than the ring."""
    g = gen(32)
    cases = []
    for M, K, N, group in ((9, 128, 16, 32), (21, 1111, 401, 32), (40, 4096, 2048, 64), (64, 512, 20000, 128), (150, 260, 300, 64)):
        x, codes, s = q4_case(g, M, K, N, group)
        cases.append((x.cuda(), mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, group)))
    want = [mt.linear_forward_q4(x, w) for x, w in cases]
    got = [[mt.linear_forward_q4(x, w) for x, w in cases] for _ in range(30)]
    for turn in got:
        assert all(torch.equal(a, b) for a, b in zip(turn, want))
    assert mt.engine.device_status() == 0


def test_linear_forward_q4_without_inputs_takes_any_number_of_rows(mt):
    none = mt.quantize_q4(torch.empty(0, 3, device="cuda"))
    bias = torch.randn(3, device="cuda")
    y = mt.linear_forward_q4(torch.empty(1100000, 0, device="cuda"), none, bias=bias, relu=True)
    assert torch.equal(y, bias.clamp_min(0).expand(1100000, 3))

# ---- 4 bits: entries of x of every size beside each other ---------------------------------

def ladder(g, M, K, N, group, low, high):
    """x whose entries' exponents are spread over [low, high], and weights that are 0 (code 8) in
    output n for every entry above the n-th of N thresholds: y[:, n] is a sum of the entries below."""
    e = torch.randint(low, high + 1, (M, K), generator=g)
    e[:, 0] = high
    x = torch.ldexp((torch.rand(M, K, generator=g) + 1) * torch.where(torch.rand(M, K, generator=g) < 0.5, -1.0, 1.0), e)
    codes = torch.randint(0, 16, (N, K), generator=g)
    limit = low + (high - low) * (torch.arange(N) + 1) // N
    codes[(e.amax(0)[None, :] > limit[:, None])] = 8
    s = (0.01 * torch.exp(rand(g, N, -(-K // group)))).to(torch.bfloat16)
    return x, codes, s


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 40, 200])
@pytest.mark.parametrize("low,high", [(-14, 0), (-35, 10), (-40, 40), (-60, 120), (-85, 125)])
@pytest.mark.parametrize("K,group", [(128, 32), (1000, 64), (4100, 128)])
def test_linear_forward_q4_small_entries_beside_large_ones(mt, M, low, high, K, group):
    """The error is held against |x| |W| alone: a large entry that meets weight 0 is no excuse."""
    g = gen(M + K + high)
    x, codes, s = ladder(g, M, K, 40, group, low, high)
    w = mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, group)
    W = R.q4_weight(codes, s, group)
    err = host(mt.linear_forward_q4(x.cuda(), w)).double() - x.double() @ W
    assert R.worst(err, x.double().abs() @ W.abs()) <= R.q4_bound(M, K, group)


def test_linear_forward_q4_one_large_entry_on_a_zero_weight(mt):
    """One entry of 1e12 on weight 0 beside 127 ones: the ones are the result, at any number of rows."""
    codes = torch.full((16, 128), 9, dtype=torch.int64)
    codes[:, 0] = 8
    w = mt.Q4Weight(R.q4_pack(codes, 128).cuda(), torch.ones(16, 1, dtype=torch.bfloat16, device="cuda"), 128, 128)
    for M in (1, 2, 4, 7, 8, 9, 200):
        x = torch.ones(M, 128, device="cuda")
        x[:, 0] = 1e12
        assert torch.equal(host(mt.linear_forward_q4(x, w)), torch.full((M, 16), 127.0))


@pytest.mark.parametrize("M", [1, 4, 8])
def test_linear_forward_q4_spread_entries_in_long_rows(mt, M):
    """Several launches over K, several passes over the digits, bias and ReLU at the end of both."""
    g, N = gen(M), 24
    K = 20000 if M == 1 else 14000
    x, codes, s = ladder(g, M, K, N, 32, -60, 60)
    bias = rand(g, N) * 2.0 ** 40
    w = mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, 32)
    y = host(mt.linear_forward_q4(x.cuda(), w, bias=bias.cuda(), relu=True)).double()
    assert "gemv" in mt.engine.last_path() or M > 4
    W = R.q4_weight(codes, s, 32)
    want, mag = x.double() @ W + bias.double(), x.double().abs() @ W.abs() + bias.double().abs()
    assert R.worst(y - want.clamp_min(0), mag) <= R.q4_bound(M, K, 32)


@pytest.mark.parametrize("e,scale", [(-90, 0), (-118, 0), (-130, 0), (-60, -60), (-40, -80), (-20, -104)])
def test_linear_forward_q4_tiny_results(mt, e, scale):
    """Rows of x with a single value, y = s * (c - 8) * x down to a float's smallest numbers, by a tiny x
    or a tiny s: at most six roundings (a conversion, the scale's product and the sum of four lanes,
    once per number), where y is not a normal number each of them to a multiple of 2^-147 at worst."""
    M, K, N, group = 4, 160, 40, 32
    g = gen(-e)
    x = torch.zeros(M, K)
    x[torch.arange(M), torch.tensor([3, 60, 101, 159])] = torch.ldexp(torch.rand(M, generator=g) + 1, torch.tensor(e))
    codes = torch.randint(0, 16, (N, K), generator=g)
    s = torch.ldexp(1 + torch.rand(N, K // group, generator=g), torch.tensor(scale)).to(torch.bfloat16)
    w = mt.Q4Weight(R.q4_pack(codes, K).cuda(), s.cuda(), K, group)
    want = x.double() @ R.q4_weight(codes, s, group)
    for rows in (1, 4):
        err = (host(mt.linear_forward_q4(x[:rows].cuda(), w)).double() - want[:rows]).abs()
        assert R.worst((err - 6 * 2.0 ** -148).clamp_min(0), want[:rows]) <= 7


@pytest.mark.parametrize("K", [2, 3, 4, 5])
@pytest.mark.parametrize("how", ["dy transposed", "gamma strided", "gamma broadcast"])
def test_rms_norm_backward_many_short_strided_rows(mt, K, how):
    """More row groups than a grid has in y."""
    rows, g = 160000, gen(K)
    h, gamma, dy = rand(g, rows, K, scale=2.0), 1 + rand(g, K, scale=0.1), rand(g, rows, K)
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(1) + 1e-6)).float()
    dyd, gd = dy.cuda(), gamma.cuda()
    if how == "dy transposed":
        dyd = strided(dy, "transposed")
    elif how == "gamma strided":
        gd = gamma.repeat_interleave(2).cuda()[::2]
    else:
        gamma = gamma[:1].expand(K)
        gd = gamma[:1].cuda().expand(K)
    dx, dgamma = mt.rms_norm_backward(dyd, h.cuda(), gd, rstd.cuda())
    want, mag, want_g, mag_g = R.rms_norm_backward(dy, h, gamma, rstd, None)
    assert R.worst(host(dx) - want, mag) <= 50
    assert R.worst(host(dgamma) - want_g, mag_g) <= rows + 3
    assert torch.equal(mt.rms_norm_backward(dyd, h.cuda(), gd, rstd.cuda(), need_dgamma=False)[0], dx)


# ---- no part of a float is lost, by every way through the products ------------------------
# Sums over thousands of terms may be off by so much that a lost third part (2^-16 of an operand)
# would pass. Here every sum has one term, at a place that differs from sum to sum.

@pytest.mark.parametrize("M,K,N,cut", [(130, 260, 200, "bn=128 whole=4 splits=1"), (1100, 70, 90, "bn=128 whole=0 splits=9"),
                                       (300, 5000, 4100, "bn=256 whole=340 splits=1"), (700, 2100, 2300, "bn=256 whole=74 splits=6")])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_linear_weight_grad_q8_keeps_every_bit_by_every_cut(mt, M, K, N, cut, fmt):
    """dY with one value per column: the third and the second part meet in an accumulator, then the
    first, each sum truncated (2 u); zeros are added after that."""
    q, dy = wgrad_input(gen(M + N), M, K, N, fmt, mt)
    at, n = (torch.arange(N) * 37 + 5) % M, torch.arange(N)
    one = torch.zeros(M, N)
    one[at, n] = dy[at, n]
    dW, db = mt.linear_weight_grad_q8(q, one.cuda())
    assert mt.engine.last_path().endswith(cut)
    want = host(mt.dequantize_q8(q)).double()[at].t() * one[at, n].double()
    assert R.worst(host(dW) - want, want) <= 3
    assert torch.equal(host(db)[0], one[at, n])


def one_value_rows(g, M, K):
    x = torch.zeros(M, K)
    x[torch.arange(M), (torch.arange(M) * 37 + 5) % K] = rand(g, M) * torch.exp(5 * rand(g, M))
    return x


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N,cut", [(200, 300, 300, "bn=128 whole=4 splits=1"), (500, 1300, 4800, "bn=128 whole=74 splits=11"),
                                       (1030, 700, 2600, "bn=256 whole=55 splits=1"), (200, 4000, 4097, "bn=256 whole=0 splits=4"),
                                       (9, 1111, 401, "batch"), (21, 4000, 700, "batch"), (40, 300, 20000, "batch"),
                                       (64, 1111, 401, "batch"), (150, 4000, 700, "batch")])
def test_linear_forward_q4_keeps_every_bit_by_every_cut(mt, M, K, N, cut, group):
    """Rows of x with one value: as above, and the product with the scale."""
    g = gen(M + K + N + group)
    _, codes, s = q4_case(g, 1, K, N, group)
    x = one_value_rows(g, M, K)
    w = mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, group)
    y = host(mt.linear_forward_q4(x.cuda(), w))
    assert cut in mt.engine.last_path()
    at = x.abs().argmax(1)
    want = x[torch.arange(M), at].double()[:, None] * R.q4_weight(codes, s, group)[at]
    assert R.worst(y - want, want) <= 7


@pytest.mark.parametrize("K", [64, 4096, 20000])
def test_rms_norm_range_of_its_statistics(mt, K):
    """Rows up to where the sum of squares is beyond a float's range, and past it."""
    top = 2.0 ** 63.9 / K ** 0.5
    x = torch.stack([torch.full((K,), top), torch.full((K,), 1.1 * 2.0 ** 64 / K ** 0.5)])
    out = mt.rms_norm(x.cuda(), torch.ones(K, device="cuda"))
    assert R.worst(host(out.rstd[:1]) - 1 / x[0, 0].double(), 1 / x[0, :1].double()) <= norm_bound(K)
    assert float(out.rstd[1]) == 0 and torch.equal(host(out.y[1]), torch.zeros(K))


@pytest.mark.parametrize("e", [-105, -112, -118, -125])
def test_products_of_tiny_entries(mt, e):
    """One term per sum, entries around 2^e: what their third part cannot hold is below 2^-133 each, and an
    accumulator of y / 2048 rounds to a multiple of 2^-138 where y is that small."""
    g, K, N, group = gen(-e), 300, 200, 64
    _, codes, s = q4_case(g, 1, K, N, group)
    W = R.q4_weight(codes, s, group)
    w = mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, group)
    for M in (5, 40, 200):
        x, at = torch.zeros(M, K), (torch.arange(M) * 37 + 5) % K
        x[torch.arange(M), at] = torch.ldexp(torch.rand(M, generator=g) + 1, torch.tensor(e))
        want = x.double() @ W
        err = (host(mt.linear_forward_q4(x.cuda(), w)).double() - want).abs()
        assert R.worst((err - 2.0 ** -133 * W[at].abs() - 4 * 2.0 ** -138).clamp_min(0), want) <= 7
    q, dy = mt.quantize_q8(rand(g, 200, 300).cuda()), torch.zeros(200, 130)
    at = (torch.arange(130) * 37 + 5) % 200
    dy[at, torch.arange(130)] = torch.ldexp(torch.rand(130, generator=g) + 1, torch.tensor(e))
    xv = host(mt.dequantize_q8(q)).double()[at].t()
    want = xv * dy.sum(0).double()
    err = (host(mt.linear_weight_grad_q8(q, dy.cuda())[0]).double() - want).abs()
    assert R.worst((err - 2.0 ** -133 * xv.abs() - 4 * 2.0 ** -149).clamp_min(0), want) <= 3


def test_calls_behind_one_that_found_no_memory(mt):
    """Scratch of 400 GB is refused by an error of that call; the calls behind it, torch's among them, do
    not meet it again."""
    q = mt.quantize_q8(torch.ones(2 ** 20, 1, device="cuda"))
    dY = torch.ones(1, 1, device="cuda").expand(2 ** 20, 2 ** 16)
    for again in (lambda: mt.quantize_q8(torch.ones(4, 64, device="cuda")).codes, lambda: torch.ones(4, device="cuda") + 1,
                  lambda: mt.matmul(torch.ones(64, 64, device="cuda"), torch.ones(64, 64, device="cuda")),
                  lambda: mt.linear_weight_grad_q8(q, dY[:, :8])[0]):
        with pytest.raises(RuntimeError, match="memory"):
            mt.linear_weight_grad_q8(q, dY)
        again()
    torch.cuda.synchronize()


def test_linear_forward_q4_passes_follow_the_values_at_replay(mt):
    """How often few rows go through the weights is decided by x on the GPU: a captured call follows x,
    and equal calls give equal bits."""
    g, K, N = gen(41), 1000, 77
    for M in (1, 3):
        spread, codes, s = ladder(g, M, K, N, 64, -80, 120)
        w = mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, 64)
        inputs = [spread.cuda(), rand(g, M, K).cuda(), torch.zeros(M, K, device="cuda"), spread.cuda() * 0.5]
        want = [mt.linear_forward_q4(x, w) for x in inputs]
        x = inputs[1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mt.linear_forward_q4(x, w)
        for v, expected in zip(inputs * 2, want * 2):
            x.copy_(v)
            graph.replay()
            assert torch.equal(y, expected)


@pytest.mark.parametrize("scale,e", [(-133, 120), (-126, 30), (60, -40), (97, -60), (105, -90), (112, -20)])
@pytest.mark.parametrize("M", [1, 4, 9, 200])
def test_linear_forward_q4_scales_of_any_size(mt, M, scale, e):
    """Scales from the least bfloat16 to 2^113, whose products with x are ordinary floats."""
    g, K, N, group = gen(scale + 200), 300, 40, 128
    codes = torch.randint(0, 16, (N, K), generator=g)
    s = torch.ldexp(1 + torch.rand(N, 3, generator=g), torch.tensor(scale)).to(torch.bfloat16)
    x = torch.ldexp(rand(g, M, K), torch.tensor(e))
    w = mt.Q4Weight(R.q4_pack(codes, K).cuda(), s.cuda(), K, group)
    W = R.q4_weight(codes, s, group)
    err = host(mt.linear_forward_q4(x.cuda(), w)).double() - x.double() @ W
    assert R.worst(err, x.double().abs() @ W.abs()) <= R.q4_bound(M, K, group)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N,path", [(1, 45000, 130, "batch"), (2, 22000, 300, "batch"), (3, 23000, 17, "batch"), (4, 20000, 70, "batch"),
                                        (8, 20000, 130, "batch"), (5, 5000, 6000, "batch"), (1, 11000, 40, "gemv rows=1 x 1"),
                                        (3, 9000, 33, "gemv rows=2 x 2"), (4, 5000, 33, "gemv rows=2 x 2"), (7, 5000, 33, "gemv rows=3 x 3"),
                                        (4, 4500, 33, "gemv rows=4 x 1"), (7, 4500, 33, "gemv rows=4 x 2"), (8, 9000, 33, "gemv rows=2 x 4")])
def test_linear_forward_q4_few_long_rows(mt, M, K, N, path, group):
    """Either side of the rows and lengths at which few rows become a batch, and rows that share a CTA by
    four, three or two (four rows of 5000 inputs take 242,944 bytes of shared memory, 232,448 are there)."""
    g = gen(M + K)
    x, codes, s = ladder(g, M, K, N, group, -30, 20)
    bias = rand(g, N) * 2.0 ** 10
    w = mt.Q4Weight(pack_fast(codes, K).cuda(), s.cuda(), K, group)
    y = host(mt.linear_forward_q4(x.cuda(), w, bias=bias.cuda())).double()
    assert path in mt.engine.last_path()
    W = R.q4_weight(codes, s, group)
    err, mag = y - x.double() @ W - bias.double(), x.double().abs() @ W.abs() + bias.double().abs()
    assert R.worst(err, mag) <= R.q4_bound(M, K, group)
