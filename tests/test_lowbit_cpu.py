"""CPU tests of the low-bit operators: the reference forms of the GPU tests against planted
mistakes, and the refusals, which come before anything touches a device."""
import ctypes

import pytest
import torch

import lowbit_ref as R
import minitensor_b200 as mt
from minitensor_b200 import engine, lowbit


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def q8(rows, cols, dtype=torch.int8):
    return mt.Q8Tensor(t(rows, cols, dtype=dtype), t(rows, -(-cols // 32), dtype=torch.uint8))


def q4(k, n, group=64):
    return mt.Q4Weight(t(n, 64 * -(-k // 128), dtype=torch.uint8), t(n, -(-k // group), dtype=torch.bfloat16), k, group)


def refuses(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


# ---- the reference forms ----------------------------------------------------------------

def test_reference_8_bit_scale_is_the_smallest_that_clips_nothing():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 100, generator=g) * torch.exp(5 * torch.randn(6, 1, generator=g))
    for fmt in ("int8", "e4m3"):
        b = R.q8_scale_bytes(x, fmt)
        amax = torch.nn.functional.pad(x.double().abs(), (0, 28)).view(6, 4, 32).amax(2)
        top = R.TOP[fmt] * torch.exp2(b.double() - 127)
        assert (amax <= top).all() and (amax > top / 2).all()
        v = R.q8_values(R.q8_codes(x, b, fmt).float(), b.to(torch.uint8))
        half = torch.exp2(b.double() - 128).repeat_interleave(32, 1)[:, :100]
        if fmt == "int8":
            assert ((v - x).abs() <= half).all()
        else:
            assert ((v - x).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, half * 2.0 ** -9)).all()


def test_reference_4_bit_order():
    codes = torch.randint(0, 16, (3, 200), generator=torch.Generator().manual_seed(1))
    words = R.q4_pack(codes, 200).view(torch.int32).view(3, 2, 16)
    for k in (0, 1, 2, 7, 8, 31, 32, 100, 127, 128, 199):
        s, r = divmod(k, 128)
        word = int(words[1, s, 4 * (r % 32 // 8) + r // 32]) & 0xFFFFFFFF
        assert (word >> (4 * (r % 8 // 2) + 16 * (r % 2))) & 15 == int(codes[1, k])


def test_reference_backward_is_the_gradient_of_the_forward():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 9, generator=g, dtype=torch.float64, requires_grad=True)
    gamma = torch.randn(9, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(4, 9, generator=g, dtype=torch.float64)
    h, rstd, y = R.rms_norm(x, None, gamma, 1e-3)
    dx, dgamma = torch.autograd.grad((y * dy).sum(), (x, gamma))
    want, _, want_g, _ = R.rms_norm_backward(dy, x.detach(), gamma.detach(), rstd.detach(), None)
    assert torch.allclose(dx, want, rtol=1e-10) and torch.allclose(dgamma, want_g, rtol=1e-10)


def test_bounds_catch_planted_mistakes():
    """A dropped low part, a shifted scale and a missing row are each beyond the bounds that
    the GPU tests use."""
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(1, 64, generator=g), torch.randn(1, 50, generator=g)
    want = x.double().t() @ dy.double()
    high = (dy.view(torch.int32) & -65536).view(torch.float32)
    mid = dy - high
    mid = (mid.view(torch.int32) & -65536).view(torch.float32)
    assert R.worst(x.double().t() @ (high + mid).double() - want, want) > 3
    X, DY = torch.randn(300, 33, generator=g), torch.randn(300, 70, generator=g)
    W, mag = X.double().t() @ DY.double(), X.double().abs().t() @ DY.double().abs()
    assert R.worst(X[:299].double().t() @ DY[:299].double() - W, mag) > 308


def test_bounds_of_single_terms_catch_a_lost_third_part():
    """Without its third part most floats are beyond the bounds for sums of one term, whatever the other
    operand; sums of many terms hide it."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(4000, generator=g) * torch.exp(5 * torch.randn(4000, generator=g))
    high = (x.view(torch.int32) & -65536).view(torch.float32)
    mid = ((x - high).view(torch.int32) & -65536).view(torch.float32)
    off = (x.double() - high.double() - mid.double()).abs() / (R.U * x.double().abs())
    assert (off > 7).double().mean() > 0.9
    assert torch.equal((x - high - mid).to(torch.bfloat16).float(), x - high - mid)   # and the third part is all of the rest


def digit_values(x, sets):
    """x [K] as the sum of `sets` fixed-point numbers of steps 2^(e - 29 - 31 j), 2^e the largest entry's
    power of two, in 64 bits where each number and its remainder are exact."""
    e = torch.floor(torch.log2(x.abs().max().double()))
    v, total = x.double() * 2.0 ** (29 - e), torch.zeros_like(x, dtype=torch.float64)
    for j in range(sets):
        X = torch.round(v)
        assert X.abs().max() <= 2 ** 30
        total += X * 2.0 ** (e - 29 - 31 * j)
        v = (v - X) * 2.0 ** 31
    return total


def test_bounds_catch_an_entry_lost_beside_a_large_one():
    """One fixed-point number for a span drops what lies far below its largest entry; that is beyond
    q4_bound, which holds an error against |x| |W|. A second number reaches 2^37 below."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(128, generator=g)
    W = torch.randint(-8, 8, (128, 40), generator=g).double()
    W[::16] = 0
    for top in (20, 35):
        y = x.clone()
        y[::16] = 2.0 ** top
        assert R.worst((digit_values(y, 1) - y.double()) @ W, y.double().abs() @ W.abs()) > R.q4_bound(1, 128, 32)
        near = y.abs() >= 2.0 ** (top - 36)
        assert torch.equal(digit_values(y, 2)[near], y.double()[near])


# ---- refusals ---------------------------------------------------------------------------

def test_rms_norm_refusals():
    refuses("2-D", mt.rms_norm, t(4), t(4))
    refuses("float32", mt.rms_norm, t(2, 4, dtype=torch.float64), t(4))
    refuses("gamma must hold 4", mt.rms_norm, t(2, 4), t(5))
    refuses("gamma must hold 4", mt.rms_norm, t(2, 4), t(2, 2))
    refuses("x's shape", mt.rms_norm, t(2, 4), t(4), residual=t(2, 5))
    refuses("no features", mt.rms_norm, t(2, 0), t(0))
    refuses("eps", mt.rms_norm, t(2, 4), t(4), eps=-1.0)
    refuses("eps", mt.rms_norm, t(2, 4), t(4), eps=float("nan"))
    refuses("8-bit format", mt.rms_norm, t(2, 4), t(4), q8="int7")
    refuses("no output", mt.rms_norm, t(2, 4), t(4), want_y=False)
    refuses("inplace", mt.rms_norm, t(2, 4), t(4), inplace=True)
    refuses("broadcast", mt.rms_norm, t(1, 4).expand(3, 4), t(4), residual=t(3, 4), inplace=True)
    base = t(2, 12)
    refuses("shares memory", mt.rms_norm, base[:, 0:8], t(8), residual=base[:, 4:12], inplace=True)


def test_rms_norm_disjoint_windows_of_one_buffer_are_not_refused():
    # Not an argument error: without a GPU the call gets as far as the launch.
    base = t(3, 16)
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    with pytest.raises(RuntimeError, match="launch"):
        mt.rms_norm(base[:, :8], t(8), residual=base[:, 8:], inplace=True)


def test_rms_norm_backward_refusals():
    refuses("2-D", mt.rms_norm_backward, t(4), t(4), t(4), t(1))
    refuses("dy's shape", mt.rms_norm_backward, t(2, 4), t(2, 5), t(4), t(2))
    refuses("dy's shape", mt.rms_norm_backward, t(2, 4), t(2, 4), t(4), t(2), dh=t(3, 4))
    refuses("rstd must hold 2", mt.rms_norm_backward, t(2, 4), t(2, 4), t(4), t(3))
    refuses("gamma must hold 4", mt.rms_norm_backward, t(2, 4), t(2, 4), t(3), t(2))
    v = engine.view
    b = ctypes.byref
    x, g, r = v(t(2, 4)), v(t(4)), v(t(2))
    part = t(3, 4)
    L = lowbit._lowbit_lib()
    rc = L.mt_rms_norm_backward(b(v(part[:2])), b(x), b(g), b(r), None, b(v(part[1:])), None, None)
    assert rc == engine.MT_EINVAL and b"shares memory" in L.mt_last_error()
    rc = L.mt_rms_norm_backward(b(x), b(v(part[:2])), b(g), b(r), None, b(v(part[:2])), None, None)
    assert rc == engine.MT_EINVAL and b"shares memory" in L.mt_last_error()
    rc = L.mt_rms_norm_backward(b(x), b(x), b(g), b(r), None, None, None, None)
    assert rc == engine.MT_EINVAL


def test_q8_tensor_refusals():
    u8 = torch.uint8
    refuses("int8 or float8", mt.Q8Tensor, t(2, 40), t(2, 2, dtype=u8))
    refuses("uint8", mt.Q8Tensor, t(2, 40, dtype=torch.int8), t(2, 2))
    refuses(r"scales must be \[2, 2\]", mt.Q8Tensor, t(2, 40, dtype=torch.int8), t(2, 1, dtype=u8))
    refuses("2-D", mt.Q8Tensor, t(40, dtype=torch.int8), t(2, dtype=u8))
    refuses("unit column stride", mt.Q8Tensor, t(40, 2, dtype=torch.int8).t(), t(2, 2, dtype=u8))
    refuses("broadcast", mt.Q8Tensor, t(1, 40, dtype=torch.int8).expand(3, 40), t(3, 2, dtype=u8))
    refuses("broadcast", mt.Q8Tensor, t(3, 40, dtype=torch.int8), t(1, 2, dtype=u8).expand(3, 2))
    assert q8(2, 40).format == "int8" and q8(2, 40, torch.float8_e4m3fn).format == "e4m3"


def test_quantize_q8_refusals():
    refuses("2-D", mt.quantize_q8, t(2, 3, 4))
    refuses("float32", mt.quantize_q8, t(2, 4, dtype=torch.bfloat16))
    refuses("format", mt.quantize_q8, t(2, 4), "e5m2")
    refuses("dtype", mt.dequantize_q8, q8(2, 4), dtype=torch.float16)
    L = lowbit._lowbit_lib()
    q = q8(2, 40)
    x = engine.view(t(2, 41))
    assert L.mt_quantize_q8(ctypes.byref(x), ctypes.byref(q._c), None) == engine.MT_EINVAL
    assert L.mt_dequantize_q8(ctypes.byref(q._c), None, 0, 40, None) == engine.MT_EINVAL
    out = t(2, 40)
    assert L.mt_dequantize_q8(ctypes.byref(q._c), out.data_ptr(), 2, 40, None) == engine.MT_EINVAL
    assert L.mt_dequantize_q8(ctypes.byref(q._c), out.data_ptr(), 0, 39, None) == engine.MT_EINVAL
    assert L.mt_dequantize_q8(ctypes.byref(q._c), q._c.codes, 0, 40, None) == engine.MT_EINVAL
    bad = lowbit.MtQ8(q._c.codes, q._c.scales, 2, 40, 39, 2, 0)
    assert L.mt_dequantize_q8(ctypes.byref(bad), out.data_ptr(), 0, 40, None) == engine.MT_EINVAL
    bad = lowbit.MtQ8(q._c.codes, q._c.scales, 2, 40, 40, 2, 2)
    assert L.mt_dequantize_q8(ctypes.byref(bad), out.data_ptr(), 0, 40, None) == engine.MT_EINVAL


def test_linear_q8_refusals():
    refuses("rows", mt.linear_weight_grad_q8, q8(3, 40), t(4, 5))
    refuses("2-D", mt.linear_weight_grad_q8, q8(3, 40), t(3))
    refuses("W must be", mt.linear_backward_q8, q8(3, 40), t(41, 5), t(3, 5))
    refuses("W must be", mt.linear_backward_q8, q8(3, 40), t(40, 6), t(3, 5))
    L = lowbit._lowbit_lib()
    q = q8(3, 40)
    dy, dw, db = t(3, 5), t(40, 5), t(5)
    v, b = engine.view, ctypes.byref

    def rc(dy_, dw_, db_=None):
        return L.mt_linear_wgrad_q8(b(q._c), b(v(dy_)), b(v(dw_)), b(v(db_)) if db_ is not None else None, None)

    assert rc(dy, t(40, 6)) == engine.MT_EINVAL
    assert rc(dy, dw, t(6)) == engine.MT_EINVAL
    assert rc(dy, t(1, 5).expand(40, 5)) == engine.MT_EINVAL
    both = t(43, 5)
    assert rc(both[:3], both[2:42]) == engine.MT_EINVAL
    assert rc(dy, both[:40], both[39]) == engine.MT_EINVAL


def test_q4_weight_refusals():
    u8, bf = torch.uint8, torch.bfloat16
    refuses("group", mt.quantize_q4, t(64, 8), 16)
    refuses("group", mt.Q4Weight, t(8, 64, dtype=u8), t(8, 4, dtype=bf), 64, 16)
    refuses("uint8", mt.Q4Weight, t(8, 64, dtype=torch.int8), t(8, 1, dtype=bf), 64, 64)
    refuses("bfloat16", mt.Q4Weight, t(8, 64, dtype=u8), t(8, 1), 64, 64)
    refuses(r"codes \[8, 64\]", mt.Q4Weight, t(8, 32, dtype=u8), t(8, 1, dtype=bf), 64, 64)
    refuses(r"scales \[8, 2\]", mt.Q4Weight, t(8, 64, dtype=u8), t(8, 1, dtype=bf), 65, 64)
    refuses("unit column", mt.Q4Weight, t(64, 8, dtype=u8).t(), t(8, 1, dtype=bf), 64, 64)
    refuses("broadcast", mt.Q4Weight, t(1, 64, dtype=u8).expand(8, 64), t(8, 1, dtype=bf), 64, 64)
    refuses("negative", mt.Q4Weight, t(8, 0, dtype=u8), t(8, 0, dtype=bf), -1, 64)


def test_linear_q4_refusals():
    w = q4(100, 8)
    refuses("features", mt.linear_forward_q4, t(3, 99), w)
    refuses("2-D", mt.linear_forward_q4, t(100), w)
    refuses("float32", mt.linear_forward_q4, t(3, 100, dtype=torch.bfloat16), w)
    refuses("bias must hold 8", mt.linear_forward_q4, t(3, 100), w, bias=t(9))
    refuses("contiguous", mt.linear_forward_q4, t(3, 100), w, bias=t(8, 2)[:, 0])
    L = lowbit._lowbit_lib()
    v, b = engine.view, ctypes.byref
    x, y = v(t(3, 100)), v(t(3, 8))
    assert L.mt_linear_fwd_q4(b(x), None, None, b(y), 0, None) == engine.MT_EINVAL
    assert L.mt_linear_fwd_q4(b(x), b(w._c), None, b(v(t(3, 9))), 0, None) == engine.MT_EINVAL
    assert L.mt_linear_fwd_q4(b(x), b(w._c), None, b(v(t(1, 8).expand(3, 8))), 0, None) == engine.MT_EINVAL
    shared = t(3, 108)
    assert L.mt_linear_fwd_q4(b(v(shared[:, :100])), b(w._c), None, b(v(shared[:, 96:104])), 0, None) == engine.MT_EINVAL
    c = w._c
    for bad in (lowbit.MtQ4(c.codes + 8, c.scales, 100, 8, 64, 64, 2), lowbit.MtQ4(c.codes, c.scales, 100, 8, 64, 72, 2),
                lowbit.MtQ4(c.codes, c.scales, 100, 8, 64, 48, 2), lowbit.MtQ4(c.codes, c.scales, 100, 8, 64, 64, 1),
                lowbit.MtQ4(c.codes, c.scales, 100, 8, 48, 64, 4), lowbit.MtQ4(None, c.scales, 100, 8, 64, 64, 2)):
        assert L.mt_linear_fwd_q4(b(x), b(bad), None, b(y), 0, None) == engine.MT_EINVAL
    assert L.mt_quantize_q4(b(v(t(99, 8))), b(c), None) == engine.MT_EINVAL
    assert L.mt_dequantize_q4(b(c), b(v(t(100, 9))), None) == engine.MT_EINVAL


def test_valid_calls_without_a_gpu_end_in_an_error():
    """Nothing is divided by the number of SMs of a GPU that is not there."""
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    w = q4(256, 64)
    for rows in (1, 8, 20, 100, 300):
        with pytest.raises(RuntimeError):
            mt.linear_forward_q4(t(rows, 256), w)
    for call in (lambda: mt.linear_weight_grad_q8(q8(300, 200), t(300, 70)), lambda: mt.quantize_q8(t(3, 64)),
                 lambda: mt.dequantize_q8(q8(3, 64)), lambda: mt.quantize_q4(t(64, 8)), lambda: mt.dequantize_q4(w),
                 lambda: mt.rms_norm(t(3, 64), t(64), q8="e4m3"), lambda: mt.rms_norm(t(3, 50000), t(50000)),
                 lambda: mt.rms_norm_backward(t(3, 64), t(3, 64), t(64), t(3))):
        with pytest.raises(RuntimeError):
            call()


def test_linear_q4_without_inputs_takes_any_number_of_rows():
    """The bias alone, on more rows than a grid has chunks: not refused (without a GPU it ends at
    the launch)."""
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    with pytest.raises(RuntimeError, match="launch|no kernel|driver|device"):
        mt.linear_forward_q4(t(1100000, 0), q4(0, 3), bias=t(3))


def test_operands_cannot_be_given_other_tensors():
    """The library reads the memory of the tensors that an operand was made of; one set later would
    not be it (and the first could be freed)."""
    for v, names in ((q8(2, 40), ("codes", "scales", "_c")), (q4(100, 8), ("codes", "scales", "in_features", "group", "_c"))):
        before = [getattr(v, n) for n in names]
        for n in names:
            with pytest.raises(AttributeError):
                setattr(v, n, getattr(v, n))
            with pytest.raises(AttributeError):
                delattr(v, n)
        assert all(getattr(v, n) is b for n, b in zip(names, before))
        assert (v._c.codes, v._c.scales) == (v.codes.data_ptr(), v.scales.data_ptr())
