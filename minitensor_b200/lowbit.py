"""Low-bit forms of Linear, and the norm that makes its input.

The reference holds every tensor in float (include/Tensor.hpp), so nothing here has a
counterpart there. Three operators around ``Linear<float>`` (include/Module.hpp:83-124):

* ``rms_norm`` / ``rms_norm_backward``: the root-mean-square norm with the residual's
  addition; its output also (or only) in 8 bits with scales.
* ``quantize_q8`` / ``linear_forward_q8`` / ``linear_backward_q8``: the forward pass saves
  Linear's input in 8 bits (a quarter of its memory), the weight gradient reads that form.
* ``quantize_q4`` / ``linear_forward_q4``: Linear with 4-bit weights and group scales, from
  one decoded token to whole prompts.

Activations, gradients and results are float32, computed to the accuracy of a float product
(entries below 2^-110 to a multiple of 2^-133, include/mtgemm.h has where); there is no TF32 form.
Like the rest of the package the functions check their arguments
(``ValueError``), launch on ``stream`` (default: torch's current stream of the operands'
device) without synchronising, and raise ``RuntimeError`` on CUDA failures. All operands
are on one device, which need not be the current one. With ``stream`` given, results are
allocated for that stream; the caller orders other streams' use of operands and results.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional

import torch

from . import engine
from .engine import MAX_DIMS, MODE_DEFAULT, _check, _gpu_present, gemm, linear_forward

Q8_BLOCK = 32
Q8_FORMATS = {"int8": 0, "e4m3": 1}
_Q8_DTYPES = {torch.int8: "int8", torch.float8_e4m3fn: "e4m3"}
_Q8_STORAGE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
Q4_GROUPS = (32, 64, 128)
Q4_SPAN = 128            # codes per 64-byte span of a weight row


class MtQ8(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("rows", ctypes.c_uint64),
                ("cols", ctypes.c_uint64), ("code_pitch", ctypes.c_uint64), ("scale_pitch", ctypes.c_uint64),
                ("format", ctypes.c_int)]


class MtQ4(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("in_", ctypes.c_uint64),
                ("out", ctypes.c_uint64), ("group", ctypes.c_uint64), ("code_pitch", ctypes.c_uint64),
                ("scale_pitch", ctypes.c_uint64)]


_lib = None


def _lowbit_lib():
    global _lib
    if _lib is None:
        L = engine.lib()
        P = Q8 = Q4 = vp = ctypes.c_void_p   # structs are passed packed (_mat) or by reference
        i, u64 = ctypes.c_int, ctypes.c_uint64
        for name, args in (("mt_rms_norm", [P, P, P, P, P, P, Q8, ctypes.c_float, vp]),
                           ("mt_rms_norm_backward", [P, P, P, P, P, P, P, vp]),
                           ("mt_quantize_q8", [P, Q8, vp]),
                           ("mt_dequantize_q8", [Q8, vp, i, u64, vp]),
                           ("mt_linear_wgrad_q8", [Q8, P, P, P, vp]),
                           ("mt_quantize_q4", [P, Q4, vp]),
                           ("mt_dequantize_q4", [Q4, P, vp]),
                           ("mt_linear_fwd_q4", [P, Q4, P, P, i, vp])):
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = i
        _lib = L
    return _lib


# ---- operands ---------------------------------------------------------------------------

class _Held:
    """Tensors with the C struct that points into their memory: no attribute can be set again,
    since the struct would go on pointing to the memory of the tensor before."""

    __slots__ = ()

    def __setattr__(self, name, value):
        raise AttributeError(f"{type(self).__name__}.{name} cannot be set: make a new {type(self).__name__}")

    def __delattr__(self, name):
        raise AttributeError(f"{type(self).__name__}.{name} cannot be deleted")


_put = object.__setattr__


class Q8Tensor(_Held):
    """A [rows, cols] tensor in 8 bits. ``codes`` (int8 or float8_e4m3fn) [rows, cols] and
    ``scales`` (uint8) [rows, ceil(cols / 32)], both with unit column stride: the code c of
    a block of 32 columns with scale byte b stands for c * 2^(b - 127); b = 255 is NaN. What the
    tensors hold may be changed in place, the tensors not."""

    __slots__ = ("codes", "scales", "_c")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype not in _Q8_DTYPES:
            raise ValueError(f"codes must be int8 or float8_e4m3fn, got {codes.dtype}")
        if scales.dtype != torch.uint8:
            raise ValueError(f"scales must be uint8, got {scales.dtype}")
        if codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("codes and scales must be 2-D")
        rows, cols = codes.shape
        if tuple(scales.shape) != (rows, -(-cols // Q8_BLOCK)):
            raise ValueError(f"scales must be [{rows}, {-(-cols // Q8_BLOCK)}] for codes [{rows}, {cols}]")
        for name, t in (("codes", codes), ("scales", scales)):
            if t.shape[1] > 1 and t.stride(1) != 1:
                raise ValueError(f"{name} must have unit column stride")
            if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
                raise ValueError(f"{name} must not have overlapping or broadcast rows")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on the same device")
        _put(self, "codes", codes)
        _put(self, "scales", scales)
        # A [n, 1] view may have any column stride; its row stride still is the pitch.
        _put(self, "_c", MtQ8(codes.data_ptr(), scales.data_ptr(), rows, cols, max(codes.stride(0), cols),
                              max(scales.stride(0), scales.shape[1]), Q8_FORMATS[_Q8_DTYPES[codes.dtype]]))

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def get_device(self) -> int:
        return self.codes.get_device()

    @property
    def format(self) -> str:
        return _Q8_DTYPES[self.codes.dtype]


class Q4Weight(_Held):
    """A Linear weight [in_features, out_features] in 4 bits: ``codes`` (uint8)
    [out, 64 * ceil(in / 128)] and ``scales`` (bfloat16) [out, ceil(in / group)], rows =
    output features. include/mtgemm.h (mt_q4) has the order of the codes in a row. What the
    tensors hold may be changed in place, the tensors not."""

    __slots__ = ("codes", "scales", "in_features", "group", "_c")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, in_features: int, group: int):
        if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16:
            raise ValueError(f"codes must be uint8 and scales bfloat16, got {codes.dtype} and {scales.dtype}")
        if group not in Q4_GROUPS:
            raise ValueError(f"group must be one of {Q4_GROUPS}, got {group}")
        if codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("codes and scales must be 2-D")
        if in_features < 0:
            raise ValueError("in_features must not be negative")
        out = codes.shape[0]
        want_c, want_s = 64 * (-(-in_features // Q4_SPAN)), -(-in_features // group)
        if codes.shape[1] != want_c or tuple(scales.shape) != (out, want_s):
            raise ValueError(f"{in_features} input features in groups of {group} need codes [{out}, {want_c}] and "
                             f"scales [{out}, {want_s}]")
        for name, t in (("codes", codes), ("scales", scales)):
            if t.shape[1] > 1 and t.stride(1) != 1:
                raise ValueError(f"{name} must have unit column stride")
            if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
                raise ValueError(f"{name} must not have overlapping or broadcast rows")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on the same device")
        pitch = codes.stride(0) if out > 1 else want_c
        for name, value in (("codes", codes), ("scales", scales), ("in_features", in_features), ("group", group),
                            ("_c", MtQ4(codes.data_ptr(), scales.data_ptr(), in_features, out, group, pitch,
                                        max(scales.stride(0), want_s)))):
            _put(self, name, value)

    @property
    def out_features(self) -> int:
        return self.codes.shape[0]

    @property
    def device(self):
        return self.codes.device

    def get_device(self) -> int:
        return self.codes.get_device()


# An mt_tensor as bytes: these operators' smallest calls are bound by the host, and packing
# takes a third of what filling a ctypes struct does.
_pack = struct.Struct(f"@PQI4x{2 * MAX_DIMS}Q").pack
_PAD = (0,) * (MAX_DIMS - 2)


def _mat(t: torch.Tensor) -> bytes:
    if t.dtype is not torch.float32:
        raise ValueError(f"expected float32, got {t.dtype}")
    dims = t.dim()
    if dims == 2:
        (r, c), (rs, cs) = t.shape, t.stride()
        return _pack(t.data_ptr(), 0, 2, r, c, *_PAD, rs, cs, *_PAD)
    if dims > MAX_DIMS:
        raise ValueError("Exceeded MAX_DIMS")
    pad = (0,) * (MAX_DIMS - dims)
    return _pack(t.data_ptr(), 0, dims, *t.shape, *pad, *t.stride(), *pad)


def _dense(t: torch.Tensor, rows: int, cols: int) -> bytes:
    """A contiguous [rows, cols] result, whose layout is known."""
    return _pack(t.data_ptr(), 0, 2, rows, cols, *_PAD, cols, 1, *_PAD)


def _opt(t):
    return None if t is None else _mat(t)


def _same_device(first, *others):
    """The operands' device index, -1 for host memory (which only a machine without a GPU
    gets as far as the library's argument checks)."""
    d = first.get_device()
    for o in others:
        if o is not None and o.get_device() != d:
            raise ValueError("all operands must be on the same device")
    if d < 0 and _gpu_present():
        raise ValueError("expected CUDA tensors, got some on the host")
    return d


def _device(d: int):
    return torch.device("cuda", d) if d >= 0 else torch.device("cpu")


def _empty(like, rows, cols):
    """An uninitialised contiguous float32 [rows, cols] on like's device."""
    if like.dtype is torch.float32 and like.is_contiguous() and like.shape == (rows, cols):
        return torch.empty_like(like)   # half the cost of naming everything
    return torch.empty((rows, cols), dtype=torch.float32, device=like.device)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # current_stream(), without the object


class _On:
    """The operands' device and the call's stream made current, so that results and scratch
    belong to them; ``.s`` is the raw stream."""

    __slots__ = ("s", "_ctx")

    def __init__(self, device, stream):
        self._ctx = None
        if device < 0:
            self.s = None
        elif stream is None:
            if device != torch.cuda.current_device():
                self._ctx = torch.cuda.device(device)
            self.s = _raw_stream(device) if _raw_stream else torch.cuda.current_stream(device).cuda_stream
        else:
            if not isinstance(stream, torch.cuda.Stream):
                stream = torch.cuda.ExternalStream(int(stream), device=device)
            elif stream.device.index != device:
                raise ValueError(f"the stream belongs to {stream.device}, the operands to cuda:{device}")
            self._ctx = torch.cuda.stream(stream)
            self.s = stream.cuda_stream

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()
        return self

    def __exit__(self, *exc):
        if self._ctx is not None:
            self._ctx.__exit__(*exc)
        return False


def _need_2d(t, name):
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {t.dim()}-D")
    if t.dtype != torch.float32:
        raise ValueError(f"{name}: expected float32, got {t.dtype}")


def _new_q8(rows, cols, fmt, d) -> Q8Tensor:
    if fmt not in Q8_FORMATS:
        raise ValueError(f"8-bit format must be one of {tuple(Q8_FORMATS)}, got {fmt!r}")
    device, blocks = _device(d), -(-cols // Q8_BLOCK)
    q = Q8Tensor.__new__(Q8Tensor)      # dense and new: nothing for the constructor to check
    codes = torch.empty((rows, cols), dtype=_Q8_STORAGE[fmt], device=device)
    scales = torch.empty((rows, blocks), dtype=torch.uint8, device=device)
    _put(q, "codes", codes)
    _put(q, "scales", scales)
    _put(q, "_c", MtQ8(codes.data_ptr(), scales.data_ptr(), rows, cols, cols, blocks, Q8_FORMATS[fmt]))
    return q


# ---- RMS norm ---------------------------------------------------------------------------

class RmsNorm(NamedTuple):
    """What ``rms_norm`` returns: the output (None unless wanted), x + residual (x itself
    without a residual), the reciprocal root mean square of each row of h, and the output in
    8 bits (None unless wanted)."""
    y: Optional[torch.Tensor]
    h: torch.Tensor
    rstd: torch.Tensor
    q8: Optional[Q8Tensor]


def rms_norm(x, gamma, residual=None, eps=1e-6, q8=None, want_y=True, inplace=False, stream=None) -> RmsNorm:
    """h = x + residual, y = h / sqrt(mean(h^2) + eps) * gamma for each row of x [rows,
    features]; gamma [features]. ``q8`` = "int8" or "e4m3" also gives y in 8 bits, as
    Linear's checkpoint; want_y=False leaves out the float form. inplace=True adds the
    residual in place: h is x's memory."""
    _need_2d(x, "x")
    if not want_y and q8 is None:
        raise ValueError("rms_norm: no output is wanted (want_y=False without q8)")
    if inplace and residual is None:
        raise ValueError("rms_norm: inplace adds a residual, and none is given")
    rows, features = x.shape
    dev = _same_device(x, gamma, residual)
    with _On(dev, stream) as on:
        q = _new_q8(rows, features, q8, dev) if q8 is not None else None
        y = _empty(x, rows, features) if want_y else None
        h = x if residual is None or inplace else _empty(x, rows, features)
        rstd = torch.empty((rows,), dtype=torch.float32, device=x.device)
        _check(_lowbit_lib().mt_rms_norm(
            _mat(x), _opt(residual), _mat(gamma),
            None if residual is None else _mat(x) if inplace else _dense(h, rows, features),
            _dense(y, rows, features) if want_y else None, _dense(rstd, 1, rows),
            ctypes.byref(q._c) if q is not None else None, eps, on.s))
    return RmsNorm(y, h, rstd, q)


def rms_norm_backward(dy, h, gamma, rstd, dh=None, need_dgamma=True, stream=None):
    """(dx, dgamma) of ``rms_norm`` from its h and rstd and the gradient dy of y. dx is the
    gradient of x and of the residual both; ``dh``, a gradient that reaches h from the
    residual stream behind the norm, is added to it. dgamma is [features], or None."""
    _need_2d(dy, "dy")
    rows, features = dy.shape
    dev = _same_device(dy, h, gamma, rstd, dh)
    with _On(dev, stream) as on:
        dx = _empty(dy, rows, features)
        dgamma = torch.empty((features,), dtype=torch.float32, device=dy.device) if need_dgamma else None
        _check(_lowbit_lib().mt_rms_norm_backward(
            _mat(dy), _mat(h), _mat(gamma), _mat(rstd), _opt(dh), _dense(dx, rows, features),
            _dense(dgamma, 1, features) if need_dgamma else None, on.s))
    return dx, dgamma


# ---- 8-bit activation checkpoints -------------------------------------------------------

def quantize_q8(x, fmt="int8", stream=None) -> Q8Tensor:
    """x [rows, cols] in 8 bits: per block of 32 columns the smallest power-of-two scale that
    clips nothing, codes rounded to nearest even."""
    _need_2d(x, "x")
    dev = _same_device(x)
    with _On(dev, stream) as on:
        q = _new_q8(x.shape[0], x.shape[1], fmt, dev)
        _check(_lowbit_lib().mt_quantize_q8(_mat(x), ctypes.byref(q._c), on.s))
    return q


def dequantize_q8(q: Q8Tensor, dtype=torch.float32, stream=None) -> torch.Tensor:
    """The values of ``q`` as float32 or bfloat16 (8 significant bits at most: bfloat16 holds
    them too)."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"dtype must be float32 or bfloat16, got {dtype}")
    dev = _same_device(q)
    with _On(dev, stream) as on:
        out = torch.empty(q.shape, dtype=dtype, device=q.device)
        _check(_lowbit_lib().mt_dequantize_q8(ctypes.byref(q._c), out.data_ptr(), int(dtype == torch.bfloat16),
                                              out.shape[1], on.s))
    return out


def linear_forward_q8(x, W, bias=None, relu=False, fmt="int8", mode=MODE_DEFAULT, stream=None):
    """``linear_forward`` of the float input, and that input in 8 bits for
    ``linear_backward_q8``: (Y, checkpoint). Keep the checkpoint in x's place."""
    dev = _same_device(x, W, bias)
    with _On(dev, stream):
        return linear_forward(x, W, bias, relu=relu, mode=mode), quantize_q8(x, fmt)


def linear_weight_grad_q8(xq: Q8Tensor, dY, need_db=True, stream=None):
    """(dW, db) of Linear from the 8-bit form of its input: dW [in, out] = x^T dY and db
    [1, out] = the column sums of dY (None with need_db=False)."""
    _need_2d(dY, "dY")
    dev = _same_device(xq, dY)
    k, n = xq.shape[1], dY.shape[1]
    with _On(dev, stream) as on:
        dW = torch.empty((k, n), dtype=torch.float32, device=dY.device)
        db = torch.empty((1, n), dtype=torch.float32, device=dY.device) if need_db else None
        _check(_lowbit_lib().mt_linear_wgrad_q8(ctypes.byref(xq._c), _mat(dY), _dense(dW, k, n),
                                                _dense(db, 1, n) if need_db else None, on.s))
    return dW, db


def linear_backward_q8(xq: Q8Tensor, W, dY, mode=MODE_DEFAULT, stream=None):
    """``linear_backward`` with Linear's input in 8 bits: (dX, dW, db). dX = dY W^T does not
    use the input and is the float product in ``mode``."""
    _need_2d(dY, "dY")
    if tuple(W.shape) != (xq.shape[1], dY.shape[1]):
        raise ValueError(f"W must be [{xq.shape[1]}, {dY.shape[1]}] for a {tuple(xq.shape)} input and a {tuple(dY.shape)} "
                         f"gradient, got {tuple(W.shape)}")
    dev = _same_device(xq, W, dY)
    with _On(dev, stream):
        dX = torch.empty((dY.shape[0], W.shape[0]), dtype=torch.float32, device=dY.device)
        gemm(dY, W.t(), dX, mode=mode)
        dW, db = linear_weight_grad_q8(xq, dY)
    return dX, dW, db


# ---- 4-bit weights ----------------------------------------------------------------------

def quantize_q4(W, group=64, stream=None) -> Q4Weight:
    """A Linear weight W [in, out] in 4 bits, one bfloat16 scale (amax / 7) per ``group`` input
    features of an output feature."""
    _need_2d(W, "W")
    if group not in Q4_GROUPS:
        raise ValueError(f"group must be one of {Q4_GROUPS}, got {group}")
    dev = _same_device(W)
    k, n = W.shape
    with _On(dev, stream) as on:
        q = Q4Weight(torch.empty((n, 64 * (-(-k // Q4_SPAN))), dtype=torch.uint8, device=W.device),
                     torch.empty((n, -(-k // group)), dtype=torch.bfloat16, device=W.device), k, group)
        _check(_lowbit_lib().mt_quantize_q4(_mat(W), ctypes.byref(q._c), on.s))
    return q


def dequantize_q4(w: Q4Weight, stream=None) -> torch.Tensor:
    """The float32 weight [in, out] that ``w`` stands for."""
    dev = _same_device(w)
    with _On(dev, stream) as on:
        W = torch.empty((w.in_features, w.out_features), dtype=torch.float32, device=w.device)
        _check(_lowbit_lib().mt_dequantize_q4(ctypes.byref(w._c), _mat(W), on.s))
    return W


def linear_forward_q4(x, w: Q4Weight, bias=None, relu=False, stream=None) -> torch.Tensor:
    """``linear_forward`` with the weight in 4 bits: x [rows, in] @ W [in, out] + bias (optional
    ReLU)."""
    _need_2d(x, "x")
    dev = _same_device(x, w, bias)
    rows, n = x.shape[0], w.codes.shape[0]
    with _On(dev, stream) as on:
        Y = torch.empty((rows, n), dtype=torch.float32, device=x.device)
        _check(_lowbit_lib().mt_linear_fwd_q4(_mat(x), ctypes.byref(w._c), _opt(bias), _dense(Y, rows, n),
                                              1 if relu else 0, on.s))
    return Y
