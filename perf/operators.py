"""Cases that measure the low-bit operators around Linear: the RMS norm that makes its
input (with an 8-bit output), the 8-bit activation checkpoint that its weight gradient
reads, and Linear with 4-bit weights.

``run`` has two forms on the same state: the plain one in elementary torch operations
(``own`` false), and the calls that a user of ``minitensor_b200`` makes (``own`` true).

8 bits: a row is cut into blocks of 32 features, the last one shorter. A block has one scale byte
b and stands for code * 2^(b - 127); b is the smallest for which no code is clipped.
4 bits: column n of a Linear weight [in, out] is row n of the codes. A code c of 0..15 stands
for (c - 8) * scale, with one bfloat16 scale for each `group` input features of that row. Rows
are padded with code 8 to spans of 128 codes (64 bytes); the 32-bit word 4 t + b of a span holds
the codes 32 b + 8 t + (0..7), even ones in its low half, odd ones in its high half.
"""
import math

import torch

own = False

EPS = 1e-6
TOP = {"int8": 127.0, "e4m3": 448.0}
STORED = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ---- cases ------------------------------------------------------------------------------

def listed():
    return [
        # The norm before one decoded token's Linear, with its residual addition: latency.
        {"name": "norm, one token", "op": "norm", "rows": 1, "features": 4096, "residual": True, "fmt": ""},
        # The norm of a training step, which saves its output as the Linear's 8-bit checkpoint.
        {"name": "norm, training step, int8", "op": "norm", "rows": 8192, "features": 4096, "residual": True,
         "fmt": "int8"},
        # Odd sizes, no residual stream (the first norm of a model), the floating 8-bit type.
        {"name": "norm, odd rows, e4m3", "op": "norm", "rows": 1027, "features": 5001, "residual": False,
         "fmt": "e4m3"},
        # The backward pass of the training step's norm; the residual stream has a gradient too.
        {"name": "norm, backward", "op": "norm_grad", "rows": 8192, "features": 4096, "residual": True},
        # A Linear's input saved for the backward pass, and read back.
        {"name": "checkpoint, save and read", "op": "save", "rows": 8192, "features": 4096, "fmt": "int8"},
        # Weight and bias gradient of the repository's Linear benchmark (batch 256, 1024 -> 4096).
        {"name": "weight grad, 256 rows", "op": "wgrad", "rows": 256, "in": 1024, "out": 4096, "fmt": "int8"},
        # Weight and bias gradient at the size of the repository's large GEMM benchmark.
        {"name": "weight grad, 8192 rows", "op": "wgrad", "rows": 8192, "in": 8192, "out": 8192, "fmt": "int8"},
        # Odd sizes in every direction, the floating 8-bit type.
        {"name": "weight grad, odd sizes, e4m3", "op": "wgrad", "rows": 777, "in": 1001, "out": 1303, "fmt": "e4m3"},
        # One decoded token through a square projection.
        {"name": "4 bits, one token", "op": "q4", "rows": 1, "in": 4096, "out": 4096, "group": 64, "bias": False},
        # One decoded token through a wide layer: more weight bytes than the L2 cache holds.
        {"name": "4 bits, one token, wide", "op": "q4", "rows": 1, "in": 8192, "out": 32768, "group": 128,
         "bias": False},
        # A small batch of sequences, one token each, odd sizes and a bias.
        {"name": "4 bits, 21 tokens, odd sizes", "op": "q4", "rows": 21, "in": 4001, "out": 11003, "group": 32,
         "bias": True},
        # A prompt.
        {"name": "4 bits, prompt", "op": "q4", "rows": 2048, "in": 4096, "out": 8192, "group": 64, "bias": True},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of its range; every third one is a multiple of 64."""
    low, high = max(1, int(low)), max(1, int(high))
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))
    n = min(max(n, low), max(low, high))
    return max(low, n // 64 * 64) if n >= 64 and rng.random() < 0.34 else n


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "save", "wgrad", "wgrad", "q4", "q4", "q4"])
    if op in ("norm", "norm_grad", "save"):
        features = _size(rng, 64, 16384)
        rows = _size(rng, 1, min(16384, 8192 * 4096 // features))
        case = {"op": op, "rows": rows, "features": features}
        if op != "save":
            case["residual"] = rng.random() < 0.5
        if op == "norm":
            case["fmt"] = rng.choice(["", "int8", "e4m3"])
        if op == "save":
            case["fmt"] = rng.choice(["int8", "e4m3"])
        return case
    if op == "wgrad":
        rows, inner = _size(rng, 16, 16384), _size(rng, 64, 8192)
        return {"op": op, "rows": rows, "in": inner, "out": _size(rng, 64, 8192), "fmt": rng.choice(["int8", "e4m3"])}
    inner, outer = _size(rng, 128, 8192), _size(rng, 128, 16384)
    rows = _size(rng, 1, min(2048, 2048 * 4096 * 8192 // (inner * outer)))
    return {"op": op, "rows": rows if rng.random() < 0.7 else 1 + rows % 8, "in": inner, "out": outer,
            "group": rng.choice([32, 64, 128]), "bias": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------

def _activations(g, rows, features):
    """Hidden states: about normal, with some features much larger than the rest."""
    x = torch.randn(rows, features, generator=g, device="cuda")
    big = torch.randn(features, generator=g, device="cuda")
    return x * torch.exp(0.5 * big + 2.0 * (big > 2.6))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows = case["op"], case["rows"]
    s = {"case": case}
    if op in ("norm", "norm_grad", "save"):
        s["x"] = _activations(g, rows, case["features"])
        s["gamma"] = 1 + 0.1 * torch.randn(case["features"], generator=g, device="cuda")
        if op == "norm" and case["residual"]:
            s["residual"] = 3 * torch.randn(rows, case["features"], generator=g, device="cuda")
        if op == "norm_grad":
            s["dy"] = 1e-3 * torch.randn(rows, case["features"], generator=g, device="cuda")
            s["dh"] = 1e-3 * torch.randn(rows, case["features"], generator=g, device="cuda") if case["residual"] else None
            s["rstd"] = torch.rsqrt(s["x"].double().square().mean(1) + EPS).float()
    elif op == "wgrad":
        s["codes"], s["scales"] = _encode8(_activations(g, rows, case["in"]), case["fmt"])
        s["dy"] = torch.randn(rows, case["out"], generator=g, device="cuda")
        s["dy"] *= 1e-3 * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
        if own:
            from minitensor_b200 import Q8Tensor
            s["q"] = Q8Tensor(s["codes"], s["scales"])
    else:
        w = torch.randn(case["out"], case["in"], generator=g, device="cuda") * case["in"] ** -0.5
        s["codes"], s["scales"] = _encode4(w, case["group"])
        del w
        s["x"] = _activations(g, rows, case["in"])
        s["b"] = torch.randn(case["out"], generator=g, device="cuda") if case["bias"] else None
        if own:
            from minitensor_b200 import Q4Weight
            s["w"] = Q4Weight(s["codes"], s["scales"], case["in"], case["group"])
    return s


# ---- the 8-bit and the 4-bit form -------------------------------------------------------

def _blocks(x):
    """[rows, features] as [rows, blocks, 32], zeros behind the last feature."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32)


def _encode8(x, fmt):
    v = _blocks(x)
    m, e = torch.frexp(v.abs().amax(2))                              # amax = m * 2^e, 0.5 <= m < 1
    tm, te = math.frexp(TOP[fmt])
    b = torch.where(m > 0, e - te + (m > tm).int() + 127, 0).clamp(0, 254)   # smallest with amax <= top * 2^(b - 127)
    v = torch.ldexp(v, (127 - b)[..., None])
    codes = (v.round() if fmt == "int8" else v).to(STORED[fmt])
    return codes.view(x.shape[0], -1)[:, :x.shape[1]].contiguous(), b.to(torch.uint8)


def _decode8(codes, scales):
    v = torch.ldexp(_blocks(codes.float()), (scales.int() - 127)[..., None])
    return v.view(codes.shape[0], -1)[:, :codes.shape[1]]


def _encode4(w, group):
    """Rows of `w` [out, in] as packed codes [out, 64 * spans] and bfloat16 scales."""
    n, k = w.shape
    groups = torch.nn.functional.pad(w, (0, -k % group)).reshape(n, -1, group)
    s = (groups.abs().amax(2) / 7).to(torch.bfloat16)
    c = torch.where(s[..., None] > 0, torch.round(groups / s.float()[..., None]), 0.0).clamp(-8, 7).int() + 8
    c = c.reshape(n, -1)[:, :k]
    c = torch.nn.functional.pad(c, (0, -k % 128), value=8).reshape(n, -1, 4, 4, 4, 2)   # span, b, t, pair, odd
    at = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], device=w.device)
    words = (c.long() << at).sum((4, 5)).transpose(2, 3)                             # span, t, b
    return words.to(torch.int32).contiguous().view(n, -1).view(torch.uint8), s


def _decode4(codes, scales, k, group):
    n = codes.shape[0]
    words = codes.view(torch.int32).view(n, -1, 4, 4).transpose(2, 3)                # span, b, t
    at = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=codes.device, dtype=torch.int32)
    c = ((words[..., None] >> at) & 15).reshape(n, -1)[:, :k]
    return (c - 8).float() * scales.float().repeat_interleave(group, 1)[:, :k]


# ---- one pass ---------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        h = s["x"] + s["residual"] if case["residual"] else s["x"]
        rstd = 1 / torch.sqrt((h * h).mean(1) + EPS)
        out = {"y": h * rstd[:, None] * s["gamma"], "rstd": rstd}
        if case["residual"]:
            out["h"] = h
        if case["fmt"]:
            out["saved"] = _decode8(*_encode8(out["y"], case["fmt"])).to(torch.bfloat16)
        return out
    if op == "norm_grad":
        xhat = s["x"] * s["rstd"][:, None]
        g = s["dy"] * s["gamma"]
        dx = (g - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        if case["residual"]:
            dx = dx + s["dh"]
        return {"dx": dx, "dgamma": (s["dy"] * xhat).sum(0)}
    if op == "save":
        return {"saved": _decode8(*_encode8(s["x"], case["fmt"])).to(torch.bfloat16)}
    if op == "wgrad":
        return {"dw": _decode8(s["codes"], s["scales"]).t() @ s["dy"], "db": s["dy"].sum(0, keepdim=True)}
    y = s["x"] @ _decode4(s["codes"], s["scales"], case["in"], case["group"]).t()
    return {"y": y + s["b"] if case["bias"] else y}


def _run_own(s):
    import minitensor_b200 as mt
    case = s["case"]
    op = case["op"]
    if op == "norm":
        r = mt.rms_norm(s["x"], s["gamma"], residual=s.get("residual"), eps=EPS, q8=case["fmt"] or None)
        out = {"y": r.y, "rstd": r.rstd}
        if case["residual"]:
            out["h"] = r.h
        if case["fmt"]:
            out["saved"] = mt.dequantize_q8(r.q8, dtype=torch.bfloat16)
        return out
    if op == "norm_grad":
        dx, dgamma = mt.rms_norm_backward(s["dy"], s["x"], s["gamma"], s["rstd"], dh=s["dh"])
        return {"dx": dx, "dgamma": dgamma}
    if op == "save":
        return {"saved": mt.dequantize_q8(mt.quantize_q8(s["x"], case["fmt"]), dtype=torch.bfloat16)}
    if op == "wgrad":
        dw, db = mt.linear_weight_grad_q8(s["q"], s["dy"])
        return {"dw": dw, "db": db}
    return {"y": mt.linear_forward_q4(s["x"], s["w"], bias=s["b"])}


# ---- floors and 64-bit values -----------------------------------------------------------

def work(case):
    op, m = case["op"], case["rows"]
    if op in ("norm", "norm_grad", "save"):
        k = case["features"]
        n = m * k
        if op == "norm":
            b = 4 * n * (4 if case["residual"] else 2) + 4 * k + 4 * m + (2 * n if case["fmt"] else 0)
            return {"bytes": b, "flops": 5 * n}
        if op == "norm_grad":
            return {"bytes": 4 * n * (4 if case["residual"] else 3) + 8 * k + 4 * m, "flops": 9 * n}
        return {"bytes": 4 * n + 2 * n, "flops": 3 * n}
    k, n = case["in"], case["out"]
    if op == "wgrad":
        return {"bytes": m * k + m * -(-k // 32) + 4 * m * n + 4 * k * n + 4 * n, "flops": 2 * m * k * n + m * n}
    groups = -(-k // case["group"])
    return {"bytes": n * 64 * -(-k // 128) + 2 * n * groups + 4 * m * k + 4 * m * n + (4 * n if case["bias"] else 0),
            "flops": 2 * m * k * n}


def _value8(x, fmt):
    """The value that each entry of `x` (64 bits) is held as, block by block of 32."""
    rows, k = x.shape
    full = torch.zeros(rows, -(-k // 32) * 32, dtype=torch.float64, device=x.device)
    full[:, :k] = x
    full = full.reshape(rows, -1, 32)
    top = full.abs().max(dim=2, keepdim=True).values
    step = torch.exp2(torch.ceil(torch.log2(top.clamp_min(1e-300) / TOP[fmt])).clamp_min(-127))
    step = torch.where(step * TOP[fmt] < top, step * 2, step)
    step = torch.where((step / 2 * TOP[fmt] >= top) & (step > 2.0 ** -127), step / 2, step)
    u = full / step
    if fmt == "int8":
        u = torch.round(u)
    else:   # 3 bits behind the leading one, 2^-9 at the least
        ulp = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
        u = torch.round(u / ulp) * ulp
    return (u * step).reshape(rows, -1)[:, :k]


def _held8(s):
    codes, scales = s["codes"], s["scales"]
    block = torch.arange(codes.shape[1], device=codes.device) // 32
    return codes.double() * torch.exp2(scales.double() - 127)[:, block]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double()
        if case["residual"]:
            h = h + s["residual"].double()
        rstd = (h.pow(2).sum(1) / h.shape[1] + EPS).rsqrt()
        y = torch.einsum("mk,m,k->mk", h, rstd, s["gamma"].double())
        out = {"y": y, "rstd": rstd}
        if case["residual"]:
            out["h"] = h
        if case["fmt"]:
            out["saved"] = _value8(y, case["fmt"])
        return out
    if op == "norm_grad":
        h, r, gamma, dy = (s[k].double() for k in ("x", "rstd", "gamma", "dy"))
        dot = torch.einsum("mk,mk,k->m", dy, h, gamma)
        dx = torch.einsum("mk,k,m->mk", dy, gamma, r) - h * (dot * r.pow(3) / h.shape[1]).unsqueeze(1)
        return {"dx": dx + s["dh"].double() if case["residual"] else dx, "dgamma": torch.einsum("mk,mk,m->k", dy, h, r)}
    if op == "save":
        return {"saved": _value8(s["x"].double(), case["fmt"])}
    if op == "wgrad":
        dy = s["dy"].double()
        return {"dw": torch.einsum("mk,mn->kn", _held8(s), dy), "db": torch.einsum("mn->n", dy).unsqueeze(0)}
    k, group = case["in"], case["group"]
    j = torch.arange(k, device="cuda")
    span, b, t, i = j // 128, j % 128 // 32, j % 32 // 8, j % 8
    word = s["codes"].view(torch.int32)[:, span * 16 + t * 4 + b].long()
    c = word.bitwise_right_shift(4 * (i // 2) + 16 * (i % 2)).bitwise_and(15) - 8
    w = c.double() * s["scales"].double()[:, j // group]
    y = torch.einsum("mk,nk->mn", s["x"].double(), w)
    return {"y": y + s["b"].double() if case["bias"] else y}
