"""Plain 64-bit forms of the low-bit operators, and bounds on what a float computation of
them may be off.

u = 2^-24 is half a step of float32. A float sum of n terms in any order is off by at most
(n - 1) u times the sum of the magnitudes (to first order), a product by u of itself.
"""
import torch

U = 2.0 ** -24
TOP = {"int8": 127.0, "e4m3": 448.0}
STORAGE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def q8_scale_bytes(x, fmt):
    """Scale bytes of x [rows, cols], found by trying every byte: the smallest b with
    amax <= top * 2^(b - 127); 255 where a block is not finite."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    pad = torch.zeros(rows, nb * 32, dtype=torch.float64)
    pad[:, :cols] = x.double()
    pad = pad.view(rows, nb, 32)
    amax = pad.abs().amax(2)
    tops = TOP[fmt] * 2.0 ** (torch.arange(255, dtype=torch.float64) - 127)
    b = (amax[..., None] > tops).sum(2)
    return torch.where(torch.isfinite(pad).all(2), b, torch.full_like(b, 255))


def q8_values(codes, scales):
    """What 8-bit codes and scale bytes stand for, in 64 bits."""
    cols = codes.shape[1]
    b = scales.double().repeat_interleave(32, 1)[:, :cols]
    v = codes.double() * torch.exp2(b - 127)
    return torch.where(b == 255, torch.full_like(v, float("nan")), v)


def q8_codes(x, b, fmt):
    """Codes of x for given scale bytes, rounded to nearest even in 64 bits."""
    u = x.double() * torch.exp2(127 - b.double().repeat_interleave(32, 1)[:, :x.shape[1]])
    if fmt == "int8":
        return torch.round(u).to(torch.int8)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(u / step) * step).float().to(torch.float8_e4m3fn)   # exact: already an e4m3 value


def q4_pack(codes, K):
    """Codes 0..15 [out, K] in the packed order, one code at a time."""
    N = codes.shape[0]
    spans = -(-K // 128)
    words = torch.zeros(N, spans * 16, dtype=torch.int64)
    full = torch.full((N, spans * 128), 8, dtype=torch.int64)
    full[:, :K] = codes
    for k in range(spans * 128):
        s, r = divmod(k, 128)
        b, r = divmod(r, 32)
        t, j = divmod(r, 8)
        words[:, s * 16 + 4 * t + b] |= full[:, k] << (4 * (j // 2) + 16 * (j % 2))
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words)
    return words.to(torch.int32).view(torch.uint8).view(N, spans * 64)


def q4_quantize(W, group):
    """(codes 0..15 [out, in], bfloat16 scales [out, groups]) of W [in, out]."""
    K, N = W.shape
    ng = -(-K // group)
    w = torch.zeros(N, ng * group)
    w[:, :K] = W.t()
    w = w.view(N, ng, group)
    s = (w.abs().amax(2) / 7).to(torch.bfloat16)
    q = torch.round(w / s.float()[..., None]).clamp(-8, 7)
    q = torch.where(s[..., None] > 0, q, torch.zeros_like(q))
    return (q.to(torch.int64) + 8).view(N, -1)[:, :K], s


def q4_weight(codes, scales, group):
    """W [in, out] in 64 bits."""
    K = codes.shape[1]
    return ((codes - 8).double() * scales.double().repeat_interleave(group, 1)[:, :K]).t()


def q4_bound(M, K, group):
    """What y = x W may be off in u times |x| |W|, W in 4 bits: relative to what each entry of x adds
    itself, as for a float product, whatever the entries beside it are.

    Up to 8 rows: the signed digits of an entry add up to 9 times it at most (a digit pair to 3.02 times
    its number, the second number of an entry to half a step of the first, 0.5 to 1 times the
    entry), and every part meets a conversion, a product with the scale, the sums over the groups,
    over four lanes, 16 warps, 5 passes and K / 1024 launches, and the bias. More rows: a tensor-core step
    aligns 17 terms to the largest and drops up to 2 u of it from each, 3 * group / 16 steps meet in
    an accumulator, then come the scale, the sum over the groups and 64 parts, and the bias."""
    few = 9 * (31 + K / group + K / 1024)
    return max(few, 102 * group / 16 + K / group + 70) if M <= 8 else 102 * group / 16 + K / group + 70


def rms_norm(x, residual, gamma, eps):
    h = x.double() + (residual.double() if residual is not None else 0)
    rstd = 1 / torch.sqrt((h * h).mean(1) + eps)
    return h, rstd, h * rstd[:, None] * gamma.double()


def rms_norm_backward(dy, h, gamma, rstd, dh):
    """(dx, dgamma) and the magnitudes that their float errors are relative to."""
    dy, h, gamma, rstd = dy.double(), h.double(), gamma.double(), rstd.double()
    xh = h * rstd[:, None]
    g = dy * gamma
    dx = rstd[:, None] * (g - xh * (g * xh).mean(1, keepdim=True))
    mag = rstd[:, None] * (g.abs() + xh.abs() * (g * xh).abs().mean(1, keepdim=True))
    if dh is not None:
        dx, mag = dx + dh.double(), mag + dh.double().abs()
    return dx, mag, (dy * xh).sum(0), (dy * xh).abs().sum(0)


def worst(err, mag):
    """The largest error in units of u times its magnitude (0 / 0 counts as 0)."""
    err, mag = err.double().abs(), mag.double().abs()
    r = torch.where(err == 0, torch.zeros_like(err), err / (U * mag))
    return float(r.max()) if r.numel() else 0.0
