"""The packed-batch operators in 64 bits, row by row as their formulas say, and how far a kernel may be from them.

Bounds. A value rounded once to bf16 is off by at most 2^-8 of itself (half a step). What the kernels hold in fp32
before that: a row's statistics are sums of at most 16384 squares, at most 256 of them one after another in a
lane, then six or eight pairwise steps: at most 264 x 2^-24 < 2^-15 of the sum, half of that (2^-16) of its
root; the few products and sums behind it add less than 8 x 2^-24. So each term of a result carries at most
2^-15 of its own magnitude, which the bounds below sum over the terms."""

import torch

F64 = torch.float64
TERM = 2.0**-15
ROUND = 2.0**-8


def normed(x, norm, eps, dims):
    """x (fp64) normalized over ``dims``, and the magnitude of what was subtracted and scaled."""
    if norm == "none":
        return x, x.abs()
    mu = x.mean(dims, keepdim=True) if norm == "layer_norm" else torch.zeros_like(x.mean(dims, keepdim=True))
    rs = 1.0 / ((x - mu).pow(2).mean(dims, keepdim=True) + eps).sqrt()
    return (x - mu) * rs, (x.abs() + x.abs().mean(dims, keepdim=True) * (norm == "layer_norm")) * rs


def sandwich_residual(hidden, residual, gate, weight, alpha, post_norm, eps):
    """(r, bound) of bf16(alpha residual + gate norm(hidden) weight); gate already one row per token."""
    p, mag = normed(hidden.to(F64), post_norm, eps, (1,))
    f = (gate.to(F64) if gate is not None else 1.0) * (weight.to(F64) if weight is not None else 1.0)
    r = alpha * residual.to(F64) + p * f
    return r, ROUND * r.abs() + TERM * ((alpha * residual.to(F64)).abs() + (mag * f).abs())


def sandwich_modulated(r, mul, add, norm, eps):
    x, mag = normed(r.to(F64), norm, eps, (1,))
    m = mul.to(F64) if mul is not None else 1.0
    a = add.to(F64) if add is not None else torch.zeros_like(x)
    y = x * m + a
    return y, ROUND * y.abs() + TERM * ((mag * m).abs() + a.abs())


def rope_axes(x, positions, axes, theta, pairs, norm, gamma, eps):
    """(y, bound, norms before rounding) of one of q and k [T, heads, D]."""
    T, heads, D = x.shape
    y = x.to(F64)
    if norm != "none":
        over = (2,) if norm == "rms_norm" else (1, 2)
        y = y / (y.pow(2).mean(over, keepdim=True) + eps).sqrt()
        if gamma is not None:
            y = y * gamma.to(F64).view(-1, D)
    theta = theta if isinstance(theta, (tuple, list)) else [theta] * len(axes)
    angles = [positions[:, i].to(F64)[:, None] * torch.tensor([th ** (-2 * j / d) for j in range(d // 2)], dtype=F64)
              for i, (d, th) in enumerate(zip(axes, theta)) if d]
    n = sum(axes)
    mag = y.abs()
    if n:
        ang = torch.cat(angles, 1)[:, None]
        lo = torch.arange(0, n, 2) if pairs == "interleaved" else torch.arange(n // 2)
        hi = lo + (1 if pairs == "interleaved" else n // 2)
        a, b = y[..., lo].clone(), y[..., hi].clone()
        y[..., lo], y[..., hi] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
        both = a.abs() + b.abs()
        mag[..., lo], mag[..., hi] = both, both
    return y, ROUND * y.abs() + TERM * mag, y.pow(2).sum(-1).sqrt()


def lora(base, x, a, b, which, scales, slices, row_scale=None):
    """(out, bound): every row against its own adapter (which < 0: the base itself). The first product's fp32 sum is
    off by at most K x 2^-24 of the sum of its terms' magnitudes, the second by r x 2^-24, and u enters it as two
    bf16 values, 2^-16 of it."""
    T, K = x.shape
    r = b.shape[2]
    x = x.to(F64)
    if row_scale is not None:
        x = x * row_scale.to(F64)[:, None]
    y, err = base.to(F64).clone(), torch.zeros(base.shape, dtype=F64)
    for e in range(a.shape[0]):
        rows = (which == e).nonzero()[:, 0]
        if not len(rows):
            continue
        s = 1.0 if scales is None else float(scales[e])
        at = 0
        for p, width in enumerate(slices):
            ap, bp = a[e, p * r : (p + 1) * r].to(F64), b[e, at : at + width].to(F64)
            u, mag = x[rows] @ ap.t() * s, x[rows].abs() @ ap.abs().t() * abs(s)
            y[rows, at : at + width] += u @ bp.t()
            err[rows, at : at + width] += (mag * (K + 8) * 2.0**-24 + u.abs() * (2.0**-16 + r * 2.0**-24)) @ bp.abs().t()
            at += width
    return y, ROUND * y.abs() * (which >= 0)[:, None] + err * (1 + ROUND)


def within(got, ref, bound, what=""):
    got = got.detach().to("cpu", F64)
    bad = ~((got - ref).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - ref).abs().max()), bad.nonzero()[:4].tolist())


def packed_ids(lengths, pad=0, order=None):
    """int32 ids of requests of these lengths, ``pad`` rows of none behind them."""
    ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lengths)] +
                    [torch.full((pad,), -1, dtype=torch.int32)])
    return ids
