"""Inputs and 64-bit results for the operators on the text side of packed batches."""

import math
from fractions import Fraction

import torch


def offsets(lens, device="cpu"):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32).to(device)


def bucket(d, buckets, max_distance, bidirectional):
    """The bucket of the distance ``key - query``, each border an inequality of whole numbers."""
    side = buckets // 2 if bidirectional else buckets
    if d > 0 and not bidirectional:
        return 0
    n, first = abs(d), side // 2
    if n < first:
        b = n
    else:  # first + floor(log(n / first) / log(max / first) * steps)
        steps = side - first
        b = first + max(i for i in range(steps) if i == 0 or Fraction(n, first) ** steps >= Fraction(max_distance, first) ** i)
    return b + (side if d > 0 else 0)


def bias_matrix(table, n, max_distance, bidirectional):
    """fp64 [heads, n, n]"""
    line = torch.tensor([bucket(d, table.shape[0], max_distance, bidirectional) for d in range(1 - n, n)])
    i = torch.arange(n)
    return table.double().cpu()[line[i[None, :] - i[:, None] + n - 1]].permute(2, 0, 1)


def attention(q, k, v, q_lens, k_lens, scale, bias=None):
    """fp64 [T, heads, D] on the CPU; ``bias(n)`` fp64 [heads, n, n]. Also the sum of p |v| of every output, over which the rounding
    of p to bf16 is spread."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    a = c = 0
    for n, m in zip(q_lens, k_lens):
        if n and m:
            kk = k[c : c + m].repeat_interleave(group, 1)
            vv = v[c : c + m].repeat_interleave(group, 1)
            s = torch.einsum("ihd,jhd->hij", q[a : a + n], kk) * scale
            if bias is not None:
                s = s + bias(n)
            p = torch.softmax(s, -1)
            out[a : a + n] = torch.einsum("hij,jhd->ihd", p, vv)
            size[a : a + n] = torch.einsum("hij,jhd->ihd", p, vv.abs())
        a, c = a + n, c + m
    return out, size


def attention_bound(size, out, score_size, terms):
    """The most an output may be off: p rounded to bf16 in the product and in its sum (2^-8 each way: at most 2^-8 of the
    weighted |v| in the product and as much again from the sum), the output's own rounding 2^-8; scores of fp32 products of ``terms`` terms,
    each off by at most (terms + 4) 2^-24 of the sum of their magnitudes, which moves every p by that factor, up and down; sums
    in fp32 over the keys and exp2's own error are below 2^-15 together at the lengths tested."""
    eps = 2.0**-8
    drift = math.expm1(2 * (terms + 4) * 2.0**-24 * score_size) + 2.0**-15
    return size * (2 * eps + drift) * (1 + eps) + out.abs() * eps + 1e-30


def row_blocks(x):
    """bf16 [M, K] (CPU) -> e4m3 codes and fp32 scales [M, ceil(K / 128)]."""
    M, K = x.shape
    y = torch.nn.functional.pad(x.float(), (0, -K % 128)).view(M, -1, 128)
    scale = y.abs().amax(-1).clamp_min(2.0**-100) * (1.0 / 448.0)  # times fp32(1 / 448)
    return (y / scale[..., None]).view(M, -1)[:, :K].contiguous().to(torch.float8_e4m3fn), scale


def spread(scales, rows, K):
    """Block scales at every element: [M, kb] (rows None) or [nb, kb]."""
    s = scales.double().repeat_interleave(128, 1)[:, :K]
    return s if rows is None else s.repeat_interleave(128, 0)[:rows]


def block_linear(codes, scales, w_codes, w_scales, bias, gelu):
    """fp64 [M, N], the most an output may be off, and the rms it may be off.

    The product of 128 codes is one matrix instruction. It adds them in groups of eight consecutive ones, in which every product is cut
    toward zero at 2^-13 of the power of two of the largest, and the sixteen groups in fp32 (seen on MI355X with powers of two: in a
    group 2^16 + 2^3 is exact, 2^16 + 2^2 is 2^16, whether the 2^16 is cancelled by a third product or not; in two groups both are
    exact). So a group is off by less than 7 2^-13 of its largest product, which is at most the product of the two largest magnitudes;
    the sums of the groups, the factor and the sum over kb blocks are 16 + 2 + kb fp32 operations, each off by 2^-23 at most of
    the sum of magnitudes (cut or rounded). The signs of what is cut are those of the products: uniform in [0, 2^-13) and independent it
    has the mean square 2^-26 / 3, seven of them in a group."""
    M, K = codes.shape
    N = w_codes.shape[0]
    x = codes.double() * spread(scales, None, K)
    w = w_codes.double() * spread(w_scales, N, K)
    y = x @ w.t()
    xg, wg = x.abs().view(M, K // 8, 8).amax(-1), w.abs().view(N, K // 8, 8).amax(-1)
    rest = (x.abs() @ w.abs().t()) * (18 + scales.shape[1]) * 2.0**-23
    off = (xg @ wg.t()) * 7 * 2.0**-13 + rest
    rms = ((xg.square() @ wg.square().t()) * (7 / 3) * 2.0**-26).sqrt() + rest
    if bias is not None:
        y = y + bias.double()
        off, rms = off + y.abs() * 2.0**-23, rms + y.abs() * 2.0**-23
    if gelu:  # its slope is at most 1.13; its own fp32 evaluation: exp2's argument, at most 64 here, rounded to 2^-24 of itself
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y.pow(3))))
        own = y.abs() * 2.0**-17 + 2.0**-40
        off, rms = 1.13 * off + own, 1.13 * rms + own
    return y, off * (1 + 2.0**-8) + y.abs() * 2.0**-8 + 1e-38, rms + y.abs() * 2.0**-8 + 1e-38


def check_block_linear(got, want, bound, rms):
    err = (got.double().cpu() - want).abs()
    bad = err > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(err.max()))
    assert float(err.square().mean().sqrt()) <= float(rms.square().mean().sqrt())
