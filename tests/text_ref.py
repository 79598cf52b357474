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
