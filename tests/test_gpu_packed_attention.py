"""Attention over packed rows (packed_cross_attention, relative_bias_attention) against 64-bit results."""

import pytest
import torch

import text_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _inputs(T, Tk, heads, k_heads, D, seed, q_std=2.0):
    g = torch.Generator().manual_seed(seed)
    q = (q_std * torch.randn(T, heads, D, generator=g)).to(BF16)
    kv = torch.randn(max(Tk, 1), 2 * k_heads, D, generator=g).to(BF16)
    return q, kv[:Tk, :k_heads], kv[:Tk, k_heads:]


def _score_size(q, k, scale):
    """The largest sum of |q| |k| of any score."""
    return float((q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * scale) if q.numel() and k.numel() else 0.0


def _check(got, q, k, v, q_lens, k_lens, scale, bias=None, bias_size=0.0):
    want, size = ref.attention(q, k, v, q_lens, k_lens, scale, bias)
    bound = ref.attention_bound(size, want, _score_size(q, k, scale) + bias_size, q.shape[-1])
    bad = (got.double().cpu() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got.double().cpu() - want).abs().max()))


CROSS = [
    # rows of the requests, keys of the requests, rows behind, heads, key heads, head_dim
    ([1], [1], 0, 1, 1, 64),
    ([1], [1], 0, 1, 1, 128),
    ([16], [512], 0, 40, 40, 128),
    ([1, 1, 1, 1], [7, 0, 300, 64], 3, 4, 4, 128),
    ([129], [65], 0, 2, 1, 128),
    ([0, 40, 0, 127, 128], [5, 63, 9, 64, 0], 70, 3, 3, 128),
    ([33, 31, 32], [129, 127, 128], 1, 6, 2, 64),
    ([200, 3, 500], [33, 700, 97], 5, 8, 2, 64),
    ([64] * 70, [3 + i for i in range(70)], 9, 2, 2, 64),
    ([2] * 130, [i % 5 for i in range(130)], 0, 2, 2, 128),
    ([1000, 24], [2000, 1], 0, 2, 2, 128),
]


@pytest.mark.parametrize("case", range(len(CROSS)))
def test_cross_attention(pkg, dev, case):
    q_lens, k_lens, pad, heads, k_heads, D = CROSS[case]
    q, k, v = _inputs(sum(q_lens) + pad, sum(k_lens) + 3, heads, k_heads, D, case)
    k, v = k.clone(), v.clone()
    k[sum(k_lens):], v[sum(k_lens):] = float("nan"), float("nan")  # nobody's keys
    got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), ref.offsets(q_lens, dev), ref.offsets(k_lens, dev))
    _check(got, q, k[: sum(k_lens)], v[: sum(k_lens)], q_lens, k_lens, D**-0.5)
    if pad:
        assert not got[-pad:].any()


BIAS = [
    # prompts, rows behind, heads, head_dim, buckets, max_distance, both directions, dtype of the table
    ([1], 0, 1, 64, 32, 128, True, torch.float32),
    ([12], 0, 64, 64, 32, 128, True, torch.float32),
    ([40, 1, 0, 300], 5, 5, 64, 32, 128, True, BF16),
    ([511, 130], 0, 3, 128, 20, 250, True, torch.float32),
    ([700], 1, 2, 64, 8, 20, True, torch.float32),
    ([257, 64], 0, 2, 64, 32, 128, False, torch.float32),
    ([5, 6, 7], 0, 2, 128, 4, 3, True, BF16),
    ([1500], 0, 1, 64, 256, 1024, True, torch.float32),
]


@pytest.mark.parametrize("case", range(len(BIAS)))
def test_relative_bias(pkg, dev, case):
    lens, pad, heads, D, buckets, far, both, dtype = BIAS[case]
    g = torch.Generator().manual_seed(50 + case)
    qkv = torch.randn(sum(lens) + pad, 3 * heads, D, generator=g)
    qkv[:, :heads] *= D**-0.5
    qkv = qkv.to(BF16)
    table = (1.5 * torch.randn(buckets, heads, generator=g)).to(dtype)
    slab = qkv.to(dev)
    parts = [slab[:, i * heads : (i + 1) * heads] for i in range(3)]
    got = pkg.relative_bias_attention(*parts, table.to(dev), ref.offsets(lens, dev), max_distance=far, bidirectional=both)
    q, k, v = (qkv[: sum(lens), i * heads : (i + 1) * heads] for i in range(3))
    _check(got[: sum(lens)], q, k, v, lens, lens, 1.0, lambda n: ref.bias_matrix(table, n, far, both), float(table.abs().max()))
    assert not got[sum(lens):].any()
