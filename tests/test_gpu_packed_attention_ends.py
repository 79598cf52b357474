"""Attention over packed rows where numbers are far from one: masks of a type's lowest value wherever they stand, scores whose
exponents are past what fp32 holds to the unit, values of one sign. No result may be NaN where the formula's is a number (a
comparison with a bound does not see one: every test here asks for it)."""

import pytest
import torch

import text_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _close(got, want, bound):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), (int((~torch.isfinite(got)).sum()), (~torch.isfinite(got)).nonzero()[:4].tolist())
    bad = (got - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got - want).abs().max()))


@pytest.mark.parametrize("n,H,D", [(3, 2, 64), (150, 2, 64), (150, 110, 64), (700, 2, 128), (700, 20, 128), (700, 20, 64)])
@pytest.mark.parametrize("scale", [1.0, 0.125, 0.3])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_masks_of_the_lowest_value(pkg, dev, n, H, D, scale, dtype):
    """Everything masked (all weigh alike), and whole tiles of keys masked in front of others: what a row has seen by then must
    vanish beside the first key that is not."""
    g = torch.Generator().manual_seed(n + H)
    q, k, v = (torch.randn(n, H, D, generator=g).mul(0.3).to(BF16) for _ in range(3))
    table = torch.randn(32, H, generator=g).to(dtype)
    low = torch.finfo(dtype).min
    tables = [torch.full_like(table, low)]
    for at in ([15, 31], list(range(12, 16)), list(range(28, 32)), list(range(16))):
        tables.append(table.clone())
        tables[-1][at] = low
    score = float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * scale
    for t in tables:
        got = pkg.relative_bias_attention(q.to(dev), k.to(dev), v.to(dev), t.to(dev), ref.offsets([n], dev), scale=scale)
        want, size = ref.attention(q, k, v, [n], [n], scale, lambda m: ref.bias_matrix(t, m, 128, True))  # noqa: B023
        _close(got, want, ref.attention_bound(size, want, score + float(table.abs().max()), D))


@pytest.mark.parametrize("T,H", [(3, 2), (200, 4), (200, 60)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("top", [2.0**20, -(2.0**20), 2.0**22, 2.0**34, -(2.0**34), 2.0**90])
def test_scores_past_the_unit(pkg, dev, T, H, D, top):
    """Scores that are whole numbers around ``top``: two numbers of q are one and the rest zero, k's are ``top`` and 0 to 5 (far above 2^24 just
    ``top``), so that their sums are exact in fp32. What is left is the rounding of the weights to bf16 (2^-8, and as much from their
    sum) and the output's."""
    g = torch.Generator().manual_seed(T + H)
    m = 300
    q = torch.zeros(T, H, D, dtype=BF16)
    q[..., 0], q[..., 48] = 1, 1
    k = torch.zeros(m, H, D, dtype=BF16)
    k[..., 0] = top
    if abs(top) < 2.0**24:
        k[..., 48] = torch.randint(0, 6, (m, H), generator=g).to(BF16)
    v = torch.randn(m, H, D, generator=g).to(BF16)
    got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), ref.offsets([T], dev), ref.offsets([m], dev), scale=1.0)
    p = torch.softmax(k[..., 48].double(), 0)  # [m, H]
    want = (p[..., None] * v.double()).sum(0)
    size = (p[..., None] * v.double().abs()).sum(0)
    eps = 2.0**-8
    # exp2, sums and the factor that joins tiles: 2^-15 together, and the exponent's own rounding, 8 2^-24, within it
    bound = size * (2 * eps + 2.0**-15) * (1 + eps) + want.abs() * eps
    _close(got, want.expand(T, H, D), bound.expand(T, H, D))


@pytest.mark.parametrize("T,H,D", [(3, 2, 64), (200, 4, 128), (200, 60, 64)])
def test_one_key_above_all(pkg, dev, T, H, D):
    """Scores of 2^32 and more, the largest of them in any tile: its value alone is left, as it is, and the mean of two that share it."""
    m = 300
    g = torch.Generator().manual_seed(D)
    q = torch.zeros(T, H, D, dtype=BF16)
    q[..., 0] = 2.0**40
    v = torch.randn(m, H, D, generator=g).to(BF16)
    for at in ([0], [299], [140], [0, 280], [40, 41]):
        k = torch.zeros(m, H, D, dtype=BF16)
        k[..., 0] = torch.randint(-100, 100, (m, 1), generator=g).to(BF16)
        k[at, :, 0] = 101
        got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), ref.offsets([T], dev), ref.offsets([m], dev), scale=1.0)
        want = v[at].double().mean(0)
        _close(got, want.expand(T, H, D), (want.abs() * 2.0**-8).expand(T, H, D))
