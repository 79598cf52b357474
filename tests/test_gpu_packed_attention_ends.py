"""Attention over packed rows where numbers are far from one: masks of a type's lowest value wherever they stand, scores whose
exponents are past what fp32 holds to the unit, values of one sign. No result may be NaN where the formula's is a number (a
comparison with a bound does not see one: every test here asks for it)."""

import pytest
import torch

import text_ref as ref
from test_gpu_packed_attention import BIAS, CROSS, _inputs, _score_size

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


@pytest.mark.parametrize("T,H,k_heads,D,m", [(1, 2, 2, 128, 512), (3, 4, 2, 64, 300), (16, 8, 8, 128, 500), (200, 40, 40, 128, 512), (200, 90, 30, 64, 333), (129, 2, 1, 128, 65)])
def test_a_mean_of_equal_values_is_that_value(pkg, dev, T, H, k_heads, D, m):
    """Every key has the same v, so that the weights do not matter as long as their sum is that of the weights which multiply v: product and
    sum are then off by fp32's rounding of ``m`` additions alone, 512 2^-24 = 2^-15, far less than the half step of 2^-9 at which v, a bf16
    number, would be rounded to another. Scores that rise by up to 2^8 from tile to tile (a maximum that is held), and that fall."""
    g = torch.Generator().manual_seed(m)
    q = torch.rand(T, H, D, generator=g).add(0.5).to(BF16)
    v = torch.randn(1, k_heads, D, generator=g).to(BF16).expand(m, k_heads, D).contiguous()
    noise = 0.1 * torch.randn(m, k_heads, D, generator=g)
    for slope in (0.0, 0.02, 0.04, -0.04, 0.5):
        k = (noise + torch.linspace(0, slope, m)[:, None, None]).to(BF16)
        got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), ref.offsets([T], dev), ref.offsets([m], dev), scale=1.0).cpu()
        assert torch.equal(got, v[0].repeat_interleave(H // k_heads, 0).expand(T, H, D)), (slope, int((got != v[0].repeat_interleave(H // k_heads, 0)).sum()))
        if k_heads == H:
            n = min(T, m)
            table = torch.randn(32, H, generator=g).to(dev)
            got = pkg.relative_bias_attention(q[:n].to(dev), k[:n].to(dev), v[:n].to(dev), table, ref.offsets([n], dev)).cpu()
            assert torch.equal(got, v[:n]), slope


@pytest.mark.parametrize("T,H,D", [(8, 8, 128), (200, 40, 128), (200, 90, 64)])
@pytest.mark.parametrize("mean", [0.0, 4.0])
def test_the_error_is_that_of_rounded_weights(pkg, dev, T, H, D, mean):
    """The root mean square over all outputs. A weight p_j is rounded to bf16 by at most 2^-8 of itself, uniformly at worst: a mean square of
    2^-16 / 3 of p_j^2; the sum has the same rounded weights, so that the output is off by sum_j p_j d_j (v_j - o): 2^-16 / 3 of
    sum_j p_j^2 (v_j - o)^2. The output's own rounding is 2^-16 / 3 of o^2 at most. What fp32 leaves is below 2^-13 of sum_j p_j |v_j|. A mean of all values
    moves o and its rounding, and the first term not at all."""
    m = 300
    g = torch.Generator().manual_seed(T + D)
    q = torch.randn(T, H, D, generator=g).mul(2).to(BF16)
    k = torch.randn(m, H, D, generator=g).to(BF16)
    v = (torch.randn(m, H, D, generator=g) + mean).to(BF16)
    got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), ref.offsets([T], dev), ref.offsets([m], dev)).double().cpu()
    p = torch.softmax((q.double().transpose(0, 1) @ k.double().permute(1, 2, 0)) * D**-0.5, -1)  # [H, T, m]
    vd = v.double().transpose(0, 1)
    o = p @ vd
    p2 = p.square()
    spread = (p2 @ vd.square() - 2 * o * (p2 @ vd) + o.square() * p2.sum(-1, keepdim=True)).clamp_min(0)
    bar = (2.0**-16 / 3 * (spread + o.square())).sqrt() + 2.0**-13 * (p @ vd.abs())
    err = got.transpose(0, 1) - o
    assert float(err.square().mean().sqrt()) <= float(bar.square().mean().sqrt())


@pytest.mark.parametrize("T,H,D", [(3, 2, 64), (16, 8, 128), (200, 40, 128), (200, 90, 64)])
def test_late_keys_that_dominate_within_the_held_maximum(pkg, dev, T, H, D):
    """The first keys (a tile of any kind) score 0, all later ones the same 2^x with x from 0.01 to 5.5 in steps: their weights round alike, by
    up to 2^-8, which only a sum of the same rounded weights takes out again. All have the same v, which has to come out."""
    m = 512
    g = torch.Generator().manual_seed(D)
    q = torch.zeros(T, H, D, dtype=BF16)
    q[..., 3] = 1
    v = torch.randn(1, H, D, generator=g).to(BF16).expand(m, H, D).contiguous()
    for i in range(24):
        k = torch.zeros(m, H, D, dtype=BF16)
        k[128:, :, 3] = 0.01 + 0.23 * i
        got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), ref.offsets([T], dev), ref.offsets([m], dev), scale=1.0).cpu()
        assert torch.equal(got, v[:1].expand(T, H, D)), i


@pytest.mark.parametrize("case", range(len(CROSS)))
def test_cross_attention_gives_numbers(pkg, dev, case):
    q_lens, k_lens, pad, heads, k_heads, D = CROSS[case]
    q, k, v = _inputs(sum(q_lens) + pad, sum(k_lens) + 3, heads, k_heads, D, case)
    k, v = k.clone(), v.clone()
    k[sum(k_lens):], v[sum(k_lens):] = float("nan"), float("nan")  # nobody's keys
    got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), ref.offsets(q_lens, dev), ref.offsets(k_lens, dev))
    want, size = ref.attention(q, k[: sum(k_lens)], v[: sum(k_lens)], q_lens, k_lens, D**-0.5)
    _close(got, want, ref.attention_bound(size, want, _score_size(q, k[: sum(k_lens)], D**-0.5), D))


@pytest.mark.parametrize("case", range(len(BIAS)))
def test_relative_bias_gives_numbers(pkg, dev, case):
    lens, pad, heads, D, buckets, far, both, dtype = BIAS[case]
    g = torch.Generator().manual_seed(50 + case)
    qkv = torch.randn(sum(lens) + pad, 3 * heads, D, generator=g)
    qkv[:, :heads] *= D**-0.5
    slab = qkv.to(BF16).to(dev)
    table = (1.5 * torch.randn(buckets, heads, generator=g)).to(dtype)
    got = pkg.relative_bias_attention(*(slab[:, i * heads : (i + 1) * heads] for i in range(3)), table.to(dev), ref.offsets(lens, dev), max_distance=far,
                                      bidirectional=both)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("T,H,D", [(30, 2, 64), (30, 4, 128), (500, 2, 64), (500, 40, 64), (500, 40, 128)])
def test_wrong_offsets_touch_nothing_outside(pkg, dev, T, H, D):
    """Descending, negative and too large offsets, with every tensor the middle of a larger one: what is around the inputs is NaN and never read,
    what is around the output stays. (The kernel holds each offset inside its tensor.)"""
    Tk = 90
    g = torch.Generator().manual_seed(T)

    def middle(rows, fill):
        slab = torch.full((rows + 80, 3 * H, D), fill, dtype=BF16, device=dev)
        return slab, slab[40 : rows + 40, H : 2 * H]

    (_, q), (_, k), (_, v), (slab, out) = middle(T, float("nan")), middle(Tk, float("nan")), middle(Tk, float("nan")), middle(T, 7.0)
    for t in (q, k, v):
        t.copy_(torch.randn(t.shape, generator=g))
    table = torch.randn(32, H, device=dev)
    wrong = [([0, 400000, 20], [0, 90, 90]), ([T, 0, T], [90, 0, 50]), ([-5, 7, 2**31 - 1], [-(2**31), 2**31 - 1, 12]), ([0, 10, T], [80, 20, 500]),
             ([0, T, T], [0, 2**31 - 1, 2**31 - 1])]
    for qo, ko in wrong:
        qo, ko = (torch.tensor(o, dtype=torch.int32, device=dev) for o in (qo, ko))
        for call in (lambda: pkg.packed_cross_attention(q, k, v, qo, ko, out=out), lambda: pkg.relative_bias_attention(q, q, q, table, qo, out=out)):  # noqa: B023
            out.fill_(7.0)
            call()
            assert torch.isfinite(out).all()
            out.fill_(7.0)
            assert bool((slab == 7).all())
