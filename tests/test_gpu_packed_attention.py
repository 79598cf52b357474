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
    # as many heads as take tiles of 128 rows
    ([129], [65], 0, 60, 30, 128),
    ([33, 31, 32], [129, 127, 128], 1, 90, 30, 64),
    ([200, 3, 500], [33, 700, 97], 5, 24, 6, 64),
    ([1000, 24], [2000, 1], 0, 10, 10, 128),
    ([100, 200, 0], [0, 300, 128], 30, 40, 8, 128),
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
    # as many heads as take tiles of 128 rows
    ([40, 1, 0, 300], 5, 40, 64, 32, 128, True, BF16),
    ([511, 130], 0, 15, 128, 20, 250, True, torch.float32),
    ([700], 1, 30, 64, 8, 20, True, torch.float32),
    ([257, 64], 0, 48, 64, 32, 128, False, torch.float32),
    ([1500], 0, 12, 64, 256, 1024, True, torch.float32),
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


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens,pad,heads", [([3, 1, 9], [40, 0, 7], 4, 4), ([200, 90], [130, 65], 7, 4), ([200, 90], [130, 65], 7, 50)])
def test_codes_are_those_of_the_bf16_output(pkg, dev, q_lens, k_lens, pad, heads, D):
    q, k, v = (t.to(dev) for t in _inputs(sum(q_lens) + pad, sum(k_lens), heads, heads // 2, D, 7))
    qo, ko = ref.offsets(q_lens, dev), ref.offsets(k_lens, dev)
    out = pkg.packed_cross_attention(q, k, v, qo, ko)
    got = pkg.packed_cross_attention(q, k, v, qo, ko, quant="mx")
    want = pkg.adaln_kernels.adaln_quant_2d(out.view(out.shape[0], -1), None, None, eps=0.0, norm_type="none", quant="mx")
    assert torch.equal(got.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("T", [5, 300])
def test_given_outputs_and_layouts(pkg, dev, T):
    """A given output keeps the rows behind the last request and may be q; heads and rows of the inputs in any order."""
    lens, k_lens, H, D = [T - 4, 1], [70, 33], 4, 64
    q, k, v = (t.to(dev) for t in _inputs(T, 103, H, H, D, T))
    qo, ko = ref.offsets(lens, dev), ref.offsets(k_lens, dev)
    want = pkg.packed_cross_attention(q, k, v, qo, ko)
    out = torch.full((T, 2 * H, D), 7.0, dtype=BF16, device=dev)
    got = pkg.packed_cross_attention(q, k, v, qo, ko, out=out[:, H:])
    assert got.data_ptr() == out[:, H:].data_ptr()
    assert torch.equal(got[: T - 3], want[: T - 3]) and bool((out[T - 3 :] == 7).all()) and bool((out[:, :H] == 7).all())
    slab = torch.cat([q, q], 1)
    pkg.packed_cross_attention(slab[:, :H], k, v, qo, ko, out=slab[:, :H])
    assert torch.equal(slab[: T - 3, :H], want[: T - 3]) and torch.equal(slab[:, H:], q) and torch.equal(slab[T - 3 :, :H], q[T - 3 :])
    head_major = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (q, k, v)]
    assert torch.equal(pkg.packed_cross_attention(*head_major, qo, ko), want)
    table = torch.randn(32, H, device=dev)
    bias = pkg.relative_bias_attention(q, q, q, table, qo)
    assert torch.equal(pkg.relative_bias_attention(*(head_major[0],) * 3, table, qo), bias)
    again = q.clone()
    pkg.relative_bias_attention(again, q, q, table, qo, out=again)
    assert torch.equal(again[: T - 3], bias[: T - 3]) and torch.equal(again[T - 3 :], q[T - 3 :])


@pytest.mark.parametrize("T,H,D", [(4, 2, 128), (200, 2, 128), (200, 40, 128), (4, 2, 64), (200, 90, 64)])
def test_scores_at_the_ends_of_their_range(pkg, dev, T, H, D):
    """A maximum that rises with every tile, scores of ten thousand, of minus infinity and of NaN."""
    g = torch.Generator().manual_seed(T)
    m = 300
    q = torch.rand(T, H, D, generator=g).add(0.5).to(BF16)
    k = torch.randn(m, H, D, generator=g).to(BF16)
    v = torch.randn(m, H, D, generator=g).to(BF16)
    k = (k.float() * 0.1 + torch.linspace(-8, 8, m)[:, None, None]).to(BF16)  # rising
    one = [ref.offsets([T], dev), ref.offsets([m], dev)]

    def check(q, k, v, scale):
        got = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), *one, scale=scale)
        _check(got, q, k, v, [T], [m], scale)

    check(q, k, v, 1.0)
    check(q, k.flip(0), v, 1.0)
    check((q.float() * 8).to(BF16), k, v, 2.0)
    check(q, k, v, 2.0**-20)
    low = k.clone()
    low[7], low[290] = float("-inf"), float("-inf")  # (q is positive: their scores are -inf)
    got = pkg.packed_cross_attention(q.to(dev), low.to(dev), v.to(dev), *one, scale=0.05)
    keep = [i for i in range(m) if i not in (7, 290)]
    _check(got, q, k[keep], v[keep], [T], [m - 2], 0.05)
    low[:] = float("-inf")  # no key at all
    assert not pkg.packed_cross_attention(q.to(dev), low.to(dev), v.to(dev), *one, scale=0.05).any()
    bad = q.clone()
    bad[1, 0, 3], bad[2, 1] = float("nan"), float("inf")
    got = pkg.packed_cross_attention(bad.to(dev), k.to(dev), v.to(dev), *one, scale=0.05).cpu()
    want = pkg.packed_cross_attention(q.to(dev), k.to(dev), v.to(dev), *one, scale=0.05).cpu()
    assert got[1, 0].isnan().all() and got[2, 1].isnan().all()
    got[1, 0], got[2, 1] = want[1, 0], want[2, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("n,H", [(3, 2), (150, 2), (150, 110)])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_tables_that_mask(pkg, dev, n, H, dtype):
    """A type's lowest value as a mask, which weighs alike where nothing else is there, and minus infinity, which leaves out."""
    g = torch.Generator().manual_seed(n)
    D = 64
    q, k, v = (torch.randn(n, H, D, generator=g).mul(0.3).to(BF16) for _ in range(3))
    table = torch.randn(32, H, generator=g).to(dtype)

    def check(table, size):
        got = pkg.relative_bias_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), ref.offsets([n], dev))
        _check(got, q, k, v, [n], [n], 1.0, lambda m: ref.bias_matrix(table, m, 128, True), size)

    lowest = table.clone()
    lowest[16:] = torch.finfo(dtype).min  # nothing behind the query
    check(lowest, float(table.float().abs().max()))
    lowest[:] = torch.finfo(dtype).min  # nothing anywhere: all weigh alike
    check(lowest, 0.0)
    out = table.clone()
    out[0] = float("-inf")  # not itself
    out[20:] = float("-inf")
    if n > 1:
        check(out, float(table.float().abs().max()))
    far = table.float()
    far[15], far[31] = -20000.0, 20000.0  # a far bias too large to be taken off the maximum
    far = far.to(dtype)
    check(far, 20000.0 if n > 91 else float(table.float().abs().max()))


def test_no_rows_no_keys_no_requests(pkg, dev):
    q, k, v = (t.to(dev) for t in _inputs(6, 10, 2, 2, 64, 1))
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    assert not pkg.packed_cross_attention(q, k, v, none, none).any()
    assert pkg.packed_cross_attention(q[:0], k, v, none, none).shape == (0, 2, 64)
    qo, ko = ref.offsets([6], dev), ref.offsets([0], dev)
    assert not pkg.packed_cross_attention(q, k[:0], v[:0], qo, ko).any()
    table = torch.randn(32, 2, device=dev)
    assert not pkg.relative_bias_attention(q, q, q, table, none).any()
    assert pkg.relative_bias_attention(q[:0], q[:0], q[:0], table, none).shape == (0, 2, 64)
    empty = pkg.packed_cross_attention(q[:0], k, v, none, none, quant="mx")
    assert empty.codes.shape == (0, 128) and empty.scales.shape == (0, 4)


@pytest.mark.parametrize("T,H", [(30, 2), (500, 2), (500, 40)])
def test_offsets_that_are_wrong_stay_inside(pkg, dev, T, H):
    """Descending, negative and too large: some rows or other, no access out of bounds (the kernel holds every offset inside its tensor)."""
    q, k, v = (t.to(dev) for t in _inputs(T, 90, H, H, 64, 3))
    for qo, ko in (([0, 400000, 20], [0, 90, 90]), ([T, 0, T], [90, 0, 50]), ([-5, 7, 2**31 - 1], [-(2**31), 2**31 - 1, 12]), ([0, 10, T], [80, 20, 500])):
        out = pkg.packed_cross_attention(q, k, v, torch.tensor(qo, dtype=torch.int32, device=dev), torch.tensor(ko, dtype=torch.int32, device=dev))
        torch.cuda.synchronize()
        assert out.shape == q.shape
    pkg.relative_bias_attention(q, q, q, torch.randn(32, H, device=dev), torch.tensor([3, 400000, -1], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()


def test_rows_far_apart(pkg, dev):
    """Elements beyond 2^31 from the tensor's first."""
    rows, ss, H, D = 1100, 1 << 21, 20, 64
    slab = torch.empty(rows, ss, dtype=BF16, device=dev)
    q, k, v = (slab[:, i * H * D : (i + 1) * H * D].view(rows, H, D) for i in range(3))
    small = [t.to(dev) for t in _inputs(rows, rows, H, H, D, 9)]
    for t, s in zip((q, k, v), small):
        t.copy_(s)
    for lens in ([700, 400], [20] * 55):
        o = ref.offsets(lens, dev)
        assert torch.equal(pkg.packed_cross_attention(q, k, v, o, o), pkg.packed_cross_attention(*small, o, o))
    del slab, q, k, v
    torch.cuda.empty_cache()


def test_other_streams_and_replayed_graphs(pkg, dev):
    """On a stream of its own beside other calls, and captured: replays follow offsets, queries and tables that were changed in place."""
    q, k, v = (t.to(dev) for t in _inputs(300, 200, 4, 4, 64, 5))
    table = torch.randn(32, 4, device=dev)
    qo, ko, bo = ref.offsets([100, 150], dev), ref.offsets([64, 130], dev), ref.offsets([3, 200, 90], dev)
    eager = lambda: (pkg.packed_cross_attention(q, k, v, qo, ko), pkg.relative_bias_attention(q, q, q, table, bo))  # noqa: E731
    want = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = eager()
    mine = eager()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, other, mine))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(eager())
    for a, b in (([100, 150], [64, 130]), ([1, 299], [0, 200]), ([200, 0], [3, 9])):
        qo.copy_(ref.offsets(a))
        ko.copy_(ref.offsets(b))
        bo.copy_(ref.offsets([a[0], 50, 20]))
        table.mul_(-1.5)
        q.mul_(0.75)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = eager()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for out in outs for x, y in zip(out, want))
