"""Q/K norm and rotary positions on several axes given per token, against 64 bits."""

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _inputs(T, hq, hk, D, norm, seed, axes=3, far=200):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(T, hq, D, generator=g).to(torch.bfloat16)
    k = (2 * torch.randn(T, hk, D, generator=g)).to(torch.bfloat16)
    pos = torch.randint(0, far, (T, axes), generator=g, dtype=torch.int32)
    n = {"none": 0, "rms_norm": 1}.get(norm)
    gam = [None if n == 0 else 1 + 0.1 * torch.randn((h if n is None else n) * D, generator=g) for h in (hq, hk)]
    return q, k, pos, *gam


def _check(pkg, dev, q, k, pos, gq, gk, ids=None, axes=(44, 42, 42), theta=10000.0, pairs="interleaved", norm="none", eps=EPS):
    to = lambda v: None if v is None else v.to(dev)  # noqa: E731
    R = 1 if ids is None else int(ids.max()) + 1
    oq, ok, kmax = pkg.qk_norm_rope_axes(to(q), to(k), to(pos), axes=axes, theta=theta, rope_pairs=pairs, norm=norm, q_gamma=to(gq),
                                         k_gamma=to(gk), eps=eps, request_ids=to(ids), requests=None if ids is None else R,
                                         want_max=True)
    ids = torch.zeros(len(q), dtype=torch.int32) if ids is None else ids
    live = ids >= 0
    for x, gamma, got in ((q, gq, oq), (k, gk, ok)):
        want, bound, norms = ref.rope_axes(x, pos, axes, theta, pairs, norm, gamma, eps)
        ref.within(got[live.to(dev)], want[live], bound[live], "q or k")
        assert not got[~live.to(dev)].any()
    for i in range(R):
        mine = (ids == i)
        want = norms[mine].amax(0) if mine.any() else torch.zeros(k.shape[1], dtype=torch.float64)
        ref.within(kmax[i], want * (1 + 2.0**-8), want * 2 * ref.TERM, "kmax")
        if mine.any():  # a bound on the rows as they were written
            assert bool((ok[mine.to(dev)].double().pow(2).sum(-1).sqrt().amax(0) <= kmax[i]).all())
    return oq, ok, kmax


@pytest.mark.parametrize("norm", ["none", "rms_norm", "rms_norm_across_heads"])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("D,axes", [(32, (16,)), (32, (12, 10, 10)), (64, (8, 12, 12)), (64, (64,)), (128, (44, 42, 42)),
                                    (128, (0, 32, 32)), (256, (64, 96, 96)), (256, (2, 2, 2, 2, 2, 2, 2, 2))])
def test_heads_axes_and_norms(pkg, dev, D, axes, pairs, norm):
    ids = ref.packed_ids([9, 0, 4], 2)
    args = _inputs(15, 6, 3, D, norm, D + len(axes), axes=len(axes))
    _check(pkg, dev, *args, ids=ids, axes=axes, pairs=pairs, norm=norm)


@pytest.mark.parametrize("T,hq,hk,D", [(1, 40, 40, 128), (1, 1, 1, 32), (7, 40, 8, 128), (300, 12, 12, 128), (64, 17, 5, 64),
                                       (130, 64, 64, 256), (33, 128, 1, 128), (1560, 40, 40, 128), (5, 512, 3, 32)])
@pytest.mark.parametrize("norm", ["rms_norm", "rms_norm_across_heads"])
def test_rows_and_heads(pkg, dev, T, hq, hk, D, norm):
    axes = (D - 4 * (D // 6), 2 * (D // 6), 2 * (D // 6))
    _check(pkg, dev, *_inputs(T, hq, hk, D, norm, T + hq), axes=axes, norm=norm)


def test_far_negative_and_fractional_positions(pkg, dev):
    q, k, _, _, _ = _inputs(40, 4, 4, 128, "none", 3)
    pos = torch.randint(-(2**31), 2**31 - 1, (40, 3), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    _check(pkg, dev, q, k, pos, None, None)
    pos = torch.randn(40, 3, generator=torch.Generator().manual_seed(2)) * 1000
    _check(pkg, dev, q, k, pos, None, None, theta=(10000.0, 500.0, 1.0))


def test_position_zero_is_the_identity(pkg, dev):
    q, k, pos, _, _ = _inputs(30, 5, 5, 64, "none", 4, axes=2)
    oq, ok = pkg.qk_norm_rope_axes(q.to(dev), k.to(dev), torch.zeros_like(pos).to(dev), axes=(16, 16))
    assert torch.equal(oq.cpu(), q) and torch.equal(ok.cpu(), k)


def test_the_grid_gives_what_the_tables_give(pkg, dev):
    """Raster positions of a grid turn K as the framework's own tables do; the table pass rounds to bf16 between norm
    and rotation, so its values may be a further 2^-8 of either term away."""
    grid = (2, 5, 7)
    S, N = 70, 40
    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn(S, N * 128, device=dev, generator=g).to(torch.bfloat16)
    gamma = 1 + 0.1 * torch.randn(N * 128, device=dev, generator=g)
    pos = torch.stack(torch.meshgrid(*(torch.arange(n, device=dev) for n in grid), indexing="ij"), -1).view(-1, 3).int()
    got, _ = pkg.qk_norm_rope_axes(x.view(S, N, 128), None, pos, norm="rms_norm_across_heads", q_gamma=gamma, eps=EPS)
    cos, sin = pkg.rope_tables(grid, device=dev)
    tab = x.clone()
    pkg.attention_ops.qk_rmsnorm_rope_(tab, gamma, cos=cos, sin=sin, eps=EPS)
    want, bound, _ = ref.rope_axes(x.cpu().view(S, N, 128), pos.cpu(), (44, 42, 42), 1e4, "interleaved", "rms_norm_across_heads",
                                   gamma.cpu(), EPS)
    ref.within(got, want, bound)
    pair = want.view(S, N, 64, 2).pow(2).sum(-1, keepdim=True).sqrt().expand(-1, -1, -1, 2).reshape(want.shape)
    ref.within(tab.view(S, N, 128), want, bound + 2 * ref.ROUND * pair)


def test_a_long_batch(pkg, dev):
    """Rows of a long batch of strided views, at its requests' borders and its end."""
    T, hq, hk = 20000, 40, 8
    g = torch.Generator(device=dev).manual_seed(6)
    slab = torch.randn(T, (hq + 2 * hk) * 128, device=dev, generator=g).to(torch.bfloat16)
    q, k = slab[:, : hq * 128].view(T, hq, 128), slab[:, hq * 128 : (hq + hk) * 128].view(T, hk, 128)
    pos = torch.randint(0, 200, (T, 3), device=dev, generator=g, dtype=torch.int32)
    ids = (torch.arange(T, device=dev) // 4999).int()
    gq, gk = torch.randn(hq * 128, device=dev, generator=g), torch.randn(hk * 128, device=dev, generator=g)
    kw = dict(norm="rms_norm_across_heads", q_gamma=gq, k_gamma=gk)
    oq, ok, kmax = pkg.qk_norm_rope_axes(q, k, pos, request_ids=ids, requests=5, want_max=True, **kw)
    for at in (0, 4990, 19990):
        sl = slice(at, at + 10)
        for x, gamma, got in ((q, gq, oq), (k, gk, ok)):
            want, bound, _ = ref.rope_axes(x[sl].cpu(), pos[sl].cpu(), (44, 42, 42), 1e4, "interleaved", "rms_norm_across_heads",
                                           gamma.cpu(), EPS)
            ref.within(got[sl], want, bound)
    n = ok.double().pow(2).sum(-1).sqrt()
    for i in range(5):
        top = n[ids == i].amax(0)
        assert bool((top <= kmax[i]).all()) and bool((kmax[i] <= top * (1 + 2.0**-6)).all())


@pytest.mark.parametrize("T", [6, 900])
def test_in_place_and_rows_of_no_request(pkg, dev, T):
    hq, hk, live = 40, 40, T - 3
    q, k, pos, gq, gk = (t.to(dev) for t in _inputs(T, hq, hk, 128, "rms_norm_across_heads", 12))
    q[live:], k[live:] = float("nan"), 3.0
    ids = ref.packed_ids([live], 3).to(dev)
    kw = dict(norm="rms_norm_across_heads", q_gamma=gq, k_gamma=gk, request_ids=ids, requests=1, want_max=True)
    oq, ok, kmax = pkg.qk_norm_rope_axes(q, k, pos, **kw)
    assert not oq[live:].any() and bool(kmax.isfinite().all())
    slab = torch.cat([q.flatten(1), k.flatten(1), torch.full((T, 64), 9.0, dtype=torch.bfloat16, device=dev)], 1)
    vq, vk = slab[:, : hq * 128].view(T, hq, 128), slab[:, hq * 128 : (hq + hk) * 128].view(T, hk, 128)
    rq, rk, kmax2 = pkg.qk_norm_rope_axes(vq, vk, pos, q_out=vq, k_out=vk, **kw)
    assert rq is vq and torch.equal(vq[:live], oq[:live]) and torch.equal(vk[:live], ok[:live]) and torch.equal(kmax, kmax2)
    assert bool(vq[live:].isnan().all()) and bool((vk[live:] == 3.0).all()) and bool((slab[:, -64:] == 9.0).all())
    # head-major outputs; one of the two given
    hm = torch.full((hq, T, 128), 5.0, dtype=torch.bfloat16, device=dev)
    rq, rk, _ = pkg.qk_norm_rope_axes(q, k, pos, q_out=hm.permute(1, 0, 2), **kw)
    assert torch.equal(hm.permute(1, 0, 2)[:live], oq[:live]) and bool((hm[:, live:] == 5.0).all()) and torch.equal(rk, ok)


def test_not_a_number_stays_in_its_row(pkg, dev):
    q, k, pos, _, _ = (None if t is None else t.to(dev) for t in _inputs(8, 4, 4, 128, "none", 14))
    want = pkg.qk_norm_rope_axes(q, k, pos, axes=(32, 32, 32), norm="rms_norm")
    q[3, 1, 0], q[5, 2, 127] = float("nan"), float("inf")
    got, _ = pkg.qk_norm_rope_axes(q, k, pos, axes=(32, 32, 32), norm="rms_norm")
    assert bool(got[3, 1].isnan().all())
    keep = torch.ones(8, 4, dtype=torch.bool, device=dev)
    keep[3, 1] = keep[5, 2] = False
    assert torch.equal(got[keep], want[0][keep])
    # without a norm, an infinity in a channel that is not turned touches that channel alone
    got, _ = pkg.qk_norm_rope_axes(q, k, pos, axes=(32, 32, 32))
    assert got[5, 2, 127].isinf() and bool(got[5, 2, :127].isfinite().all())


def test_no_rows(pkg, dev):
    e = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=dev)
    pos = torch.empty(0, 3, dtype=torch.int32, device=dev)
    q, k, kmax = pkg.qk_norm_rope_axes(e, e, pos, want_max=True)
    assert q.shape == k.shape == (0, 4, 128) and kmax.shape == (1, 4) and not kmax.any()


def test_rows_past_four_gigabytes(pkg, dev):
    T, ld = 40000, 1 << 16
    wide = torch.empty(T * ld, dtype=torch.bfloat16, device=dev).as_strided((T, ld), (ld, 1))
    ids = torch.full((T,), -1, dtype=torch.int32, device=dev)
    rows = torch.tensor([0, 20000, T - 1], device=dev)
    ids[rows] = 0
    x = torch.randn(3, 256, device=dev).to(torch.bfloat16)
    wide[rows, :256] = x
    pos = torch.arange(T * 3, device=dev, dtype=torch.int32).view(T, 3)
    view = wide[:, :256].unflatten(1, (2, 128))
    pkg.qk_norm_rope_axes(view, None, pos, request_ids=ids, q_out=view)
    want, _ = pkg.qk_norm_rope_axes(x.view(3, 2, 128), None, pos[rows])
    assert torch.equal(wide[rows, :256].view(3, 2, 128), want)


def test_graph_replays_with_other_requests(pkg, dev):
    T = 90
    q, k, pos, gq, gk = (t.to(dev) for t in _inputs(T, 8, 4, 128, "rms_norm", 17))
    ids = ref.packed_ids([50, 30], 10).to(dev)
    call = lambda: pkg.qk_norm_rope_axes(q, k, pos, norm="rms_norm", q_gamma=gq, k_gamma=gk, request_ids=ids, requests=3,  # noqa: E731
                                         want_max=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        ids.copy_(torch.randint(-1, 3, (T,), generator=g, dtype=torch.int32))
        pos.copy_(torch.randint(0, 99, (T, 3), generator=g, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("norm", ["rms_norm", "rms_norm_across_heads"])
def test_the_norm_alone(pkg, dev, norm):
    q, k, _, gq, gk = _inputs(20, 5, 3, 128, norm, 19)
    oq, ok = pkg.qk_norm_rope_axes(q.to(dev), k.to(dev), None, axes=(), norm=norm, q_gamma=gq.to(dev), k_gamma=gk.to(dev), eps=EPS)
    for x, gamma, got in ((q, gq, oq), (k, gk, ok)):
        want, bound, _ = ref.rope_axes(x, torch.zeros(20, 0), (), 1.0, "halves", norm, gamma, EPS)
        ref.within(got, want, bound)


def test_bases_as_tensors_are_read_at_every_call(pkg, dev):
    q, k, pos, _, _ = (None if t is None else t.to(dev) for t in _inputs(40, 4, 2, 128, "none", 23))
    theta, eps = torch.tensor(10000.0), torch.tensor(EPS)
    for base in (10000.0, 500.0):
        theta.fill_(base)
        for pair in ((theta, EPS), (base, eps)):
            got = pkg.qk_norm_rope_axes(q, k, pos, theta=pair[0], eps=pair[1])
            assert all(torch.equal(a, b) for a, b in zip(got, pkg.qk_norm_rope_axes(q, k, pos, theta=base)))


@pytest.mark.parametrize("T,hq,hk,D,axes", [(1, 1, 1, 32, (16, 16)), (301, 32, 4, 64, (8, 12, 12)), (301, 32, 32, 64, (32, 16, 16)), (77, 16, 16, 64, (16,)),
                                            (1030, 16, 1, 128, (44, 42, 42)), (65, 5, 16, 128, (64, 16)), (130, 8, 3, 256, (16, 0, 96)), (9, 3, 64, 32, (16,))])
@pytest.mark.parametrize("norm", ["none", "rms_norm"])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_without_the_bound(pkg, dev, pairs, norm, T, hq, hk, D, axes):
    """Short rows that share neither a weight nor maxima."""
    q, k, pos, gq, gk = _inputs(T, hq, hk, D, norm, T + hq, axes=len(axes))
    ids = torch.randint(-1, 3, (T,), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    to = lambda v: None if v is None else v.to(dev)  # noqa: E731
    got = pkg.qk_norm_rope_axes(to(q), to(k), to(pos), axes=axes, rope_pairs=pairs, norm=norm, q_gamma=to(gq), k_gamma=to(gk), eps=EPS, request_ids=to(ids))
    live = ids >= 0
    for x, gamma, y in zip((q, k), (gq, gk), got):
        want, bound, _ = ref.rope_axes(x, pos, axes, 10000.0, pairs, norm, gamma, EPS)
        ref.within(y[live.to(dev)], want[live], bound[live], "q or k")
        assert not y[~live.to(dev)].any()


@pytest.mark.parametrize("norm", ["none", "rms_norm_across_heads"])
def test_a_batch_of_no_requests(pkg, dev, norm):
    """``requests=0``: every row belongs to none, with the bound as without it."""
    T, hq, hk = 70, 4, 2
    q, k, pos, gq, gk = (None if t is None else t.to(dev) for t in _inputs(T, hq, hk, 128, norm, 29))
    kw = dict(norm=norm, q_gamma=gq, k_gamma=gk, request_ids=torch.zeros(T, dtype=torch.int32, device=dev), requests=0)
    for want_max in (False, True):
        for _ in range(4):  # what the allocator hands out next holds no zeros
            old = [torch.full_like(t, float("nan")) for t in (q, k)]
            del old
            oq, ok, *rest = pkg.qk_norm_rope_axes(q, k, pos, want_max=want_max, **kw)
            assert not oq.any() and not ok.any()
            assert not want_max or rest[0].shape == (0, hk)
    q_out = torch.full_like(q, 5.0)
    _, ok, kmax = pkg.qk_norm_rope_axes(q, k, pos, want_max=True, q_out=q_out, **kw)
    assert bool((q_out == 5.0).all()) and not ok.any() and kmax.shape == (0, hk)


@pytest.mark.parametrize("norm", ["rms_norm", "rms_norm_across_heads"])
def test_rows_whose_mean_square_is_subnormal(pkg, dev, norm):
    """Without eps, rows of 2^-64 normalize like any others: their mean square is held to 2^-150, 2^-22 of itself."""
    q, k, pos, gq, gk = _inputs(33, 5, 3, 128, norm, 31)
    tiny = lambda x: (x.float() * 2.0**-64).to(torch.bfloat16)  # noqa: E731
    _check(pkg, dev, tiny(q), tiny(k), pos, gq, gk, norm=norm, eps=0.0)


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_a_weight_of_one_head_at_an_odd_float(pkg, dev, pairs):
    q, k, pos, gq, gk = (t.to(dev) for t in _inputs(20, 3, 2, 128, "rms_norm", 37))
    want = pkg.qk_norm_rope_axes(q, k, pos, rope_pairs=pairs, norm="rms_norm", q_gamma=gq, k_gamma=gk)
    buf = torch.zeros(300, device=dev)
    buf[1:129], buf[150:278] = gq, gk
    got = pkg.qk_norm_rope_axes(q, k, pos, rope_pairs=pairs, norm="rms_norm", q_gamma=buf[1:129], k_gamma=buf[150:278])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("hq,hk,D", [(23, 20, 128), (22, 3, 128), (32, 32, 128), (31, 29, 128), (64, 16, 64), (36, 40, 128), (40, 40, 128), (48, 48, 128),
                                     (45, 6, 128), (64, 64, 128), (60, 8, 128), (30, 32, 256), (1, 60, 128), (65, 3, 128), (128, 128, 128), (512, 400, 32)])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("norm", ["rms_norm", "rms_norm_across_heads"])
def test_rows_of_every_width(pkg, dev, hq, hk, D, pairs, norm):
    """Up to 16384 channels in both layouts of the pairs, Q and K of equal and of unequal widths; requests that meet inside
    a workgroup's eight rows."""
    axes = {32: (8, 8), 64: (8, 12, 12), 128: (44, 42, 42), 256: (64, 96, 80)}[D]
    ids = ref.packed_ids([5, 9, 0, 18], 3)
    ids[20] = -1
    _check(pkg, dev, *_inputs(35, hq, hk, D, norm, hq + hk, axes=len(axes)), ids=ids, axes=axes, pairs=pairs, norm=norm)
