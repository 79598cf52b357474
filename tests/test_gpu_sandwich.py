"""The norms around a sub-layer's gated residual sum, with each row's request's modulation, against 64 bits."""

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _inputs(T, H, R, seed, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    h = (torch.randn(T, H, generator=g) * 3 + shift).to(torch.bfloat16)
    res = torch.randn(T, H, generator=g).to(torch.bfloat16)
    w = 1 + 0.1 * torch.randn(H, generator=g)
    mod = torch.randn(R, 3, H, generator=g)
    return h, res, w, mod[:, 0], 1 + 0.5 * mod[:, 1], mod[:, 2]


def _check(pkg, dev, h, res, w, gate, mul, add, ids, alpha=1.0, post="rms_norm", norm="layer_norm", eps=EPS):
    row = ids.long()
    pick = lambda v: None if v is None else (v[row] if v.dim() == 2 else v.expand(len(row), -1))  # noqa: E731
    to = lambda v: None if v is None else v.to(dev)  # noqa: E731
    live = ids >= 0
    r, y = pkg.adaln_sandwich(h.to(dev), res.to(dev), to(mul), to(add), eps=eps, post_norm=post, post_weight=to(w), gate=to(gate),
                              residual_scale=alpha, norm_type=norm, request_ids=ids.to(dev))
    want, bound = ref.sandwich_residual(h, res, pick(gate), w, alpha, post, eps)
    ref.within(r[live.to(dev)], want[live], bound[live], "residual")
    want, bound = ref.sandwich_modulated(r.cpu(), pick(mul), pick(add), norm, eps)
    ref.within(y[live.to(dev)], want[live], bound[live], "modulated")
    assert not r[~live.to(dev)].any() and not y[~live.to(dev)].any()
    return r, y


@pytest.mark.parametrize("lengths,pad,H", [
    ([1], 0, 32), ([1], 3, 5120), ([2, 1, 4], 0, 96), ([1] * 9, 2, 512), ([3, 0, 70], 5, 544), ([257], 0, 1536),
    ([130, 127], 1, 5120), ([5, 9], 0, 13824), ([3, 4], 1, 16384), ([700, 400, 900], 48, 5120),
])
def test_against_64_bits(pkg, dev, lengths, pad, H):
    ids = ref.packed_ids(lengths, pad)
    h, res, w, gate, mul, add = _inputs(len(ids), H, len(lengths), 7 * H + len(ids))
    _check(pkg, dev, h, res, w, gate, mul, add, ids, alpha=0.75)


@pytest.mark.parametrize("post", ["none", "rms_norm", "layer_norm"])
@pytest.mark.parametrize("norm", ["none", "rms_norm", "layer_norm"])
@pytest.mark.parametrize("H", [160, 5120])
def test_norms(pkg, dev, post, norm, H):
    ids = ref.packed_ids([17, 20], 3)
    h, res, w, gate, mul, add = _inputs(40, H, 2, 5, shift=2.0)
    _check(pkg, dev, h, res, w, gate, mul, add, ids, post=post, norm=norm)


@pytest.mark.parametrize("left_out", ["weight", "gate", "mul", "add", "all"])
def test_vectors_left_out_or_shared(pkg, dev, left_out):
    ids = ref.packed_ids([6, 5], 1)
    h, res, w, gate, mul, add = _inputs(12, 1280, 2, 9)
    w, gate, mul, add = (None if left_out in (n, "all") else v
                         for n, v in (("weight", w), ("gate", gate), ("mul", mul), ("add", add)))
    _check(pkg, dev, h, res, w, gate, mul, add, ids, alpha=-1.5)
    one = lambda v: None if v is None else v[0].contiguous()  # noqa: E731
    _check(pkg, dev, h, res, w, one(gate), mul, one(add), ids)


def test_requests_in_any_order_and_ids_that_name_none(pkg, dev):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(-2, 5, (333,), generator=g, dtype=torch.int32)
    h, res, w, gate, mul, add = _inputs(333, 5120, 4, 11)
    ids4 = torch.where(ids >= 4, torch.tensor(-1, dtype=torch.int32), ids)  # 4 names no request: as -1
    r, y = _check(pkg, dev, h, res, w, gate, mul, add, ids4)
    r2, y2 = pkg.adaln_sandwich(h.to(dev), res.to(dev), mul.to(dev), add.to(dev), eps=EPS, post_weight=w.to(dev), gate=gate.to(dev),
                                request_ids=ids.to(dev))
    assert torch.equal(r, r2) and torch.equal(y, y2)


@pytest.mark.parametrize("H", [96, 5120])
@pytest.mark.parametrize("T", [5, 300])
def test_quantized_outputs_are_those_of_the_bf16_output(pkg, dev, H, T):
    """MX and ROW codes of exactly the bf16 output, by the quantizer that has its own tests."""
    ids = ref.packed_ids([T - 2], 2).to(dev)
    h, res, w, gate, mul, add = (t.to(dev) for t in _inputs(T, H, 1, 21))
    kw = dict(eps=EPS, post_weight=w, gate=gate, request_ids=ids)
    r, y = pkg.adaln_sandwich(h, res, mul, add, **kw)
    for quant in ("mx", "row"):
        r2, q = pkg.adaln_sandwich(h, res, mul, add, quant=quant, **kw)
        assert torch.equal(r, r2)
        want = pkg.adaln_modulate(y, eps=EPS, norm_type="none", quant=quant)
        live = T - 2
        if quant == "mx":
            assert torch.equal(q.codes.view(torch.uint8)[:live], want.codes.view(torch.uint8)[:live])
            assert torch.equal(q.scales[:live], want.scales[:live])
            assert not q.codes.view(torch.uint8)[live:].any() and not q.scales[live:].any()
        else:
            assert torch.equal(q.view(torch.uint8)[:live], want.view(torch.uint8)[:live])
            assert not q.view(torch.uint8)[live:].any()


@pytest.mark.parametrize("quant", ["none", "mx", "row"])
@pytest.mark.parametrize("T", [12, 600])
def test_rows_of_no_request_stay_in_given_outputs(pkg, dev, quant, T):
    """Padding rows hold NaN and reach nothing; the given outputs keep what they had there."""
    H, live = 5120, T - 5
    ids = ref.packed_ids([live], 5).to(dev)
    h, res, w, gate, mul, add = (t.to(dev) for t in _inputs(T, H, 1, 31))
    h[live:], res[live:] = float("nan"), float("nan")
    kw = dict(eps=EPS, post_weight=w, gate=gate, request_ids=ids, quant=quant)
    r, y = pkg.adaln_sandwich(h, res, mul, add, **kw)
    ro = torch.full_like(r, 7.0)
    fill = lambda t: torch.full(t.shape, 3, dtype=torch.uint8, device=dev)  # noqa: E731
    if quant == "none":
        out, raw = (o := torch.full_like(y, 5.0)), [(o, y)]
    elif quant == "mx":
        out = pkg.MXTensor(fill(y.codes).view(torch.float8_e4m3fn), fill(y.scales))
        raw = [(out.codes.view(torch.uint8), y.codes.view(torch.uint8)), (out.scales, y.scales)]
    else:
        out = fill(y).view(torch.float8_e4m3fn)
        raw = [(out.view(torch.uint8), y.view(torch.uint8))]
    before = [t[live:].clone() for t, _ in raw]
    got_r, got = pkg.adaln_sandwich(h, res, mul, add, residual_out=ro, out=out, **kw)
    assert got_r is ro and torch.equal(ro[:live], r[:live]) and bool((ro[live:] == 7.0).all())
    for (t, want), b in zip(raw, before):
        assert torch.equal(t[:live], want[:live]) and torch.equal(t[live:], b)
    # one output given: the other is allocated, its rest zero
    ro.fill_(7.0)
    _, y2 = pkg.adaln_sandwich(h, res, mul, add, residual_out=ro, **kw)
    assert bool((ro[live:] == 7.0).all())
    for t, want in zip(y2 if quant == "mx" else (y2,), y if quant == "mx" else (y,)):
        assert torch.equal(t.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("T", [3, 400])
def test_in_place_strided_and_sliced_modulation(pkg, dev, T):
    H, R = 5120, 3
    g = torch.Generator(device=dev).manual_seed(5)
    wide = torch.randn(T, 2 * H + 64, device=dev, generator=g).to(torch.bfloat16)
    h, res = wide[:, :H], wide[:, H + 32 : 2 * H + 32]
    mod = torch.randn(R, 6, H, device=dev, generator=g)
    ids = (torch.arange(T, device=dev) * R // T).to(torch.int32)
    kw = dict(eps=EPS, request_ids=ids)
    want = pkg.adaln_sandwich(h.contiguous(), res.contiguous(), mod[:, 1].contiguous(), mod[:, 0].contiguous(),
                              gate=mod[:, 2].contiguous(), **kw)
    got = pkg.adaln_sandwich(h, res, mod[:, 1], mod[:, 0], gate=mod[:, 2], **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    h2, r2 = h.contiguous(), res.contiguous()
    pkg.adaln_sandwich(h2, r2, mod[:, 1], mod[:, 0], gate=mod[:, 2], residual_out=r2, out=h2, **kw)
    assert torch.equal(r2, want[0]) and torch.equal(h2, want[1])


def test_no_rows(pkg, dev):
    e = torch.empty(0, 64, dtype=torch.bfloat16, device=dev)
    r, y = pkg.adaln_sandwich(e, e, eps=EPS, quant="mx")
    assert r.shape == (0, 64) and y.codes.shape == (0, 64) and y.scales.shape == (0, 2)


def test_extreme_values(pkg, dev):
    """Zero rows, the largest finite values and infinities: what fp32 gives for the formulas, row by row."""
    H = 512
    h = torch.zeros(6, H, dtype=torch.bfloat16)
    res = torch.zeros(6, H, dtype=torch.bfloat16)
    h[1] = 1e15
    h[2, 0] = float("inf")
    res[3, 5] = float("nan")
    res[4] = -2.0**100
    h[5] = 2.0**-60
    r, y = pkg.adaln_sandwich(h.to(dev), res.to(dev), eps=EPS, norm_type="rms_norm")
    r, y = r.cpu().float(), y.cpu().float()
    assert not r[0].any() and not y[0].any()
    assert torch.equal(r[1], torch.ones(H)) and torch.equal(y[1], torch.ones(H))
    assert r[2, 0].isnan()
    assert r[3, 5].isnan() and not r[3, :5].any() and y[3].isnan().all()
    assert bool((r[4] == -2.0**100).all())
    assert bool(((r[5] - 2.0**-60 * 1e3).abs() <= 2.0**-60 * 1e3 * 2.0**-7).all())


def test_rows_past_four_gigabytes(pkg, dev):
    """A row stride that puts rows beyond 2^32 bytes."""
    T, H, ld = 40000, 256, 1 << 16
    wide = torch.empty(T * ld, dtype=torch.bfloat16, device=dev).as_strided((T, ld), (ld, 1))
    ids = torch.full((T,), -1, dtype=torch.int32, device=dev)
    rows = torch.tensor([0, 20000, T - 1], device=dev)
    ids[rows] = 0
    x = torch.randn(3, 2, H, device=dev).to(torch.bfloat16)
    wide[rows, :H], wide[rows, 512 : 512 + H] = x[:, 0], x[:, 1]
    r, y = pkg.adaln_sandwich(wide[:, :H], wide[:, 512 : 512 + H], eps=EPS, request_ids=ids)
    want = pkg.adaln_sandwich(x[:, 0].contiguous(), x[:, 1].contiguous(), eps=EPS)
    assert torch.equal(r[rows], want[0]) and torch.equal(y[rows], want[1])
    assert not y[ids < 0].any()


def test_graph_replays_with_other_requests(pkg, dev):
    T, H, R = 70, 5120, 4
    h, res, w, gate, mul, add = (t.to(dev) for t in _inputs(T, H, R, 41))
    ids = ref.packed_ids([20, 30], 20).to(dev)
    call = lambda: pkg.adaln_sandwich(h, res, mul, add, eps=EPS, post_weight=w, gate=gate, request_ids=ids, quant="mx")  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, y = call()
    for seed in range(3):
        ids.copy_(torch.randint(-1, R, (T,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32))
        h.copy_(torch.randn(T, H, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        r2, y2 = call()
        torch.cuda.synchronize()
        assert torch.equal(r, r2) and torch.equal(y.codes.view(torch.uint8), y2.codes.view(torch.uint8))
        assert torch.equal(y.scales, y2.scales)


def test_on_another_stream(pkg, dev):
    h, res, w, gate, mul, add = (t.to(dev) for t in _inputs(500, 5120, 1, 51))
    want = pkg.adaln_sandwich(h, res, mul, add, eps=EPS, gate=gate)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.adaln_sandwich(h, res, mul, add, eps=EPS, gate=gate)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("T", [9, 700])
@pytest.mark.parametrize("H", [96, 5120])
def test_without_a_residual_or_without_a_second_output(pkg, dev, T, H):
    ids = ref.packed_ids([T - 2], 2)
    h, res, w, gate, mul, add = _inputs(T, H, 1, 61)
    h[T - 1] = float("inf")
    to = lambda t: t.to(dev)  # noqa: E731
    kw = dict(eps=EPS, post_weight=to(w), gate=to(gate), request_ids=to(ids))
    r, y = pkg.adaln_sandwich(to(h), None, to(mul), to(add), residual_scale=3.0, **kw)
    want, bound = ref.sandwich_residual(h, torch.zeros_like(h), gate.expand(T, H), w, 1.0, "rms_norm", EPS)
    ref.within(r[: T - 2], want[: T - 2], bound[: T - 2])
    want, bound = ref.sandwich_modulated(r.cpu(), mul.expand(T, H), add.expand(T, H), "layer_norm", EPS)
    ref.within(y[: T - 2], want[: T - 2], bound[: T - 2])
    assert not r[T - 2 :].any() and not y[T - 2 :].any()
    full, _ = pkg.adaln_sandwich(to(h), to(res), to(mul), to(add), **kw)
    alone, none = pkg.adaln_sandwich(to(h), to(res), norm_type=None, **kw)
    assert none is None and torch.equal(alone, full)
    ro = torch.full_like(full, 2.0)
    pkg.adaln_sandwich(to(h), to(res), norm_type=None, residual_out=ro, **kw)
    assert torch.equal(ro[: T - 2], full[: T - 2]) and bool((ro[T - 2 :] == 2.0).all())


@pytest.mark.parametrize("T", [5, 600])
@pytest.mark.parametrize("norm", ["layer_norm", "rms_norm"])
def test_rows_whose_variance_is_subnormal(pkg, dev, norm, T):
    """Without eps, rows of 3 x 2^-66 normalize like any others: their mean square (2^-129) is held to 2^-150, 2^-21 of itself."""
    ids = ref.packed_ids([T])
    h, res, w, gate, mul, add = _inputs(T, 512, 1, 71)
    tiny = (h.float() * 2.0**-66).to(torch.bfloat16)
    _check(pkg, dev, tiny, res, w, gate, mul, add, ids, post=norm, eps=0.0)
    _check(pkg, dev, torch.zeros_like(h), tiny, None, None, mul, add, ids, post="none", norm=norm, eps=0.0)


@pytest.mark.parametrize("T", [6, 700])
def test_one_row_of_vectors_serves_one_request(pkg, dev, T):
    """Vectors ``[1, H]`` are those of request 0: a row with another id belongs to none. Beside vectors of several
    requests, and as ``[H]``, they serve every one."""
    H = 96
    ids = (torch.arange(T) % 3 - 1).to(torch.int32)  # -1, 0, 1
    h, res, w, gate, mul, add = _inputs(T, H, 1, 73)
    _check(pkg, dev, h, res, w, gate, mul, add, torch.where(ids == 0, ids, -1))
    to = lambda v: v.to(dev)  # noqa: E731
    kw = dict(eps=EPS, post_weight=to(w), request_ids=to(ids))
    mine = (ids == 0).to(dev)
    r, y = pkg.adaln_sandwich(to(h), to(res), to(mul), to(add), gate=to(gate), **kw)
    assert not r[~mine].any() and not y[~mine].any() and bool(r[mine].any(1).all())
    every = pkg.adaln_sandwich(to(h), to(res), to(mul)[0], to(add)[0], gate=to(gate)[0], **kw)
    assert torch.equal(every[0][mine], r[mine]) and torch.equal(every[1][mine], y[mine])
    mixed = pkg.adaln_sandwich(to(h), to(res), to(mul).expand(2, H).contiguous(), to(add), gate=to(gate), **kw)
    assert all(torch.equal(a, b) for a, b in zip(every, mixed)) and bool(every[0][(ids == 1).to(dev)].any(1).all())


@pytest.mark.parametrize("post,norm", [("rms_norm", "layer_norm"), ("layer_norm", "rms_norm"), ("none", "none"), ("layer_norm", "layer_norm")])
@pytest.mark.parametrize("H", [32, 512, 544, 1024, 1056, 1536, 2048, 2080, 2592, 3040, 3104, 3616, 4096, 4128, 4608, 4640, 5088])
def test_many_rows_of_every_length(pkg, dev, H, post, norm):
    """More rows than two for every CU, in rows of one to ten pieces of 512 with whole and ragged last ones; requests
    that end inside a workgroup's eight rows, and rows of none between them."""
    ids = ref.packed_ids([1, 300, 0, 205, 83], 9)
    ids[[40, 41, 320]] = -1
    h, res, w, gate, mul, add = _inputs(len(ids), H, 5, H + 1, shift=0.5)
    _check(pkg, dev, h, res, w, gate, mul, add, ids, alpha=-0.5, post=post, norm=norm)


@pytest.mark.parametrize("H", [96, 1536, 2592, 4640, 5120, 5152])
def test_many_quantized_rows_are_those_of_the_bf16_output(pkg, dev, H):
    T, live = 611, 607
    ids = ref.packed_ids([200, 407], 4).to(dev)
    h, res, w, gate, mul, add = (t.to(dev) for t in _inputs(T, H, 2, H))
    kw = dict(eps=EPS, post_norm="none", gate=gate, request_ids=ids)
    r, y = pkg.adaln_sandwich(h, res, mul, add, **kw)
    for quant in ("mx", "row"):
        r2, q = pkg.adaln_sandwich(h, res, mul, add, quant=quant, **kw)
        want = pkg.adaln_modulate(y, eps=EPS, norm_type="none", quant=quant)
        assert torch.equal(r, r2)
        for got, full in zip(q if quant == "mx" else (q,), want if quant == "mx" else (want,)):
            got, full = got.view(torch.uint8), full.view(torch.uint8)
            assert torch.equal(got[:live], full[:live]) and not got[live:].any()


@pytest.mark.parametrize("H", [1536, 4640, 5120, 13824])
def test_many_rows_in_place_strided_and_sliced_modulation(pkg, dev, H):
    T, R = 700, 3
    g = torch.Generator(device=dev).manual_seed(15)
    wide = torch.randn(T, 2 * H + 64, device=dev, generator=g).to(torch.bfloat16)
    h, res = wide[:, :H], wide[:, H + 32 : 2 * H + 32]
    mod = torch.randn(R, 6, H, device=dev, generator=g)
    ids = (torch.arange(T, device=dev) * (R + 1) // T - 1).to(torch.int32)
    kw = dict(eps=EPS, request_ids=ids)
    want = pkg.adaln_sandwich(h.contiguous(), res.contiguous(), mod[:, 1].contiguous(), mod[:, 0].contiguous(), gate=mod[:, 2].contiguous(), **kw)
    got = pkg.adaln_sandwich(h, res, mod[:, 1], mod[:, 0], gate=mod[:, 2], **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    h2, r2 = h.contiguous(), res.contiguous()
    pkg.adaln_sandwich(h2, r2, mod[:, 1], mod[:, 0], gate=mod[:, 2], residual_out=r2, out=h2, **kw)
    live = ids >= 0
    assert torch.equal(r2[live], want[0][live]) and torch.equal(h2[live], want[1][live])
    assert torch.equal(r2[~live], res[~live]) and torch.equal(h2[~live], h[~live])
    # the sum over hidden, the second output over the residual
    h2, r2 = h.contiguous(), res.contiguous()
    pkg.adaln_sandwich(h2, r2, mod[:, 1], mod[:, 0], gate=mod[:, 2], residual_out=h2, out=r2, **kw)
    assert torch.equal(h2[live], want[0][live]) and torch.equal(r2[live], want[1][live])


@pytest.mark.parametrize("T,H", [(600, 5152), (1100, 8192), (1030, 13824), (601, 16384)])
def test_many_rows_longer_than_a_wave_holds(pkg, dev, T, H):
    """A workgroup goes through several rows: requests change between them, and some belong to none."""
    ids = torch.randint(-1, 3, (T,), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    h, res, w, gate, mul, add = _inputs(T, H, 3, 81)
    _check(pkg, dev, h, res, w, gate, mul, add, ids, post="layer_norm")


def test_a_workgroup_of_more_rows_than_it_looks_up_at_once(pkg, dev):
    """17000 rows of 5152: more than 64 to each of 256 workgroups. Every row as in a batch of 250."""
    T, H = 17000, 5152
    g = torch.Generator(device=dev).manual_seed(83)
    h, res = (torch.randn(T, H, device=dev, generator=g).to(torch.bfloat16) for _ in range(2))
    gate, mul, add = (torch.randn(4, H, device=dev, generator=g) for _ in range(3))
    ids = torch.randint(-1, 4, (T,), device=dev, generator=g, dtype=torch.int32)
    r, y = pkg.adaln_sandwich(h, res, mul, add, eps=EPS, gate=gate, quant="mx", request_ids=ids)
    for at in range(0, T, 250):
        s = slice(at, at + 250)
        r2, y2 = pkg.adaln_sandwich(h[s], res[s], mul, add, eps=EPS, gate=gate, quant="mx", request_ids=ids[s].clone())
        assert torch.equal(r[s], r2) and torch.equal(y.codes.view(torch.uint8)[s], y2.codes.view(torch.uint8)) and torch.equal(y.scales[s], y2.scales)
