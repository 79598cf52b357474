"""Low-rank adapters of many requests beside a shared projection, against 64 bits."""

import pytest
import torch

import packed_ref as ref

pytestmark = pytest.mark.gpu


def _mx(pkg, dev, x):
    return pkg.adaln_modulate(x.to(dev), eps=0.0, norm_type="none", quant="mx")


def _inputs(T, K, slices, n, r, seed):
    g = torch.Generator().manual_seed(seed)
    N = sum(slices)
    base = torch.randn(T, N, generator=g).to(torch.bfloat16)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16)
    a = (torch.randn(n, len(slices) * r, K, generator=g) * K**-0.5).to(torch.bfloat16)
    b = (torch.randn(n, N, r, generator=g) * r**-0.5).to(torch.bfloat16)
    scales = 1 + 0.3 * torch.randn(n, generator=g)
    return base, x, a, b, scales


def _check(pkg, dev, base, x, a, b, scales, slices, adapters, ids=None, kind="bf16", rows=None):
    to = lambda v: None if v is None else v.to(dev)  # noqa: E731
    row_scale = None
    if kind == "bf16":
        xd, xr = x.to(dev), x
    elif kind == "mx":
        xd = _mx(pkg, dev, x)
        xr = xd.dequantize(torch.float32).cpu()
    else:
        xd = pkg.row_quantize_packed(x.to(dev))
        raw = xd.view(torch.uint8).cpu()
        xr = raw[:, :-4].contiguous().view(torch.float8_e4m3fn).float()
        row_scale = raw[:, -4:].contiguous().view(torch.float32)[:, 0]
    out = pkg.lora_add(to(base), xd, to(a), to(b), to(adapters), scales=to(scales), slices=slices, request_ids=to(ids))
    if ids is None:
        which, live = adapters, torch.ones(len(base), dtype=torch.bool)
    else:
        live = (ids >= 0) & (ids < len(adapters))
        which = torch.where(live, adapters[ids.clamp(0, len(adapters) - 1).long()], -1)
    which = torch.where(which < a.shape[0], which, -1)
    want, bound = ref.lora(base, xr, a, b, which, scales, slices, row_scale)
    live_d = live.to(dev)
    ref.within(out[live_d], want[live], bound[live])
    assert not out[~live_d].any()
    return out


@pytest.mark.parametrize("kind", ["bf16", "mx", "row"])
@pytest.mark.parametrize("T,K,slices,n,r", [
    (1, 32, (8,), 1, 16), (1, 5120, (5120,), 3, 16), (5, 96, (72,), 2, 32), (16, 5120, (1024,), 8, 64), (33, 416, (264,), 2, 48),
    (64, 160, (64, 128, 64), 3, 16), (129, 1536, (192, 64), 4, 80), (31, 256, (2568,), 1, 256), (70, 1024, (128,) * 8, 2, 32),
    (300, 640, (512, 512, 512), 5, 128),
])
def test_against_64_bits(pkg, dev, kind, T, K, slices, n, r):
    base, x, a, b, scales = _inputs(T, K, slices, n, r, T + K + r)
    adapters = torch.randint(-1, n, (T,), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    adapters[0] = 0
    _check(pkg, dev, base, x, a, b, scales, slices, adapters, kind=kind)


@pytest.mark.parametrize("kind", ["bf16", "mx", "row"])
@pytest.mark.parametrize("lengths,pad,K,slices,r", [
    ([1024], 0, 128, (64,), 16), ([700, 500], 7, 256, (136,), 32), ([1, 1023, 1], 0, 384, (256, 64), 32), ([300] * 5, 3, 640, (192,), 48),
    ([1025], 0, 1152, (128, 64, 64), 64), ([600, 0, 900], 100, 2560, (320,), 128), ([2000], 48, 512, (512,), 96),
    ([900, 200], 0, 256, (72,), 144), ([1100, 300], 1, 416, (1088,), 80), ([257] * 8, 0, 896, (128,) * 4, 32),
])
def test_many_rows(pkg, dev, kind, lengths, pad, K, slices, r):
    ids = ref.packed_ids(lengths, pad)
    base, x, a, b, scales = _inputs(len(ids), K, slices, 3, r, K + r)
    adapters = torch.tensor([i % 4 - 1 for i in range(1, len(lengths) + 1)], dtype=torch.int32)
    _check(pkg, dev, base, x, a, b, scales, slices, adapters, ids, kind=kind)


@pytest.mark.parametrize("kind", ["bf16", "mx"])
def test_many_rows_of_mixed_adapters(pkg, dev, kind):
    T, n = 1500, 7
    base, x, a, b, scales = _inputs(T, 384, (192,), n, 32, 78)
    adapters = torch.randint(-1, n, (T,), generator=torch.Generator().manual_seed(7), dtype=torch.int32)
    _check(pkg, dev, base, x, a, b, scales, (192,), adapters, kind=kind)
    x[7], base[9] = float("nan"), float("inf")
    ids = torch.zeros(T, dtype=torch.int32)
    ids[1203:] = -1
    to = lambda t: t.to(dev)  # noqa: E731
    xd = to(x) if kind == "bf16" else _mx(pkg, dev, x)
    view = torch.full((T, 200), 5.0, dtype=torch.bfloat16, device=dev)
    view[:, 8:] = to(base)
    out = pkg.lora_add(view[:, 8:], xd, to(a), to(b), to(adapters[:1]) * 0, request_ids=to(ids), out=view[:, 8:])
    assert bool(out[7].isnan().all()) and bool(out[9].isinf().all())
    assert torch.equal(out[1203:].cpu(), base[1203:]) and bool((view[:, :8] == 5.0).all())
    rest = torch.ones(T, dtype=torch.bool)
    rest[[7, 9]] = False
    assert bool(out[rest.to(dev)].isfinite().all())


@pytest.mark.parametrize("kind", ["bf16", "mx"])
@pytest.mark.parametrize("lengths,pad", [([1], 0), ([1] * 40, 3), ([100, 28], 0), ([130, 1, 0, 200], 17), ([500], 12)])
def test_requests(pkg, dev, kind, lengths, pad):
    ids = ref.packed_ids(lengths, pad)
    n = 3
    base, x, a, b, scales = _inputs(len(ids), 1280, (640, 640), n, 32, len(ids))
    adapters = torch.tensor([i % (n + 1) - 1 for i in range(1, len(lengths) + 1)], dtype=torch.int32)
    _check(pkg, dev, base, x, a, b, scales, (640, 640), adapters, ids, kind=kind)


def test_rows_in_any_order_and_ids_that_do_not_exist(pkg, dev):
    T, n = 333, 6
    base, x, a, b, scales = _inputs(T, 512, (256,), n, 32, 77)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(-3, 12, (T,), generator=g, dtype=torch.int32)
    adapters = torch.randint(-2, n + 3, (10,), generator=g, dtype=torch.int32)  # ids 10 and 11 name no request
    _check(pkg, dev, base, x, a, b, scales, (256,), adapters, ids)


def test_many_adapters_in_one_tile(pkg, dev):
    T = n = 64
    base, x, a, b, scales = _inputs(T, 2048, (512,), n, 16, 5)
    _check(pkg, dev, base, x, a, b, scales, (512,), torch.randperm(n, generator=torch.Generator().manual_seed(1)).int())


def test_an_adapter_that_outweighs_its_base(pkg, dev):
    """u enters the second product to 2^-16 of itself: nothing of the output's own precision is lost where the base
    is small or cancels."""
    base, x, a, b, _ = _inputs(200, 1024, (256,), 1, 64, 9)
    _check(pkg, dev, base * 0, x, a, b * 16, None, (256,), torch.zeros(200, dtype=torch.int32))


def test_not_a_number_reaches_its_own_row_alone(pkg, dev):
    T, n = 48, 2
    base, x, a, b, scales = (t.to(dev) for t in _inputs(T, 256, (128,), n, 16, 11))
    ids = torch.arange(T, dtype=torch.int32, device=dev) % n
    want = pkg.lora_add(base, x, a, b, ids, scales=scales)
    x2 = x.clone()
    x2[5, 17], x2[6, 0], x2[40] = float("nan"), float("inf"), float("nan")
    ids2 = ids.clone()
    ids2[40] = -1  # no adapter: its activation is not used
    got = pkg.lora_add(base, x2, a, b, ids2, scales=scales)
    keep = torch.ones(T, dtype=torch.bool, device=dev)
    keep[[5, 6, 40]] = False
    assert torch.equal(got[keep], want[keep]) and bool(got[5].isnan().all()) and not bool(got[6].isfinite().any())
    assert torch.equal(got[40], base[40])
    a2, b2 = a.clone(), b.clone()
    a2[1], b2[1] = float("nan"), float("inf")  # an adapter that no row uses
    got = pkg.lora_add(base, x, a2, b2, torch.zeros_like(ids), scales=scales)
    assert torch.equal(got[ids == 0], want[ids == 0]) and bool(got.isfinite().all())


@pytest.mark.parametrize("kind", ["bf16", "mx"])
def test_in_place_strided_and_rows_of_no_request(pkg, dev, kind):
    T, K, N, live = 75, 544, 136, 70
    base, x, a, b, scales = (t.to(dev) for t in _inputs(T, K, (N,), 3, 32, 13))
    x[live:] = float("nan") if kind == "bf16" else 1.0
    ids = ref.packed_ids([30, 40], T - live).to(dev)
    adapters = torch.tensor([2, -1], dtype=torch.int32, device=dev)
    xi = x if kind == "bf16" else _mx(pkg, dev, x)
    kw = dict(scales=scales, request_ids=ids)
    want = pkg.lora_add(base, xi, a, b, adapters, **kw)
    assert not want[live:].any() and torch.equal(want[30:live], base[30:live])
    wide = torch.full((T, N + 24), 9.0, dtype=torch.bfloat16, device=dev)
    wide[:, 8 : N + 8] = base
    view = wide[:, 8 : N + 8]
    wx = torch.zeros(T, K + 32, dtype=x.dtype, device=dev)
    wx[:, 16 : K + 16] = x
    xs = wx[:, 16 : K + 16]
    if kind == "mx":
        codes = torch.zeros(T, K + 32, dtype=torch.uint8, device=dev)
        codes[:, 16 : K + 16] = xi.codes.view(torch.uint8)
        xs = pkg.MXTensor(codes[:, 16 : K + 16].view(torch.float8_e4m3fn), xi.scales)
    got = pkg.lora_add(view, xs, a, b, adapters, out=view, **kw)
    assert got is view and torch.equal(view[:live], want[:live]) and torch.equal(view[live:], base[live:])
    assert bool((wide[:, :8] == 9.0).all()) and bool((wide[:, N + 8 :] == 9.0).all())


def test_every_mx_scale_and_code(pkg, dev):
    """Codes times their block's scale enter the product exactly: one code per row against ones."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 0x7F) != 0x7F]
    s = torch.arange(16, 247, dtype=torch.uint8)
    grid = torch.cartesian_prod(torch.arange(len(s)), torch.arange(len(codes)))
    T, K = len(grid), 32
    x = torch.zeros(T, K, dtype=torch.uint8)
    x[:, 5] = codes[grid[:, 1]]
    xs = s[grid[:, 0]].view(T, 1).contiguous()
    a = torch.zeros(1, 16, K, dtype=torch.bfloat16)
    a[0, 3] = 1.0
    b = torch.zeros(1, 8, 16, dtype=torch.bfloat16)
    b[0, 2, 3] = 1.0
    mx = pkg.MXTensor(x.view(torch.float8_e4m3fn).to(dev), xs.to(dev))
    out = pkg.lora_add(torch.zeros(T, 8, dtype=torch.bfloat16, device=dev), mx, a.to(dev), b.to(dev),
                       torch.zeros(T, dtype=torch.int32, device=dev)).cpu()
    want = mx.dequantize(torch.float32).cpu().double()[:, 5].to(torch.bfloat16)
    assert torch.equal(out[:, 2], want) and not out[:, [0, 1, 3, 4, 5, 6, 7]].any()


def test_stacked_adapters_of_different_ranks(pkg, dev):
    g = torch.Generator().manual_seed(19)
    K, slices = 320, (128, 64)
    mk = lambda r, w: (torch.randn(r, K, generator=g).to(torch.bfloat16), torch.randn(w, r, generator=g).to(torch.bfloat16))  # noqa: E731
    adapters = [[mk(1, 128), None], [mk(20, 128), mk(7, 64)], [None, mk(33, 64)]]
    a, b = pkg.stack_adapters(adapters, K, slices, device=dev)
    assert a.shape == (3, 2 * 48, K) and b.shape == (3, 192, 48)
    base = torch.randn(9, 192, generator=g).to(torch.bfloat16)
    x = torch.randn(9, K, generator=g).to(torch.bfloat16)
    which = torch.arange(9, dtype=torch.int32) % 3
    _check(pkg, dev, base, x, a.cpu(), b.cpu(), None, slices, which)
    want = base[0, :128].double() + x[0].double() @ adapters[0][0][0].double().t() @ adapters[0][0][1].double().t()
    got = pkg.lora_add(base.to(dev), x.to(dev), a, b, which.to(dev), slices=slices)[0].cpu().double()
    assert float((got[:128] - want).abs().max()) <= 2.0**-7 * float(want.abs().max())
    assert torch.equal(got[128:].to(torch.bfloat16), base[0, 128:])


def test_no_rows_and_equal_calls(pkg, dev):
    base, x, a, b, scales = (t.to(dev) for t in _inputs(1500, 5120, (640,), 4, 64, 23))
    e = torch.empty(0, dtype=torch.int32, device=dev)
    assert pkg.lora_add(base[:0], x[:0], a, b, e).shape == (0, 640)
    ids = (torch.arange(1500, device=dev) // 400).int()
    first = pkg.lora_add(base, x, a, b, ids, scales=scales)
    assert all(torch.equal(first, pkg.lora_add(base, x, a, b, ids, scales=scales)) for _ in range(3))


def test_rows_past_four_gigabytes(pkg, dev):
    T, ld, N = 40000, 1 << 16, 64
    wide = torch.empty(T * ld, dtype=torch.bfloat16, device=dev).as_strided((T, ld), (ld, 1))
    _, _, a, b, _ = (t.to(dev) for t in _inputs(1, 128, (N,), 1, 16, 29))
    rows = torch.tensor([0, 20000, T - 1], device=dev)
    ids = torch.full((T,), -1, dtype=torch.int32, device=dev)
    ids[rows] = 0
    adapters = torch.zeros(1, dtype=torch.int32, device=dev)
    base, x = torch.randn(3, N, device=dev).to(torch.bfloat16), torch.randn(3, 128, device=dev).to(torch.bfloat16)
    wide[rows, :N], wide[rows, 1024:1152] = base, x
    view = wide[:, :N]
    pkg.lora_add(view, wide[:, 1024:1152], a, b, adapters, request_ids=ids, out=view)
    want = pkg.lora_add(base, x, a, b, torch.zeros(3, dtype=torch.int32, device=dev))
    assert torch.equal(wide[rows, :N], want)


def test_graph_replays_with_other_adapters_and_two_graphs(pkg, dev):
    """Replays read the ids anew; two graphs, and eager calls between, hold workspaces of their own."""
    T = 100
    base, x, a, b, scales = (t.to(dev) for t in _inputs(T, 2560, (512,), 3, 32, 31))
    ids = torch.zeros(T, dtype=torch.int32, device=dev)
    call = lambda: pkg.lora_add(base, x, a, b, ids, scales=scales)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for seed in range(3):
        ids.copy_(torch.randint(-1, 3, (T,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32))
        for graph in graphs:
            graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("T", [9, 1100])
def test_a_batch_of_no_requests(pkg, dev, T):
    """No adapter ids at all: every row belongs to no request."""
    base, x, a, b, scales = (t.to(dev) for t in _inputs(T, 128, (64,), 2, 16, 37))
    none = torch.empty(0, dtype=torch.int32, device=dev)
    for ids in (torch.full((T,), -1, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int32, device=dev)):
        out = pkg.lora_add(base, x, a, b, none, scales=scales, request_ids=ids)
        assert out.shape == base.shape and not out.any()
        given = torch.full_like(base, 3.0)
        pkg.lora_add(base, x, a, b, none, scales=scales, request_ids=ids, out=given)
        assert bool((given == 3.0).all())


@pytest.mark.parametrize("zero_rest", [0, 1])
@pytest.mark.parametrize("T,rank", [(9, 16), (1100, 16), (1100, 144)])
def test_more_rows_than_requests_without_request_ids(pkg, dev, T, rank, zero_rest):
    """The C entry point without request_ids: row t is request t, and the rows behind the last request read no adapter id."""
    R, K, N = T - 5, 128, 64
    base, x, a, b, scales = (t.to(dev) for t in _inputs(T, K, (N,), 2, rank, 41))
    ids = (torch.arange(T, device=dev) % 3 - 1).int()  # (ids behind the last request, too: what they say is not used)
    want = pkg.lora_add(base, x, a, b, ids, scales=scales)
    out = torch.full_like(base, 3.0)
    lib = pkg._lib.load()
    size = lib.wanmi_lora_workspace(T, K, 1, rank)
    work = torch.empty(size, dtype=torch.uint8, device=dev)
    p = lambda t: t.data_ptr()  # noqa: E731
    pkg._lib.call("wanmi_lora_add", 0, p(x), None, None, K, p(a), p(b), p(scales), p(ids), None, R, 2, T, K, N, rank, 1, pkg.lora._widths((N,)), p(base), N,
                  p(out), N, zero_rest, p(work), size)
    assert torch.equal(out[:R], want[:R]) and bool((out[R:] == (0.0 if zero_rest else 3.0)).all())


@pytest.mark.parametrize("kind", ["bf16", "mx", "row"])
@pytest.mark.parametrize("K,slices,r", [
    (1664, (256,), 16),  # 13 pairs of steps of K in two splits, the second one shorter
    (2944, (192,), 32), (2944, (64, 128), 64), (2944, (136,), 128),  # 23 pairs in three, the last one shorter
    (5120, (256,), 32), (5120, (128, 64, 64), 64), (5120, (320,), 128),  # 40 pairs in four
    (13824, (64,), 32), (13824, (128,), 96), (13824, (72,), 128), (13824, (64,), 160),  # 108 pairs in six
])
def test_many_rows_in_several_splits_of_k(pkg, dev, kind, K, slices, r):
    ids = ref.packed_ids([500, 0, 413, 200], 5)
    base, x, a, b, scales = _inputs(len(ids), K, slices, 3, r, K + r)
    adapters = torch.tensor([1, 0, -1, 2], dtype=torch.int32)
    _check(pkg, dev, base, x, a, b, scales, slices, adapters, ids, kind=kind)
