"""The operators for packed batches as they are used together: Wan blocks over several requests at once, against the
single-request block of :mod:`block` run for each request alone.

The two paths share every GEMM and differ in where they round: q and k once instead of twice, 2^-8 of a value, and
fp32 sums in another order. What follows re-quantizes to e4m3, whose steps are up to 2^-3 of a value: two inputs that
differ by a share d fall on different codes with probability d / step and are then a step apart, a mean square of
(d / step) step^2 = d step. With d = 2^-8 that is an RMS of sqrt(2^-8 2^-3) = 2.2e-2 of what is quantized, hence of the
block's update out - h, which is linear in the last quantized tensor (the block against its oracle has
measured 2.3e-2). Independent over blocks, it grows with their square root. An element of the update sums the changes of
hundreds of codes, times the gate of its channel: it is near-normal with a deviation of that channel, which is as
many times the mean one as its gate is of the gates' root mean square (the timestep embedding is N(0, 1) here, so up to
its largest entry), and six of these bound the largest of < 10^6 elements. The bars allow 1.4 times the deviation."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DIM, HEADS, FFN = 512, 4, 1024
GRIDS = [(1, 6, 8), (2, 5, 7), (1, 1, 1), (3, 10, 10)]


def _setup(pkg, dev, blocks=2, pad=6, seed=3):
    blk = pkg.block
    g = torch.Generator(device=dev).manual_seed(seed)
    ws = [blk.random_block_weights(dev, g, dim=DIM, ffn=FFN, heads=HEADS, std=0.04, qk_gamma_mean=1.0, keep_raw=False)[0] for _ in range(blocks)]
    lengths = [f * h * w for f, h, w in GRIDS]
    packed = pkg.PackedRequests.from_lengths(lengths, sum(lengths) + pad, dev)
    h = torch.randn(packed.rows, DIM, device=dev, generator=g).to(torch.bfloat16)
    h[sum(lengths):] = float("nan")
    temb = torch.randn(len(GRIDS), 6, DIM, device=dev, generator=g)
    ctx = [torch.randn(20 + 13 * i, DIM, device=dev, generator=g).to(torch.bfloat16) for i in range(len(GRIDS))]
    crosses = [[blk.project_cross_kv(w, c) for c in ctx] for w in ws]
    return ws, packed, packed.grid_positions(GRIDS), h, temb, crosses


def _close(got, ref, what, temb, blocks=1):
    got, ref = got.double().flatten(), ref.double().flatten()
    sigma = 1.4 * (blocks * 2.0**-8 * 2.0**-3) ** 0.5
    rms = ref.square().mean().sqrt()
    off = float((got - ref).square().mean().sqrt() / rms)
    most = float((got - ref).abs().max() / rms)
    gates = float(temb.abs().max() / temb.square().mean().sqrt())
    assert off <= sigma and most <= 6 * sigma * gates, (what, off, most, sigma, gates)


def test_each_request_gets_what_it_gets_alone(pkg, dev):
    ws, packed, pos, h, temb, crosses = _setup(pkg, dev)
    out = pkg.packed_dit_forward(ws, h, temb, packed, pos, crosses)
    for i, (a, b) in enumerate(packed.spans()):
        rope = pkg.rope_tables(GRIDS[i], device=dev)
        want = pkg.block.dit_forward(ws, h[a:b].contiguous(), temb[i], rope, [c[i] for c in crosses])
        _close(out[a:b] - h[a:b], want - h[a:b], i, temb, blocks=2)
    assert not out[packed.rows - 6:].any()


def _adapters(pkg, dev, seed):
    g = torch.Generator().manual_seed(seed)

    def one(k, widths, r):
        return [(torch.randn(r, k, generator=g) * k**-0.5, torch.randn(n, r, generator=g) * 0.5) for n in widths]

    def stack(k, widths):
        a, b = pkg.stack_adapters([one(k, widths, 16), one(k, widths, 5)], k, widths, device=dev)
        return pkg.packed_block.Adapters(a, b, torch.tensor([0.7, 1.1], device=dev))

    return pkg.packed_block.BlockAdapters(stack(DIM, (DIM,) * 3), stack(DIM, (DIM,)), stack(DIM, (DIM,)), stack(DIM, (DIM,)), stack(FFN, (DIM,)))


def test_adapters_reach_their_own_requests(pkg, dev):
    """With adapters on some requests: those without get the bits of a batch without adapters, those with get what they
    get in a batch of their own, and it is not what they get without."""
    ws, packed, pos, h, temb, crosses = _setup(pkg, dev, blocks=1)
    ad = _adapters(pkg, dev, 5)
    ids = torch.tensor([1, -1, -1, 0], dtype=torch.int32, device=dev)
    plain = pkg.packed_block_forward(ws[0], h, temb, packed, pos, crosses[0])
    out = pkg.packed_block_forward(ws[0], h, temb, packed, pos, crosses[0], adapters=ad, adapter_ids=ids)
    none = pkg.packed_block_forward(ws[0], h, temb, packed, pos, crosses[0], adapters=ad, adapter_ids=ids * 0 - 1)
    for i, (a, b) in enumerate(packed.spans()):
        alone = pkg.PackedRequests.from_lengths([b - a], device=dev)
        want = pkg.packed_block_forward(ws[0], h[a:b].contiguous(), temb[i : i + 1], alone, pos[a:b].contiguous(), [crosses[0][i]],
                                        adapters=ad, adapter_ids=ids[i : i + 1].clone())
        _close(out[a:b] - h[a:b], want - h[a:b], i, temb)
        if int(ids[i]) < 0:
            assert torch.equal(out[a:b], none[a:b])
        else:
            change = (out[a:b] - plain[a:b]).float().norm() / (plain[a:b] - h[a:b]).float().norm()
            assert float(change) > 0.1
    _close(none[: packed.rows - 6] - h[: packed.rows - 6], plain[: packed.rows - 6] - h[: packed.rows - 6], "no adapters", temb)


def test_captured_and_replayed_with_other_adapters_and_steps(pkg, dev):
    ws, packed, pos, h, temb, crosses = _setup(pkg, dev, blocks=1)
    ad = _adapters(pkg, dev, 6)
    ids = torch.tensor([1, -1, 0, 0], dtype=torch.int32, device=dev)
    call = lambda: pkg.packed_block_forward(ws[0], h, temb, packed, pos, crosses[0], adapters=ad, adapter_ids=ids)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        ids.copy_(torch.randint(-1, 2, (4,), generator=g, dtype=torch.int32))
        temb.copy_(torch.randn(temb.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_forward_changes_none_of_its_inputs(pkg, dev):
    ws, packed, pos, h, temb, crosses = _setup(pkg, dev, blocks=1)
    before = [t.clone() for t in (h, temb, pos, packed.request_ids)]
    first = pkg.packed_block_forward(ws[0], h, temb, packed, pos, crosses[0])
    again = pkg.packed_block_forward(ws[0], h, temb, packed, pos, crosses[0])
    assert torch.equal(first, again)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (h, temb, pos, packed.request_ids)))


def test_requests_without_rows_and_a_batch_without_any(pkg, dev):
    ws, _, _, h, temb, crosses = _setup(pkg, dev, blocks=1)
    grids = [(0, 5, 7), (2, 5, 7), (1, 0, 3)]
    packed = pkg.PackedRequests.from_lengths([0, 70, 0], 72, dev)
    got = pkg.packed_dit_forward(ws, h[:72], temb[:3], packed, packed.grid_positions(grids), [crosses[0][:3]])
    alone = pkg.PackedRequests.from_lengths([70], 72, dev)
    want = pkg.packed_dit_forward(ws, h[:72], temb[1:2], alone, alone.grid_positions(grids[1:2]), [crosses[0][1:2]])
    assert torch.equal(got, want)
    none = pkg.PackedRequests.from_lengths([0, 0], 0, dev)
    empty = pkg.packed_dit_forward(ws, h[:0], temb[:2], none, none.grid_positions(grids[::2]), [crosses[0][:2]])
    assert empty.shape == (0, DIM)
    idle = pkg.PackedRequests.from_lengths([0], 5, dev)
    assert not pkg.packed_dit_forward(ws, h[-5:], temb[:1], idle, idle.grid_positions(grids[:1]), [crosses[0][:1]]).any()
