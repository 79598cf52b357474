"""Every tile of the products with block-scaled 8-bit weights and every way to share out their sums, against 64-bit results."""

import pytest
import torch

import text_ref as ref
from fp8_tiles import TILES
from test_gpu_fp8_block import _to, _weight, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N", TILES)
def test_every_tile(pkg, dev, M, K, N):
    """From bf16, from codes whose scales lie block by block, and row by row, with a bias and GELU or neither."""
    g = torch.Generator().manual_seed(M + K + N)
    gelu = (M + N // 8) % 2 == 1
    x, w = _x(M, K, g), _weight(pkg, N, K, g, bias=gelu)
    codes, scales = ref.row_blocks(x)
    want = ref.block_linear(codes, scales, w.codes, w.scales, w.bias, gelu)
    c, s = codes.to(dev), scales.to(dev)
    outs = [pkg.fp8_block_linear(arg, _to(w, dev), activation="gelu" if gelu else None)
            for arg in (x.to(dev), pkg.FP8BlockTensor(c, s.t().contiguous().t()), pkg.FP8BlockTensor(c, s))]
    ref.check_block_linear(outs[0], *want)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("M,K,N", [(333, 4112, 5096), (500, 1040, 5128), (1000, 1040, 5120), (2000, 528, 5000)])
def test_graphs_and_streams_of_the_larger_tiles(pkg, dev, M, K, N):
    """The same bits in every run, beside other calls, and in two replayed graphs with other rows."""
    g = torch.Generator().manual_seed(M)
    x, w = _x(M, K, g).to(dev), _to(_weight(pkg, N, K, g), dev)
    want = pkg.fp8_block_linear(x, w, activation="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [pkg.fp8_block_linear(x, w, activation="gelu") for _ in range(3)]
    mine = [pkg.fp8_block_linear(x, w, activation="gelu") for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in other + mine)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(pkg.fp8_block_linear(x, w))
    for seed in range(3):
        x.copy_(_x(M, K, torch.Generator().manual_seed(seed)))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = pkg.fp8_block_linear(x, w)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)


@pytest.mark.parametrize("M,K,N", [(333, 4112, 5096), (500, 272, 5128), (1000, 1040, 5120), (2000, 528, 5000), (40, 5120, 640)])
def test_nothing_is_written_beside_the_output(pkg, dev, M, K, N):
    """The output as rows and columns in the middle of a larger tensor."""
    g = torch.Generator().manual_seed(N)
    x, w = _x(M, K, g).to(dev), _to(_weight(pkg, N, K, g), dev)
    slab = torch.full((M + 6, N + 24), 7.0, dtype=torch.bfloat16, device=dev)
    out = slab[3 : M + 3, 8 : N + 8]
    want = pkg.fp8_block_linear(x, w)
    assert torch.equal(pkg.fp8_block_linear(x, w, out=out), want)
    out.fill_(7.0)
    assert bool((slab == 7).all())
