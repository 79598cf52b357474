"""Products with block-scaled 8-bit weights (fp8_block_linear, quantize_fp8_blocks) against 64-bit results."""

import pytest
import torch

import text_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _x(M, K, g, zero_block=True):
    x = torch.randn(M, K, generator=g) * (0.25 + 2 * torch.rand(M, 1, generator=g))
    if zero_block:
        x[M // 2, : min(K, 128)] = 0  # a block of zeros
    return x.to(BF16)


def _weight(pkg, N, K, g, bias=True):
    w = pkg.quantize_weight_fp8_blocks(torch.randn(K, N, generator=g) * K**-0.5, 0.1 * torch.randn(N, generator=g) if bias else None)
    # scales that are no power of two and far apart
    return w._replace(scales=w.scales * torch.exp2(4 * torch.rand(w.scales.shape, generator=g) - 2))


def _to(w, dev):
    return w._replace(codes=w.codes.to(dev), scales=w.scales.to(dev), bias=None if w.bias is None else w.bias.to(dev))


@pytest.mark.parametrize("M,K", [(1, 16), (3, 128), (5, 144), (65, 640), (1000, 5120), (130, 1520), (2, 13824)])
def test_quantize(pkg, dev, M, K):
    g = torch.Generator().manual_seed(M + K)
    x = _x(M, K, g) * torch.exp2(torch.randint(-60, 60, (M, 1), generator=g)).to(BF16)
    # values that a division puts onto the border between two codes
    x[0, :16] = torch.tensor([448.0, 17, 19, 21, 27, 33, 34, 38, 42, 50, 54, 66, 68, 76, 2.0**-10, -17], dtype=BF16) if K < 128 else x[0, :16]
    got = pkg.quantize_fp8_blocks(x.to(dev))
    codes, scales = ref.row_blocks(x)
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.codes.cpu().view(torch.uint8), codes.view(torch.uint8))


SIZES = [(1, 16, 8), (1, 5120, 640), (3, 128, 128), (16, 400, 264), (17, 1024, 72), (33, 2064, 136), (64, 640, 256), (65, 256, 64), (100, 1552, 200),
         (129, 640, 1000), (300, 144, 5120), (700, 1024, 2048), (2000, 528, 5000), (4100, 256, 4360), (4000, 400, 8192), (1000, 1040, 5120), (2100, 1040, 8200)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("form", ["bf16", "codes", "codes_rows"])
def test_linear(pkg, dev, M, K, N, form):
    g = torch.Generator().manual_seed(M * 7 + K + N)
    gelu = (M + K // 16) % 2 == 1
    x, w = _x(M, K, g), _weight(pkg, N, K, g, bias=M % 3 != 0)
    codes, scales = ref.row_blocks(x)
    if form == "bf16":
        arg = x.to(dev)
    else:
        s = scales.to(dev)
        arg = pkg.FP8BlockTensor(codes.to(dev), s.t().contiguous().t() if form == "codes" else s)
    got = pkg.fp8_block_linear(arg, _to(w, dev), activation="gelu" if gelu else None)
    ref.check_block_linear(got, *ref.block_linear(codes, scales, w.codes, w.scales, w.bias, gelu))


def _one(pkg, dev, M, K, N, seed=1):
    g = torch.Generator().manual_seed(seed)
    return _x(M, K, g).to(dev), _to(_weight(pkg, N, K, g), dev)


@pytest.mark.parametrize("M", [1, 4, 16, 100, 700])
def test_layouts_and_given_outputs(pkg, dev, M):
    K, N = 272, 136
    x, w = _one(pkg, dev, M, K, N)
    want = pkg.fp8_block_linear(x, w)
    out = torch.full((M + 1, N + 8), 7.0, dtype=BF16, device=dev)
    assert torch.equal(pkg.fp8_block_linear(x, w, out=out[:M, :N]), want)
    assert torch.equal(out[:M, :N], want) and bool((out[M:] == 7).all()) and bool((out[:, N:] == 7).all())
    wide = torch.randn(M, K + 40, device=dev).to(BF16)
    wide[:, 8 : K + 8] = x
    assert torch.equal(pkg.fp8_block_linear(wide[:, 8 : K + 8], w), want)
    q = pkg.quantize_fp8_blocks(x)
    wide = torch.zeros(M, K + 48, dtype=torch.uint8, device=dev)
    wide[:, 16 : K + 16] = q.codes.view(torch.uint8)
    codes = wide.view(torch.float8_e4m3fn)[:, 16 : K + 16]
    for scales in (q.scales, q.scales.contiguous(), q.scales.repeat(1, 2)[:, ::2] * 0 + q.scales, torch.stack([q.scales, q.scales], 2)[:, :, 1]):
        assert torch.equal(pkg.fp8_block_linear(pkg.FP8BlockTensor(codes, scales), w), want)
    same = pkg.FP8BlockTensor(q.codes, q.scales[:1].expand(M, 3))  # one scale for all rows
    assert torch.equal(pkg.fp8_block_linear(same, w), pkg.fp8_block_linear(pkg.FP8BlockTensor(q.codes, same.scales.contiguous()), w))
    if M % 4 == 0:
        assert torch.equal(pkg.fp8_block_linear(x.view(2, M // 4, 2, K), w), want.view(2, M // 4, 2, N))
        q4 = pkg.quantize_fp8_blocks(x.view(2, M // 4, 2, K))
        assert q4.codes.shape == (2, M // 4, 2, K) and torch.equal(pkg.fp8_block_linear(q4, w), want.view(2, M // 4, 2, N))
    assert torch.equal(pkg.fp8_block_linear(x[0], w), pkg.fp8_block_linear(x[:1], w)[0])
    assert pkg.fp8_block_linear(x[:0], w).shape == (0, N) and pkg.quantize_fp8_blocks(x[:0]).scales.shape == (0, 3)


@pytest.mark.parametrize("M", [3, 16, 100, 600])
def test_values_at_the_ends_of_their_range(pkg, dev, M):
    """Blocks with an infinity or a NaN are NaN, and with them their rows alone; the smallest and largest values; GELU far out."""
    K, N = 384, 128
    x, w = _one(pkg, dev, M, K, N, 3)
    want = pkg.fp8_block_linear(x, w)
    bad = x.clone()
    bad[0, 130], bad[2, 5], bad[2, 6] = float("inf"), float("nan"), float("-inf")
    got = pkg.fp8_block_linear(bad, w)
    assert got[0].isnan().all() and got[2].isnan().all()
    keep = [i for i in range(M) if i not in (0, 2)]
    assert torch.equal(got[keep], want[keep])
    q = pkg.quantize_fp8_blocks(bad)
    assert q.codes[0, 128:256].float().isnan().all() and not q.codes[0, :128].float().isnan().any() and q.codes[2, :128].float().isnan().all()
    tiny = x.clone()
    tiny[0] = 2.0**-120  # below the smallest scale times a code: rounds to codes of it
    tiny[1] = 0
    codes, scales = ref.row_blocks(tiny.cpu())
    wc = _to(w, "cpu")
    ref.check_block_linear(pkg.fp8_block_linear(tiny, w._replace(bias=None)), *ref.block_linear(codes, scales, wc.codes, wc.scales, None, False))
    assert not pkg.fp8_block_linear(tiny, w._replace(bias=None))[1].any()
    big = (x.float() * 2.0**60).to(BF16)
    codes, scales = ref.row_blocks(big.cpu())
    ref.check_block_linear(pkg.fp8_block_linear(big, w), *ref.block_linear(codes, scales, wc.codes, wc.scales, wc.bias, False))
    y = pkg.fp8_block_linear(big, w, activation="gelu")
    assert not y.isnan().any()
    lin = pkg.fp8_block_linear(big, w)
    assert torch.equal(y[lin > 100], lin[lin > 100]) and not y[lin < -100].any()


@pytest.mark.parametrize("M,K,N", [(2, 640, 256), (40, 5120, 640), (150, 5120, 512), (300, 400, 4096), (5000, 400, 4096)])
def test_graphs_streams_and_repeats(pkg, dev, M, K, N):
    """Few rows, parts of a sum, and tiles of each kind: the same bits in every run, beside other calls, and replayed with other rows."""
    x, w = _one(pkg, dev, M, K, N, 5)
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


def test_codes_beyond_four_gigabytes(pkg, dev):
    """Rows whose codes, values and outputs lie beyond 2^31 and 2^32 bytes from the first; the last rows against the same rows alone."""
    M, K, N = 270000, 16384, 8
    g = torch.Generator().manual_seed(2)
    w = _to(_weight(pkg, N, K, g), dev)
    tail = _x(513, K, g).to(dev)
    x = torch.zeros(M, K, dtype=BF16, device=dev)
    x[-513:] = tail
    got = pkg.fp8_block_linear(x, w)
    codes, scales = ref.row_blocks(tail.cpu())
    wc = _to(w, "cpu")
    ref.check_block_linear(got[-513:], *ref.block_linear(codes, scales, wc.codes, wc.scales, wc.bias, False))
    assert torch.equal(got[: M - 513], w.bias.to(BF16).expand(M - 513, N))
    del x, got
    torch.cuda.empty_cache()
    M, K, N = 150000, 128, 16384  # outputs
    x = _x(M, K, g, zero_block=False).to(dev)
    w = _to(_weight(pkg, N, K, g), dev)
    got = pkg.fp8_block_linear(x, w)
    codes, scales = ref.row_blocks(x[-300:].cpu())
    wc = _to(w, "cpu")
    ref.check_block_linear(got[-300:], *ref.block_linear(codes, scales, wc.codes, wc.scales, wc.bias, False))
    del x, got
    torch.cuda.empty_cache()
