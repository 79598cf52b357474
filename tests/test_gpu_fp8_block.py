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
         (129, 640, 1000), (300, 144, 5120), (700, 1024, 2048), (2000, 528, 5000), (4100, 256, 4360), (4000, 400, 8192)]


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
