"""Attention over packed rows whose heads lie far apart: head-major tensors of long clips, each head's rows one behind the other."""

import pytest
import torch

import text_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("T,D", [(75600, 128), (65600, 64), (32768, 128)])
def test_head_major_tensors_of_long_clips(pkg, dev, T, D):
    """Heads 2^22 elements apart and more, of q, k and v."""
    H = 2
    g = torch.Generator(device=dev).manual_seed(T)
    major = [torch.randn(H, T, D, device=dev, generator=g).to(BF16).transpose(0, 1) for _ in range(3)]
    assert major[0].stride(1) >= 1 << 22
    rows = [t.contiguous() for t in major]
    table = torch.randn(32, H, device=dev, generator=g)
    for lens in ([300] * (T // 300), [20] * (T // 20)):
        o = ref.offsets(lens, dev)
        assert torch.equal(pkg.packed_cross_attention(*major, o, o), pkg.packed_cross_attention(*rows, o, o))
        assert torch.equal(pkg.relative_bias_attention(*major, table, o), pkg.relative_bias_attention(*rows, table, o))


def test_heads_beyond_four_gigabytes(pkg, dev):
    H, D, T, far = 2, 64, 200, 1 << 25
    slab = torch.empty(H, far, 3 * D, dtype=BF16, device=dev)  # 25 GB, of which the heads' first rows are touched
    slab[:, :T] = torch.randn(H, T, 3 * D, device=dev).to(BF16)
    q, k, v = (slab[:, :T, i * D : (i + 1) * D].transpose(0, 1) for i in range(3))
    assert q.stride(1) > 1 << 32
    for lens in ([150, 50], [2] * 100):
        o = ref.offsets(lens, dev)
        assert torch.equal(pkg.packed_cross_attention(q, k, v, o, o), pkg.packed_cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), o, o))
    del slab, q, k, v
    torch.cuda.empty_cache()
