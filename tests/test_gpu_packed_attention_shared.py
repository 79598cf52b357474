"""Attention over packed rows in tiles of 32 rows whose keys the waves share out: few rows over long texts."""

import pytest
import torch

import text_ref as ref
from attention_forms import SHARED
from test_gpu_packed_attention import _inputs, _score_size

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _call(pkg, dev, case):
    q_lens, k_lens, pad, heads, k_heads, D = SHARED[case]
    q, k, v = _inputs(sum(q_lens) + pad, sum(k_lens), heads, k_heads, D, 30 + case)
    return (q, k, v), [t.to(dev) for t in (q, k, v)], ref.offsets(q_lens, dev), ref.offsets(k_lens, dev)


@pytest.mark.parametrize("case", range(len(SHARED)))
def test_results_codes_and_given_outputs(pkg, dev, case):
    """Against 64 bits; as MX codes, those of the bf16 output; into columns of a larger tensor and into q itself, rows behind the last request left."""
    q_lens, k_lens, pad, heads, k_heads, D = SHARED[case]
    (q, k, v), gpu, qo, ko = _call(pkg, dev, case)
    n, T = sum(q_lens), sum(q_lens) + pad
    got = pkg.packed_cross_attention(*gpu, qo, ko)
    want, size = ref.attention(q, k, v, q_lens, k_lens, D**-0.5)
    assert torch.isfinite(got).all()
    assert not ((got.double().cpu() - want).abs() > ref.attention_bound(size, want, _score_size(q, k, D**-0.5), D)).any()
    mx = pkg.packed_cross_attention(*gpu, qo, ko, quant="mx")
    as_mx = pkg.adaln_kernels.adaln_quant_2d(got.view(T, -1), None, None, eps=0.0, norm_type="none", quant="mx")
    assert torch.equal(mx.codes.view(torch.uint8), as_mx.codes.view(torch.uint8)) and torch.equal(mx.scales, as_mx.scales)
    slab = torch.full((T + 2, 3 * heads, D), 7.0, dtype=BF16, device=dev)
    out = slab[1 : T + 1, heads : 2 * heads]
    pkg.packed_cross_attention(*gpu, qo, ko, out=out)
    assert torch.equal(out[:n], got[:n]) and bool((out[n:] == 7).all())
    out.fill_(7.0)
    assert bool((slab == 7).all())
    own = gpu[0].clone()
    pkg.packed_cross_attention(own, *gpu[1:], qo, ko, out=own)
    assert torch.equal(own[:n], got[:n]) and torch.equal(own[n:], gpu[0][n:])
    major = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in gpu]
    assert torch.equal(pkg.packed_cross_attention(*major, qo, ko), got)


@pytest.mark.parametrize("lens,H,D", [([100], 12, 64), ([1024], 12, 64), ([90, 80, 100], 4, 128), ([200, 1], 8, 64)])
def test_prompts_with_a_bias(pkg, dev, lens, H, D):
    n = sum(lens)
    g = torch.Generator().manual_seed(n)
    qkv = torch.randn(n + 3, 3 * H, D, generator=g)
    qkv[:, :H] *= D**-0.5
    qkv = qkv.to(BF16)
    table = 1.5 * torch.randn(32, H, generator=g)
    slab = qkv.to(dev)
    got = pkg.relative_bias_attention(*(slab[:, i * H : (i + 1) * H] for i in range(3)), table.to(dev), ref.offsets(lens, dev))
    q, k, v = (qkv[:n, i * H : (i + 1) * H] for i in range(3))
    want, size = ref.attention(q, k, v, lens, lens, 1.0, lambda m: ref.bias_matrix(table, m, 128, True))
    assert torch.isfinite(got).all() and not got[n:].any()
    bound = ref.attention_bound(size, want, _score_size(q, k, 1.0) + float(table.abs().max()), D)
    assert not ((got[:n].double().cpu() - want).abs() > bound).any()


def test_replayed_graphs(pkg, dev):
    """Replays follow queries and offsets that were changed in place, in two graphs."""
    _, (q, k, v), qo, ko = _call(pkg, dev, 3)
    graphs, outs = [], []
    pkg.packed_cross_attention(q, k, v, qo, ko)
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(pkg.packed_cross_attention(q, k, v, qo, ko))
    for a, b in (([3, 1, 9], [140, 0, 170]), ([0, 17, 0], [1, 300, 9]), ([5, 5, 5], [0, 0, 310])):
        qo.copy_(ref.offsets(a))
        ko.copy_(ref.offsets(b))
        q.mul_(0.75)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = pkg.packed_cross_attention(q, k, v, qo, ko)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)
