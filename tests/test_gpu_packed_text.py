"""The operators on the text side as they are used together: prompts through an encoder layer with a relative position bias and
block-scaled weights, their keys and values for a block, and the block's cross-attention over packed texts.

The block's bars are those of the packed blocks against single ones: what is quantized behind an attention that rounds in
another order is off by (2^-8 2^-3)^(1/2) of itself, the square root of the blocks as often."""

import sys

import pytest
import torch

import text_ref as ref
from test_gpu_packed_block import DIM, FFN, GRIDS, HEADS, _adapters, _close, _setup

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _texts(dev, lens=(20, 33, 0, 59), pad=5, seed=4):
    g = torch.Generator(device=dev).manual_seed(seed)
    ctx = torch.randn(sum(lens) + pad, DIM, device=dev, generator=g).to(BF16)
    return lens, ctx


@pytest.mark.parametrize("together", [True, False])
def test_packed_texts_give_what_each_text_gives_alone(pkg, dev, together, monkeypatch):
    """packed_dit_forward with the texts packed, against one cross-attention per request, whose text is never empty. Self-attention
    all together as for short requests, or request by request as for long ones."""
    monkeypatch.setattr(sys.modules[pkg.PackedRequests.__module__], "_TOGETHER", 3600 if together else 0)
    ws, packed, pos, h, temb, _ = _setup(pkg, dev)
    lens, ctx = _texts(dev, (20, 33, 7, 59))
    text = pkg.PackedRequests.from_lengths(lens, ctx.shape[0], dev)
    one = [[pkg.block.project_cross_kv(w, ctx[a:b]) for a, b in text.spans()] for w in ws]
    want = pkg.packed_dit_forward(ws, h, temb, packed, pos, one)
    got = pkg.packed_dit_forward(ws, h, temb, packed, pos, [pkg.project_packed_cross_kv(w, ctx, text) for w in ws])
    n = sum(packed.lengths)
    _close(got[:n] - h[:n], want[:n] - h[:n], "packed texts", temb, blocks=2)
    assert not got[n:].any()
    mixed = pkg.packed_dit_forward(ws, h, temb, packed, pos, [one[0], pkg.project_packed_cross_kv(ws[1], ctx, text)])
    _close(mixed[:n] - h[:n], want[:n] - h[:n], "one block packed", temb, blocks=2)


def test_an_empty_text_changes_with_no_other(pkg, dev):
    """A request whose text is empty attends to nothing: its rows have the bits that they have in a batch whose other texts differ."""
    ws, packed, pos, h, temb, _ = _setup(pkg, dev, blocks=1)
    lens, ctx = _texts(dev)
    w = ws[0]
    a = pkg.packed_block_forward(w, h, temb, packed, pos, pkg.project_packed_cross_kv(w, ctx, pkg.PackedRequests.from_lengths(lens, ctx.shape[0], dev)))
    other = (3, 1, 0, 100)
    b = pkg.packed_block_forward(w, h, temb, packed, pos, pkg.project_packed_cross_kv(w, ctx, pkg.PackedRequests.from_lengths(other, ctx.shape[0], dev)))
    spans = list(packed.spans())
    assert torch.equal(a[spans[2][0] : spans[2][1]], b[spans[2][0] : spans[2][1]])
    assert not torch.equal(a[: spans[0][1]], b[: spans[0][1]])
    assert not torch.isnan(a.float()).any()


def _block_weights(pkg, dev, seed=11):
    """A block whose projections are all block-scaled, and the same with every weight dequantized and MX-quantized."""
    g = torch.Generator(device=dev).manual_seed(seed)
    w, raw = pkg.block.random_block_weights(dev, g, dim=DIM, ffn=FFN, heads=HEADS, std=0.04, qk_gamma_mean=1.0)
    names = ("qkv", "o", "q2", "k2", "v2", "o2", "up", "down")
    fp8 = {n: pkg.quantize_weight_fp8_blocks(raw[n + "_w"].float(), raw[n + "_b"]) for n in names}
    mx = {n: pkg.quantize_weight_mx(f.dequantize(BF16).t().contiguous(), f.bias) for n, f in fp8.items()}
    return w._replace(**fp8), w._replace(**mx)


def test_a_block_of_block_scaled_weights(pkg, dev):
    """Against the same block with MX weights made of the same values. Both quantize activations to e4m3, on different scales, and the MX
    weights are rounded once more: each operand is off by up to half a step, 2^-4 of itself, uniformly: an RMS of 2^-4 / sqrt(3) 2 / 1.5 per
    operand at most (the step is up to 2^-3 of a value in [1, 2) 2^e, of mean square 7 / 3 against 1 / 12 of the step's square): 2^-3
    / sqrt(12) / sqrt(7 / 3) = 2.4e-2. Three roundings apart in each of the five products on the way, independent: sqrt(15)
    2.4e-2 = 9.2e-2 of the update."""
    fp8, mx = _block_weights(pkg, dev)
    _, packed, pos, h, temb, _ = _setup(pkg, dev, blocks=1)
    lens, ctx = _texts(dev)
    text = pkg.PackedRequests.from_lengths(lens, ctx.shape[0], dev)
    got = pkg.packed_block_forward(fp8, h, temb, packed, pos, pkg.project_packed_cross_kv(fp8, ctx, text))
    want = pkg.packed_block_forward(mx, h, temb, packed, pos, pkg.project_packed_cross_kv(mx, ctx, text))
    n = sum(packed.lengths)
    up, ref_up = (got[:n] - h[:n]).double(), (want[:n] - h[:n]).double()
    assert float((up - ref_up).norm() / ref_up.norm()) <= 9.2e-2
    # weights of both kinds in one block, request by request, with adapters
    ids = torch.tensor([1, -1, 0, 0], dtype=torch.int32, device=dev)
    one = [pkg.block.project_cross_kv(mx, ctx[a:b] if b > a else ctx[:1]) for a, b in text.spans()]
    for kinds in (dict(o=mx.o, up=mx.up), dict(q2=mx.q2, down=mx.down), dict(qkv=mx.qkv, o2=mx.o2)):
        both = fp8._replace(**kinds)
        got = pkg.packed_block_forward(both, h, temb, packed, pos, one, adapters=_adapters(pkg, dev, 5), adapter_ids=ids)
        want = pkg.packed_block_forward(mx, h, temb, packed, pos, one, adapters=_adapters(pkg, dev, 5), adapter_ids=ids)
        up, ref_up = (got[:n] - h[:n]).double(), (want[:n] - h[:n]).double()
        assert float((up - ref_up).norm() / ref_up.norm()) <= 9.2e-2, kinds.keys()


def test_no_text_at_all(pkg, dev):
    """Every request's text empty, without a row of context: as rows of context that belong to no text."""
    _, packed, pos, h, temb, _ = _setup(pkg, dev, blocks=1)
    _, ctx = _texts(dev)
    none = [0] * len(packed.lengths)
    for w in _block_weights(pkg, dev):
        kv = pkg.project_packed_cross_kv(w, ctx[:0], pkg.PackedRequests.from_lengths(none, 0, dev))
        assert kv.k.shape == kv.v.shape == (0, HEADS, 128)
        got = pkg.packed_block_forward(w, h, temb, packed, pos, kv)
        rows = pkg.project_packed_cross_kv(w, ctx, pkg.PackedRequests.from_lengths(none, ctx.shape[0], dev))
        assert torch.equal(got, pkg.packed_block_forward(w, h, temb, packed, pos, rows))


def _encoder(pkg, x, offsets, p):
    """One layer of a text encoder on packed prompts: RMSNorm, attention with a relative position bias, RMSNorm, GELU-gated FFN."""
    norm = lambda t, g: pkg.adaln_kernels.adaln_quant_2d(t, g, None, eps=1e-6, norm_type="rms_norm", quant="none")  # noqa: E731
    T = x.shape[0]
    qkv = pkg.fp8_block_linear(norm(x, p["g1"]), p["qkv"]).view(T, 3 * HEADS, DIM // HEADS)
    q, k, v = (qkv[:, i * HEADS : (i + 1) * HEADS] for i in range(3))
    o = pkg.relative_bias_attention(q, k, v, p["table"], offsets, out=q)
    x = x + pkg.fp8_block_linear(o.reshape(T, DIM), p["o"])
    a = norm(x, p["g2"])
    return x + pkg.fp8_block_linear(pkg.fp8_block_linear(a, p["gate"], activation="gelu") * pkg.fp8_block_linear(a, p["up"]), p["down"])


def _encoder_weights(pkg, dev, seed=21):
    g = torch.Generator().manual_seed(seed)
    w = lambda k, n: pkg.quantize_weight_fp8_blocks((torch.randn(k, n, generator=g) * k**-0.5).to(dev))  # noqa: E731
    qkv = torch.randn(DIM, 3 * DIM, generator=g) * DIM**-0.5
    qkv[:, :DIM] *= (DIM // HEADS) ** -0.5  # the scores of such an encoder are not scaled
    return dict(qkv=pkg.quantize_weight_fp8_blocks(qkv.to(dev)), o=w(DIM, DIM), gate=w(DIM, FFN), up=w(DIM, FFN), down=w(FFN, DIM),
                table=torch.randn(32, HEADS, generator=g).to(dev), g1=(1 + 0.1 * torch.randn(DIM, generator=g)).to(dev),
                g2=(1 + 0.1 * torch.randn(DIM, generator=g)).to(dev))


def test_prompts_through_the_encoder_and_the_block(pkg, dev):
    """Packed prompts get what each gets alone, up to sums in another order (the rows choose the tile and the parts of a sum); all get what the
    layer gives in fp64, up to the activations' rounding; and the whole path is captured and replayed with other prompts and lengths."""
    p = _encoder_weights(pkg, dev)
    g = torch.Generator(device=dev).manual_seed(22)
    lens, rows = [150, 33, 90], 300
    x = torch.randn(rows, DIM, device=dev, generator=g).to(BF16)
    offsets = ref.offsets(lens, dev)
    out = _encoder(pkg, x, offsets, p)
    for i, n in enumerate(lens):
        a = int(offsets[i])
        alone = _encoder(pkg, x[a : a + n].contiguous(), ref.offsets([n], dev), p)
        err = (alone - out[a : a + n]).double().norm() / out[a : a + n].double().norm()
        assert float(err) <= 2.2e-2, (i, float(err))  # rounding behind sums in another order: (2^-8 2^-3)^(1/2)
    # against the same layer in fp64, on dequantized weights: the activations' e4m3 alone, 2.4e-2 a product, four products deep and the residual on top
    d = {k: v.dequantize(torch.float64) if isinstance(v, pkg.FP8BlockWeight) else v.double() for k, v in p.items()}

    def norm(t, gamma):
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gamma

    for i, n in enumerate(lens):
        a = int(offsets[i])
        t = x[a : a + n].double()
        q, k, v = (norm(t, d["g1"]) @ d["qkv"].t()).view(n, 3, HEADS, -1).permute(1, 2, 0, 3)
        s = torch.softmax(q @ k.transpose(1, 2) + ref.bias_matrix(p["table"], n, 128, True).to(dev), -1) @ v
        t = t + s.transpose(0, 1).reshape(n, DIM) @ d["o"].t()
        b = norm(t, d["g2"])
        t = t + (torch.nn.functional.gelu(b @ d["gate"].t(), approximate="tanh") * (b @ d["up"].t())) @ d["down"].t()
        err = float((out[a : a + n].double() - t).norm() / t.norm())
        assert err <= 4.8e-2, (i, err)

    fp8, _ = _block_weights(pkg, dev)
    _, packed, pos, h, temb, _ = _setup(pkg, dev, blocks=1)
    text_offsets = ref.offsets([100, 0, 60, 90], dev)

    def call():
        states = _encoder(pkg, x, text_offsets, p)
        text = pkg.PackedRequests((100, 0, 60, 90), rows, torch.empty(0), text_offsets)
        return pkg.packed_block_forward(fp8, h, temb, packed, pos, pkg.project_packed_cross_kv(fp8, states, text))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed, texts in enumerate(([100, 0, 60, 90], [1, 200, 0, 99], [75, 75, 75, 75])):
        x.copy_(torch.randn(rows, DIM, generator=torch.Generator().manual_seed(seed)))
        text_offsets.copy_(ref.offsets(texts))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(got, want), texts
