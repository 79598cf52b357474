"""What the operators on the text side refuse, on the CPU: shapes, types, layouts and sizes are said to be wrong before anything
is launched, and host tensors are never computed. Also the choice of tiles (csrc/fp8_plan.h) and the buckets, over their range."""

import ctypes
import pathlib
import subprocess

import pytest
import torch

import text_ref as ref

BF, F32, I32, E4 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn
T, TK, H, D = 6, 9, 4, 64


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def codes(*shape):
    return z(*shape, dtype=torch.uint8).view(E4)


def off(n=3):
    return torch.zeros(n, dtype=I32)


def _cross(pkg, q=None, k=None, v=None, q_offsets=None, k_offsets=None, **kw):
    one = lambda t, *shape: z(*shape) if t is None else t  # noqa: E731
    return pkg.packed_cross_attention(one(q, T, H, D), one(k, TK, H, D), one(v, TK, H, D), off() if q_offsets is None else q_offsets,
                                      off() if k_offsets is None else k_offsets, **kw)


def _bias(pkg, q=None, k=None, v=None, table=None, offsets=None, **kw):
    one = lambda t: z(T, H, D) if t is None else t  # noqa: E731
    return pkg.relative_bias_attention(one(q), one(k), one(v), z(32, H, dtype=F32) if table is None else table, off() if offsets is None else offsets, **kw)


CROSS = [
    (dict(q=z(T, H, D, dtype=F32)), "bfloat16"), (dict(k=z(TK, H, D, dtype=torch.float16)), "bfloat16"), (dict(q=z(T, H * D)), "shape"), (dict(q=1), "Tensor"),
    (dict(k=z(TK, H, 128)), "shape"), (dict(v=z(TK, H, 128)), "shape"), (dict(v=z(TK, 2, D)), "shape"), (dict(v=z(TK - 1, H, D)), "rows"),
    (dict(k=z(TK, 3, D), v=z(TK, 3, D)), "heads"), (dict(k=z(TK, 0, D), v=z(TK, 0, D)), "heads"), (dict(q=z(T, 0, D)), "heads"),
    (dict(q=z(T, H, 2 * D)[..., ::2]), "unit stride"), (dict(q=z(T, H, D + 4)[..., :D]), "aligned"), (dict(q=z(T * H * D + 4)[4:].view(T, H, D)), "aligned"),
    (dict(k=z(1, H, D).expand(TK, H, D)), "overlap"), (dict(q=z(T, 1, D).expand(T, H, D)), "overlap"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=2.0**-70), "scale"),
    (dict(quant="row"), "quant"), (dict(q_offsets=off().long()), "int32"), (dict(q_offsets=off(4)), "shape"), (dict(k_offsets=off(2)), "shape"),
    (dict(q_offsets=off(0), k_offsets=off(0)), "entry"), (dict(q_offsets=off(6)[::2]), "contiguous"), (dict(q_offsets=None, k_offsets=off(3).view(3, 1)), "shape"),
    (dict(out=z(T, H, D), quant="mx"), "quant"), (dict(out=z(T, H, D, dtype=F32)), "bfloat16"), (dict(out=z(T, H * D)), "shape"),
    (dict(out=z(T, 2 * H, D)[:, ::2]), "side by side"), (dict(out=z(T, H * D + 8)[:, : H * D].view(T, H, D)), "side by side"),
    (dict(out=z(T * H * D + 8)[4 : 4 + T * H * D].view(T, H, D)), "aligned"),
]


@pytest.mark.parametrize("case", range(len(CROSS)))
def test_cross_attention_refuses(pkg, case):
    kw, match = CROSS[case]
    with pytest.raises(ValueError, match=match):
        _cross(pkg, **kw)


def test_other_head_widths_are_not_there(pkg):
    for d in (32, 80, 256):
        with pytest.raises(NotImplementedError):
            _cross(pkg, q=z(T, H, d), k=z(TK, H, d), v=z(TK, H, d))


def _over(t, dtype, *shape):
    raw = t.view(-1).view(torch.uint8)
    n = torch.empty((), dtype=dtype).element_size() * torch.Size(shape).numel()
    return raw[:n].view(dtype).view(shape)


def test_attention_outputs_over_the_inputs(pkg):
    """The rows of q are read before they are written, element for element; everything else is read by other workgroups as well."""
    big = z(4 * T, H, D)
    for name, shape, dtype in (("k", (TK, H, D), BF), ("v", (TK, H, D), BF), ("q_offsets", (3,), I32), ("k_offsets", (3,), I32)):
        with pytest.raises(ValueError, match="overlaps|may not be"):
            _cross(pkg, **{name: _over(big, dtype, *shape)}, out=_over(big, BF, T, H, D))
    for name, shape, dtype in (("k", (T, H, D), BF), ("v", (T, H, D), BF), ("table", (32, H), F32), ("offsets", (3,), I32)):
        with pytest.raises(ValueError, match="overlaps|may not be"):
            _bias(pkg, **{name: _over(big, dtype, *shape)}, out=_over(big, BF, T, H, D))
    with pytest.raises(ValueError, match="overlaps"):
        _cross(pkg, q=big[1 : T + 1], out=big[:T])
    slab = z(T, 3 * H, D)
    for q, out in ((big[:T], big[:T]), (slab[:, :H], slab[:, :H]), (slab[:, :H], slab[:, H : 2 * H])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            _cross(pkg, q=q, out=out)


BIAS = [
    (dict(k=z(T - 1, H, D), v=z(T - 1, H, D)), "rows and heads"), (dict(k=z(T, 2, D), v=z(T, 2, D)), "rows and heads"),
    (dict(table=z(32, H, dtype=torch.float16)), "table"), (dict(table=None, offsets=off().long()), "int32"), (dict(table=z(32, H + 1, dtype=F32)), "table"),
    (dict(table=z(H, 32, dtype=F32).t()), "contiguous"), (dict(table=z(32, dtype=F32)), "table"), (dict(table=z(31, H, dtype=F32)), "buckets"),
    (dict(table=z(2, H, dtype=F32)), "buckets"), (dict(table=z(258, H, dtype=F32), max_distance=1000), "at most 128"), (dict(max_distance=8), "exceed"),
    (dict(max_distance=0), "exceed"), (dict(max_distance=4000), "at most 1024"), (dict(max_distance=10**15), "at most 1024"), (dict(table=z(1, H, dtype=F32), bidirectional=False), "buckets"), (dict(scale=0.0), "scale"),
    (dict(scale=2.0**25), "scale"), (dict(offsets=off(0)), "entry"),
]


@pytest.mark.parametrize("case", range(len(BIAS)))
def test_relative_bias_refuses(pkg, case):
    kw, match = BIAS[case]
    with pytest.raises(ValueError, match=match):
        _bias(pkg, **kw)


def test_buckets(pkg):
    """The first distance of each bucket against the definition at every distance, borders on whole numbers among them."""
    for buckets, far, both in ((32, 128, True), (32, 128, False), (20, 250, True), (64, 64, True), (8, 512, True), (4, 3, True), (256, 1024, True), (2, 5, False), (128, 1024, False)):
        starts = list(pkg.packed_attention._bucket_starts(buckets, far, both))
        for n in range(0, 1500, 1 if far < 300 else 3):
            want = ref.bucket(-n, buckets, far, both)
            assert sum(n >= s for s in starts) - 1 == want, (buckets, far, both, n)
    assert list(pkg.packed_attention._bucket_starts(32, 128, True)) == [0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91]


def _weight(pkg, N=64, K=144, **kw):
    w = dict(codes=codes(N, K), scales=z(-(-N // 128), -(-K // 128), dtype=F32), bias=z(N, dtype=F32))
    return pkg.FP8BlockWeight(**{**w, **kw})


def test_linear_refuses(pkg):
    x, s = z(T, 144), z(T, 2, dtype=F32)
    t = pkg.FP8BlockTensor(codes(T, 144), s)
    for arg, w, kw, match in (
        (x, "w", {}, "FP8BlockWeight"), (x, pkg.MXWeight(codes(64, 144), s), {}, "FP8BlockWeight"), (x, _weight(pkg, codes=z(64, 144)), {}, "float8"),
        (x, _weight(pkg, codes=codes(64, 288)[:, :144]), {}, "contiguous"), (x, _weight(pkg, scales=z(1, 1, dtype=F32)), {}, "shape"),
        (x, _weight(pkg, scales=z(1, 2)), {}, "float32"), (x, _weight(pkg, bias=z(32, dtype=F32)), {}, "shape"), (x, _weight(pkg, bias=z(64)), {}, "float32"),
        (x, _weight(pkg, N=68), {}, "multiple of 8"), (x, _weight(pkg, N=0), {}, "multiple of 8"), (x, _weight(pkg, bias=z(65, dtype=F32)[1:]), {}, "aligned"),
        (z(T, 128), _weight(pkg), {}, "K=144"), (z(T, 136), _weight(pkg, K=136), {}, "multiple of 16"), (z(T, 144, dtype=F32), _weight(pkg), {}, "bf16"), (5, _weight(pkg), {}, "bf16"),
        (z(T, 288)[:, ::2], _weight(pkg), {}, "contiguous"), (z(T, 148)[:, :144], _weight(pkg), {}, "aligned"), (z(1, 144).expand(T, 144), _weight(pkg), {}, "contiguous"),
        (pkg.FP8BlockTensor(z(T, 144), s), _weight(pkg), {}, "float8"), (pkg.FP8BlockTensor(codes(T, 144), z(T, 1, dtype=F32)), _weight(pkg), {}, "shape"),
        (pkg.FP8BlockTensor(codes(T, 144), z(T, 2)), _weight(pkg), {}, "float32"), (pkg.FP8BlockTensor(codes(T, 152)[:, :144], s), _weight(pkg), {}, "aligned"),
        (x, _weight(pkg), dict(activation="silu"), "activation"), (x, _weight(pkg), dict(out=z(T, 32)), "shape"), (x, _weight(pkg), dict(out=z(T, 64, dtype=F32)), "bfloat16"),
        (x, _weight(pkg), dict(out=z(T, 68)[:, :64]), "aligned"), (x, _weight(pkg), dict(out=_over(x, BF, T, 64)), "overlaps|may not be"),
    ):
        with pytest.raises(ValueError, match=match):
            pkg.fp8_block_linear(arg, w, **kw)
    out = z(T, 64)
    for name, shape, dtype in (("codes", (64, 144), E4), ("scales", (1, 2), F32), ("bias", (64,), F32)):
        big = z(64, 144)
        with pytest.raises(ValueError, match="overlaps|may not be"):
            pkg.fp8_block_linear(x, _weight(pkg, **{name: _over(big, dtype, *shape)}), out=_over(big, BF, T, 64))
    for arg in (x, t, x.view(2, 3, 144), pkg.FP8BlockTensor(codes(2, 3, 144), s.view(2, 3, 2)), x[0]):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            pkg.fp8_block_linear(arg, _weight(pkg))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.fp8_block_linear(x, _weight(pkg), out=out)


def test_quantizers_refuse(pkg):
    for x in (z(T, 144, dtype=F32), z(T, 140), z(T, 0), z(()), 3, z(T, 288)[:, ::2], z(T, 148)[:, :144]):
        with pytest.raises(ValueError):
            pkg.quantize_fp8_blocks(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.quantize_fp8_blocks(z(T, 144))
    with pytest.raises(ValueError):
        pkg.quantize_weight_fp8_blocks(z(3, 4, 5))


def test_weights_by_blocks(pkg):
    """Codes and scales of every block, the partial ones at both ends too, and what they stand for."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(300, 200, generator=g) * torch.exp2(torch.randint(-20, 20, (300, 1), generator=g).float())
    w[:128, 128:] = 0
    q = pkg.quantize_weight_fp8_blocks(w, torch.arange(200.0))
    assert q.codes.shape == (200, 300) and q.scales.shape == (2, 3) and torch.equal(q.bias, torch.arange(200.0))
    for i in range(2):
        for j in range(3):
            block = w[128 * j : 128 * j + 128, 128 * i : 128 * i + 128].t()
            scale = block.abs().max().clamp_min(2.0**-100) * (1.0 / 448.0)
            assert q.scales[i, j] == scale
            assert torch.equal(q.codes[128 * i : 128 * i + 128, 128 * j : 128 * j + 128].float(), (block / scale).to(E4).float())
    off_by = (q.dequantize() - w.t()).abs()
    step = q.scales.repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :300]
    # half a step: 2^-4 of the value, or of the smallest normal 2^-6 below it; the scale's own rounding moves a code by 2^-23 of it
    assert bool((off_by <= (2.0**-4 + 2.0**-22) * torch.maximum(w.t().abs(), step * 2.0**-6)).all())


def test_packed_texts_that_do_not_fit(pkg):
    packed = pkg.PackedRequests.from_lengths([2, 3], 6, "cpu")
    assert packed.offsets.tolist() == [0, 2, 5] and packed.offsets.dtype == I32
    kv = lambda n: pkg.PackedCrossKV(z(9, 1, 128), z(9, 1, 128), off(n))  # noqa: E731
    args = dict(h=z(6, 128), temb=z(2, 6, 128, dtype=F32), packed=packed, positions=torch.zeros(6, 3, dtype=I32), tables=z(1, 6, 128, dtype=F32))
    for crosses in ([kv(4)], [kv(2)], [kv(3), kv(3)], [kv(0)]):
        with pytest.raises(ValueError, match="crosses"):
            pkg.packed_dit_forward([None], crosses=crosses, **args)
    with pytest.raises(ValueError, match="offsets"):
        pkg.packed_dit_forward([None], crosses=[kv(3)], **{**args, "packed": packed._replace(offsets=None)})
    w = pkg.block.BlockWeights(*[None] * 15)
    for context, text in ((z(5, 128), packed), (z(6), packed), (z(6, 128), packed._replace(offsets=None))):
        with pytest.raises(ValueError, match="context"):
            pkg.project_packed_cross_kv(w, context, text)


def test_c_entry_points_refuse_before_any_launch(pkg):
    """Sizes, options and null pointers: an argument error, no GPU call (there is none here)."""
    lib = pkg._lib.load()
    arg, unsupported = pkg._lib.WANMI_ERR_ARG, pkg._lib.WANMI_ERR_UNSUPPORTED

    def cross(q=16, k=16, ss=256, hs=64, qo=16, ko=16, R=2, T=4, Tk=4, heads=4, kh=2, D=64, scale=0.5, out=16, o_ss=256):
        return lib.wanmi_packed_cross_attention(q, ss, hs, k, ss, hs, k, ss, hs, qo, ko, R, T, Tk, heads, kh, D, scale, out, o_ss, None, 1, None)

    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(out=None), dict(q=8), dict(k=24), dict(out=8), dict(ss=12), dict(hs=4), dict(ss=-256), dict(ss=1 << 22),
               dict(ss=32), dict(R=-1), dict(R=1 << 20), dict(T=-1), dict(T=1 << 28), dict(Tk=-1), dict(Tk=1 << 28), dict(heads=0), dict(kh=0), dict(kh=3), dict(heads=2048, o_ss=1 << 20),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-30), dict(o_ss=128), dict(o_ss=264),
               dict(T=(1 << 28) - 1, heads=64, o_ss=4096, kh=64)):
        assert cross(**kw) == arg, kw
    assert cross(D=96) == unsupported and cross(T=0, q=None, out=None) == 0

    starts = (ctypes.c_int * 4)(0, 1, 2, 5)

    def bias(q=16, T=4, table=16, starts=starts, side=4, D=64, offsets=16, o_ss=256, scale=1.0):
        return lib.wanmi_relative_bias_attention(q, 256, 64, q, 256, 64, q, 256, 64, offsets, 2, T, 4, D, scale, table, 0, starts, side, 1, 16, o_ss, 1, None)

    for kw in (dict(q=None), dict(table=None), dict(starts=None), dict(side=0), dict(side=129), dict(starts=(ctypes.c_int * 4)(0, 2, 1, 5)), dict(starts=(ctypes.c_int * 4)(-1, 2, 3, 5)),
               dict(starts=(ctypes.c_int * 4)(0, 1, 2, 1025)), dict(offsets=None), dict(o_ss=64), dict(scale=0.0)):
        assert bias(**kw) == arg, kw
    assert bias(D=128 + 64) == unsupported and bias(T=0, q=None, table=None) == 0

    def quantize(x=16, ldx=144, M=4, K=144, codes=16, scales=16):
        return lib.wanmi_fp8_block_quantize(x, ldx, M, K, codes, scales, 1, M, None)

    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(x=8), dict(codes=8), dict(ldx=128), dict(ldx=148), dict(M=-1), dict(M=1 << 27), dict(K=0), dict(K=136),
               dict(K=1 << 22, ldx=1 << 22), dict(M=(1 << 26) - 4)):
        assert quantize(**kw) == arg, kw
    assert quantize(M=0, x=None) == 0

    def linear(x=16, xs=16, ldx=144, xs_row=1, w=16, ws=16, b=16, M=4, N=64, K=144, out=16, ldo=64, work=16, size=1 << 40):
        return lib.wanmi_fp8_block_linear(x, xs, ldx, xs_row, M, w, ws, b, M, N, K, 0, out, ldo, work, size, None)

    for kw in (dict(x=None), dict(w=None), dict(ws=None), dict(out=None), dict(x=8), dict(w=8), dict(b=8), dict(out=8), dict(ldx=128), dict(ldx=152), dict(ldx=1 << 23), dict(ldo=56), dict(ldo=68),
               dict(ldo=1 << 24), dict(M=-1), dict(M=1 << 27), dict(N=0), dict(N=68), dict(N=1 << 24), dict(K=0), dict(K=152), dict(xs=None, M=100, size=0), dict(xs=None, M=100, work=None),
               dict(M=100, xs_row=2, size=16), dict(xs=None, M=100, work=8), dict(M=(1 << 27) - 1, N=1 << 20, ldo=1 << 20), dict(M=(1 << 27) - 1, K=4096, ldx=4096)):
        assert linear(**kw) == arg, kw
    assert linear(M=0, x=None) == 0
    size = lib.wanmi_fp8_block_workspace
    assert size(0, 64, 144, 1, 0) == 0 and size(4, 64, 144, 1, 0) == 0 and size(16, 64, 144, 0, 2) == 0 and size(5, 64, 144, 1, 0) >= 5 * (144 + 8)
    assert size(4096, 8192, 256, 0, 1) == 0 and size(4096, 8192, 256, 0, 2) >= 4096 * 8


def test_the_choice_of_tiles(tmp_path):
    """Over the range of sizes: the parts of a sum are never empty and at most eight, their workspace stays below the product's operands and
    output several times over, and a product of more rows is never estimated cheaper by more than its parts' launch."""
    root = pathlib.Path(__file__).resolve().parents[1]
    (tmp_path / "main.cc").write_text(r"""
#include "fp8_plan.h"
#include <cstdio>
using namespace wanmi;
int main() {
  long checked = 0, bad = 0;
  for (int64_t N : {8, 64, 640, 2568, 5120, 13824, 15360, 1 << 20})
    for (int64_t KB : {1, 2, 3, 5, 33, 40, 108, 864}) {
      int64_t before = 0;
      for (int64_t M = 17; M <= 33000; M += M < 600 ? 1 : 61) {
        const Fp8Plan p = fp8_plan(M, N, KB);
        ++checked;
        const bool deep = p.tiles == kFp8Tiles64 || p.tiles == kFp8Tiles128Deep;
        if (p.splits < 1 || p.splits > 8 || p.splits > KB || (p.splits > 1 && !deep) || p.cost + 3800 + 8 * M * N / 6000 < before || p.splits * M * N * 4 > (1LL << 40)) {
          if (bad++ < 5) printf("M=%ld N=%ld KB=%ld: tiles %d, %d parts, %ld after %ld\n", (long)M, (long)N, (long)KB, p.tiles, p.splits, (long)p.cost, (long)before);
        }
        before = p.cost;
      }
    }
  printf("%ld checked, %ld bad\n", checked, bad);
}
""")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{root / 'vllm-omni-neuron_amd' / 'csrc'}", str(tmp_path / "main.cc"), "-o",
                    str(tmp_path / "main")], check=True)
    out = subprocess.run([str(tmp_path / "main")], check=True, capture_output=True, text=True, timeout=120).stdout
    assert out.endswith(" 0 bad\n"), out
