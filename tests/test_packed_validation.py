"""Refusals of the operators for packed batches (CPU only): a wrong type, shape, layout or option raises before anything is
launched, and well-formed host tensors are refused as such. The C entry points refuse bad sizes without touching the GPU."""

import ctypes

import pytest
import torch

BF = torch.bfloat16
T, H = 6, 64


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def ids(n=T):
    return torch.zeros(n, dtype=torch.int32)


def f(*shape):
    return torch.zeros(*shape)


@pytest.mark.parametrize("kw,match", [
    (dict(hidden=f(T, H)), "hidden"), (dict(hidden=z(T, H, 1)), "hidden"), (dict(hidden=z(T, 40)), "multiple of 32"),
    (dict(hidden=z(T, 32 * 513)), "16384"), (dict(hidden=z(T, 2 * H)[:, ::2]), "unit stride"), (dict(hidden=z(T, H + 4)[:, :H]), "16-byte"),
    (dict(residual=z(T + 1, H)), "residual"), (dict(residual=f(T, H)), "residual"), (dict(residual=z(1, H).expand(T, H)), "overlap"),
    (dict(mul=z(2, H)), "mul"), (dict(mul=f(2, H + 4)), "mul"), (dict(mul=f(3, H), add=f(2, H)), "add has 2 rows"), (dict(gate=f(2, 2, H)), "gate"),
    (dict(gate=f(H + 1)[1:]), "aligned"), (dict(gate=f(2, H), request_ids=None), "need request_ids"),
    (dict(post_weight=f(H + 1)), "post_weight"), (dict(post_norm="group"), "post_norm"), (dict(norm_type="group"), "norm_type"),
    (dict(quant="fp4"), "quant"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(request_ids=torch.zeros(T, dtype=torch.int64)), "request_ids"), (dict(request_ids=ids(T + 1)), "request_ids"),
    (dict(out=f(T, H)), "out"), (dict(quant="mx", out=z(T, H)), "MXTensor"), (dict(residual_out=z(T, H + 1)), "residual_out"),
    (dict(norm_type=None, quant="mx"), "no second output"), (dict(norm_type=None, mul=f(H)), "no second output"),
])
def test_sandwich(pkg, kw, match):
    args = dict(hidden=z(T, H), residual=z(T, H), mul=None, add=None, eps=1e-6, request_ids=ids())
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        pkg.adaln_sandwich(args.pop("hidden"), args.pop("residual"), args.pop("mul"), args.pop("add"), **args)


def test_sandwich_outputs_that_overlap(pkg):
    buf = z(T + 1, H)
    with pytest.raises(ValueError, match="overlaps"):
        pkg.adaln_sandwich(buf[:T], z(T, H), eps=1e-6, out=buf[1:])
    with pytest.raises(ValueError, match="share memory"):
        pkg.adaln_sandwich(z(T, H), z(T, H), eps=1e-6, out=buf[:T], residual_out=buf[:T])


def _qk(pkg, **kw):
    args = dict(q=z(T, 4, 64), k=z(T, 2, 64), positions=torch.zeros(T, 2, dtype=torch.int32), axes=(16, 16))
    args.update(kw)
    return pkg.qk_norm_rope_axes(args.pop("q"), args.pop("k"), args.pop("positions"), **args)


@pytest.mark.parametrize("kw,match", [
    (dict(q=z(T, 256)), "q must be"), (dict(q=f(T, 4, 64)), "q must be"), (dict(k=z(T + 1, 2, 64)), "k must have"), (dict(k=z(T, 2, 32)), "k must have"),
    (dict(q=z(T, 4, 128)[:, :, ::2]), "unit stride"), (dict(q=z(T, 4, 68)[:, :, :64]), "16-byte"),
    (dict(axes=(16, 15)), "axes"), (dict(axes=(64, 16)), "axes"), (dict(axes=(2,) * 9), "axes"), (dict(axes=(-16, 32)), "axes"),
    (dict(theta=0.0), "theta"), (dict(theta=(1.0,)), "theta"), (dict(theta=float("inf")), "theta"), (dict(rope_pairs="thirds"), "rope_pairs"),
    (dict(norm="layer_norm"), "norm"), (dict(eps=-1.0), "eps"), (dict(q_gamma=f(64)), "without a norm"),
    (dict(norm="rms_norm", q_gamma=f(256)), "q_gamma"), (dict(norm="rms_norm_across_heads", q_gamma=f(64)), "q_gamma"),
    (dict(norm="rms_norm", q_gamma=z(64)), "q_gamma"), (dict(k=None, norm="rms_norm", k_gamma=f(64)), "need k"), (dict(k=None, k_out=z(T, 2, 64)), "need k"),
    (dict(positions=torch.zeros(T, 2, dtype=torch.int64)), "positions"), (dict(positions=torch.zeros(T, 3, dtype=torch.int32)), "positions"),
    (dict(positions=torch.zeros(2, T, dtype=torch.int32).t()), "contiguous"), (dict(positions=None), "positions"),
    (dict(request_ids=ids(3)), "request_ids"), (dict(k=None, want_max=True), "want_max"), (dict(want_max=True, request_ids=ids()), "want_max"),
    (dict(requests=-1, request_ids=ids()), "requests"), (dict(requests=2), "need request_ids"),
    (dict(q_out=z(T, 4, 32)), "q_out"), (dict(q_out=z(1, 4, 64).expand(T, 4, 64)), "share memory"),
])
def test_qk_axes(pkg, kw, match):
    with pytest.raises(ValueError, match=match):
        _qk(pkg, **kw)


def test_qk_axes_unsupported_and_overlapping(pkg):
    for kw in (dict(q=z(T, 4, 80), k=None), dict(axes=(10, 10)), dict(q=z(T, 257, 64))):
        with pytest.raises(NotImplementedError):
            _qk(pkg, **kw)
    slab = z(T, 8 * 64)
    q, k = slab[:, :256].view(T, 4, 64), slab[:, 256:384].view(T, 2, 64)
    with pytest.raises(ValueError, match="overlaps"):
        _qk(pkg, q=q, k=k, q_out=slab[:, 128:384].view(T, 4, 64))
    with pytest.raises(ValueError, match="may not be"):
        _qk(pkg, q=z(T, 2, 64), k=(k2 := z(T, 2, 64)), q_out=k2)
    with pytest.raises(ValueError, match="share memory"):
        _qk(pkg, q=z(T, 2, 64), q_out=(o := z(T, 2, 64)), k_out=o)
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # in place on views of one slab: accepted, but for the device
        _qk(pkg, q=q, k=k, q_out=q, k_out=k)


def _lora(pkg, **kw):
    args = dict(base=z(T, 128), x=z(T, 96), a=z(2, 32, 96), b=z(2, 128, 32), adapter_ids=ids())
    args.update(kw)
    return pkg.lora_add(args.pop("base"), args.pop("x"), args.pop("a"), args.pop("b"), args.pop("adapter_ids"), **args)


@pytest.mark.parametrize("kw,match", [
    (dict(base=f(T, 128)), "base"), (dict(base=z(T, 132)[:, :128]), "16-byte"), (dict(x=z(T + 1, 96)), "x must"), (dict(x=f(T, 96)), "activation"),
    (dict(x=z(T, 100)[:, :96]), "16-byte"), (dict(a=z(2, 32, 64)), "do not fit"), (dict(a=z(3, 32, 96)), "do not fit"), (dict(a=f(2, 32, 96)), "a must"),
    (dict(a=z(2, 96, 32).transpose(1, 2)), "contiguous"), (dict(b=z(2, 120, 32)), "do not fit"), (dict(a=z(2, 24, 96), b=z(2, 128, 24)), "rank"),
    (dict(a=z(2, 1040, 96), b=z(2, 128, 1040)), "rank"), (dict(x=z(T, 80), a=z(2, 32, 80)), "multiple of 32"),
    (dict(base=z(T, 120), b=z(2, 120, 32), slices=(60, 60)), "multiples of 64"), (dict(slices=(64, 32)), "slices"), (dict(slices=(64, 64)), "do not fit"),
    (dict(slices=()), "slices"), (dict(slices=(128, 0)), "slices"), (dict(scales=f(3)), "scales"), (dict(scales=z(2)), "scales"),
    (dict(adapter_ids=ids(5)), "adapter_ids"), (dict(adapter_ids=torch.zeros(T, dtype=torch.int64)), "adapter_ids"), (dict(request_ids=ids(5)), "request_ids"),
    (dict(out=z(T, 120)), "out"), (dict(out=f(T, 128)), "out"), (dict(a=z(0, 32, 96), b=z(0, 128, 32)), "do not fit"),
])
def test_lora(pkg, kw, match):
    with pytest.raises(ValueError, match=match):
        _lora(pkg, **kw)


def test_lora_outputs_that_overlap_and_host_tensors(pkg):
    x = z(T, 128)
    with pytest.raises(ValueError, match="may not be"):
        _lora(pkg, x=x, a=z(2, 32, 128), out=x)
    buf = z(T + 1, 128)
    with pytest.raises(ValueError, match="overlaps"):
        _lora(pkg, base=buf[:T], out=buf[1:])
    base = z(T, 128)
    for kw in (dict(), dict(base=base, out=base)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            _lora(pkg, **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.adaln_sandwich(z(T, H), z(T, H), eps=1e-6)


def test_stacks_and_packings(pkg):
    with pytest.raises(ValueError, match="no adapters"):
        pkg.stack_adapters([], 32, (64,), device="cpu")
    with pytest.raises(ValueError, match="parts"):
        pkg.stack_adapters([[None]], 32, (64, 64), device="cpu")
    with pytest.raises(ValueError, match="for 32 -> 64"):
        pkg.stack_adapters([[(z(4, 32), z(64, 5))]], 32, (64,), device="cpu")
    a, b = pkg.stack_adapters([[(torch.ones(3, 32), torch.ones(64, 3))], [None]], 32, (64,), device="cpu")
    assert a.shape == (2, 16, 32) and b.shape == (2, 64, 16) and float(a.sum()) == 96 and float(b.sum()) == 192
    p = pkg.PackedRequests.from_lengths([2, 0, 3], 7, "cpu")
    assert p.request_ids.tolist() == [0, 0, 2, 2, 2, -1, -1] and list(p.spans()) == [(0, 2), (2, 2), (2, 5)]
    assert p.grid_positions([(1, 1, 2), (0, 4, 4), (3, 1, 1)]).tolist() == [[0, 0, 0], [0, 0, 1], [0, 0, 0], [1, 0, 0], [2, 0, 0], [0, 0, 0], [0, 0, 0]]
    for bad in ([], [-1]):
        with pytest.raises(ValueError):
            pkg.PackedRequests.from_lengths(bad, device="cpu")
    with pytest.raises(ValueError, match="do not fit"):
        pkg.PackedRequests.from_lengths([4, 4], 7, "cpu")
    with pytest.raises(ValueError, match="do not hold"):
        p.grid_positions([(1, 1, 2), (0, 4, 4), (3, 1, 2)])


def test_c_entry_points_refuse_before_any_launch(pkg):
    """Sizes, options and null pointers: an argument error, no GPU call (there is none here)."""
    lib = pkg._lib.load()
    arg, unsupported = pkg._lib.WANMI_ERR_ARG, pkg._lib.WANMI_ERR_UNSUPPORTED

    def sandwich(T=4, H=64, ld=64, lg=0, requests=1, eps=1e-6, post=2, norm=1, quant=0, p=16, ids=None):
        return lib.wanmi_adaln_sandwich(p, ld, p, ld, None, p, lg, None, 0, None, 0, ids, requests, 1.0, T, H, eps, post, norm, quant, 1, p, p, None, None)

    for kw in (dict(T=-1), dict(T=1 << 32), dict(H=48), dict(H=0), dict(ld=32), dict(ld=68), dict(lg=32), dict(lg=66), dict(requests=-1), dict(requests=0),
               dict(eps=-1.0), dict(post=3), dict(norm=-1), dict(quant=3), dict(quant=1), dict(p=None), dict(p=8)):
        assert sandwich(**kw) == arg, kw
    assert sandwich(H=16416) == unsupported
    assert sandwich(T=0, p=None) == 0

    dims, freqs = (ctypes.c_int * 2)(16, 16), (ctypes.c_double * 16)()

    def qk(T=4, D=64, qh=2, kh=2, ts=128, axes=2, dims=dims, pairs=0, norm=0, eps=1e-6, requests=1, p=16, kmax=None):
        return lib.wanmi_qk_norm_rope_axes(p, ts, D, qh, None, p, ts, D, p, ts, D, kh, None, p, ts, D, T, D, p, 0, axes, dims, freqs, pairs, norm, eps, None,
                                           requests, 1, kmax, None)

    odd = (ctypes.c_int * 2)(16, 15)
    wide = (ctypes.c_int * 2)(64, 16)
    for kw in (dict(T=-1), dict(qh=0), dict(kh=-1), dict(ts=4), dict(axes=9), dict(axes=-1), dict(dims=odd), dict(dims=wide), dict(dims=None), dict(pairs=2), dict(norm=3),
               dict(eps=-1.0), dict(requests=0), dict(p=None), dict(p=8), dict(kh=0, kmax=16)):
        assert qk(**kw) == arg, kw
    assert qk(D=48) == unsupported and qk(qh=300) == unsupported and qk(dims=(ctypes.c_int * 2)(16, 8)) == unsupported
    assert qk(T=0, p=None) == 0

    widths = (ctypes.c_int64 * 2)(64, 64)

    def lora(T=4, K=96, N=128, r=32, parts=2, widths=widths, n=2, requests=2, ldx=96, ldb=128, p=16, size=1 << 20):
        return lib.wanmi_lora_add(p, None, None, ldx, p, p, None, p, None, requests, n, T, K, N, r, parts, widths, p, ldb, p, ldb, 1, p, size, None)

    for kw in (dict(T=-1), dict(K=80), dict(K=0), dict(N=124), dict(r=24), dict(r=0), dict(r=2048), dict(parts=0), dict(parts=9), dict(widths=None), dict(N=192),
               dict(widths=(ctypes.c_int64 * 2)(96, 32)), dict(widths=(ctypes.c_int64 * 2)(128, 64)), dict(n=0), dict(requests=-1), dict(ldx=64), dict(ldx=100), dict(ldb=64),
               dict(ldb=132), dict(p=None), dict(p=8), dict(size=16)):
        assert lora(**kw) == arg, kw
    assert lora(T=0, p=None) == 0
    assert lib.wanmi_lora_workspace(0, 96, 1, 16) == 0 and lib.wanmi_lora_workspace(4, 96, 2, 32) >= 4 * 4 * 64


def test_more_rows_than_a_launch_holds(pkg):
    """A launch has fewer than 2^32 lanes: more rows are an argument error, not a failed launch."""
    lib = pkg._lib.load()
    arg = pkg._lib.WANMI_ERR_ARG
    dims, freqs, widths = (ctypes.c_int * 1)(16), (ctypes.c_double * 8)(), (ctypes.c_int64 * 1)(64)
    for T in (1 << 26, (1 << 26) - 7):
        assert lib.wanmi_adaln_sandwich(16, 64, 16, 64, None, None, 0, None, 0, None, 0, None, 1, 1.0, T, 64, 1e-6, 2, 1, 0, 1, 16, 16, None, None) == arg
        assert lib.wanmi_qk_norm_rope_axes(16, 64, 64, 1, None, 16, 64, 64, None, 0, 0, 0, None, None, 0, 0, T, 64, 16, 0, 1, dims, freqs, 0, 0, 1e-6,
                                           None, 1, 1, None, None) == arg
    assert lib.wanmi_lora_add(16, None, None, 96, 16, 16, None, 16, None, 1 << 28, 1, 1 << 28, 96, 64, 16, 1, widths, 16, 64, 16, 64, 1, 16, 1 << 62, None) == arg
    assert lib.wanmi_qk_norm_rope_axes(16, 64, 64, 1, None, 16, 64, 64, 16, 64, 64, 2, None, 16, 64, 64, 0, 64, 16, 0, 1, dims, freqs, 0, 0, 1e-6,
                                       16, 1 << 30, 1, 16, None) == arg


def _over(t, dtype, *shape):
    """A tensor of this type and shape over the first bytes of ``t``."""
    raw = t.view(-1).view(torch.uint8)
    n = torch.empty((), dtype=dtype).element_size()
    for s in shape:
        n *= s
    return raw[:n].view(dtype).view(shape)


def test_sandwich_outputs_over_the_other_inputs(pkg):
    """What every row still reads: the vectors and the ids; and the scales of the codes, over anything."""
    big = {name: f(2 * T, H) for name in ("mul", "add", "gate", "post_weight", "request_ids")}
    arg = dict(mul=big["mul"][:2], add=big["add"][:2], gate=big["gate"][:2], post_weight=big["post_weight"][0], request_ids=_over(big["request_ids"], torch.int32, T))
    for name in big:
        over = _over(big[name], BF, T, H)
        for kw in (dict(out=over), dict(residual_out=over)):
            args = dict(arg)
            with pytest.raises(ValueError, match="overlaps|may not be"):
                pkg.adaln_sandwich(z(T, H), z(T, H), args.pop("mul"), args.pop("add"), eps=1e-6, **args, **kw)
    codes = z(T, H, dtype=torch.uint8).view(torch.float8_e4m3fn)
    kw = dict(eps=1e-6, quant="mx", request_ids=arg["request_ids"], gate=arg["gate"])
    hidden, residual, ro = z(T, H), z(T, H), z(T, H)
    for t in (big["gate"], big["request_ids"], hidden, residual, ro, codes):
        scales = _over(t, torch.uint8, T, H // 32)
        with pytest.raises(ValueError, match="overlaps|may not be|share memory"):
            pkg.adaln_sandwich(hidden, residual, residual_out=ro, out=pkg.MXTensor(codes, scales), **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # apart from each other: accepted, but for the device
        pkg.adaln_sandwich(hidden, residual, residual_out=residual, out=pkg.MXTensor(codes, z(T, H // 32, dtype=torch.uint8)), **kw)


def test_lora_outputs_over_the_other_inputs(pkg):
    """The ids and scales that the rows of other workgroups still read."""
    buf = {name: f(T, 128) for name in ("scales", "adapter_ids", "request_ids")}
    arg = dict(scales=_over(buf["scales"], torch.float32, 2), adapter_ids=_over(buf["adapter_ids"], torch.int32, T),
               request_ids=_over(buf["request_ids"], torch.int32, T))
    for name in buf:
        with pytest.raises(ValueError, match="overlaps|may not be"):
            _lora(pkg, out=_over(buf[name], BF, T, 128), **arg)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _lora(pkg, out=z(T, 128), **arg)


def test_qk_axes_outputs_over_the_other_inputs(pkg):
    """The positions, ids and weights that the rows of other workgroups still read, for either output."""
    buf = {name: f(T, 256) for name in ("positions", "request_ids", "q_gamma", "k_gamma")}
    arg = dict(positions=_over(buf["positions"], torch.int32, T, 2), request_ids=_over(buf["request_ids"], torch.int32, T), requests=2,
               q_gamma=_over(buf["q_gamma"], torch.float32, 64), k_gamma=_over(buf["k_gamma"], torch.float32, 64), norm="rms_norm")
    for name in buf:
        for out in (dict(q_out=_over(buf[name], BF, T, 4, 64)), dict(k_out=_over(buf[name], BF, T, 2, 64))):
            with pytest.raises(ValueError, match="overlaps|may not be"):
                _qk(pkg, **arg, **out)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _qk(pkg, q_out=z(T, 4, 64), k_out=z(T, 2, 64), **arg)


def test_qk_axes_weights_across_heads_at_an_odd_float(pkg):
    """They are read 16 bytes a lane; a weight of one head may lie anywhere."""
    for kw, what in ((dict(q_gamma=f(257)[1:]), "q_gamma"), (dict(q_gamma=f(256), k_gamma=f(130)[2:]), "k_gamma")):
        with pytest.raises(ValueError, match=f"{what} must be 16-byte aligned"):
            _qk(pkg, norm="rms_norm_across_heads", **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _qk(pkg, norm="rms_norm", q_gamma=f(65)[1:])
    lib, dims, freqs = pkg._lib.load(), (ctypes.c_int * 1)(16), (ctypes.c_double * 8)()
    for gq, gk in ((20, None), (None, 24), (32, 36)):
        assert lib.wanmi_qk_norm_rope_axes(16, 64, 64, 1, gq, 16, 64, 64, 16, 64, 64, 1, gk, 16, 64, 64, 4, 64, 16, 0, 1, dims, freqs, 0, 2, 1e-6,
                                           None, 1, 1, None, None) == pkg._lib.WANMI_ERR_ARG


@pytest.mark.parametrize("name", ["mul", "add", "gate"])
def test_sandwich_vectors_without_dimensions(pkg, name):
    args = dict(mul=None, add=None, gate=None)
    args[name] = torch.tensor(1.0)
    with pytest.raises(ValueError, match=name):
        pkg.adaln_sandwich(z(T, H), z(T, H), args["mul"], args["add"], gate=args["gate"], eps=1e-6)


def test_packed_forward_refuses_what_does_not_fit(pkg):
    packed = pkg.PackedRequests.from_lengths([2, 3], 6, "cpu")
    args = dict(h=z(6, 128), temb=f(2, 6, 128), packed=packed, positions=torch.zeros(6, 3, dtype=torch.int32), crosses=[[None, None]])
    none = pkg.packed_block.BlockAdapters()
    for kw, match in ((dict(h=z(5, 128)), "do not fit"), (dict(positions=torch.zeros(6, 2, dtype=torch.int32)), "do not fit"), (dict(temb=f(1, 6, 128)), "crosses"),
                      (dict(crosses=[[None]]), "crosses"), (dict(crosses=[]), "crosses"), (dict(adapter_ids=ids(3)), "adapter_ids"),
                      (dict(adapters=[none, none], adapter_ids=ids(2)), "adapters")):
        with pytest.raises(ValueError, match=match):
            pkg.packed_dit_forward([None], **{**args, **kw}, tables=f(1, 6, 128))
    with pytest.raises(ValueError, match="1 entries for 2 blocks"):
        pkg.packed_dit_forward([None] * 2, **{**args, "crosses": [[None] * 2] * 2}, adapters=[none], tables=f(2, 6, 128))


def test_qk_axes_refuses_before_it_clears_the_bounds(pkg):
    """With a bound asked for, too: null pointers, strides and alignment are argument errors, no launch."""
    lib, dims, freqs = pkg._lib.load(), (ctypes.c_int * 1)(16), (ctypes.c_double * 8)()

    def qk(q=16, k=16, ts=64, pos=16, gq=None):
        return lib.wanmi_qk_norm_rope_axes(q, ts, 64, 1, gq, 16, 64, 64, k, 64, 64, 1, None, 16, 64, 64, 4, 64, pos, 0, 1, dims, freqs, 0, 2, 1e-6,
                                           None, 1, 1, 16, None)

    for kw in (dict(q=None), dict(k=None), dict(ts=4), dict(ts=-64), dict(q=8), dict(pos=None), dict(gq=20)):
        assert qk(**kw) == pkg._lib.WANMI_ERR_ARG, kw
