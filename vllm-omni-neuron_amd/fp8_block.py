"""Products with 8-bit weights that have one fp32 scale per block of 128 x 128, on gfx950.

The format of checkpoints that are quantized block by block: e4m3 codes ``[N, K]`` and fp32 scales ``[ceil(N / 128), ceil(K / 128)]``
(:class:`FP8BlockWeight`), and activations with one fp32 scale for each 128 of a row (:class:`FP8BlockTensor`). Such weights run as
they are: neither their codes nor their scales are rounded again, as they would be to the power-of-two scales per 32 of an
:class:`.MXWeight`. The reference has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

BLOCK = 128
_ACTIVATIONS = {None: 0, "gelu": 1}


class FP8BlockTensor(NamedTuple):
    """An activation: e4m3fn codes ``[..., K]`` and an fp32 scale per 128 codes ``[..., ceil(K / 128)]``; code i of a row stands for
    ``codes[i] * scales[i // 128]``. :func:`quantize_fp8_blocks` lays the scales out block by block (their strides are
    ``(1, rows)``), which the product reads as they are; of any other strides it makes such a copy first."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.codes.shape

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        f = self.scales.repeat_interleave(BLOCK, dim=-1)[..., : self.codes.shape[-1]]
        return (self.codes.to(torch.float32) * f).to(dtype)


class FP8BlockWeight(NamedTuple):
    """A projection weight: e4m3fn codes ``[N, K]``, fp32 scales ``[ceil(N / 128), ceil(K / 128)]``, fp32 ``bias [N]`` or None."""

    codes: torch.Tensor
    scales: torch.Tensor
    bias: torch.Tensor | None = None

    @property
    def out_features(self) -> int:
        return self.codes.shape[0]

    @property
    def in_features(self) -> int:
        return self.codes.shape[1]

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """``[N, K]``"""
        N, K = self.codes.shape
        f = self.scales.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
        return (self.codes.to(torch.float32) * f).to(dtype)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def quantize_weight_fp8_blocks(weight_kn: torch.Tensor, bias: torch.Tensor | None = None) -> FP8BlockWeight:
    """Reference-layout weight ``[K, N]`` (``x @ W``) -> :class:`FP8BlockWeight`, once at load time. A block's scale is its largest
    magnitude (at least 2^-100) times fp32(1 / 448)."""
    if weight_kn.dim() != 2:
        raise ValueError("weight must be [K, N]")
    K, N = weight_kn.shape
    w = torch.nn.functional.pad(weight_kn.t().to(torch.float32), (0, -K % BLOCK, 0, -N % BLOCK)).view(_blocks(N), BLOCK, _blocks(K), BLOCK)
    scales = w.abs().amax((1, 3)).clamp_min(2.0**-100) * (1.0 / 448.0)
    codes = (w / scales[:, None, :, None]).view(_blocks(N) * BLOCK, -1)[:N, :K].contiguous().to(torch.float8_e4m3fn)
    return FP8BlockWeight(codes, scales, None if bias is None else bias.reshape(-1).to(torch.float32).contiguous())


def _check_rows(x: torch.Tensor, what: str) -> tuple:
    """``[..., K]`` as two dimensions with 16-byte aligned rows: the tensor and its row stride."""
    K = x.shape[-1] if x.dim() else 0
    if x.dim() < 1 or K < 16 or K % 16:
        raise ValueError(f"{what}: K={K} must be a multiple of 16")
    if x.dim() != 2:
        x = x.reshape(-1, K)
    ld = x.stride(0) if x.shape[0] > 1 else K
    if x.stride(1) != 1 or ld < K or ld * x.element_size() % 16 or x.data_ptr() % 16:
        raise ValueError(f"{what} rows must be contiguous and 16-byte aligned")
    return x, ld


def quantize_fp8_blocks(x: torch.Tensor) -> FP8BlockTensor:
    """bf16 ``[..., K]`` (K a multiple of 16) -> :class:`FP8BlockTensor`: a block's scale is its largest magnitude (at least
    2^-100) times fp32(1 / 448), the codes are ``x / scale`` to the nearest. A block that holds an infinity or a NaN is NaN throughout."""
    if not isinstance(x, torch.Tensor) or x.dtype != torch.bfloat16:
        raise ValueError("x must be a bf16 tensor [..., K]")
    lead = x.shape[:-1]
    x2, ld = _check_rows(x, "x")
    _lib.require_gpu(x2, what="quantize_fp8_blocks")
    M, K = x2.shape
    codes = torch.empty((M, K), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((_blocks(K), M), dtype=torch.float32, device=x.device)
    if M:
        _lib.call("wanmi_fp8_block_quantize", x2.get_device(), _lib.ptr(x2), ld, M, K, _lib.ptr(codes), _lib.ptr(scales), 1, M)
    scales = scales.t()
    return FP8BlockTensor(codes, scales) if len(lead) == 1 else FP8BlockTensor(codes.view(*lead, K), scales.reshape(*lead, _blocks(K)))


def _check_weight(w: FP8BlockWeight) -> None:
    if not isinstance(w, FP8BlockWeight):
        raise ValueError("weight must be an FP8BlockWeight (see quantize_weight_fp8_blocks)")
    _lib.expect(w.codes, "weight.codes", dtype=torch.float8_e4m3fn, shape=(None, None))
    N, K = w.codes.shape
    _lib.expect(w.scales, "weight.scales", dtype=torch.float32, shape=(_blocks(N), _blocks(K)))
    _lib.expect(w.bias, "weight.bias", dtype=torch.float32, shape=(N,), optional=True)
    if N < 8 or N % 8:
        raise ValueError(f"N={N} must be a multiple of 8")
    if w.codes.data_ptr() % 16 or (w.bias is not None and w.bias.data_ptr() % 16):
        raise ValueError("weight codes and bias must be 16-byte aligned")


def fp8_block_linear(x, weight: FP8BlockWeight, *, activation: str | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ W^T + bias)`` with the scales of each block of 128 along the sum applied in fp32; bf16 ``[..., N]``.

    ``x``: bf16 ``[..., K]``, quantized on the way as :func:`quantize_fp8_blocks` does it, or an :class:`FP8BlockTensor`. K a multiple of 16, N
    of 8 (the last blocks may be partial). ``activation``: None or ``"gelu"`` (its tanh form). ``out``: bf16 ``[rows, N]`` with rows a
    multiple of 8 elements apart. Any number of rows. Up to 16 of them take one launch that reads the weight once at the memory's
    rate, up to 4 in bf16 are quantized inside it; more in bf16 take a launch for that and a workspace for the codes, and middling
    sizes, whose tiles would not fill the chip, share out the sum and add its parts in another. Inference only: no gradient."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    y = _linear_plain(x, weight, _ACTIVATIONS[activation]) if out is None else None
    return _linear_checked(x, weight, _ACTIVATIONS[activation], out) if y is None else y


def _launch(dev: int, px, ps, ld: int, s_row: int, s_blk: int, pw, psw, pb, M: int, N: int, K: int, gelu: int, y: torch.Tensor, ldo: int) -> None:
    size = _lib.load().wanmi_fp8_block_workspace(M, N, K, int(ps is None), s_row)
    work = torch.empty(size, dtype=torch.uint8, device=y.device) if size else None
    _lib.call("wanmi_fp8_block_linear", dev, px, ps, ld, s_row, s_blk, pw, psw, pb, M, N, K, gelu, y.data_ptr(), ldo, _lib.ptr(work), size)


def _linear_plain(x, weight, gelu: int):
    """:func:`fp8_block_linear` for arguments of ordinary form (two dimensions, contiguous rows); None if any is not."""
    try:
        if type(weight) is not FP8BlockWeight:
            return None
        wc, wsc, wb = weight
        N, K = wc.shape
        dev = wc.get_device()
        kb = (K + 127) >> 7
        if N < 8 or N & 7 or K < 16 or K & 15 or dev < 0:
            return None
        ps, s_row, s_blk = None, 0, 0
        if type(x) is FP8BlockTensor:
            codes, scales = x
            M = codes.shape[0]
            px = _lib.plain_ptr(codes, torch.float8_e4m3fn, (M, K), dev)
            if scales.dtype is not torch.float32 or scales.shape != (M, kb) or scales.get_device() != dev:
                return None
            s_row, s_blk = scales.stride()
            ps = scales.data_ptr()
        else:
            M = x.shape[0]
            px = _lib.plain_ptr(x, torch.bfloat16, (M, K), dev)
        pw = _lib.plain_ptr(wc, torch.float8_e4m3fn, (N, K), dev)
        psw = _lib.plain_ptr(wsc, torch.float32, ((N + 127) >> 7, kb), dev)
        pb = _lib.plain_ptr(wb, torch.float32, (N,), dev)
    except (AttributeError, IndexError, TypeError, ValueError):
        return None
    if M < 1 or None in (px, pw, psw) or -1 in (px, pw, psw, pb):
        return None
    y = torch.empty((M, N), dtype=torch.bfloat16, device=wc.device)
    _launch(dev, px, ps, K, s_row if M > 1 else 1, s_blk, pw, psw, pb, M, N, K, gelu, y, N)
    return y


def _linear_checked(x, weight, gelu: int, out):
    _check_weight(weight)
    N, K = weight.codes.shape
    scales = None
    if isinstance(x, FP8BlockTensor):
        codes, scales = x
        _lib.expect(codes, "x.codes", dtype=torch.float8_e4m3fn, contiguous=False)
        if codes.dim() < 1:
            raise ValueError("x.codes must be [..., K]")
        lead = codes.shape[:-1]
        _lib.expect(scales, "x.scales", dtype=torch.float32, shape=(*lead, _blocks(codes.shape[-1])), contiguous=False)
    elif isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16:
        codes, lead = x, x.shape[:-1]
    else:
        raise ValueError("x must be a bf16 tensor [..., K] or an FP8BlockTensor")
    if codes.dim() < 1 or codes.shape[-1] != K:
        raise ValueError(f"x {list(codes.shape)} does not match the weight's K={K}")
    codes, ld = _check_rows(codes, "x")
    M = codes.shape[0]
    s_row = s_blk = 0
    if scales is not None:
        if len(lead) != 1:
            scales = scales.reshape(M, _blocks(K))
        s_row, s_blk = (scales.stride(0) if M > 1 else 1), scales.stride(1)
    if out is not None:
        _lib.expect(out, "out", dtype=torch.bfloat16, shape=(M, N), contiguous=False, row_contiguous=True)
        if (M > 1 and (out.stride(0) < N or out.stride(0) % 8)) or out.data_ptr() % 16:
            raise ValueError("out rows must be 16-byte aligned")
        _lib.refuse_input(out, "out", codes, scales, weight.codes, weight.scales, weight.bias)
    dev = _lib.require_gpu(codes, scales, weight.codes, weight.scales, weight.bias, out, what="fp8_block_linear")
    y = torch.empty((M, N), dtype=torch.bfloat16, device=dev) if out is None else out
    if M:
        p = _lib.ptr
        _launch(codes.get_device(), p(codes), p(scales), ld, s_row, s_blk, p(weight.codes), p(weight.scales), p(weight.bias), M, N, K, gelu, y,
                y.stride(0) if M > 1 else N)
    return y if len(lead) == 1 else y.reshape(*lead, N)
