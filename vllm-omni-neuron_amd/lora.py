"""Low-rank adapters of many requests beside a shared projection, on gfx950.

:func:`lora_add` adds each row's ``scale * B (A x)`` to what a projection such as :func:`.mxfp8_linear` made of the
same activation. Which adapter a row uses is read from GPU tensors, so nothing is sorted or planned on the host
and a captured HIP graph may be replayed with other adapters. :func:`stack_adapters` lays adapters of
different ranks out for it. The reference serves one set of weights and has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .common_types import MXTensor
from .row_mx_kernels import _as_mx_2d

_MAX_PARTS = 8


def _check_slices(slices, N: int) -> tuple:
    slices = (N,) if slices is None else tuple(int(w) for w in slices)
    if not 1 <= len(slices) <= _MAX_PARTS or any(w <= 0 for w in slices) or sum(slices) != N:
        raise ValueError(f"slices {slices}: 1 to {_MAX_PARTS} widths that sum to {N}")
    if len(slices) > 1 and any(w % 64 for w in slices):
        raise ValueError(f"slices {slices} must be multiples of 64")
    return slices


def _workspace(T: int, K: int, parts: int, rank: int) -> int:
    return _lib.load().wanmi_lora_workspace(T, K, parts, rank)


@functools.lru_cache(maxsize=64)
def _fits(slices: tuple, N: int) -> bool:
    """Whether :func:`_check_slices` takes these widths as they are."""
    try:
        return all(type(w) is int for w in slices) and _check_slices(slices, N) == slices
    except (TypeError, ValueError):
        return False


@functools.lru_cache(maxsize=64)
def _widths(slices: tuple):
    return (ctypes.c_int64 * len(slices))(*slices)


def stack_adapters(adapters, in_features: int, slices, *, device):
    """Adapters of one projection -> the ``(a, b)`` stacks of :func:`lora_add`, made once.

    ``adapters``: a list; each adapter a list with an entry per slice, ``(a [r, in_features], b [width, r])`` or None
    (that part is not adapted). Ranks may differ; all are padded with zeros to the largest, rounded up to 16."""
    slices = _check_slices(slices, sum(int(w) for w in slices))
    if not adapters:
        raise ValueError("no adapters")
    rank = 16
    for i, parts in enumerate(adapters):
        if len(parts) != len(slices):
            raise ValueError(f"adapter {i} has {len(parts)} parts for {len(slices)} slices")
        for part, width in zip(parts, slices):
            if part is None:
                continue
            a, b = part
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != in_features or tuple(b.shape) != (width, a.shape[0]):
                raise ValueError(f"adapter {i}: a {list(a.shape)} and b {list(b.shape)} for {in_features} -> {width}")
            rank = max(rank, -(-a.shape[0] // 16) * 16)
    a_all = torch.zeros((len(adapters), len(slices), rank, in_features), dtype=torch.bfloat16, device=device)
    b_all = torch.zeros((len(adapters), sum(slices), rank), dtype=torch.bfloat16, device=device)
    for i, parts in enumerate(adapters):
        at = 0
        for s, (part, width) in enumerate(zip(parts, slices)):
            if part is not None:
                r = part[0].shape[0]
                a_all[i, s, :r] = part[0].to(device=device, dtype=torch.bfloat16)
                b_all[i, at : at + width, :r] = part[1].to(device=device, dtype=torch.bfloat16)
            at += width
    return a_all.view(len(adapters), len(slices) * rank, in_features), b_all


def lora_add(base: torch.Tensor, x, a: torch.Tensor, b: torch.Tensor, adapter_ids: torch.Tensor, *,
             scales: torch.Tensor | None = None, slices=None, request_ids: torch.Tensor | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = bf16(base[t] + scales[e] * (x[t] @ a[e].T) @ b[e].T)``, e the adapter of row t's request.

    ``base`` bf16 ``[T, N]``: the shared projection's output. ``x``: its activation, bf16 ``[T, K]``, an
    :class:`MXTensor` or ROW-packed ``[T, K + 4]``. ``a`` bf16 ``[adapters, len(slices) * r, K]`` and ``b`` bf16
    ``[adapters, N, r]``, contiguous (:func:`stack_adapters`), r a multiple of 16, K of 32, N of 8; ``scales`` fp32
    ``[adapters]`` (None: ones). ``slices``: the column counts of a fused projection's parts (Q, K, V), multiples of 64:
    the columns of part p take the ranks ``p * r`` to ``(p + 1) * r`` of ``a``.

    ``adapter_ids`` int32: one per request, ``[R]``, with ``request_ids`` int32 ``[T]``; without ``request_ids`` one per row,
    ``[T]``. A negative adapter (or one that does not exist) leaves the row as ``base`` has it. A row whose request id
    is negative (or not below R) belongs to no request and is not computed: left as it is in a given ``out``, zeros
    in one allocated here. ``out`` may be ``base``.

    Both sums are fp32, and the output is rounded once; between them ``u = scales[e] * (x[t] @ a[e].T)`` enters the
    second product as two bf16 values, to 2^-16 of itself. From 1024 rows on, K that is a multiple of 128 is faster than K
    that is not (1.2 to 1.8 times at 32760 rows and K about 5000). A ROW-packed ``x`` is unpacked by a launch of its own first.
    """
    if out is None and (slices is None or type(slices) is tuple):
        done = _add_plain(base, x, a, b, adapter_ids, scales, slices, request_ids)
        if done is not None:
            return done
    return _add_checked(base, x, a, b, adapter_ids, scales, slices, request_ids, out)


def _add_plain(base, x, a, b, adapter_ids, scales, slices, request_ids):
    """:func:`lora_add` for arguments of ordinary form (contiguous rows, bf16 or MX activations, ``out`` allocated here);
    None if any is not."""
    try:
        T, N = shape = base.shape
        dev = base.get_device()
        n, R, K = a.shape
        r = b.shape[2]
        slices = (N,) if slices is None else slices
        parts = len(slices)
        if not 0 < r <= 1024 or r & 15 or R != parts * r or K & 31 or N & 7 or not _fits(slices, N):
            return None
        if type(x) is MXTensor:
            px, psx = _lib.plain_ptr(x.codes, torch.float8_e4m3fn, (T, K), dev), _lib.plain_ptr(x.scales, torch.uint8, (T, K >> 5), dev)
        else:
            px, psx = _lib.plain_ptr(x, torch.bfloat16, (T, K), dev), None
        pb = _lib.plain_ptr(base, torch.bfloat16, shape, dev)
        pA = _lib.plain_ptr(a, torch.bfloat16, (n, R, K), dev)
        pB = _lib.plain_ptr(b, torch.bfloat16, (n, N, r), dev)
        ps = _lib.plain_ptr(scales, torch.float32, (n,), dev)
        pq = _lib.plain_ptr(request_ids, torch.int32, (T,), dev)
        requests = T if request_ids is None else adapter_ids.shape[0]
        pe = _lib.plain_ptr(adapter_ids, torch.int32, (requests,), dev)
    except (AttributeError, IndexError, TypeError, ValueError):
        return None
    if dev < 0 or T == 0 or n < 1 or None in (px, pA, pB, pe) or -1 in (px, psx, pb, pA, pB, ps, pq, pe):
        return None
    out = torch.empty_like(base)
    size = _workspace(T, K, parts, r)
    work = torch.empty(size, dtype=torch.uint8, device=base.device)
    _lib.call("wanmi_lora_add", dev, px, psx, None, K, pA, pB, ps, pe, pq, requests, n, T, K, N, r, parts, _widths(slices), pb, N,
              out.data_ptr(), N, 1, work.data_ptr(), size)
    return out


def _add_checked(base, x, a, b, adapter_ids, scales, slices, request_ids, out):
    _lib.expect(base, "base", dtype=torch.bfloat16, shape=(None, None), contiguous=False, row_contiguous=True)
    T, N = base.shape
    if isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16:
        _lib.expect(x, "x", dtype=torch.bfloat16, shape=(T, None), contiguous=False, row_contiguous=True)
        codes, x_scales, row_scale = x, None, None
    else:
        codes, x_scales, row_scale, lead = _as_mx_2d(x)
        if tuple(lead) != (T,):
            raise ValueError(f"x must hold {T} rows, got {list(lead)}")
        if not x_scales.is_contiguous():
            raise ValueError("x's scales must be contiguous")
    K = codes.shape[1]
    for name, t in (("a", a), ("b", b)):
        _lib.expect(t, name, dtype=torch.bfloat16, shape=(None, None, None))
    n, R, r = a.shape[0], a.shape[1], b.shape[2]
    slices = _check_slices(slices, N)
    if n < 1 or tuple(a.shape) != (n, len(slices) * r, K) or tuple(b.shape) != (n, N, r):
        raise ValueError(f"a {list(a.shape)} and b {list(b.shape)} do not fit x [{T}, {K}], base [{T}, {N}] and "
                         f"{len(slices)} slices")
    if r < 16 or r % 16 or r > 1024:
        raise ValueError(f"rank {r} must be a multiple of 16, at most 1024 (pad with zeros: stack_adapters)")
    if K < 32 or K % 32 or N < 8 or N % 8:
        raise ValueError(f"K={K} must be a multiple of 32, N={N} of 8")
    _lib.expect(scales, "scales", dtype=torch.float32, shape=(n,), optional=True)
    _lib.request_rows(request_ids, T)
    _lib.expect(adapter_ids, "adapter_ids", dtype=torch.int32, shape=(T if request_ids is None else None,))
    item = codes.element_size()
    ldx, ldb = codes.stride(0) if T > 1 else K, base.stride(0) if T > 1 else N
    if ldx < K or ldx * item % 16 or codes.data_ptr() % 16:
        raise ValueError("x rows must be 16-byte aligned")
    if ldb < N or ldb % 8 or base.data_ptr() % 16:
        raise ValueError("base rows must be 16-byte aligned")
    if a.data_ptr() % 16 or b.data_ptr() % 16:
        raise ValueError("a and b must be 16-byte aligned")
    if out is not None:
        _lib.expect(out, "out", dtype=torch.bfloat16, shape=(T, N), contiguous=False, row_contiguous=True)
        if (T > 1 and (out.stride(0) < N or out.stride(0) % 8)) or out.data_ptr() % 16:
            raise ValueError("out rows must be 16-byte aligned")
        _lib.refuse_overlap(out, "out", base)
        _lib.refuse_input(out, "out", codes, x_scales, row_scale, a, b, scales, adapter_ids, request_ids)
    _lib.require_gpu(base, codes, x_scales, row_scale, a, b, scales, adapter_ids, request_ids, out, what="lora_add")
    zero_rest = out is None
    if out is None:
        out = torch.empty((T, N), dtype=torch.bfloat16, device=base.device)
    if T == 0:
        return out
    size = _workspace(T, K, len(slices), r)
    work = torch.empty(size, dtype=torch.uint8, device=base.device)
    p = _lib.ptr
    _lib.call("wanmi_lora_add", base.get_device(), p(codes), p(x_scales), p(row_scale), ldx, p(a), p(b), p(scales), p(adapter_ids), p(request_ids),
              T if request_ids is None else adapter_ids.shape[0], n, T, K, N, r, len(slices), _widths(slices), p(base), ldb, p(out),
              out.stride(0) if T > 1 else N, int(zero_rest), p(work), size)
    return out
