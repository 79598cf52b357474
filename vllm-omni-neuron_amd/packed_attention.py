"""Attention over packed rows on gfx950: the text side of a batch of requests.

:func:`packed_cross_attention` lets the rows of every request look at its own text, whatever its length, in one launch.
:func:`relative_bias_attention` is the self-attention of the text encoder in front of it, over packed prompts, with a learned
bias by buckets of relative distance. Where a request's rows and keys begin and end is read from GPU tensors of offsets, so
that a captured HIP graph may be replayed with other lengths. The reference serves one request per forward and
has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .common_types import MXTensor

_MAX_SIDE, _MAX_SATURATION = 128, 1024
_MIN_SCALE, _MAX_SCALE = 2.0**-64, 2.0**24


@functools.lru_cache(maxsize=64)
def _bucket_starts(buckets: int, max_distance: int, bidirectional: bool):
    """The smallest distance of each bucket of one direction: the first half hold one distance each, the
    others grow by equal ratios up to ``max_distance``. The borders are ``first * (max_distance / first)^(i / steps)`` rounded up,
    found in whole numbers: some of them are whole, where a logarithm in floating point may fall on either side."""
    if buckets < (4 if bidirectional else 2) or (bidirectional and buckets % 2):
        raise ValueError(f"{buckets} buckets: at least 2 a direction, an even number for both")
    side = buckets // 2 if bidirectional else buckets
    first = side // 2
    if side > _MAX_SIDE or max_distance <= first:
        raise ValueError(f"{side} buckets of one direction (at most {_MAX_SIDE}) up to distance {max_distance}, which must exceed {first}")
    steps = side - first
    starts = list(range(first))
    n = first
    for i in range(steps):
        while n**steps * first**i < max_distance**i * first**steps:
            n += 1
            if n > _MAX_SATURATION:
                raise ValueError(f"bucket {first + i} of {side} up to distance {max_distance} starts behind {_MAX_SATURATION}: at most {_MAX_SATURATION}")
        starts.append(n)
    return (ctypes.c_int * side)(*starts)


def _rows(t, what: str, heads: int | None, head_dim: int | None) -> None:
    _lib.expect(t, what, dtype=torch.bfloat16, shape=(None, heads, head_dim), contiguous=False, row_contiguous=True)


def _strides(t) -> tuple:
    """Row and head strides; those of a dimension of one element, which nothing reads, as a contiguous tensor has them."""
    T, H, D = t.shape
    return (t.stride(0) if T > 1 else H * D), (t.stride(1) if H > 1 else D)


def _check(q, k, v, scale, out, quant, what: str) -> float:
    _rows(q, "q", None, None)
    T, heads, head_dim = q.shape
    _rows(k, "k", None, head_dim)
    _rows(v, "v", k.shape[1], head_dim)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"k holds {k.shape[0]} rows, v {v.shape[0]}")
    if head_dim not in (64, 128):
        raise NotImplementedError(f"{what}: head_dim {head_dim}: 64 or 128")
    if heads < 1 or k.shape[1] < 1 or heads % k.shape[1]:
        raise ValueError(f"{heads} query heads over {k.shape[1]} key heads")
    scale = head_dim**-0.5 if scale is None else float(scale)
    if not _MIN_SCALE <= scale <= _MAX_SCALE:
        raise ValueError(f"scale {scale} must be between 2^-64 and 2^24")
    for name, t in (("q", q), ("k", k), ("v", v)):
        ss, hs = _strides(t)
        if ss % 8 or hs % 8 or t.data_ptr() % 16:
            raise ValueError(f"{name}'s rows and heads must be 16-byte aligned")
        if (t.shape[0] > 1 and ss < head_dim) or (t.shape[1] > 1 and hs < head_dim):
            raise ValueError(f"{name}'s rows or heads overlap")
    if quant not in ("none", "mx"):
        raise ValueError(f"unknown quant {quant!r}")
    if out is not None:
        if quant != "none":
            raise ValueError("out takes bf16: quant must be 'none'")
        _lib.expect(out, "out", dtype=torch.bfloat16, shape=(T, heads, head_dim), contiguous=False, row_contiguous=True)
        ss, hs = _strides(out)
        if ss % 16 or (heads > 1 and hs != head_dim) or ss < heads * head_dim or out.data_ptr() % 16:
            raise ValueError("out must have its heads side by side and 16-byte aligned rows, a multiple of 16 elements apart")
        # a tile reads its rows of q before it writes them, and nobody else reads them
        _lib.refuse_overlap(out, "out", q)
        _lib.refuse_input(out, "out", k, v)
    return scale


def _plain(q, k, v, scale):
    """The shapes, strides and pointers of ordinary arguments (several rows and heads, on one GPU, aligned) in one look, or None:
    :func:`_check` says what is wrong with them or takes them as they are."""
    try:
        (T, heads, D), (Tk, k_heads, Dk), vs = q.shape, k.shape, v.shape
        dev = q.get_device()
        strides, pointers = [], []
        for t in (q, k, v):
            ss, hs, es = t.stride()
            p = t.data_ptr()
            if t.dtype is not torch.bfloat16 or t.get_device() != dev or es != 1 or ss & 7 or hs & 7 or p & 15 or ss < D or hs < D:
                return None
            strides.append((ss, hs))
            pointers.append(p)
        scale = D**-0.5 if scale is None else scale
        if D != Dk or vs != k.shape or dev < 0 or D not in (64, 128) or T < 2 or Tk < 2 or k_heads < 1 or heads % k_heads or type(scale) is not float:
            return None
        if heads < 2 or k_heads < 2 or not _MIN_SCALE <= scale <= _MAX_SCALE:
            return None
    except (AttributeError, RuntimeError, TypeError, ValueError):
        return None
    return dev, T, heads, D, Tk, k_heads, strides, pointers, scale


def _offsets(t, what: str, n: int | None = None) -> int:
    _lib.expect(t, what, dtype=torch.int32, shape=(n,))
    if t.shape[0] < 1:
        raise ValueError(f"{what} needs one entry more than there are requests")
    return t.shape[0] - 1


def packed_cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
                           *, scale: float | None = None, quant: str = "none", out: torch.Tensor | None = None):
    """Each request's rows of ``q`` over its own rows of ``k`` and ``v``: ``softmax(scale * q k^T) v`` per head, all requests in one launch.

    ``q`` bf16 ``[T, heads, D]``, ``k`` and ``v`` bf16 ``[Tk, k_heads, D]`` with D 64 or 128, ``heads`` a multiple of ``k_heads`` (query
    head h reads key head ``h // (heads // k_heads)``); rows and heads may be strided (column blocks of a fused
    projection). ``q_offsets`` and ``k_offsets`` int32 ``[R + 1]`` on the GPU, ascending from 0: request r has the rows
    ``q_offsets[r]`` to ``q_offsets[r + 1]`` and the keys ``k_offsets[r]`` to ``k_offsets[r + 1]``
    (:attr:`.PackedRequests.offsets`). ``scale``: ``D ** -0.5`` if None.

    Returns bf16 ``[T, heads, D]``, or with ``quant="mx"`` an :class:`MXTensor` ``[T, heads * D]`` as the MX projections read it.
    The rows of a request without keys are zeros. Rows behind the last request are zeros too in an output allocated here and
    left as they are in a given ``out``, which may be ``q``. Offsets are held inside the tensors: wrong ones give wrong
    rows, and no access out of bounds. The softmax has a running maximum (no bound on scores is needed) and fp32 sums; its weights enter the
    second product as bf16. Inference only: no gradient.
    """
    if out is None and quant == "none":
        plain = _plain(q, k, v, scale)
        if plain is not None:
            dev, T, heads, head_dim, Tk, k_heads, strides, pointers, s = plain
            n = q_offsets.shape if isinstance(q_offsets, torch.Tensor) else ()
            pq, pk = (_lib.plain_ptr(t, torch.int32, n, dev) if isinstance(t, torch.Tensor) else None for t in (q_offsets, k_offsets))
            if len(n) == 1 and n[0] and pq not in (None, -1) and pk not in (None, -1):
                out = torch.empty((T, heads, head_dim), dtype=torch.bfloat16, device=q.device)
                _lib.call("wanmi_packed_cross_attention", dev, pointers[0], *strides[0], pointers[1], *strides[1], pointers[2], *strides[2], pq, pk,
                          n[0] - 1, T, Tk, heads, k_heads, head_dim, s, out.data_ptr(), heads * head_dim, None, 1)
                return out
    scale = _check(q, k, v, scale, out, quant, "packed_cross_attention")
    requests = _offsets(q_offsets, "q_offsets")
    _offsets(k_offsets, "k_offsets", requests + 1)
    if out is not None:
        _lib.refuse_input(out, "out", q_offsets, k_offsets)
    _lib.require_gpu(q, k, v, q_offsets, k_offsets, out, what="packed_cross_attention")
    T, heads, head_dim = q.shape
    zero_rest = out is None
    scales = None
    if quant == "mx":
        out = torch.empty((T, heads * head_dim), dtype=torch.float8_e4m3fn, device=q.device)
        scales = torch.empty((T, heads * head_dim // 32), dtype=torch.uint8, device=q.device)
        ldo = heads * head_dim
    else:
        if out is None:
            out = torch.empty((T, heads, head_dim), dtype=torch.bfloat16, device=q.device)
        ldo = _strides(out)[0]
    if T:
        p = _lib.ptr
        _lib.call("wanmi_packed_cross_attention", q.get_device(), p(q), *_strides(q), p(k), *_strides(k), p(v), *_strides(v), p(q_offsets),
                  p(k_offsets), requests, T, k.shape[0], heads, k.shape[1], head_dim, scale, p(out), ldo, p(scales), int(zero_rest))
    return out if scales is None else MXTensor(out, scales)


def relative_bias_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, offsets: torch.Tensor, *,
                            max_distance: int = 128, bidirectional: bool = True, scale: float = 1.0,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """Self-attention of packed prompts with a learned bias by buckets of relative distance: per head
    ``softmax(scale * q_i k_j + table[bucket(j - i), h]) v_j`` over the tokens j of row i's own prompt.

    ``q``, ``k``, ``v`` bf16 ``[T, heads, D]``, D 64 or 128 (rows and heads may be strided); ``table`` fp32 or bf16 ``[buckets, heads]``, the
    weight of the embedding that holds the bias; ``offsets`` int32 ``[R + 1]`` on the GPU, ascending from 0: prompt r is the rows
    ``offsets[r]`` to ``offsets[r + 1]``. ``scale`` 1: such an encoder's scores are not scaled.

    Half of a direction's buckets hold one distance each, the others grow by equal ratios up to ``max_distance``, and the last
    holds everything beyond. ``bidirectional``: the first half of the table is for keys at or before the query, the second for those
    after it. Otherwise every bucket is for the keys before, and all later ones take bucket 0 (they are not masked). A bias of minus
    infinity leaves a key out, and a row that has no other is zeros; the lowest finite value of a type masks too, and a row of
    nothing else weighs all its keys alike.

    Returns bf16 ``[T, heads, D]``. Rows behind the last prompt are zeros in an output allocated here and left as they are in a
    given ``out``, which may be ``q``. Inference only: no gradient.
    """
    if out is None:
        plain = _plain(q, k, v, scale)
        if plain is not None:
            dev, T, heads, head_dim, Tk, k_heads, strides, pointers, s = plain
            if Tk == T and k_heads == heads and isinstance(table, torch.Tensor) and isinstance(offsets, torch.Tensor) and table.dim() == 2:
                n = offsets.shape
                po = _lib.plain_ptr(offsets, torch.int32, n, dev)
                pt = _lib.plain_ptr(table, table.dtype, (table.shape[0], heads), dev)
                if len(n) == 1 and n[0] and po != -1 and pt != -1 and table.dtype in (torch.float32, torch.bfloat16):
                    starts = _bucket_starts(table.shape[0], int(max_distance), bool(bidirectional))
                    out = torch.empty((T, heads, head_dim), dtype=torch.bfloat16, device=q.device)
                    _lib.call("wanmi_relative_bias_attention", dev, pointers[0], *strides[0], pointers[1], *strides[1], pointers[2], *strides[2], po,
                              n[0] - 1, T, heads, head_dim, s, pt, int(table.dtype is torch.bfloat16), starts, len(starts), int(bool(bidirectional)),
                              out.data_ptr(), heads * head_dim, 1)
                    return out
    scale = _check(q, k, v, scale, out, "none", "relative_bias_attention")
    T, heads, head_dim = q.shape
    if k.shape[1] != heads or k.shape[0] != T:
        raise ValueError(f"k and v {list(k.shape)} must have the rows and heads of q {list(q.shape)}")
    if not isinstance(table, torch.Tensor) or table.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("table must be an fp32 or bf16 tensor [buckets, heads]")
    _lib.expect(table, "table", dtype=table.dtype, shape=(None, heads))
    starts = _bucket_starts(table.shape[0], int(max_distance), bool(bidirectional))
    requests = _offsets(offsets, "offsets")
    if out is not None:
        _lib.refuse_input(out, "out", table, offsets)
    _lib.require_gpu(q, k, v, table, offsets, out, what="relative_bias_attention")
    zero_rest = out is None
    if out is None:
        out = torch.empty((T, heads, head_dim), dtype=torch.bfloat16, device=q.device)
    if T:
        p = _lib.ptr
        _lib.call("wanmi_relative_bias_attention", q.get_device(), p(q), *_strides(q), p(k), *_strides(k), p(v), *_strides(v), p(offsets), requests,
                  T, heads, head_dim, scale, p(table), int(table.dtype is torch.bfloat16), starts, len(starts), int(bool(bidirectional)),
                  p(out), _strides(out)[0], int(zero_rest))
    return out
