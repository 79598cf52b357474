"""The Wan2.2 DiT blocks over a packed batch: several requests of different sizes, timesteps and adapters at once.

The rows of all requests lie one behind the other in one ``[rows, dim]`` tensor (:class:`PackedRequests`), so that a
weight is read once for all of them and small requests fill the chip together: a block of dim 5120 on 16 requests of
16 tokens takes 0.82 ms and 3.95 one request after another, 8 of 390 tokens 1.50 and 2.47, 4 of 1560 2.12 and 2.62, 2 of 7800
6.22 and 6.42. Attention runs request by request, and one request alone is faster through :func:`.block.dit_forward`
(7800 tokens: 3.30 here, 3.22 there). Per request differ the modulation
(one row of the timestep embedding each), the grid (positions given per token), the text context and the
low-rank adapters. A block is that of :mod:`.block` with each request's own

    q, k, v = a @ Wqkv + b (+ adapters)                               MXFP8 GEMM, lora_add
    q, k = RoPE(RMS_heads(q, k) g) at the rows' positions, max||k||      qk_norm_rope_axes
    o = MX(attention(q, k, v)) request by request                      constant-max attention
    y = o @ Wo + b (+ adapters)                                        MXFP8 GEMM, lora_add
    h1 = h + gate[q] * y;  a2 = MX(LN_affine(h1))                       adaln_sandwich
    ... the cross-attention and the FFN likewise, each sum with the norm that follows it in one pass:
    h3 = h2 + c_gate[q] * ffn;  a1 of the next block = MX(LN(h3) * (1 + scale[q]) + shift[q])

The reference serves one request per forward; what it computes for one is what a request gets here, up to the
rounding of q and k between norm and rotation, which this path does not make.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import attention_ops as ops
from .adaln_kernels import adaln_sandwich
from .block import HEAD_DIM, BlockWeights, modulation
from .common_types import MXTensor
from .lora import lora_add
from .row_mx_kernels import mxfp8_linear


class PackedRequests(NamedTuple):
    """Requests of ``lengths`` tokens, one behind the other in a batch of ``rows`` rows; the rows behind the last
    request belong to none. ``request_ids`` int32 ``[rows]``: each row's request, -1 for those."""

    lengths: tuple
    rows: int
    request_ids: torch.Tensor

    @classmethod
    def from_lengths(cls, lengths, rows: int | None = None, device="cuda") -> "PackedRequests":
        lengths = tuple(int(n) for n in lengths)
        if not lengths or min(lengths) < 0:
            raise ValueError(f"lengths must be non-negative, at least one: got {lengths}")
        total = sum(lengths)
        rows = total if rows is None else int(rows)
        if rows < total:
            raise ValueError(f"{total} tokens do not fit {rows} rows")
        ids = torch.full((rows,), -1, dtype=torch.int32)
        ids[:total] = torch.repeat_interleave(torch.arange(len(lengths), dtype=torch.int32), torch.tensor(lengths))
        return cls(lengths, rows, ids.to(device))

    def spans(self):
        """``(first row, row behind the last)`` of every request."""
        at = 0
        for n in self.lengths:
            yield at, at + n
            at += n

    def grid_positions(self, grids) -> torch.Tensor:
        """int32 ``[rows, 3]``: frame, row and column of every token in its request's latent grid ``(F, H, W)``, raster order
        (zeros for rows of no request)."""
        grids = [tuple(int(v) for v in grid) for grid in grids]
        if len(grids) != len(self.lengths) or any(f * h * w != n for (f, h, w), n in zip(grids, self.lengths)):
            raise ValueError(f"grids {grids} do not hold {self.lengths} tokens")
        pos = torch.zeros((self.rows, 3), dtype=torch.int32)
        for (a, b), grid in zip(self.spans(), grids):
            pos[a:b] = torch.stack(torch.meshgrid(*(torch.arange(n, dtype=torch.int32) for n in grid), indexing="ij"), -1).view(-1, 3)
        return pos.to(self.request_ids.device)


class Adapters(NamedTuple):
    """The stacked adapters of one projection (:func:`.stack_adapters`) and their scales, fp32 ``[adapters]`` or None."""

    a: torch.Tensor
    b: torch.Tensor
    scales: torch.Tensor | None = None


class BlockAdapters(NamedTuple):
    """Adapters of a block's projections (None: that projection has none). ``qkv`` in three slices of ``dim`` columns.

    The FFN's up projection takes none: its GELU and quantization are in the GEMM's epilogue. Nor do the text's K and V,
    which :func:`.block.project_cross_kv` projects once per generation: an adapter of theirs can be merged into the
    weights that it is given, request by request."""

    qkv: Adapters | None = None
    o: Adapters | None = None
    q2: Adapters | None = None
    o2: Adapters | None = None
    down: Adapters | None = None


def packed_modulation(tables: torch.Tensor, temb: torch.Tensor) -> torch.Tensor:
    """:func:`.modulation` for every request: tables ``[blocks, 6, dim]``, ``temb`` ``[R, 6, dim]`` -> fp32
    ``[blocks, R, 6, dim]``."""
    return torch.stack([modulation(tables, t) for t in temb], dim=1)


def _project(x, weight, adapters: Adapters | None, ids, packed: PackedRequests, slices=None) -> torch.Tensor:
    y = mxfp8_linear(x, weight)
    if adapters is None:
        return y
    if ids is None:
        raise ValueError("adapters need adapter_ids, one per request")
    return lora_add(y, x, adapters.a, adapters.b, ids, scales=adapters.scales, slices=slices, request_ids=packed.request_ids, out=y)


def _attend(packed: PackedRequests, dim: int, device, one) -> MXTensor:
    """``one(i, first, end, codes)`` -> the request's :class:`MXTensor` written to ``codes``, for each request that has rows."""
    codes = torch.zeros((packed.rows, dim), dtype=torch.uint8, device=device)
    scales = torch.zeros((packed.rows, dim // 32), dtype=torch.uint8, device=device)
    for i, (a, b) in enumerate(packed.spans()):
        if b > a:
            scales[a:b] = one(i, a, b, codes[a:b]).scales
    return MXTensor(codes.view(torch.float8_e4m3fn), scales)


def _sublayers(w: BlockWeights, h, a1: MXTensor, mod, packed, positions, crosses, adapters: BlockAdapters, ids, eps: float):
    """One block from its first normalized input to its FFN's output: ``(h2, ffn)``, whose gated sum is the block's result."""
    rows, dim = h.shape
    heads, scale = dim // HEAD_DIM, HEAD_DIM**-0.5
    sandwich = dict(eps=eps, post_norm="none", quant="mx", request_ids=packed.request_ids)

    qkv = _project(a1, w.qkv, adapters.qkv, ids, packed, slices=(dim, dim, dim))
    q, k, v = (qkv[:, i * dim : (i + 1) * dim].view(rows, heads, HEAD_DIM) for i in range(3))
    _, _, kmax = ops.qk_norm_rope_axes(q, k, positions, norm="rms_norm_across_heads", q_gamma=w.norm_q.view(-1), k_gamma=w.norm_k.view(-1), eps=eps,
                                       request_ids=packed.request_ids, requests=len(packed.lengths), want_max=True, q_out=q, k_out=k)

    def self_attention(i, a, b, codes):
        vt, _ = ops.transpose_heads(v[a:b])
        return ops.attention_core(q[a:b], k[a:b], vt, kmax[i], scale, ops.OUT_MX, out=codes)

    y = _project(_attend(packed, dim, h.device, self_attention), w.o, adapters.o, ids, packed)
    h1, a2 = adaln_sandwich(y, h, w.norm2_weight, w.norm2_bias, gate=mod[:, 2], **sandwich)

    sumsq = torch.empty((rows, dim // 128), dtype=torch.float32, device=h.device) if adapters.q2 is None else None
    if sumsq is not None:
        q2 = mxfp8_linear(a2, w.q2, row_sumsq=sumsq, sumsq_cols=dim).view(rows, heads, HEAD_DIM)
    else:
        q2 = _project(a2, w.q2, adapters.q2, ids, packed).view(rows, heads, HEAD_DIM)
        ops.qk_norm_rope_axes(q2, None, None, axes=(), norm="rms_norm_across_heads", q_gamma=w.norm_q2.view(-1), eps=eps,
                              request_ids=packed.request_ids, q_out=q2)

    def cross_attention(i, a, b, codes):
        prep = None if sumsq is None else ops.QPrep(sumsq[a:b], w.norm_q2, eps=eps)
        return ops.attention_core(q2[a:b], crosses[i].k, crosses[i].vt, crosses[i].kmax, scale, ops.OUT_MX, out=codes, q_prep=prep)

    y = _project(_attend(packed, dim, h.device, cross_attention), w.o2, adapters.o2, ids, packed)
    h2, a3 = adaln_sandwich(y, h1, mod[:, 4], mod[:, 3], **sandwich)
    inter = mxfp8_linear(a3, w.up, epilogue="gelu_mx")
    return h2, _project(inter, w.down, adapters.down, ids, packed)


def packed_dit_forward(blocks, h: torch.Tensor, temb: torch.Tensor, packed: PackedRequests, positions: torch.Tensor, crosses,
                       eps: float = 1e-6, adapters=None, adapter_ids: torch.Tensor | None = None,
                       tables: torch.Tensor | None = None) -> torch.Tensor:
    """The block loop of one DiT forward over a packed batch.

    ``h`` bf16 ``[rows, dim]``; ``temb`` ``[R, 6, dim]``, one per request; ``positions`` int32 ``[rows, 3]``
    (:meth:`PackedRequests.grid_positions`); ``crosses``: per block, per request the cross-attention's K/V
    (:func:`.block.project_cross_kv` of the request's text). ``adapters``: per block a :class:`BlockAdapters` (or None);
    ``adapter_ids`` int32 ``[R]``: the adapter of each request, -1 for none. Returns bf16 ``[rows, dim]``; rows of no request
    are zeros. The norm before a block is formed with the sum at the end of the one before it."""
    rows, dim = h.shape
    count = len(packed.lengths)
    if rows != packed.rows or tuple(positions.shape) != (rows, 3):
        raise ValueError(f"h {list(h.shape)} and positions {list(positions.shape)} do not fit {packed.rows} rows")
    if tuple(temb.shape) != (count, 6, dim) or len(crosses) != len(blocks) or any(len(c) != count for c in crosses):
        raise ValueError(f"temb and every block's crosses need one entry for each of {count} requests")
    if adapters and len(adapters) != len(blocks):
        raise ValueError(f"adapters: {len(adapters)} entries for {len(blocks)} blocks (None where a block has none)")
    if adapter_ids is not None and tuple(adapter_ids.shape) != (count,):
        raise ValueError(f"adapter_ids must be [{count}], got {list(adapter_ids.shape)}")
    if tables is None:
        tables = torch.stack([w.scale_shift_table for w in blocks])
    mods = packed_modulation(tables, temb)  # shift, 1 + scale, gate, c_shift, 1 + c_scale, c_gate of every request
    common = dict(eps=eps, post_norm="none", request_ids=packed.request_ids)
    ffn, gate = h, None
    h = None
    for i, w in enumerate(blocks):
        h, a1 = adaln_sandwich(ffn, h, mods[i][:, 1], mods[i][:, 0], gate=gate, quant="mx", **common)
        h, ffn = _sublayers(w, h, a1, mods[i], packed, positions, crosses[i], (adapters[i] if adapters else None) or BlockAdapters(),
                            adapter_ids, eps)
        gate = mods[i][:, 5]
    return adaln_sandwich(ffn, h, gate=gate, norm_type=None, **common)[0]


def packed_block_forward(w: BlockWeights, h: torch.Tensor, temb: torch.Tensor, packed: PackedRequests, positions: torch.Tensor,
                         crosses, eps: float = 1e-6, adapters: BlockAdapters | None = None,
                         adapter_ids: torch.Tensor | None = None) -> torch.Tensor:
    """One block over a packed batch (:func:`packed_dit_forward` with one block); ``crosses``: one :class:`.block.CrossKV` per request."""
    return packed_dit_forward([w], h, temb, packed, positions, [crosses], eps, None if adapters is None else [adapters], adapter_ids)
