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

The texts can be packed like the rows (:func:`project_packed_cross_kv`): the cross-attention of all requests is then one launch
(:func:`.packed_cross_attention`) in place of one each, and so is the self-attention of requests that are not long: 16 requests of 16 tokens
take 0.41 ms in place of 0.88, 8 of 390 1.28 and 1.56, 4 of 1560 2.13 and 2.17 (and their texts' keys and values 0.43 ms a
block in place of 0.77 for 16 texts of 512 tokens). A projection whose weight is an :class:`.FP8BlockWeight` runs as
:func:`.fp8_block_linear` on bf16 rows in place of MX codes.

The reference serves one request per forward; what it computes for one is what a request gets here, up to the
rounding of q and k between norm and rotation, which this path does not make.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import attention_ops as ops
from .adaln_kernels import adaln_quant_2d, adaln_sandwich
from .block import HEAD_DIM, BlockWeights, modulation
from .common_types import MXTensor
from .fp8_block import FP8BlockWeight, fp8_block_linear, quantize_fp8_blocks
from .lora import lora_add
from .packed_attention import packed_cross_attention
from .row_mx_kernels import mxfp8_linear


class _Requests(NamedTuple):
    lengths: tuple
    rows: int
    request_ids: torch.Tensor


class PackedRequests(_Requests):
    """Requests of ``lengths`` tokens, one behind the other in a batch of ``rows`` rows; the rows behind the last
    request belong to none. ``request_ids`` int32 ``[rows]``: each row's request, -1 for those. Beside these three fields
    ``offsets`` int32 ``[requests + 1]``, which packed texts need: each request's first row, and the row behind the last one's."""

    offsets: torch.Tensor | None = None

    def __new__(cls, lengths: tuple, rows: int, request_ids: torch.Tensor, offsets: torch.Tensor | None = None):
        self = super().__new__(cls, lengths, rows, request_ids)
        self.offsets = offsets
        return self

    def _replace(self, **fields) -> "PackedRequests":
        """A copy with other fields. Other ``lengths`` come without offsets unless theirs are given."""
        offsets = fields.pop("offsets", None if "lengths" in fields else self.offsets)
        made = super()._replace(**fields)
        made.offsets = offsets
        return made

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
        offsets = torch.tensor((0, *lengths), dtype=torch.int64).cumsum(0).to(torch.int32)
        return cls(lengths, rows, ids.to(device), offsets.to(device))

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


class PackedCrossKV(NamedTuple):
    """The cross-attention's keys (normalized) and values of packed texts: bf16 ``[rows, heads, 128]`` each, and the texts' offsets int32
    ``[requests + 1]``."""

    k: torch.Tensor
    v: torch.Tensor
    offsets: torch.Tensor


def project_packed_cross_kv(w: BlockWeights, context: torch.Tensor, text: PackedRequests, eps: float = 1e-6) -> PackedCrossKV:
    """:func:`.block.project_cross_kv` for the texts of all requests at once, their tokens one behind the other: ``context`` bf16 ``[rows,
    dim]``, ``text`` says which rows are whose (:meth:`PackedRequests.from_lengths` of the texts' lengths, 0 for an empty text)."""
    if context.dim() != 2 or context.shape[0] != text.rows or text.offsets is None:
        raise ValueError(f"context {list(context.shape)} does not fit {text.rows} packed rows with offsets")
    mx = blocks = None
    parts = []
    for weight in (w.k2, w.v2):
        if isinstance(weight, FP8BlockWeight):
            blocks = quantize_fp8_blocks(context) if blocks is None else blocks
            parts.append(fp8_block_linear(blocks, weight))
        else:
            mx = adaln_quant_2d(context.contiguous(), None, None, eps=0.0, norm_type="none", quant="mx") if mx is None else mx
            parts.append(mxfp8_linear(mx, weight))
    k, v = parts
    ops.qk_rmsnorm_rope_(k, w.norm_k2, eps=eps)
    heads = k.shape[1] // HEAD_DIM
    return PackedCrossKV(k.view(text.rows, heads, HEAD_DIM), v.view(text.rows, heads, HEAD_DIM), text.offsets)


# With packed texts, self-attention too is one launch for all requests, as long as none has more rows than this: few rows then
# share the chip instead of waiting for one another, while the constant-max kernel is the faster one on long rows. A block of dim 5120, all together
# against one by one, us: 16 x 16 tokens 411 / 593, 64 x 16 1004 / 1729, 8 x 390 1265 / 1423, 4 x 1560 2108 / 2148, one of 1560 707 / 694,
# 2 x 3600 2765 / 2778, 2 x 7800 6782 / 6275.
_TOGETHER = 3600


def _quant(weight) -> str:
    """The form in which a projection takes its input from the norm before it."""
    return "none" if isinstance(weight, FP8BlockWeight) else "mx"


def _linear(x, weight) -> torch.Tensor:
    return fp8_block_linear(x, weight) if isinstance(weight, FP8BlockWeight) else mxfp8_linear(x, weight)


def _up(x, w: BlockWeights):
    """GELU(up projection), as the down projection reads it."""
    if not isinstance(w.up, FP8BlockWeight):
        return mxfp8_linear(x, w.up, epilogue="gelu_mx" if _quant(w.down) == "mx" else "gelu_bf16")
    y = fp8_block_linear(x, w.up, activation="gelu")
    return y if _quant(w.down) == "none" else adaln_quant_2d(y, None, None, eps=0.0, norm_type="none", quant="mx")


def _project(x, weight, adapters: Adapters | None, ids, packed: PackedRequests, slices=None) -> torch.Tensor:
    y = _linear(x, weight)
    if adapters is None:
        return y
    if ids is None:
        raise ValueError("adapters need adapter_ids, one per request")
    return lora_add(y, x, adapters.a, adapters.b, ids, scales=adapters.scales, slices=slices, request_ids=packed.request_ids, out=y)


def _attend(packed: PackedRequests, dim: int, device, quant: str, one):
    """``one(i, first, end, out_mode, out)`` -> the request's output written to ``out``, for each request that has rows: all of them
    together as an :class:`MXTensor` or bf16 ``[rows, dim]``, the other rows zeros."""
    out = torch.zeros((packed.rows, dim), dtype=torch.uint8 if quant == "mx" else torch.bfloat16, device=device)
    scales = torch.zeros((packed.rows, dim // 32), dtype=torch.uint8, device=device) if quant == "mx" else None
    for i, (a, b) in enumerate(packed.spans()):
        if b > a:
            got = one(i, a, b, ops.OUT_MX if quant == "mx" else ops.OUT_TOKEN, out[a:b])
            if scales is not None:
                scales[a:b] = got.scales
    return out if scales is None else MXTensor(out.view(torch.float8_e4m3fn), scales)


def _attend_packed(q, k, v, q_offsets, k_offsets, scale: float, weight):
    """All requests' attention in one launch, as the projection ``weight`` reads it."""
    o = packed_cross_attention(q, k, v, q_offsets, k_offsets, scale=scale, quant=_quant(weight))
    return o if isinstance(o, MXTensor) else o.view(q.shape[0], -1)


def _sublayers(w: BlockWeights, h, a1: MXTensor, mod, packed, positions, crosses, adapters: BlockAdapters, ids, eps: float):
    """One block from its first normalized input to its FFN's output: ``(h2, ffn)``, whose gated sum is the block's result."""
    rows, dim = h.shape
    heads, scale = dim // HEAD_DIM, HEAD_DIM**-0.5
    sandwich = dict(eps=eps, post_norm="none", request_ids=packed.request_ids)
    texts = crosses if isinstance(crosses, PackedCrossKV) else None

    qkv = _project(a1, w.qkv, adapters.qkv, ids, packed, slices=(dim, dim, dim))
    q, k, v = (qkv[:, i * dim : (i + 1) * dim].view(rows, heads, HEAD_DIM) for i in range(3))
    together = texts is not None and max(packed.lengths) <= _TOGETHER
    *_, kmax = ops.qk_norm_rope_axes(q, k, positions, norm="rms_norm_across_heads", q_gamma=w.norm_q.view(-1), k_gamma=w.norm_k.view(-1), eps=eps,
                                     request_ids=packed.request_ids, requests=len(packed.lengths), want_max=not together, q_out=q, k_out=k)

    def self_attention(i, a, b, mode, out):
        vt, _ = ops.transpose_heads(v[a:b])
        return ops.attention_core(q[a:b], k[a:b], vt, kmax[i], scale, mode, out=out)

    if together:
        o = _attend_packed(q, k, v, packed.offsets, packed.offsets, scale, w.o)
    else:
        o = _attend(packed, dim, h.device, _quant(w.o), self_attention)
    y = _project(o, w.o, adapters.o, ids, packed)
    h1, a2 = adaln_sandwich(y, h, w.norm2_weight, w.norm2_bias, gate=mod[:, 2], quant=_quant(w.q2), **sandwich)

    # the attention request by request normalizes q as it loads it, from sums that the MX projection leaves
    fused = adapters.q2 is None and texts is None and not isinstance(w.q2, FP8BlockWeight)
    sumsq = torch.empty((rows, dim // 128), dtype=torch.float32, device=h.device) if fused else None
    if sumsq is not None:
        q2 = mxfp8_linear(a2, w.q2, row_sumsq=sumsq, sumsq_cols=dim).view(rows, heads, HEAD_DIM)
    else:
        q2 = _project(a2, w.q2, adapters.q2, ids, packed).view(rows, heads, HEAD_DIM)
        ops.qk_norm_rope_axes(q2, None, None, axes=(), norm="rms_norm_across_heads", q_gamma=w.norm_q2.view(-1), eps=eps,
                              request_ids=packed.request_ids, q_out=q2)

    def cross_attention(i, a, b, mode, out):
        prep = None if sumsq is None else ops.QPrep(sumsq[a:b], w.norm_q2, eps=eps)
        return ops.attention_core(q2[a:b], crosses[i].k, crosses[i].vt, crosses[i].kmax, scale, mode, out=out, q_prep=prep)

    if texts is None:
        o2 = _attend(packed, dim, h.device, _quant(w.o2), cross_attention)
    else:
        o2 = _attend_packed(q2, texts.k, texts.v, packed.offsets, texts.offsets, scale, w.o2)
    y = _project(o2, w.o2, adapters.o2, ids, packed)
    h2, a3 = adaln_sandwich(y, h1, mod[:, 4], mod[:, 3], quant=_quant(w.up), **sandwich)
    return h2, _project(_up(a3, w), w.down, adapters.down, ids, packed)


def packed_dit_forward(blocks, h: torch.Tensor, temb: torch.Tensor, packed: PackedRequests, positions: torch.Tensor, crosses,
                       eps: float = 1e-6, adapters=None, adapter_ids: torch.Tensor | None = None,
                       tables: torch.Tensor | None = None) -> torch.Tensor:
    """The block loop of one DiT forward over a packed batch.

    ``h`` bf16 ``[rows, dim]``; ``temb`` ``[R, 6, dim]``, one per request; ``positions`` int32 ``[rows, 3]``
    (:meth:`PackedRequests.grid_positions`); ``crosses``: per block, per request the cross-attention's K/V
    (:func:`.block.project_cross_kv` of the request's text), or per block a :class:`PackedCrossKV` of all requests' texts. Weights may be
    :class:`.FP8BlockWeight` in place of :class:`.MXWeight`, each for itself. ``adapters``: per block a :class:`BlockAdapters` (or None);
    ``adapter_ids`` int32 ``[R]``: the adapter of each request, -1 for none. Returns bf16 ``[rows, dim]``; rows of no request
    are zeros. The norm before a block is formed with the sum at the end of the one before it.

    Captured into a graph, a replay follows adapter ids, adapters, positions and the offsets of packed texts that were changed in place. Other
    row lengths need :class:`PackedCrossKV` in every block and no request above 3600 rows at the capture (each attention is then one launch, which
    reads its lengths on the GPU), and ``request_ids``, ``offsets`` and positions changed together; otherwise the rows of a request are those
    of ``packed.lengths`` at the capture."""
    rows, dim = h.shape
    count = len(packed.lengths)
    if rows != packed.rows or tuple(positions.shape) != (rows, 3):
        raise ValueError(f"h {list(h.shape)} and positions {list(positions.shape)} do not fit {packed.rows} rows")
    if len(crosses) == len(blocks) and any(isinstance(c, PackedCrossKV) for c in crosses):
        if packed.offsets is None:
            raise ValueError("packed texts need the requests' offsets (PackedRequests.from_lengths)")
        per_block = [c.offsets.shape[0] - 1 if isinstance(c, PackedCrossKV) else len(c) for c in crosses]
    else:
        per_block = [len(c) for c in crosses]
    if tuple(temb.shape) != (count, 6, dim) or len(crosses) != len(blocks) or any(n != count for n in per_block):
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
        h, a1 = adaln_sandwich(ffn, h, mods[i][:, 1], mods[i][:, 0], gate=gate, quant=_quant(w.qkv), **common)
        h, ffn = _sublayers(w, h, a1, mods[i], packed, positions, crosses[i], (adapters[i] if adapters else None) or BlockAdapters(),
                            adapter_ids, eps)
        gate = mods[i][:, 5]
    return adaln_sandwich(ffn, h, gate=gate, norm_type=None, **common)[0]


def packed_block_forward(w: BlockWeights, h: torch.Tensor, temb: torch.Tensor, packed: PackedRequests, positions: torch.Tensor,
                         crosses, eps: float = 1e-6, adapters: BlockAdapters | None = None,
                         adapter_ids: torch.Tensor | None = None) -> torch.Tensor:
    """One block over a packed batch (:func:`packed_dit_forward` with one block); ``crosses``: one :class:`.block.CrossKV` per request, or a
    :class:`PackedCrossKV`."""
    return packed_dit_forward([w], h, temb, packed, positions, [crosses], eps, None if adapters is None else [adapters], adapter_ids)
