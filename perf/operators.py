"""Measured cases of the operators for packed batches: several requests of different sizes in one call.

A server packs the tokens of its requests into one ``[rows, ...]`` tensor; ``request_ids`` names the
request of every row, and the rows behind the last request (padding up to a fixed capacity) carry -1
and come back as zeros. Three operators, each at the sizes of the Wan2.2-A14B block (dim 5120, 40
heads x 128, FFN 13824) and of its token counts: a latent frame at 480 x 832 (1560 tokens), one at
720 x 1280 (3600), short clips (7800), 81 frames (32760), 512 text tokens.

``rope``      Q/K RMSNorm and rotary positions on several axes, given per token
``sandwich``  norm behind a sub-layer, gate, residual scale and sum, norm and modulation before the next
``lora``      low-rank adapters of many requests beside a shared projection

``own`` selects the package's kernels; otherwise ``run`` is the plain 32-bit form in torch.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6
WIDTH, HEIGHT = 52, 30  # latent patches of a 480 x 832 frame: a frame's tokens in raster order


def _pkg():
    import __graft_entry__

    return __graft_entry__.load_package()


# ---------------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------------
def listed():
    wan = {"q_heads": 40, "k_heads": 40, "head_dim": 128, "axes": "44,42,42", "pairs": "interleaved",
           "norm": "rms_norm_across_heads"}
    return [
        # a handful of tokens (a warm-up or a preview patch): only latency counts
        {"name": "rope_16", "kind": "rope", "tokens": 16, "pad": 0, "requests": 1, **wan},
        # three small pictures in one batch with room behind the last
        {"name": "rope_1560", "kind": "rope", "tokens": 1560, "pad": 104, "requests": 3, **wan},
        # grouped key heads, a norm per head, rotate-half pairs over half of the head, as image models beside Wan have it
        {"name": "rope_gqa_7799", "kind": "rope", "tokens": 7799, "pad": 9, "requests": 5, "q_heads": 32, "k_heads": 4,
         "head_dim": 64, "axes": "8,12,12", "pairs": "halves", "norm": "rms_norm"},
        # two clips packed to the length of 81 frames at 480p
        {"name": "rope_32760", "kind": "rope", "tokens": 32760, "pad": 0, "requests": 2, **wan},
        # one token for each of seven requests: latency
        {"name": "sandwich_7", "kind": "sandwich", "tokens": 7, "pad": 0, "requests": 7, "hidden": 5120, "pre": "layer_norm",
         "quant": "none"},
        # three small pictures, with the codes that the MX projections read
        {"name": "sandwich_mx_1560", "kind": "sandwich", "tokens": 1560, "pad": 104, "requests": 3, "hidden": 5120,
         "pre": "layer_norm", "quant": "mx"},
        # short clips, an RMSNorm on both sides, a narrower model
        {"name": "sandwich_7799", "kind": "sandwich", "tokens": 7799, "pad": 1, "requests": 5, "hidden": 1536,
         "pre": "rms_norm", "quant": "none"},
        # two clips packed to the length of 81 frames at 480p
        {"name": "sandwich_32760", "kind": "sandwich", "tokens": 32760, "pad": 0, "requests": 2, "hidden": 5120,
         "pre": "layer_norm", "quant": "none"},
        # sixteen requests of one token, eight adapters: what an adapter's weights cost to read
        {"name": "lora_16", "kind": "lora", "tokens": 16, "pad": 0, "requests": 16, "adapters": 8, "rank": 16, "k": 5120,
         "slices": "5120", "x": "bf16"},
        # the text context of eight requests at the cross-attention's projections
        {"name": "lora_text_4096", "kind": "lora", "tokens": 4096, "pad": 0, "requests": 8, "adapters": 8, "rank": 32, "k": 5120,
         "slices": "5120", "x": "mx"},
        # the fused QKV projection of short clips, each part with its own adapter
        {"name": "lora_qkv_7799", "kind": "lora", "tokens": 7799, "pad": 9, "requests": 5, "adapters": 4, "rank": 64, "k": 5120,
         "slices": "5120,5120,5120", "x": "mx"},
        # the FFN's down projection at 81 frames
        {"name": "lora_down_32760", "kind": "lora", "tokens": 32760, "pad": 0, "requests": 3, "adapters": 2, "rank": 128,
         "k": 13824, "slices": "5120", "x": "mx"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Token counts over the logarithm of the range, any number of requests, every type and layout."""
    kind = rng.choice(["rope", "sandwich", "lora"])
    tokens = _log_int(rng, 1, 30000)
    case = {"kind": kind, "tokens": tokens, "pad": rng.choice([0, rng.randrange(200)]),
            "requests": min(tokens, _log_int(rng, 1, 64))}
    if kind == "rope":
        head_dim = rng.choice([64, 128, 128, 256])
        k_heads = rng.randrange(1, 5120 // head_dim + 1)
        q_heads = k_heads * rng.randrange(1, 5120 // head_dim // k_heads + 1)
        half = head_dim // 2
        axes = rng.choice([[half // 2, half // 4, half // 4], [half, half // 2, half // 2], [head_dim],
                           [head_dim - 4 * (head_dim // 6), 2 * (head_dim // 6), 2 * (head_dim // 6)], [half, half]])
        case.update(q_heads=q_heads, k_heads=k_heads, head_dim=head_dim, axes=",".join(map(str, axes)),
                    pairs=rng.choice(["interleaved", "halves"]),
                    norm=rng.choice(["none", "rms_norm", "rms_norm_across_heads"]))
    elif kind == "sandwich":
        case.update(hidden=32 * _log_int(rng, 8, 160), pre=rng.choice(["layer_norm", "rms_norm"]),
                    quant=rng.choice(["none", "none", "mx"]))
    else:
        slices = rng.choice(["5120", "1024", "1536,512,512", "5120,5120,5120", "13824", "2568"])
        case.update(adapters=_log_int(rng, 1, 12), rank=16 * _log_int(rng, 1, 8), k=32 * _log_int(rng, 8, 432), slices=slices,
                    x=rng.choice(["bf16", "mx"]))
        # no more than the down projection at 81 frames, and the plain form computes every adapter for every row
        K, N, r = case["k"], sum(_ints(slices)), case["rank"]
        cost = 2 * r * (len(_ints(slices)) * K + N)
        tokens = min(tokens, int(1.5e11 / cost), int(1.1e9 / (2 * K + 4 * N)), 32760 // case["adapters"])
        case.update(tokens=tokens, requests=min(case["requests"], tokens))
    return case


def work(case):
    """Each input read once, each output written once (an adapter's weights once if a request uses it)."""
    T, rows = case["tokens"], case["tokens"] + case["pad"]
    if case["kind"] == "rope":
        n = T * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        return {"bytes": 4 * n + 2 * (rows - T) * n // T + 12 * rows, "flops": 8 * n}
    if case["kind"] == "sandwich":
        H = case["hidden"]
        out = {"none": 2.0, "mx": 1.0 + 1 / 32}[case["quant"]]
        return {"bytes": T * H * (4 + 2 + out) + (rows - T) * H * (2 + out) + 12 * case["requests"] * H, "flops": 16 * T * H}
    widths = _ints(case["slices"])
    N, K, r, n = sum(widths), case["k"], case["rank"], min(case["adapters"], case["requests"])
    x = 2.0 if case["x"] == "bf16" else 1.0 + 1 / 32
    return {"bytes": T * K * x + 2 * T * N + 2 * rows * N + 2 * n * r * (len(widths) * K + N),
            "flops": 2 * T * r * (len(widths) * K + N)}


def _ints(text):
    return [int(v) for v in text.split(",")]


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _lengths(case, rng):
    """The requests' lengths: unequal ones of at least one token that sum to the case's tokens."""
    R, T = case["requests"], case["tokens"]
    share = [rng.uniform(0.3, 1.7) for _ in range(R)]
    lens = [1 + int((T - R) * s / sum(share)) for s in share]
    lens[-1] += T - sum(lens)
    return lens


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = _lengths(case, rng)
    R, rows = case["requests"], case["tokens"] + case["pad"]
    ids = torch.full((rows,), -1, dtype=torch.int32)
    ids[: case["tokens"]] = torch.repeat_interleave(torch.arange(R, dtype=torch.int32), torch.tensor(lens))
    s = {"case": case, "ids": ids.to(DEV)}

    def rnd(*shape, std=1.0, mean=0.0, dtype=F32):
        return (mean + std * torch.randn(*shape, device=DEV, generator=g)).to(dtype)

    if case["kind"] == "rope":
        hq, hk, d, axes = case["q_heads"], case["k_heads"], case["head_dim"], _ints(case["axes"])
        # q and k are column blocks of the projection's output, as a fused QKV projection leaves them
        slab = rnd(rows, (hq + 2 * hk) * d, dtype=BF16)
        s["q"] = slab[:, : hq * d].view(rows, hq, d)
        s["k"] = slab[:, hq * d : (hq + hk) * d].view(rows, hk, d)
        # every request's own grid, in raster order: frame, row, column
        starts = torch.tensor([0] + lens).cumsum(0)[:-1]
        local = torch.arange(rows) - torch.cat([torch.repeat_interleave(starts, torch.tensor(lens)),
                                                torch.zeros(case["pad"], dtype=torch.int64)])
        pos = torch.stack([local // (WIDTH * HEIGHT), local // WIDTH % HEIGHT, local % WIDTH], 1)
        s["pos"] = pos[:, 3 - len(axes) :].to(torch.int32).contiguous().to(DEV)
        s["axes"] = tuple(axes)
        # the axis and the frequency of every pair, which a program keeps
        s["axis"] = torch.tensor([a for a, dim in enumerate(axes) for _ in range(dim // 2)], device=DEV)
        s["freq"] = torch.tensor([10000.0 ** (-2 * j / dim) for dim in axes for j in range(dim // 2)], dtype=F64, device=DEV)
        n = {"none": 0, "rms_norm": 1, "rms_norm_across_heads": None}[case["norm"]]
        s["gq"], s["gk"] = (None if n == 0 else rnd((h if n is None else n) * d, std=0.1, mean=1.0) for h in (hq, hk))
    elif case["kind"] == "sandwich":
        H = case["hidden"]
        s["h"], s["res"] = rnd(rows, H, std=3.0, dtype=BF16), rnd(rows, H, dtype=BF16)
        s["w"] = rnd(H, std=0.1, mean=1.0)
        s["gate"], s["add"] = rnd(R, H), rnd(R, H, std=0.5)
        s["mul"] = rnd(R, H, std=0.5, mean=1.0)
        s["alpha"] = 0.75
    else:
        widths, K, r, n = _ints(case["slices"]), case["k"], case["rank"], case["adapters"]
        s["base"] = rnd(rows, sum(widths), dtype=BF16)
        x = rnd(rows, K, dtype=BF16)
        s["x"] = x if case["x"] == "bf16" else _mx(x)
        s["a"] = rnd(n, len(widths) * r, K, std=K**-0.5, dtype=BF16)
        s["b"] = rnd(n, sum(widths), r, std=0.5 * r**-0.5, dtype=BF16)
        s["scales"] = rnd(n, std=0.2, mean=1.0)
        # every adapter has a request while there are enough; the last of four or more requests has none
        which = [i % n for i in range(R)]
        if R >= 3 and R > n:
            which[-1] = -1
        s["adapter"] = torch.tensor(which, dtype=torch.int32, device=DEV)
        s["widths"] = tuple(widths)
        s["parts"] = torch.arange(len(widths), device=DEV)
        s["part"] = torch.repeat_interleave(s["parts"], torch.tensor(widths, device=DEV))  # of every column
        s["all"] = torch.arange(n, dtype=torch.int32, device=DEV)
    return s


def _mx(y):
    """bf16 ``[..., K]`` as e4m3 codes and one power-of-two scale (biased exponent) per 32 of them."""
    y = y.to(BF16)
    blocks = y.view(*y.shape[:-1], -1, 32)
    e = ((blocks.view(torch.int16).to(torch.int32) & 0x7FFF) >> 7).amax(-1)
    e = (e - 7).clamp_min(0)
    codes = torch.ldexp(blocks.float(), (127 - e)[..., None]).to(torch.float8_e4m3fn)
    return codes.view(y.shape), e.to(torch.uint8)


def _values(codes, scales, dtype):
    """What codes and scales stand for; exact in bf16 and wider."""
    shape = codes.shape
    f = torch.exp2(scales.to(F32) - 127.0).to(dtype)
    return (codes.view(*shape[:-1], -1, 32).to(dtype) * f[..., None]).view(shape)


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return {"rope": _rope, "sandwich": _sandwich, "lora": _lora}[s["case"]["kind"]](s)


def _rope(s):
    case = s["case"]
    if own:
        return _pkg().qk_norm_rope_axes(s["q"], s["k"], s["pos"], axes=s["axes"], theta=10000.0, rope_pairs=case["pairs"],
                                        norm=case["norm"], q_gamma=s["gq"], k_gamma=s["gk"], eps=EPS, request_ids=s["ids"])
    angle = s["pos"].to(F64)[:, s["axis"]] * s["freq"]
    cos, sin = angle.cos().to(F32)[:, None], angle.sin().to(F32)[:, None]
    return tuple(_rope_one(x, gamma, cos, sin, case, s["ids"]) for x, gamma in ((s["q"], s["gq"]), (s["k"], s["gk"])))


def _rope_one(x, gamma, cos, sin, case, ids):
    y = x.to(F32)
    if case["norm"] == "rms_norm":
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * gamma
    elif case["norm"] == "rms_norm_across_heads":
        y = y * torch.rsqrt(y.square().mean((1, 2), keepdim=True) + EPS) * gamma.view(x.shape[1], x.shape[2])
    n = 2 * cos.shape[-1]
    turn, rest = y[..., :n], y[..., n:]
    if case["pairs"] == "interleaved":
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = turn[..., : n // 2], turn[..., n // 2 :]
        turn = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    y = torch.cat([turn, rest], -1) if rest.shape[-1] else turn
    return torch.where(ids[:, None, None] >= 0, y, 0.0).to(BF16)


def _sandwich(s):
    case = s["case"]
    if own:
        r, y = _pkg().adaln_sandwich(s["h"], s["res"], s["mul"], s["add"], post_norm="rms_norm", post_weight=s["w"],
                                     gate=s["gate"], residual_scale=s["alpha"], norm_type=case["pre"], quant=case["quant"],
                                     eps=EPS, request_ids=s["ids"])
        return r, (_values(y.codes, y.scales, BF16) if case["quant"] == "mx" else y)
    row = s["ids"].clamp_min(0).long()
    live = (s["ids"] >= 0)[:, None]
    h = s["h"].to(F32)
    p = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"]
    r = torch.where(live, s["alpha"] * s["res"].to(F32) + s["gate"][row] * p, 0.0).to(BF16)
    y = r.to(F32)
    if case["pre"] == "layer_norm":
        y = y - y.mean(-1, keepdim=True)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    y = torch.where(live, y * s["mul"][row] + s["add"][row], 0.0).to(BF16)
    return r, (_values(*_mx(y), BF16) if case["quant"] == "mx" else y)


def _lora(s):
    case = s["case"]
    if own:
        pkg = _pkg()
        x = s["x"] if case["x"] == "bf16" else pkg.MXTensor(*s["x"])
        return pkg.lora_add(s["base"], x, s["a"], s["b"], s["adapter"], scales=s["scales"], slices=s["widths"],
                            request_ids=s["ids"])
    # every adapter's product for all rows, then only the row's own adapter kept
    n, r, parts = case["adapters"], case["rank"], len(s["widths"])
    x = s["x"].to(F32) if case["x"] == "bf16" else _values(*s["x"], F32)
    which = torch.where(s["ids"] >= 0, s["adapter"][s["ids"].clamp_min(0).long()], -1)
    mine = which[:, None] == s["all"]
    u = (x @ s["a"].to(F32).view(n * parts * r, -1).t()).view(-1, n, parts, r)
    u = torch.where(mine[:, :, None, None], u * s["scales"][:, None, None], 0.0)
    # B with each column's part spread out: zero against the other parts' ranks
    b = torch.where((s["part"][:, None] == s["parts"])[None, :, :, None], s["b"].to(F32)[:, :, None], 0.0)
    delta = u.reshape(-1, n * parts * r) @ b.permute(0, 2, 3, 1).reshape(n * parts * r, -1)
    y = s["base"].to(F32) + delta
    return torch.where(s["ids"][:, None] >= 0, y, 0.0).to(BF16)


# ---------------------------------------------------------------------------------------------
# The same in 64 bits, from the definition
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "sandwich": _exact_sandwich, "lora": _exact_lora}[case["kind"]](s, case)


def _exact_rope(s, case):
    """Each pair as a complex number, turned by exp(i angle)."""
    angles = []
    for a, dim in enumerate(s["axes"]):
        f = torch.tensor([10000.0 ** (-2 * j / dim) for j in range(dim // 2)], dtype=F64, device=DEV)
        angles.append(s["pos"][:, a : a + 1].to(F64) * f)
    angle = torch.cat(angles, 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    m = 2 * angle.shape[1]
    out = []
    for x, gamma in ((s["q"], s["gq"]), (s["k"], s["gk"])):
        y = x.to(F64)
        if case["norm"] != "none":
            over = (2,) if case["norm"] == "rms_norm" else (1, 2)
            size = math.prod(x.shape[d] for d in over)
            y = y / (y.pow(2).sum(over, keepdim=True) / size + EPS).sqrt()
            y = y * gamma.to(F64).reshape((-1, x.shape[2]))
        if case["pairs"] == "interleaved":
            z = torch.view_as_complex(y[..., :m].reshape(*y.shape[:-1], m // 2, 2)) * turn
            y[..., :m] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(y[..., : m // 2], y[..., m // 2 : m]) * turn
            y[..., : m // 2], y[..., m // 2 : m] = z.real, z.imag
        y[s["ids"] < 0] = 0
        out.append(y)
    return tuple(out)


def _exact_sandwich(s, case):
    """Request by request. The residual sum is held in bf16, and what follows starts from it."""
    r = torch.zeros(s["h"].shape, dtype=F64, device=DEV)
    y = torch.zeros_like(r)
    carried = torch.zeros_like(s["h"])
    H = case["hidden"]
    for i in range(case["requests"]):
        at = s["ids"] == i
        h = s["h"][at].to(F64)
        h = h / (h.pow(2).sum(1, keepdim=True) / H + EPS).sqrt() * s["w"].to(F64)
        r[at] = s["res"][at].to(F64) * s["alpha"] + h * s["gate"][i].to(F64)
        carried[at] = r[at].to(BF16)
        c = carried[at].to(F64)
        if case["pre"] == "layer_norm":
            c = c - c.sum(1, keepdim=True) / H
        c = c / (c.pow(2).sum(1, keepdim=True) / H + EPS).sqrt()
        y[at] = c * s["mul"][i].to(F64) + s["add"][i].to(F64)
    if case["quant"] == "mx":
        y = _values(*_mx(y.to(BF16)), F64)
    return r, y


def _exact_lora(s, case):
    """Adapter by adapter over the rows that use it, part by part."""
    x = s["x"].to(F64) if case["x"] == "bf16" else _values(*s["x"], F64)
    y = s["base"].to(F64)
    which = s["adapter"].tolist()
    for n in range(case["adapters"]):
        mine = torch.tensor([w == n for w in which], device=DEV)
        rows = ((s["ids"] >= 0) & mine[s["ids"].clamp_min(0).long()]).nonzero()[:, 0]
        at = 0
        for p, width in enumerate(s["widths"]):
            a = s["a"][n, p * case["rank"] : (p + 1) * case["rank"]].to(F64)
            b = s["b"][n, at : at + width].to(F64)
            y[rows, at : at + width] += (x[rows] @ a.t()) @ b.t() * s["scales"][n].to(F64)
            at += width
    y[s["ids"] < 0] = 0
    return y
