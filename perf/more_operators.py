"""Measured cases of the operators on the text side of packed batches: the requests of a batch have prompts of unequal
lengths, and the rows of all of them lie one behind the other, without padding between them.

``cross``  attention of the rows of each request over the keys and values of its own text, all requests in one call
``text``   self-attention of a text encoder over packed prompts, with a learned relative position bias by buckets
``fp8``    product with a weight held in 8-bit floating point with one fp32 scale for each block of 128 x 128, the
           activation with one for each 128 of a row

The sizes are those of the Wan2.2-A14B block (dim 5120, 40 heads x 128, FFN 13824, 512 text tokens) at its token counts (a
latent frame at 480 x 832: 1560, short clips: 7800, 81 frames: 32760) and generic ones of a text encoder (64 heads x 64).

``own`` selects the package's kernels; otherwise ``run`` is the plain 32-bit form in torch.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
BLOCK = 128


def _pkg():
    import __graft_entry__

    return __graft_entry__.load_package()


# ---------------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------------
def listed():
    wan = {"q_heads": 40, "k_heads": 40, "head_dim": 128}
    enc = {"heads": 64, "head_dim": 64, "buckets": 32, "max_distance": 128}
    return [
        # a handful of rows (a warm-up or a preview patch) over a full prompt: only latency counts
        {"name": "cross_16", "kind": "cross", "tokens": 16, "pad": 0, "requests": 1, "text": 512, **wan},
        # three small pictures in one batch with room behind the last, prompts of unequal lengths
        {"name": "cross_1560", "kind": "cross", "tokens": 1560, "pad": 104, "requests": 3, "text": 300, **wan},
        # grouped key heads, text and picture tokens as context; the last request has no text
        {"name": "cross_gqa_7799", "kind": "cross", "tokens": 7799, "pad": 9, "requests": 5, "text": 769, "q_heads": 32,
         "k_heads": 4, "head_dim": 64},
        # two clips packed to the length of 81 frames at 480p
        {"name": "cross_32760", "kind": "cross", "tokens": 32760, "pad": 0, "requests": 2, "text": 512, **wan},
        # one short prompt through the encoder: latency
        {"name": "text_12", "kind": "text", "tokens": 12, "pad": 0, "requests": 1, "longest": 12, "table": "fp32", **enc},
        # the prompts and negative prompts of eight requests
        {"name": "text_2600", "kind": "text", "tokens": 2600, "pad": 24, "requests": 16, "longest": 512, "table": "bf16", **enc},
        # a few long descriptions
        {"name": "text_6001", "kind": "text", "tokens": 6001, "pad": 0, "requests": 4, "longest": 2048, "table": "fp32", **enc},
        # one row of a timestep or pooled text embedding: what the weight costs to read
        {"name": "fp8_1", "kind": "fp8", "tokens": 1, "k": 5120, "n": 5120, "x": "bf16", "activation": "none"},
        # the prompts of a small batch, widths that end inside a block
        {"name": "fp8_333", "kind": "fp8", "tokens": 333, "k": 4112, "n": 5096, "x": "bf16", "activation": "none"},
        # the FFN's up projection of one latent frame
        {"name": "fp8_up_1560", "kind": "fp8", "tokens": 1560, "k": 5120, "n": 13824, "x": "bf16", "activation": "gelu"},
        # the FFN's down projection of short clips
        {"name": "fp8_down_7799", "kind": "fp8", "tokens": 7799, "k": 13824, "n": 5120, "x": "bf16", "activation": "none"},
        # the fused QKV projection at 81 frames, the activation quantized before
        {"name": "fp8_qkv_32760", "kind": "fp8", "tokens": 32760, "k": 5120, "n": 15360, "x": "fp8", "activation": "none"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Token counts, lengths and widths over the logarithm of their ranges, any number of requests, every type."""
    kind = rng.choice(["cross", "text", "fp8"])
    if kind == "cross":
        head_dim = rng.choice([64, 128, 128])
        k_heads = _log_int(rng, 1, 40)
        q_heads = k_heads * rng.randrange(1, max(40, k_heads) // k_heads + 1)
        tokens = _log_int(rng, 1, 32000)
        return {"kind": kind, "tokens": tokens, "pad": rng.choice([0, rng.randrange(200)]),
                "requests": min(tokens, _log_int(rng, 1, 64)), "text": _log_int(rng, 1, 512 if tokens > 8000 else 2000),
                "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim}
    if kind == "text":
        requests = _log_int(rng, 1, 32)
        longest = _log_int(rng, 1, 2048 if requests <= 4 else 512)
        # between one long prompt with short ones beside it and all of them long
        tokens = longest + sum(rng.randint(1, longest) for _ in range(requests - 1))
        return {"kind": kind, "tokens": tokens, "pad": rng.choice([0, rng.randrange(100)]), "requests": requests,
                "longest": longest, "table": rng.choice(["fp32", "bf16"]), "heads": _log_int(rng, 4, 64),
                "head_dim": rng.choice([64, 64, 128]), "buckets": rng.choice([32, 32, 64, 20]),
                "max_distance": rng.choice([128, 128, 250, 64])}
    tokens, k, n = _log_int(rng, 1, 32000), 16 * _log_int(rng, 4, 864), 8 * _log_int(rng, 8, 1920)
    tokens = max(1, min(tokens, int(2.5e12 / (k * n)), int(5e8 / (k + n))))
    return {"kind": kind, "tokens": tokens, "k": k, "n": n, "x": rng.choice(["bf16", "bf16", "fp8"]),
            "activation": rng.choice(["none", "none", "gelu"])}


def _lengths(total, parts, longest, seed):
    """Unequal lengths of at least one that sum to ``total``, none above ``longest``: the case's own, whatever the inputs."""
    rng = random.Random(seed)
    lens = [1] * parts
    left = total - parts
    share = [rng.uniform(0.3, 1.7) for _ in range(parts)]
    for i, s in enumerate(share):
        lens[i] += min(longest - 1, int(left * s / sum(share)))
    rest = total - sum(lens)
    for i in range(parts):
        more = min(rest, longest - lens[i])
        lens[i] += more
        rest -= more
    return lens


def _plan(case):
    """The lengths of the requests: rows, and for ``cross`` the tokens of their texts."""
    if case["kind"] == "text":
        longest, others = case["longest"], case["requests"] - 1
        return [longest] + (_lengths(case["tokens"] - longest, others, longest, 11) if others else []), None
    rows = _lengths(case["tokens"], case["requests"], case["tokens"], 12)
    rng = random.Random(13)
    texts = [case["text"]] + [rng.randint(1, case["text"]) for _ in rows[1:]]
    if len(texts) >= 5:
        texts[-1] = 0  # an empty prompt
    return rows, texts


def work(case):
    """Each input read once, each output written once; keys and values of a text once."""
    if case["kind"] == "fp8":
        M, K, N = case["tokens"], case["k"], case["n"]
        kb, nb = -(-K // BLOCK), -(-N // BLOCK)
        x = 2 * M * K if case["x"] == "bf16" else M * K + 4 * M * kb
        return {"bytes": x + N * K + 4 * nb * kb + 4 * N + 2 * M * N, "flops": 2 * M * N * K}
    rows, texts = _plan(case)
    if case["kind"] == "cross":
        D, hq, hk = case["head_dim"], case["q_heads"], case["k_heads"]
        return {"bytes": 2 * D * (hq * (2 * case["tokens"] + case["pad"]) + 2 * hk * sum(texts)),
                "flops": 4 * D * hq * sum(a * b for a, b in zip(rows, texts))}
    D, H = case["head_dim"], case["heads"]
    return {"bytes": 2 * D * H * (4 * case["tokens"] + case["pad"]), "flops": 4 * D * H * sum(n * n for n in rows)}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _offsets(lens):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(*shape, std=1.0, dtype=F32):
        return (std * torch.randn(*shape, device=DEV, generator=g)).to(dtype)

    s = {"case": case}
    if case["kind"] == "fp8":
        M, K, N = case["tokens"], case["k"], case["n"]
        w = rnd(N, K, std=K**-0.5)
        codes, scales = _weight_blocks(w)
        del w
        s["w"], s["ws"], s["bias"] = codes, scales, rnd(N, std=0.1)
        # rows of unequal sizes, as behind a norm with a modulation
        x = (rnd(M, K) * (0.25 + 2 * torch.rand(M, 1, device=DEV, generator=g))).to(BF16)
        s["x"] = x if case["x"] == "bf16" else _row_blocks(x)
        return s
    rows, texts = _plan(case)
    s["rows"], s["texts"] = rows, texts
    s["q_offsets"] = _offsets(rows)
    if case["kind"] == "cross":
        D, hq, hk = case["head_dim"], case["q_heads"], case["k_heads"]
        s["q"] = rnd(case["tokens"] + case["pad"], hq, D, std=2.0, dtype=BF16)
        # keys and values are the column blocks of one projection
        kv = rnd(max(1, sum(texts)), 2 * hk, D, dtype=BF16)
        s["k"], s["v"] = kv[:, :hk], kv[:, hk:]
        s["k_offsets"] = _offsets(texts)
        return s
    D, H = case["head_dim"], case["heads"]
    # the encoder's scores are not scaled: its queries are small instead
    qkv = rnd(case["tokens"] + case["pad"], 3 * H, D)
    qkv[:, :H] *= D**-0.5
    qkv = qkv.to(BF16)
    s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H : 2 * H], qkv[:, 2 * H :]
    s["table"] = rnd(case["buckets"], H, std=1.5, dtype=F32 if case["table"] == "fp32" else BF16)
    return s


def _to_codes(y):
    return y.to(E4M3)


def _row_blocks(x):
    """bf16 ``[M, K]`` -> e4m3 codes and one fp32 scale per 128 of a row: the largest magnitude (at least 2^-100) / 448."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    y = torch.nn.functional.pad(x.to(F32), (0, kb * BLOCK - K)).view(M, kb, BLOCK)
    scale = y.abs().amax(-1).clamp_min(2.0**-100) / 448.0
    return _to_codes(y / scale[..., None]).view(M, kb * BLOCK)[:, :K].contiguous(), scale


def _weight_blocks(w):
    """fp32 ``[N, K]`` -> e4m3 codes and one fp32 scale per block of 128 x 128."""
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    y = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N)).view(nb, BLOCK, kb, BLOCK)
    scale = y.abs().amax((1, 3)).clamp_min(2.0**-100) / 448.0
    codes = _to_codes(y / scale[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)
    return codes[:N, :K].contiguous(), scale


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return {"cross": _cross, "text": _text, "fp8": _fp8}[s["case"]["kind"]](s)


def _softmax_values(scores, v):
    """softmax over the last dimension times ``v``; scores ``[H, a, b]``, v ``[H, b, D]``."""
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return (p / p.sum(-1, keepdim=True)) @ v


def _cross(s):
    case = s["case"]
    if own:
        return _pkg().packed_cross_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"])
    group = case["q_heads"] // case["k_heads"]
    out = torch.zeros(s["q"].shape, dtype=BF16, device=DEV)
    a = c = 0
    for n, m in zip(s["rows"], s["texts"]):
        if m:
            q = s["q"][a : a + n].to(F32).transpose(0, 1).contiguous()
            k = s["k"][c : c + m].to(F32).permute(1, 2, 0).repeat_interleave(group, 0)
            v = s["v"][c : c + m].to(F32).transpose(0, 1).repeat_interleave(group, 0)
            out[a : a + n] = _softmax_values(q @ k * case["head_dim"] ** -0.5, v).transpose(0, 1).to(BF16)
        a, c = a + n, c + m
    return out


def _bucket_starts(side, max_distance):
    """The smallest distance of each of ``side`` buckets: one distance each for the first half, the others
    logarithmic up to ``max_distance``. In whole numbers, since the borders of the logarithm lie on them."""
    first = side // 2
    starts = list(range(first))
    for b in range(first, side):
        n = first
        while (n**(side - first)) * first ** (b - first) < max_distance ** (b - first) * first ** (side - first):
            n += 1
        starts.append(n)
    return starts


def _text(s):
    case = s["case"]
    if own:
        return _pkg().relative_bias_attention(s["q"], s["k"], s["v"], s["table"], s["q_offsets"],
                                              max_distance=case["max_distance"])
    side = case["buckets"] // 2
    starts = torch.tensor(_bucket_starts(side, case["max_distance"])[1:], device=DEV)
    out = torch.zeros(s["q"].shape, dtype=BF16, device=DEV)
    a = 0
    for n in s["rows"]:
        q, k, v = (s[c][a : a + n].to(F32).transpose(0, 1).contiguous() for c in "qkv")
        i = torch.arange(n, device=DEV)
        far = i[None, :] - i[:, None]  # key - query
        bucket = torch.bucketize(far.abs(), starts, right=True) + side * (far > 0)
        bias = s["table"].to(F32)[bucket].permute(2, 0, 1)
        out[a : a + n] = _softmax_values(q @ k.transpose(1, 2).contiguous() + bias, v).transpose(0, 1).to(BF16)
        a += n
    return out


def _fp8(s):
    case = s["case"]
    if own:
        pkg = _pkg()
        x = s["x"] if case["x"] == "bf16" else pkg.FP8BlockTensor(*s["x"])
        return pkg.fp8_block_linear(x, pkg.FP8BlockWeight(s["w"], s["ws"], s["bias"]),
                                    activation=None if case["activation"] == "none" else case["activation"])
    codes, scales = _row_blocks(s["x"]) if case["x"] == "bf16" else s["x"]
    M, K = codes.shape
    N = s["w"].shape[0]
    x = codes.to(F32) * scales.repeat_interleave(BLOCK, 1)[:, :K]
    w = s["w"].to(F32) * s["ws"].repeat_interleave(BLOCK, 1)[:, :K].repeat_interleave(BLOCK, 0)[:N]
    y = x @ w.t() + s["bias"]
    if case["activation"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y.to(BF16)


# ---------------------------------------------------------------------------------------------
# The same in 64 bits, from the definition
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"cross": _exact_cross, "text": _exact_text, "fp8": _exact_fp8}[case["kind"]](s, case)


def _exact_cross(s, case):
    """Head by head: a row's weights are exp(scores) over their sum, the rows of an empty text zero."""
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    a = c = 0
    for n, m in zip(s["rows"], s["texts"]):
        for h in range(case["q_heads"] if m else 0):
            kh = h * case["k_heads"] // case["q_heads"]
            score = s["q"][a : a + n, h].to(F64) @ s["k"][c : c + m, kh].to(F64).t() / math.sqrt(case["head_dim"])
            out[a : a + n, h] = torch.softmax(score, 1) @ s["v"][c : c + m, kh].to(F64)
        a, c = a + n, c + m
    return out


def _exact_text(s, case):
    """Head by head, the bias as a vector over the distances -(n - 1) .. n - 1."""
    side, far = case["buckets"] // 2, case["max_distance"]
    first = side // 2

    def bucket(n):  # of a distance n >= 0
        if n < first:
            return n
        # the largest b with first * (far / first)^(b / steps) <= n, compared as whole numbers raised to the steps
        steps = side - first
        b = 0
        while b + 1 < steps and first**steps * far ** (b + 1) <= n**steps * first ** (b + 1):
            b += 1
        return first + b

    longest = max(s["rows"])
    index = [bucket(abs(d)) + (side if d > 0 else 0) for d in range(1 - longest, longest)]
    line = s["table"].to(F64)[torch.tensor(index, device=DEV)]
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    a = 0
    for n in s["rows"]:
        at = torch.arange(n, device=DEV)
        at = at[None, :] - at[:, None] + longest - 1
        for h in range(case["heads"]):
            q, k, v = (s[c][a : a + n, h].to(F64) for c in "qkv")
            out[a : a + n, h] = torch.softmax(q @ k.t() + line[at, h], 1) @ v
        a += n
    return out


def _exact_fp8(s, case):
    """Block of 128 after block of 128 along the sum, each with its scales."""
    codes, scales = s["x"] if case["x"] == "fp8" else _row_blocks(s["x"])
    M, K = codes.shape
    N = s["w"].shape[0]
    y = s["bias"].to(F64).expand(M, N).clone()
    for b in range(scales.shape[1]):
        at = slice(b * BLOCK, min((b + 1) * BLOCK, K))
        x = codes[:, at].to(F64) * scales[:, b, None].to(F64)
        for i in range(s["ws"].shape[0]):
            part = slice(i * BLOCK, min((i + 1) * BLOCK, N))
            y[:, part] += x @ (s["w"][part, at].to(F64).t() * s["ws"][i, b].to(F64))
    if case["activation"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y.pow(3))))
    return y
