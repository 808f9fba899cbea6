"""Workloads of the attention operators: rotary positions, the cache write that goes with them, attention for training and
attention over a key / value cache.

Every case runs in two forms on the same inputs: the framework's operators (``own`` true) and their plain form in elementary
torch operations.  ``exact`` evaluates the definitions once more in float64.

Shapes: the packed text decoder of this repository (32 heads of 64, half of each head rotated, caches of 1024 slots, prompts of
745 embeddings of which the first 730 are one image prefix), its ViT-Base stack (12 heads of 64 over 197 patches), and generic
grouped-query layers with heads of 128.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # q and k heads of a training batch, rotated as one tensor straight out of the joint projection, with the gradient
        {"name": "rotary train bf16", "op": "rotary", "type": "bf16", "batch": 4, "tokens": 2048, "heads": 64, "dim": 64, "rotary": 32,
         "interleaved": False, "stretch": 1.0, "start": 0},
        # a model in float32 with pairs of neighbours, its positions squeezed by 4 to reach 131072 tokens, a ragged token count
        {"name": "rotary far f32", "op": "rotary", "type": "f32", "batch": 2, "tokens": 745, "heads": 12, "dim": 64, "rotary": 64,
         "interleaved": True, "stretch": 4.0, "start": 130000},
        # one decode step of one sequence: latency
        {"name": "cache write step", "op": "write", "type": "f16", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 32, "dim": 64,
         "rotary": 32, "interleaved": False, "slots": 1024, "lo": 745, "hi": 745, "ragged": False},
        # a batch of prompts of different lengths, padded to the longest
        {"name": "cache write prompts", "op": "write", "type": "f16", "batch": 8, "tokens": 745, "heads": 32, "kv_heads": 32, "dim": 64,
         "rotary": 32, "interleaved": False, "slots": 1024, "lo": 0, "hi": 0, "ragged": True},
        # a small float32 layer: an image prefix, distance bias, shared heads, odd lengths
        {"name": "attention small f32", "op": "train", "type": "f32", "batch": 2, "tokens": 133, "heads": 4, "kv_heads": 2, "dim": 64,
         "causal": True, "cap": 0.0, "slopes": True, "prefix": 50, "documents": 0},
        # one layer of the ViT-Base stack at batch 128: every patch sees every patch
        {"name": "attention patches f16", "op": "train", "type": "f16", "batch": 128, "tokens": 197, "heads": 12, "kv_heads": 12, "dim": 64,
         "causal": False, "cap": 0.0, "slopes": False, "prefix": 0, "documents": 0},
        # one layer of the text decoder in training
        {"name": "attention causal bf16", "op": "train", "type": "bf16", "batch": 4, "tokens": 2048, "heads": 32, "kv_heads": 32, "dim": 64,
         "causal": True, "cap": 0.0, "slopes": False, "prefix": 0, "documents": 0},
        # documents packed into one long row, capped scores, grouped heads of 128
        {"name": "attention packed bf16", "op": "train", "type": "bf16", "batch": 1, "tokens": 8191, "heads": 16, "kv_heads": 4, "dim": 128,
         "causal": True, "cap": 50.0, "slopes": False, "prefix": 0, "documents": 7},
        # one decode step of one sequence over the prompt: latency
        {"name": "cached step", "op": "cached", "type": "f16", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 32, "dim": 64, "cap": 0.0,
         "slopes": False, "prefix": 730, "slots": 1024, "lo": 745, "hi": 745, "ragged": False},
        # one decode step of 256 sequences of different lengths
        {"name": "cached step batch", "op": "cached", "type": "f16", "batch": 256, "tokens": 1, "heads": 32, "kv_heads": 32, "dim": 64,
         "cap": 0.0, "slopes": False, "prefix": 0, "slots": 1024, "lo": 200, "hi": 1000, "ragged": False},
        # one decode step over long contexts, grouped heads of 128, capped scores
        {"name": "cached step long", "op": "cached", "type": "bf16", "batch": 4, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "cap": 30.0, "slopes": False, "prefix": 0, "slots": 32768, "lo": 20000, "hi": 32767, "ragged": False},
        # the prompts' own pass over the fresh cache: the image prefix sees itself whole, the text after it is causal
        {"name": "cached prompts", "op": "cached", "type": "f16", "batch": 8, "tokens": 745, "heads": 32, "kv_heads": 32, "dim": 64,
         "cap": 0.0, "slopes": False, "prefix": 730, "slots": 1024, "lo": 0, "hi": 0, "ragged": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "write", "train", "train", "cached", "cached"])
    kind = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    dim = rng.choice([32, 64, 64, 80, 96, 128])
    kv = rng.choice([1, 2, 4, 8, 12, 32])
    heads = kv * rng.choice([1, 1, 2, 4, 8] if kv <= 8 else [1])
    if op == "rotary":
        tokens = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(64, (1 << 25) // (tokens * heads * dim))))
        part = rng.choice([dim, dim // 2])
        return {"op": op, "type": kind, "batch": batch, "tokens": tokens, "heads": heads, "dim": dim, "rotary": part,
                "interleaved": rng.random() < 0.5, "stretch": rng.choice([1.0, 1.0, 4.0]), "start": rng.choice([0, 0, rng.randrange(1, 100000)])}
    if op == "write":
        tokens = rng.choice([1, 1, _log(rng, 2, 1000)])
        batch = _log(rng, 1, max(1, min(256, 6000 // tokens)))
        before = rng.choice([0, rng.randrange(0, 1024)])
        return {"op": op, "type": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim,
                "rotary": rng.choice([dim, dim // 2]), "interleaved": rng.random() < 0.5, "slots": min(2048, before + tokens + rng.randrange(1, 25)),
                "lo": before // 2, "hi": before, "ragged": tokens > 1 and rng.random() < 0.5}
    if op == "train":
        tokens = _log(rng, 1, min(4096, int(math.sqrt(1.2e8 / heads))))
        batch = _log(rng, 1, max(1, min(64, int(1.2e8 / (tokens * max(tokens, 64) * heads)))))
        causal = rng.random() < 0.7
        return {"op": op, "type": kind if tokens <= 1500 else rng.choice(["f16", "bf16"]), "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim,
                "causal": causal, "cap": rng.choice([0.0, 0.0, 30.0]), "slopes": rng.random() < 0.3,
                "prefix": rng.randrange(1, tokens + 1) if causal and rng.random() < 0.3 else 0,
                "documents": rng.randrange(2, 9) if tokens > 64 and rng.random() < 0.3 else 0}
    tokens = rng.choice([1, 1, 1, rng.randrange(2, 9), _log(rng, 9, 800)])
    hi = _log(rng, 1, 32000) if tokens == 1 else _log(rng, 1, 4000)
    batch = _log(rng, 1, max(1, min(256, 260000 * 128 // ((hi + tokens) * kv * dim))))
    batch = max(1, min(batch, int(2.4e8 / (tokens * heads * (hi + tokens)))))
    return {"op": op, "type": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv, "dim": dim, "cap": rng.choice([0.0, 0.0, 30.0]),
            "slopes": rng.random() < 0.3, "prefix": rng.randrange(1, hi + 2) if rng.random() < 0.3 else 0, "slots": hi + tokens + rng.randrange(0, 40),
            "lo": hi // 2, "hi": hi, "ragged": tokens > 1 and rng.random() < 0.5}


# --------------------------------------------------------------------------------------- what a case fixes besides its sizes

def _before(case):
    """Tokens of each sequence that are in the cache before the call: spread over [lo, hi]."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    r = random.Random(b * 7919 + hi)
    return [hi if i == 0 else r.randint(lo, hi) for i in range(b)]


def _counts(case):
    """New tokens of each sequence: all of them, or a ragged batch padded to the longest."""
    b, t = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [t] * b
    r = random.Random(b * 104729 + t)
    return [t if i == 0 else r.randint((t + 1) // 2, t) for i in range(b)]


def _documents(case):
    """Document of each token of a packed row, the last few tokens padding (-1)."""
    t, n = case["tokens"], case["documents"]
    r = random.Random(t * 31 + n)
    pad = r.randint(1, max(1, t // 50))
    cuts = sorted(r.sample(range(1, t - pad), n - 1))
    ids, at = [], 0
    for i, c in enumerate(cuts + [t - pad]):
        ids += [i] * (c - at)
        at = c
    return ids + [-1] * pad


def _slopes(heads):
    """Geometric slopes of a distance bias: 2^(-8 (i + 1) / heads)."""
    return [2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)]


def _causal_pairs(t, prefix):
    """Pairs (query, key) of one row of t tokens: key <= query, or key < prefix."""
    p = min(prefix, t)
    return t * (t + 1) // 2 + p * (p - 1) // 2


def work(case):
    z, d = _SIZE[case["type"]], case["dim"]
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"] * case["heads"]
        # x and the gradient read, both rotated; the angles of the rotated part once
        return {"bytes": 4 * n * d * z + case["tokens"] * case["rotary"] * 4, "flops": 2 * n * case["rotary"] * 3}
    if case["op"] == "write":
        new = sum(_counts(case))
        n = case["heads"] + 2 * case["kv_heads"]
        return {"bytes": 2 * new * n * d * z + new * case["rotary"] * 4, "flops": 3 * new * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    if case["op"] == "train":
        b, t, hq, hk = case["batch"], case["tokens"], case["heads"], case["kv_heads"]
        if case["documents"]:
            ids = _documents(case)
            sizes = {}
            for x in ids:
                sizes[x] = sizes.get(x, 0) + 1
            sizes.pop(-1, None)
            pairs, at = 0, 0
            for x in sorted(sizes):
                n = sizes[x]
                pairs += _causal_pairs(n, max(0, case["prefix"] - at)) if case["causal"] else n * n
                at += n
        else:
            pairs = _causal_pairs(t, case["prefix"]) if case["causal"] else t * t
        # q, out, its gradient and dq; k, v, dk and dv.  Two products forward; the scores again and four products backward
        return {"bytes": b * t * d * z * (4 * hq + 4 * hk), "flops": 14 * b * hq * pairs * d}
    pairs = keys = 0
    for n, c in zip(_before(case), _counts(case)):
        keys += n + c
        p = min(case["prefix"], n + c)
        pairs += sum(max(n + i + 1, p) for i in range(c))
    new = sum(_counts(case))
    return {"bytes": z * d * (2 * new * case["heads"] + 2 * keys * case["kv_heads"]), "flops": 4 * case["heads"] * pairs * d}


# --------------------------------------------------------------------------------------------------------------- inputs

def _angles(case, rows):
    """[rows, rotary / 2] angles in float64: position / stretch times 10000^(-2 i / rotary)."""
    half = case["rotary"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") * 2.0 / case["rotary"])
    return torch.outer(torch.arange(rows, dtype=torch.float64, device="cuda") / case.get("stretch", 1.0), f)


def _table(case, rows):
    """The rotation table a program keeps: float32 [rows, rotary], cosines then sines."""
    a = _angles(case, rows)
    return torch.cat([a.cos(), a.sin()], dim=1).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = _TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(kind)

    b, t, h, d = case["batch"], case["tokens"], case["heads"], case["dim"]
    s = {"case": case}
    if case["op"] == "rotary":
        s["x"] = normal(b, t, h, d).requires_grad_(True)
        s["gy"] = normal(b, t, h, d, scale=0.02)
        s["positions"] = torch.arange(case["start"], case["start"] + t, device="cuda")
        s["table"] = _table(case, case["start"] + t)
        return s
    if case["op"] == "train":
        hk = case["kv_heads"]
        s["q"], s["k"], s["v"] = (normal(b, t, n, d).requires_grad_(True) for n in (h, hk, hk))
        s["go"] = normal(b, t, h, d, scale=0.02)
        s["documents"] = torch.tensor([_documents(case)] * b, device="cuda") if case["documents"] else None
        s["prefix"] = torch.full((b,), case["prefix"], device="cuda") if case["prefix"] else None
    else:
        hk, slots = case["kv_heads"], case["slots"]
        s["k_cache"], s["v_cache"] = normal(b, hk, slots, d), normal(b, hk, slots, d)
        s["cache_len"] = torch.tensor(_before(case), device="cuda")
        s["count"] = torch.tensor(_counts(case), device="cuda") if case["ragged"] else None
        if case["op"] == "write":
            s["qkv"] = normal(b, t, (h + 2 * hk) * d)
            s["table"] = _table(case, slots)
            return s
        s["q"] = normal(b, t, h, d)
        s["prefix"] = torch.full((b,), case["prefix"], device="cuda") if case["prefix"] else None
    s["slopes"] = torch.tensor(_slopes(h), device="cuda") if case["slopes"] else None
    return s


# ------------------------------------------------------------------------------------------------------------ plain form

def _rotate(x, cos, sin, interleaved):
    """x [..., dim] float32; cos, sin broadcast over [..., rotary / 2]; the rest of the head stays."""
    half = cos.shape[-1]
    part, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, c = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - c * sin, c * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, c = part[..., :half], part[..., half:]
        turned = torch.cat([a * cos - c * sin, c * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_rotary(s):
    c = s["case"]
    half = c["rotary"] // 2
    rows = s["table"][s["positions"]][None, :, None, :]
    cos, sin = rows[..., :half], rows[..., half:]
    y = _rotate(s["x"].detach().float(), cos, sin, c["interleaved"]).to(s["x"].dtype)
    gx = _rotate(s["gy"].float(), cos, -sin, c["interleaved"]).to(s["x"].dtype)
    return [y, gx]


def _plain_write(s):
    c = s["case"]
    b, t, h, hk, d, half = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"] // 2
    x = s["qkv"].view(b, t, h + 2 * hk, d)
    at = s["cache_len"][:, None] + torch.arange(t, device="cuda")                     # [b, t] position = cache slot
    rows = s["table"][at.clamp(max=c["slots"] - 1)][:, :, None, :]
    turned = _rotate(x[:, :, : h + hk].float(), rows[..., :half], rows[..., half:], c["interleaved"]).to(x.dtype)
    q = turned[:, :, :h]
    new = torch.ones((b, t), dtype=torch.bool, device="cuda")
    if s["count"] is not None:
        new = torch.arange(t, device="cuda") < s["count"][:, None]
        q = torch.where(new[:, :, None, None], q, torch.zeros((), dtype=q.dtype, device="cuda"))
    slot = torch.where(new, at, s["cache_len"][:, None]).clamp(max=c["slots"] - 1)
    seq = torch.arange(b, device="cuda")[:, None].expand(b, t)
    first = seq * t                                                                     # padding repeats the row's first token
    pick = torch.where(new, first + torch.arange(t, device="cuda"), first).reshape(-1)
    kn = turned[:, :, h:].reshape(b * t, hk, d)[pick]
    vn = x[:, :, h + hk:].reshape(b * t, hk, d)[pick]
    s["k_cache"].transpose(1, 2)[seq.reshape(-1), slot.reshape(-1)] = kn
    s["v_cache"].transpose(1, 2)[seq.reshape(-1), slot.reshape(-1)] = vn
    return [q.contiguous(), s["k_cache"], s["v_cache"]]


def _see(s, b, tq, tk):
    """[b, tq, tk] truth values (or of a shape that broadcasts to it): which keys each query sees; and its position [b or 1, tq]."""
    c = s["case"]
    key = torch.arange(tk, device="cuda")[None, None, :]
    if c["op"] == "cached":
        at = s["cache_len"][:, None] + torch.arange(tq, device="cuda")
        n = s["count"] if s["count"] is not None else torch.full((b,), tq, device="cuda")
        see = key <= at[:, :, None]
        if s["prefix"] is not None:
            see = see | (key < s["prefix"][:, None, None])
        see = see & (key < (s["cache_len"] + n)[:, None, None])
        return see & (torch.arange(tq, device="cuda")[None, :] < n[:, None])[:, :, None], at
    at = torch.arange(tq, device="cuda")[None, :]
    see = torch.ones((1, tq, tk), dtype=torch.bool, device="cuda")
    if c["causal"]:
        see = key <= at[:, :, None]
        if s["prefix"] is not None:
            see = see | (key < s["prefix"][:, None, None])
    if s["documents"] is not None:
        doc = s["documents"]
        see = see & (doc[:, :, None] == doc[:, None, :]) & (doc >= 0)[:, :, None]
    return see, at


def _plain_scores(s, q, k, b, hk, group, tq, tk, d):
    """q [b, hk, group, tq, d], k [b, hk, tk, d], float32: the weights of the softmax [b, hk, group, tq, tk] and the slope of the cap."""
    c = s["case"]
    x = torch.matmul(q.reshape(b, hk, group * tq, d), k.transpose(2, 3).contiguous()).view(b, hk, group, tq, tk).mul_(1.0 / math.sqrt(d))
    bend = None
    if c["cap"] > 0:
        th = torch.tanh(x.mul_(1.0 / c["cap"]))
        x = th * c["cap"]
        bend = 1.0 - th * th
    see, at = _see(s, b, tq, tk)
    if s["slopes"] is not None:
        away = (at[:, :, None] - torch.arange(tk, device="cuda")[None, None, :]).abs().float()
        x = x - s["slopes"].view(1, hk, group, 1, 1) * away[:, None, None]
    x = torch.where(see[:, None, None], x, torch.full((), -math.inf, device="cuda"))
    top = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros((), device="cuda"), top))
    total = p.sum(dim=-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones((), device="cuda"), total), bend


def _plain_train(s):
    c = s["case"]
    b, t, h, hk, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    n = h // hk
    q, go = (x.detach().float().view(b, t, hk, n, d).permute(0, 2, 3, 1, 4).contiguous() for x in (s["q"], s["go"]))
    k, v = (x.detach().float().transpose(1, 2).contiguous() for x in (s["k"], s["v"]))
    p, bend = _plain_scores(s, q, k, b, hk, n, t, t, d)
    p2, g2 = p.view(b, hk, n * t, t), go.view(b, hk, n * t, d)
    out = torch.matmul(p2, v)
    dv = torch.matmul(p2.transpose(2, 3).contiguous(), g2)
    ds = torch.matmul(g2, v.transpose(2, 3).contiguous())
    ds = p2 * (ds - (ds * p2).sum(dim=-1, keepdim=True)) * (1.0 / math.sqrt(d))
    if bend is not None:
        ds = ds * bend.view(b, hk, n * t, t)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q.view(b, hk, n * t, d))
    kind = s["q"].dtype

    def rows(x):
        return x.view(b, hk, n, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(kind)

    return [rows(out), rows(dq), dk.transpose(1, 2).to(kind).contiguous(), dv.transpose(1, 2).to(kind).contiguous()]


def _plain_cached(s):
    c = s["case"]
    b, t, h, hk, d, slots = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["slots"]
    n = h // hk
    q = s["q"].float().view(b, t, hk, n, d).permute(0, 2, 3, 1, 4).contiguous()
    p, _ = _plain_scores(s, q, s["k_cache"].float(), b, hk, n, t, slots, d)
    out = torch.matmul(p.view(b, hk, n * t, slots), s["v_cache"].float())
    return out.view(b, hk, n, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(s["q"].dtype)


_PLAIN = {"rotary": _plain_rotary, "write": _plain_write, "train": _plain_train, "cached": _plain_cached}


# ------------------------------------------------------------------------------------------------------------------ run

def run(state):
    if not own:
        with torch.no_grad():
            return _PLAIN[state["case"]["op"]](state)
    import ternary_vllm_amd as tv
    c = state["case"]
    if c["op"] == "rotary":
        y = tv.rotary(state["x"], state["positions"], state["table"], interleaved=c["interleaved"])
        (gx,) = torch.autograd.grad(y, state["x"], state["gy"])
        return [y, gx]
    if c["op"] == "write":
        q = tv.rotary_cache(state["qkv"], state["table"], state["k_cache"], state["v_cache"], state["cache_len"], c["heads"],
                            interleaved=c["interleaved"], count=state["count"])
        return [q, state["k_cache"], state["v_cache"]]
    if c["op"] == "train":
        out = tv.attention(state["q"], state["k"], state["v"], causal=c["causal"], softcap=c["cap"], slopes=state["slopes"],
                           prefix=state["prefix"], documents=state["documents"])
        return [out, *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["go"])]
    return tv.cached_attention(state["q"], state["k_cache"], state["v_cache"], state["cache_len"], softcap=c["cap"], slopes=state["slopes"],
                               prefix=state["prefix"], count=state["count"])


# ---------------------------------------------------------------------------------------------------------------- exact

def _turn64(x, angles, interleaved, back=False):
    """Each pair as a complex number, times exp(+-i angle), in float64."""
    half = angles.shape[-1]
    part = x[..., : 2 * half].double()
    pair = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) if interleaved else torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous())
    pair = pair * torch.polar(torch.ones_like(angles), -angles if back else angles)
    part = torch.stack([pair.real, pair.imag], dim=-1).flatten(-2) if interleaved else torch.cat([pair.real, pair.imag], dim=-1)
    return torch.cat([part, x[..., 2 * half:].double()], dim=-1)


def _attend64(q, k, v, allowed, away, cap, slopes):
    """The definition for one sequence and one query head: q [tq, d], k, v [tk, d], float64."""
    w = (q @ k.t().contiguous()) / math.sqrt(q.shape[1])
    if cap > 0:
        w = torch.tanh(w / cap) * cap
    if slopes is not None:
        w = w - slopes * away
    w = torch.softmax(w.masked_fill(~allowed, -1e300), dim=-1) * allowed
    return w @ v


def exact(case, seed):
    s = prepare(case, seed)
    b, t, h, d = case["batch"], case["tokens"], case["heads"], case["dim"]
    if case["op"] == "rotary":
        a = _angles(case, case["start"] + t)[case["start"]:][None, :, None, :]
        return [_turn64(s["x"].detach(), a, case["interleaved"]), _turn64(s["gy"], a, case["interleaved"], back=True)]
    hk = case["kv_heads"]
    n = h // hk
    if case["op"] == "write":
        a = _angles(case, case["slots"])
        x = s["qkv"].view(b, t, h + 2 * hk, d)
        q = torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda")
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for i, (at, c) in enumerate(zip(_before(case), _counts(case))):
            turned = _turn64(x[i, :c, : h + hk], a[at: at + c, None, :], case["interleaved"])
            q[i, :c] = turned[:, :h]
            kc[i, :, at: at + c] = turned[:, h:].transpose(0, 1)
            vc[i, :, at: at + c] = x[i, :c, h + hk:].double().transpose(0, 1)
        return [q, kc, vc]
    slopes = _slopes(h)
    if case["op"] == "train":
        if b * h * max(t, 64) ** 2 > 1.5e9 or b * h > 4096:
            return None
        leaves = [s[x].detach().double().requires_grad_(True) for x in ("q", "k", "v")]
        i = torch.arange(t, device="cuda")
        allowed = torch.ones((t, t), dtype=torch.bool, device="cuda")
        if case["causal"]:
            allowed = (i[None, :] <= i[:, None]) | (i[None, :] < case["prefix"])
        if case["documents"]:
            ids = torch.tensor(_documents(case), device="cuda")
            allowed = allowed & (ids[:, None] == ids[None, :]) & (ids[:, None] >= 0)
        away = (i[:, None] - i[None, :]).abs().double()
        out = torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda")
        for x in range(b):
            for j in range(h):
                q, k, v = leaves[0][x, :, j], leaves[1][x, :, j // n], leaves[2][x, :, j // n]
                o = _attend64(q, k, v, allowed, away, case["cap"], slopes[j] if case["slopes"] else None)
                out[x, :, j] = o.detach()
                o.backward(s["go"][x, :, j].double())
        return [out] + [x.grad for x in leaves]
    if b * h * t * (case["hi"] + t) > 1.5e9 or b * h > 10000:
        return None
    out = torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda")
    for x, (at, c) in enumerate(zip(_before(case), _counts(case))):
        i, j = torch.arange(c, device="cuda")[:, None] + at, torch.arange(at + c, device="cuda")[None, :]
        allowed, away = (j <= i) | (j < case["prefix"]), (i - j).abs().double()
        for y in range(h):
            k, v = s["k_cache"][x, y // n, : at + c].double(), s["v_cache"][x, y // n, : at + c].double()
            out[x, :c, y] = _attend64(s["q"][x, :c, y].double(), k, v, allowed, away, case["cap"], slopes[y] if case["slopes"] else None)
    return out
