"""Cases of the shared-prefix attention and cache-eviction operators.

Many speech streams that read with one voice start from the same long prompt.  Its
keys and values are kept once (``prefix_k`` / ``prefix_v``); every stream has its own
static cache for the text and audio tokens after it.

* ``decode``: one query token per stream over the shared prefix and the stream's own
  valid rows, optionally adding each own row's attention weight to a running score.
* ``prefill``: the prompt tokens that follow the prefix, causal among themselves.
* ``evict``: a cache cut down to a budget of rows: the protected first rows, the most
  recent ones and those with the highest running score stay, in their order.

``listed()`` names the cases, ``prepare`` makes their inputs, ``run`` makes one pass
(the plain form in elementary torch operations, or the library's call where ``own``),
``work`` counts what a pass cannot do without and ``exact`` gives the same outputs in
64 bits from the definitions.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _decode(name, batch, heads, kv_heads, dim, prefix, low, high, slots, dtype="bf16", scores=False):
    c = {"op": "decode", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "prefix": prefix,
         "low": low, "high": high, "slots": slots, "dtype": dtype, "scores": scores}
    return {"name": name, **c} if name else c


def _prefill(name, batch, tokens, low, start, heads, kv_heads, dim, prefix, slots, dtype="bf16"):
    c = {"op": "prefill", "batch": batch, "tokens": tokens, "low": low, "start": start, "heads": heads,
         "kv_heads": kv_heads, "dim": dim, "prefix": prefix, "slots": slots, "dtype": dtype}
    return {"name": name, **c} if name else c


def _evict(name, batch, kv_heads, dim, low, high, slots, out_slots, budget, recent, protect, dtype="bf16"):
    c = {"op": "evict", "batch": batch, "kv_heads": kv_heads, "dim": dim, "low": low, "high": high, "slots": slots,
         "out_slots": out_slots, "budget": budget, "recent": recent, "protect": protect, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one stream a few tokens into its sentence: the latency of a single decode step
        _decode("decode, 1 stream", 1, 16, 8, 64, 251, 37, 37, 2048),
        # a serving batch of one voice, streams at different points of their sentences
        _decode("decode, 64 streams", 64, 16, 8, 64, 2048, 120, 1500, 2048),
        # a small batch whose caches are nearly full, weights kept for the next eviction
        _decode("decode, 16 streams, scores", 16, 16, 8, 64, 640, 700, 1024, 1024, scores=True),
        # the largest batch: a long voice prompt and caches of up to 2048 rows
        _decode("decode, 256 streams, fp16", 256, 16, 8, 64, 8192, 64, 2048, 2048, dtype="fp16"),
        # wide heads, eight query heads to a key head, odd sizes, a stream without rows of its own
        _decode("decode, odd, 8 heads a group", 13, 16, 2, 128, 777, 0, 1999, 2001, dtype="fp16", scores=True),
        # one short text after a voice prompt: time to the first token of a single request
        _prefill("prefill, 1 short text", 1, 23, 23, 0, 16, 8, 64, 300, 64),
        # a batch of texts of unequal lengths after one voice prompt
        _prefill("prefill, 64 texts", 64, 96, 17, 0, 16, 8, 64, 1024, 2048),
        # long documents after a long prefix
        _prefill("prefill, long", 4, 4096, 4000, 0, 16, 8, 64, 4096, 4096),
        # the second chunk of texts that are prefilled in pieces: wide heads, odd sizes
        _prefill("prefill, chunk, fp16", 3, 777, 700, 500, 16, 4, 128, 1500, 1300, dtype="fp16"),
        # one stream just past its budget
        _evict("evict, 1 stream", 1, 8, 64, 600, 600, 640, 768, 512, 64, 40),
        # a serving batch halves its caches
        _evict("evict, 64 streams", 64, 8, 64, 900, 2048, 2048, 1536, 1024, 256, 100),
        # long caches of wide rows in 32 bits, a quarter kept
        _evict("evict, long, fp32", 8, 2, 128, 12001, 16384, 16384, 5000, 4096, 511, 33, dtype="fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("decode", "prefill", "evict"))
    dtype = rng.choice(("bf16", "fp16"))
    heads, kv_heads, dim = rng.choice(((16, 8, 64), (8, 8, 64), (16, 4, 64), (16, 2, 64), (6, 2, 64), (2, 1, 64),
                                       (16, 4, 128), (8, 8, 128), (10, 2, 128), (8, 1, 128)))
    if op == "decode":
        batch = _log(rng, 1, 256)
        prefix = _log(rng, 1, 8192)
        slots = _log(rng, 16, 2048)
        high = rng.randint(1, slots)
        # no more key rows (own, and queries x prefix) than the largest listed case
        while batch * kv_heads * high * dim > 256 * 8 * 1056 * 64 or batch * heads * prefix * dim > 256 * 16 * 8192 * 64:
            batch = (batch + 1) // 2
        return _decode(None, batch, heads, kv_heads, dim, prefix, rng.randint(0, high), high, slots, dtype,
                       rng.random() < 0.5)
    if op == "prefill":
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, 4096)
        start = rng.choice((0, 0, _log(rng, 1, 2048)))
        prefix = _log(rng, 1, 4096)
        while batch * heads * tokens * (prefix + start + tokens / 2) * dim > 4 * 16 * 4096 * 6144 * 64:
            batch, tokens = (batch // 2, tokens) if batch > 1 else (1, tokens // 2)
        slots = start + tokens + rng.randint(0, 500)
        return _prefill(None, batch, tokens, rng.randint(1, tokens), start, heads, kv_heads, dim, prefix, slots, dtype)
    batch = _log(rng, 1, 64)
    slots = _log(rng, 40, 16384)
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    while batch * kv_heads * slots * dim * (2 if dtype == "fp32" else 1) > 64 * 8 * 1024 * 64:
        batch, slots = ((batch + 1) // 2, slots) if batch > 1 else (1, slots // 2)
    high = rng.randint(slots // 2, slots)
    budget = rng.randint(max(1, high // 8), high)
    recent = rng.randint(0, budget)
    return _evict(None, batch, kv_heads, dim, rng.randint(high // 2, high), high, slots, budget + rng.randint(0, 64),
                  budget, recent, rng.randint(0, budget - recent), dtype)


def _lengths(low, high, batch, g):
    """`batch` lengths spread evenly over low..high, in an order that the seed decides (a lone stream has `high`)."""
    if batch == 1:
        return torch.tensor([high], device="cuda")
    spread = low + (torch.arange(batch, device="cuda") * (high - low)) // (batch - 1)
    return spread[torch.randperm(batch, generator=g, device="cuda")]


def _length_list(low, high, batch):
    return [high] if batch == 1 else [low + (i * (high - low)) // (batch - 1) for i in range(batch)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(t)

    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    s = {"op": case["op"], "k": normal(b, hk, case["slots"], d), "v": normal(b, hk, case["slots"], d)}
    if case["op"] == "evict":
        s["kv_len"] = _lengths(case["low"], case["high"], b, g)
        # running attention weights are heavy-tailed: most rows get little, a few get much
        s["scores"] = torch.exp(2.0 * torch.randn(b, hk, case["slots"], generator=g, device="cuda"))
        s["scores"] *= torch.arange(case["slots"], device="cuda") < s["kv_len"][:, None, None]
        s["k_out"] = torch.zeros(b, hk, case["out_slots"], d, dtype=t, device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
        s["scores_out"] = torch.zeros(b, hk, case["out_slots"], device="cuda")
        s["kept"] = torch.zeros(b, hk, case["budget"], dtype=torch.int32, device="cuda")
        return {**s, "budget": case["budget"], "recent": case["recent"], "protect": case["protect"]}
    s["prefix_k"], s["prefix_v"] = normal(hk, case["prefix"], d), normal(hk, case["prefix"], d)
    if case["op"] == "decode":
        s["q"] = normal(b, case["heads"], d)
        s["kv_len"] = _lengths(case["low"], case["high"], b, g)
        s["scores"] = torch.zeros(b, hk, case["slots"], device="cuda") if case["scores"] else None
        return s
    s["q"] = normal(b, case["tokens"], case["heads"], d)
    s["q_len"] = _lengths(case["low"], case["tokens"], b, g)
    s["kv_len"] = s["q_len"] + case["start"]
    return s


@functools.lru_cache(maxsize=None)
def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "kani-tts-2-openai-server_b200"))
    from kani_tts_b200 import fused_kernels
    return fused_kernels


def run(s):
    if own:
        lib = _library()
        if s["op"] == "decode":
            out = lib.prefix_decode_attention(s["q"], s["k"], s["v"], s["kv_len"], s["prefix_k"], s["prefix_v"],
                                              scores=s["scores"])
            return out if s["scores"] is None else (out, s["scores"])
        if s["op"] == "prefill":
            return lib.prefix_prefill_attention(s["q"], s["k"], s["v"], s["kv_len"], s["prefix_k"], s["prefix_v"],
                                                q_len=s["q_len"])
        new_len = lib.evict_cache(s["k"], s["v"], s["scores"], s["kv_len"], s["budget"], s["recent"], s["protect"],
                                  k_out=s["k_out"], v_out=s["v_out"], scores_out=s["scores_out"], kept_out=s["kept"])
        return s["k_out"], s["v_out"], s["scores_out"], s["kept"], new_len
    return {"decode": _plain_decode, "prefill": _plain_prefill, "evict": _plain_evict}[s["op"]](s)


def _weights(logits, seen):
    """Softmax over the last dimension of what `seen` allows; a row that sees nothing gets zeros."""
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    return e / total.masked_fill(total == 0, 1.0)


def _plain_decode(s):
    q, pk, pv = s["q"], s["prefix_k"].float(), s["prefix_v"].float()
    b, hk, slots, d = s["k"].shape
    p = pk.shape[1]
    q32 = q.float().view(b, hk, -1, d) * d ** -0.5                                  # [B, Hk, G, D]
    of_prefix = torch.matmul(q32.transpose(0, 1).reshape(hk, -1, d), pk.transpose(1, 2))
    of_prefix = of_prefix.view(hk, b, -1, p).transpose(0, 1)                        # [B, Hk, G, P]
    logits = torch.cat([of_prefix, torch.matmul(q32, s["k"].float().transpose(2, 3))], -1)
    at = torch.arange(slots, device=q.device) < s["kv_len"][:, None]
    seen = torch.cat([at.new_ones(b, p), at], 1)[:, None, None]
    w = _weights(logits, seen)
    out = torch.matmul(w[..., :p].transpose(0, 1).reshape(hk, -1, p), pv).view(hk, b, -1, d).transpose(0, 1)
    out = out + torch.matmul(w[..., p:], s["v"].float())
    out = out.reshape(q.shape).to(q.dtype)
    if s["scores"] is None:
        return out
    s["scores"] += w[..., p:].sum(2)
    return out, s["scores"]


def _plain_prefill(s):
    q, pk, pv = s["q"], s["prefix_k"].float(), s["prefix_v"].float()
    b, tokens, heads, d = q.shape
    hk, slots = s["k"].shape[1:3]
    p, g = pk.shape[1], heads // hk
    q32 = q.float().view(b, tokens, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * tokens, d) * d ** -0.5
    logits = torch.cat([torch.matmul(q32, pk.transpose(1, 2)), torch.matmul(q32, s["k"].float().transpose(2, 3))], -1)
    i, j = torch.arange(tokens, device=q.device), torch.arange(slots, device=q.device)
    real = i < s["q_len"][:, None]                                                  # [B, T]
    last = (s["kv_len"] - s["q_len"])[:, None] + i                                  # the row that token i wrote
    seen = torch.cat([real[..., None].expand(b, tokens, p), real[..., None] & (j <= last[..., None])], -1)
    seen = seen[:, None, None].expand(b, 1, g, tokens, p + slots).reshape(b, 1, g * tokens, p + slots)
    w = _weights(logits, seen)
    out = torch.matmul(w[..., :p], pv) + torch.matmul(w[..., p:], s["v"].float())
    return out.view(b, hk, g, tokens, d).permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype)


def _plain_evict(s):
    scores, n = s["scores"], s["kv_len"][:, None, None]
    slots, out_slots = scores.shape[2], s["k_out"].shape[2]
    new_len = s["kv_len"].clamp_max(s["budget"])
    j = torch.arange(slots, device=scores.device)
    always = (j < s["protect"]) | (j >= n - s["recent"]) | (n <= s["budget"])
    rank = scores.masked_fill(always, math.inf).masked_fill(j >= n, -math.inf)
    order = rank.sort(dim=2, descending=True, stable=True).indices                  # ties: the lowest slot first
    place = torch.empty_like(order).scatter_(2, order, j.expand_as(order).contiguous())
    keep = place < new_len[:, None, None]
    # kept slots first, in their order
    kept = (~keep).to(torch.uint8).sort(dim=2, stable=True).indices[..., :s["budget"]]
    row = torch.arange(kept.shape[2], device=scores.device)
    valid = row < new_len[:, None, None]
    s["kept"].copy_(kept.masked_fill(~valid, -1))
    for new, old in ((s["k_out"], s["k"]), (s["v_out"], s["v"])):
        at = kept[..., None].expand(*kept.shape, old.shape[3])
        new[:, :, :kept.shape[2]] = torch.where(valid[..., None], old.gather(2, at), new[:, :, :kept.shape[2]])
    s["scores_out"].zero_()
    s["scores_out"][..., :kept.shape[2]] = scores.gather(2, kept).masked_fill(~valid, 0.0)
    return s["k_out"], s["v_out"], s["scores_out"], s["kept"], new_len


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    row = 2 * d * e                                                                 # one slot's key and value
    if case["op"] == "evict":
        lengths = _length_list(case["low"], case["high"], b)
        rows = sum(min(n, case["budget"]) for n in lengths)
        # scores of the valid rows in; kept rows in and out; the new scores and the kept slots out
        return {"bytes": hk * (4 * sum(lengths) + 2 * rows * row + b * 4 * (case["out_slots"] + case["budget"])) + 16 * b,
                "flops": 0}
    h = case["heads"]
    if case["op"] == "decode":
        own_rows = sum(_length_list(case["low"], case["high"], b))
        return {"bytes": hk * row * (own_rows + case["prefix"]) + 2 * b * h * d * e + 8 * b
                + (8 * hk * own_rows if case["scores"] else 0),
                "flops": 4 * h * d * (own_rows + b * case["prefix"])}
    lengths = _length_list(case["low"], case["tokens"], b)
    pairs = sum(n * (case["prefix"] + case["start"]) + n * (n + 1) // 2 for n in lengths)
    return {"bytes": hk * row * (case["prefix"] + sum(n + case["start"] for n in lengths))
            + h * d * e * (sum(lengths) + b * case["tokens"]) + 16 * b,
            "flops": 4 * h * d * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    b, hk, d = case["batch"], case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        kept = torch.full((b, hk, case["budget"]), -1, dtype=torch.int32)
        k_out, v_out = s["k_out"].cpu().double(), s["v_out"].cpu().double()
        scores_out = torch.zeros(b, hk, case["out_slots"], dtype=torch.float64)
        lengths, scores = s["kv_len"].tolist(), s["scores"].cpu()
        k, v = s["k"].cpu(), s["v"].cpu()
        for i, n in enumerate(lengths):
            for h in range(hk):
                if n <= case["budget"]:
                    stay = list(range(n))
                else:
                    first, last = case["protect"], n - case["recent"]
                    most = case["budget"] - case["protect"] - case["recent"]
                    value = scores[i, h].tolist()
                    best = sorted(range(first, last), key=lambda j: (-value[j], j))[:most]
                    stay = list(range(first)) + sorted(best) + list(range(last, n))
                at = torch.tensor(stay, dtype=torch.int64)
                kept[i, h, :len(stay)] = at.int()
                k_out[i, h, :len(stay)] = k[i, h, at].double()
                v_out[i, h, :len(stay)] = v[i, h, at].double()
                scores_out[i, h, :len(stay)] = scores[i, h, at].double()
        return k_out, v_out, scores_out, kept, s["kv_len"].clamp_max(case["budget"])

    g, p = case["heads"] // hk, case["prefix"]
    pk, pv = s["prefix_k"].double(), s["prefix_v"].double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    scores = torch.zeros(b, hk, case["slots"], dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(s["kv_len"][i])
        for h in range(hk):
            keys = torch.cat([pk[h], s["k"][i, h, :n].double()])
            values = torch.cat([pv[h], s["v"][i, h, :n].double()])
            if case["op"] == "decode":
                w = torch.softmax(s["q"][i, h * g:(h + 1) * g].double() @ keys.T / math.sqrt(d), -1)
                out[i, h * g:(h + 1) * g] = w @ values
                scores[i, h, :n] = w[:, p:].sum(0)
                continue
            m = int(s["q_len"][i])
            sees = p + n - m + 1 + torch.arange(m, device="cuda")                  # keys that token t sees
            hidden = torch.arange(p + n, device="cuda") >= sees[:, None]
            for a in range(h * g, (h + 1) * g):
                logits = (s["q"][i, :m, a].double() @ keys.T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
                out[i, :m, a] = torch.softmax(logits, -1) @ values
    return (out, scores) if case["op"] == "decode" and case["scores"] else out
