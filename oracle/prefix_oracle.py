"""Definitions, in 64 bits, of attention behind a shared prefix and of cache eviction.

Each attention function returns the output and the two quantities that rounding
bounds need: ``mass`` = sum_j w_j |v_j| per output element and ``dot`` = the largest
sum_d |q_d k_jd| * scale of a query over the rows that it sees (0 where it sees none).
"""
from __future__ import annotations

import torch


def _attend(q, keys, values, scale):
    """q [G, D] over keys / values [N, D], all double: (out, mass, dot, weights)."""
    if keys.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, z.clone(), torch.zeros(q.shape[0], dtype=q.dtype), q.new_zeros(q.shape[0], 0)
    w = torch.softmax(q @ keys.T * scale, -1)
    return w @ values, w @ values.abs(), (q.abs() @ keys.abs().T * scale).amax(-1), w


def prefix_decode_attention(q, k, v, kv_len, pk, pv, plen, scale):
    """q [B, Hq, D]; k, v [B, Hk, S, D]; pk, pv [Hk, P, D] -> out, mass, dot [B, Hq], scores [B, Hk, S]."""
    b, hq, d = q.shape
    hk = k.shape[1]
    g = hq // hk
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    mass, dot = torch.zeros_like(out), torch.zeros(b, hq, dtype=torch.float64)
    scores = torch.zeros(b, hk, k.shape[2], dtype=torch.float64)
    q, k, v, pk, pv = (x.detach().cpu().double() for x in (q, k, v, pk, pv))
    for i in range(b):
        n = int(kv_len[i])
        for h in range(hk):
            a = slice(h * g, (h + 1) * g)
            out[i, a], mass[i, a], dot[i, a], w = _attend(
                q[i, a], torch.cat([pk[h, :plen], k[i, h, :n]]), torch.cat([pv[h, :plen], v[i, h, :n]]), scale)
            scores[i, h, :n] = w[:, plen:].sum(0)
    return out, mass, dot, scores


def prefix_prefill_attention(q, k, v, kv_len, q_len, pk, pv, plen, scale):
    """q [B, T, Hq, D] -> out, mass, dot [B, T, Hq]; token i sees own rows up to kv_len - q_len + i."""
    b, t, hq, d = q.shape
    hk = k.shape[1]
    g = hq // hk
    out = torch.zeros(b, t, hq, d, dtype=torch.float64)
    mass, dot = torch.zeros_like(out), torch.zeros(b, t, hq, dtype=torch.float64)
    q, k, v, pk, pv = (x.detach().cpu().double() for x in (q, k, v, pk, pv))
    for i in range(b):
        n, m = int(kv_len[i]), int(q_len[i])
        for j in range(m):
            last = n - m + j + 1
            for h in range(hk):
                a = slice(h * g, (h + 1) * g)
                out[i, j, a], mass[i, j, a], dot[i, j, a], _ = _attend(
                    q[i, j, a], torch.cat([pk[h, :plen], k[i, h, :last]]), torch.cat([pv[h, :plen], v[i, h, :last]]),
                    scale)
    return out, mass, dot


def evict(scores, n: int, budget: int, recent: int, protect: int) -> list[int]:
    """The kept slots, ascending, of one stream and KV head (scores: a list of floats)."""
    if n <= budget:
        return list(range(n))
    low = float("-inf")

    def order(j):
        s = scores[j]
        return (1, 0.0, j) if s != s else (0, -max(s, low), j)       # NaN after every number

    middle = sorted(range(protect, n - recent), key=order)[:budget - protect - recent]
    return list(range(protect)) + sorted(middle) + list(range(n - recent, n))
