"""The step form of the shared-prefix decode attention behind the launch that feeds it.

In a decode step that launch is ``fused_rope_kv_write``: it writes q and each stream's
newest row, and it lets the attention start before it has written either (its short-call
kernel releases its dependents first thing).  Here both are NaN until then, so an early
read shows; the result has to be the plain call's bit for bit.
"""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200 import fused_kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"

CASES = [
    # streams, heads, kv heads, dim, prefix rows, in use, slots, shortest and longest length
    (1, 16, 8, 64, 0, 0, 64, 1, 1),             # the newest row is the only one
    (1, 16, 8, 64, 251, 251, 300, 37, 37),
    (2, 16, 8, 64, 40, 33, 2500, 2200, 2500),   # in the last of many tiles
    (5, 16, 2, 128, 77, 70, 40, 1, 40),
    (16, 16, 8, 64, 640, 640, 400, 300, 400),
    (33, 8, 8, 64, 10, 1, 70, 1, 70),           # more streams than the writer's own early launch takes
    (64, 16, 8, 64, 100, 100, 300, 1, 300),     # 512 blocks: the rings of three stages
    (200, 4, 2, 64, 30, 30, 50, 1, 50),
    (130, 16, 2, 64, 2100, 2000, 33, 1, 33),    # behind a launch of the prefix's own
    (70, 8, 2, 128, 2000, 2000, 40, 1, 40),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_step_behind_the_launch_that_writes_q_and_the_newest_row(case, dtype):
    b, hq, hk, d, p, plen, s, low, high = case
    g = torch.Generator(device=DEV).manual_seed(7)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    k, v, pk, pv = normal(b, hk, s, d), normal(b, hk, s, d), normal(hk, p, d), normal(hk, p, d)
    n = torch.randint(low, high + 1, (b,), generator=g, device=DEV)
    slot, pos = (n - 1).view(b, 1), torch.randint(0, 5000, (b, 1), generator=g, device=DEV)
    inv_freq = (10000.0 ** (-torch.arange(d // 2, device=DEV) / (d // 2))).float()
    used = torch.tensor([plen], device=DEV) if p else None
    prefix = (pk, pv) if p else (None, None)
    rows, streams = torch.arange(b, device=DEV), slot.view(-1)
    q_out = torch.empty(b, 1, hq, d, dtype=dtype, device=DEV)
    scores = torch.rand(b, hk, s, generator=g, device=DEV)
    qkv = torch.empty(b, 1, (hq + 2 * hk) * d, dtype=dtype, device=DEV)
    q, kn, vn = qkv.split([hq * d, hk * d, hk * d], dim=-1)
    kept = scores.clone()

    def step(prefix_final):
        K.fused_rope_kv_write(q.view(b, 1, hq, d), kn.view(b, 1, hk, d), vn.view(b, 1, hk, d), inv_freq, pos, k, v, slot,
                              q_out=q_out)
        return K.prefix_decode_attention(q_out, k, v, n, *prefix, used, scores=scores, prefix_final=prefix_final)

    def unwritten():
        q_out.fill_(float("nan"))
        k[rows, :, streams] = float("nan")
        v[rows, :, streams] = float("nan")
        scores.copy_(kept)

    qkv.copy_(normal(*qkv.shape))
    step(True)                               # warm up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        from_graph = step(True)
    for _ in range(8):
        qkv.copy_(normal(*qkv.shape))
        results = []
        for form in ("step", "graph"):
            unwritten()
            torch.cuda.synchronize()
            if form == "step":
                out = step(True)
            else:
                graph.replay()
                out = from_graph.clone()
            torch.cuda.synchronize()
            results.append((out, scores.clone()))
        scores.copy_(kept)
        want = K.prefix_decode_attention(q_out, k, v, n, *prefix, used, scores=scores)
        assert torch.isfinite(want).all()
        for out, sc in results:
            assert torch.equal(out, want) and torch.equal(sc, scores)
