"""A query row's attention does not depend on the rows computed beside it.

The tensor-core kernel keeps one query row per thread.  The rows of a warp are tokens of
one prompt, or, where the prefix is computed for the whole batch, different streams.  A
row whose logits are all NaN, or all -inf over its first tiles, has no finite maximum;
the rows next to it have to give what they give without it, bit for bit, and that is
held to the definition with the bounds of ``test_gpu_prefix_attention``.
"""
from __future__ import annotations

import math

import pytest
import torch

from kani_tts_b200 import fused_kernels as K
from oracle import prefix_oracle as O
from test_gpu_prefix_attention import check_out, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 64

# dtype, rise of the logits from one tile of 64 keys to the next in powers of two: past
# what the type holds as a weight relative to the first tile's maximum
RISES = [(torch.float16, 20), (torch.bfloat16, 20), (torch.bfloat16, 144)]


def rising_keys(p, rise, dtype, g):
    """Keys [1, p, D] whose logits with a query of ones are `rise` powers of two higher in
    each tile of 64 than in the one before, for four tiles, and again from there."""
    level = (torch.arange(p) // 64 % 4).float() * rise * math.log(2.0)
    k = level.view(1, p, 1) / (D - 1) + 0.01 * torch.randn(1, p, D, generator=g)
    k[..., 0] = 0.0
    return k.to(dtype)


def queries(n, dtype):
    """[n, D]: ones, a little more from row to row; dimension 0 is free."""
    q = (1.0 + torch.arange(n).view(n, 1) / 256).expand(n, D).clone()
    q[:, 0] = 0.0
    return q.to(dtype)


def odd_queries(q, pk, what, rows):
    """(queries with odd rows, keys): "nan": every logit of the rows is NaN; "-inf": those of
    each first tile of four are -inf (products past fp32's range), the others as before."""
    q, pk = q.clone(), pk.clone()
    if what == "nan":
        q[rows] = float("nan")
    else:
        q[rows, 0] = -1e30
        pk[:, torch.arange(pk.shape[1]) // 64 % 4 == 0, 0] = 1e30
    return q, pk


CASES = [(t, r, w) for t, r in RISES for w in ("nan", "-inf") if w == "nan" or t == torch.bfloat16]


@pytest.mark.parametrize("dtype,rise,what", CASES, ids=str)
def test_prompt_rows(dtype, rise, what):
    g = torch.Generator().manual_seed(91)
    t, p, odd = 70, 320, [3, 40, 69]
    q, pk = queries(t, dtype), rising_keys(p, rise, dtype, g)
    pv, k, v = make((1, p, D), g, dtype), make((1, 1, t, D), g, dtype, 0.01), make((1, 1, t, D), g, dtype)
    k[..., 0] = 0.0
    bad, pk = odd_queries(q, pk, what, odd)
    rest = [x.to(DEV) for x in (k, v, torch.tensor([t]), pk, pv)]
    clean = K.prefix_prefill_attention(q.view(1, t, 1, D).to(DEV), *rest, scale=1.0)[0, :, 0]
    out = K.prefix_prefill_attention(bad.view(1, t, 1, D).to(DEV), *rest, scale=1.0)[0, :, 0]
    ref, mass, dot = O.prefix_prefill_attention(q.view(1, t, 1, D), k, v, [t], [t], pk, pv, p, 1.0)
    check_out(clean, ref[0, :, 0], mass[0, :, 0], dot[0, :, 0], p + t, 6.0)
    live = [i for i in range(t) if i not in odd]
    assert torch.equal(out[live], clean[live])
    if what == "nan":
        assert out[odd].isnan().all()
    else:
        # the keys whose logits are -inf weigh nothing: the definition over the others (a
        # query of 0 in dimension 0, since theirs are 0 there)
        seen = torch.arange(p) // 64 % 4 != 0
        ref, mass, dot = O.prefix_prefill_attention(q.view(1, t, 1, D), k, v, [t], [t], pk[:, seen], pv[:, seen],
                                                    int(seen.sum()), 1.0)
        check_out(out[odd], ref[0, odd, 0], mass[0, odd, 0], dot[0, odd, 0], p + t, 6.0)


@pytest.mark.parametrize("dtype,rise,what", CASES, ids=str)
@pytest.mark.parametrize("b", [64, 300])
def test_streams_of_one_batch(dtype, rise, what, b):
    """The prefix computed once for the batch (128 MB of prefix rows times streams or more):
    a warp's rows are streams."""
    g = torch.Generator().manual_seed(92)
    p = -(-(128 << 20) // (b * D * 4)) // 64 * 64 + 64
    q, pk = queries(b, dtype), rising_keys(p, rise, dtype, g)
    pv, k, v = make((1, p, D), g, dtype), make((b, 1, 9, D), g, dtype, 0.01), make((b, 1, 9, D), g, dtype)
    k[..., 0] = 0.0
    odd = [5, 31, 33, b - 1]
    bad, pk = odd_queries(q, pk, what, odd)
    lens = [i % 10 for i in range(b)]
    rest = [x.to(DEV) for x in (k, v, torch.tensor(lens), pk, pv)]
    clean = K.prefix_decode_attention(q.view(b, 1, D).to(DEV), *rest, scale=1.0)[:, 0]
    out = K.prefix_decode_attention(bad.view(b, 1, D).to(DEV), *rest, scale=1.0)[:, 0]
    ref, mass, dot, _ = O.prefix_decode_attention(q.view(b, 1, D), k, v, lens, pk, pv, p, 1.0)
    check_out(clean, ref[:, 0], mass[:, 0], dot[:, 0], p + 9, 6.0)
    live = [i for i in range(b) if i not in odd]
    assert torch.equal(out[live], clean[live])
    if what == "nan":
        assert out[odd].isnan().all()
    else:
        seen = torch.arange(p) // 64 % 4 != 0
        ref, mass, dot, _ = O.prefix_decode_attention(q.view(b, 1, D), k, v, lens, pk[:, seen], pv[:, seen],
                                                      int(seen.sum()), 1.0)
        check_out(out[odd], ref[odd, 0], mass[odd, 0], dot[odd, 0], p + 9, 6.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(8, 1, 64), (6, 2, 128)])
def test_heads_of_one_group(hq, hk, d, dtype):
    """A NaN query head beside the others of its group: the group's heads are rows of one
    product, in the streams' own rows and in the prompt pass."""
    g = torch.Generator().manual_seed(93)
    b, p, s = 5, 130, 200
    q = make((b, hq, d), g, dtype)
    pk, pv = make((hk, p, d), g, dtype), make((hk, p, d), g, dtype)
    k, v = make((b, hk, s, d), g, dtype), make((b, hk, s, d), g, dtype)
    lens = [200, 0, 64, 17, 129]
    odd = [1, hq - 1]
    live = [h for h in range(hq) if h not in odd]
    bad = q.clone()
    bad[:, odd] = float("nan")
    rest = [x.to(DEV) for x in (k, v, torch.tensor(lens), pk, pv)]
    ref, mass, dot, add = O.prefix_decode_attention(q, k, v, lens, pk, pv, p, d ** -0.5)
    scores = torch.zeros(b, hk, s, device=DEV)
    out = K.prefix_decode_attention(bad.to(DEV), *rest, scores=scores)
    assert out[:, odd].isnan().all()
    check_out(out[:, live], ref[:, live], mass[:, live], dot[:, live], p + s, 6.0)
    t = 9
    q4 = make((b, t, hq, d), g, dtype)
    lens = [200, 9, 64, 17, 129]
    rest[2] = torch.tensor(lens, device=DEV)
    ref, mass, dot = O.prefix_prefill_attention(q4, k, v, lens, [t] * b, pk, pv, p, d ** -0.5)
    bad4 = q4.clone()
    bad4[:, :, odd] = float("nan")
    clean, out = (K.prefix_prefill_attention(x.to(DEV), *rest) for x in (q4, bad4))
    check_out(clean, ref, mass, dot, p + s, 6.0)
    assert out[:, :, odd].isnan().all()
    assert torch.equal(out[:, :, live], clean[:, :, live])
