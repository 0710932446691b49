"""Eviction from the static caches on the GPU: which rows stay is exact, rows move bit for bit."""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200 import _lib
from kani_tts_b200 import fused_kernels as K
from oracle import prefix_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def inputs(b, hk, s, d, lens, dtype, seed, kind="random"):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(b, hk, s, d, generator=g).to(dtype), torch.randn(b, hk, s, d, generator=g).to(dtype)
    sc = torch.exp(2 * torch.randn(b, hk, s, generator=g))
    if kind == "ties":
        sc = torch.randint(0, 3, (b, hk, s), generator=g).float()
    elif kind == "equal":
        sc = torch.full((b, hk, s), 0.25)
    elif kind == "close":                                   # neighbours in the last bits
        sc = (torch.full((b, hk, s), 1.5).view(torch.int32) + torch.randint(0, 5, (b, hk, s), generator=g).int()).view(torch.float32)
    elif kind == "odd":                                     # zeros of both signs, infinities, NaN, negatives, subnormals
        pool = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), -1.0, 1e-42, -1e-42, 2.0])
        sc = pool[torch.randint(0, len(pool), (b, hk, s), generator=g)]
    for i, n in enumerate(lens):
        if kind != "odd":
            sc[i, :, n:] = 0
    return k, v, sc


CASES = [
    # batch, kv heads, slots, dim, lengths, budget, recent, protect
    (1, 8, 640, 64, [600], 512, 64, 40),
    (3, 2, 100, 64, [100, 50, 0], 50, 10, 5),
    (2, 1, 33, 128, [33, 32], 32, 0, 0),
    (2, 2, 257, 64, [257, 256], 1, 0, 0),
    (2, 2, 257, 64, [257, 256], 1, 1, 0),
    (2, 2, 257, 64, [257, 256], 1, 0, 1),
    (2, 3, 300, 64, [300, 299], 200, 200, 0),
    (2, 3, 300, 64, [300, 299], 200, 0, 200),
    (1, 2, 70, 64, [70], 0, 0, 0),
    (4, 2, 2049, 64, [2049, 1024, 1025, 2048], 1024, 256, 100),
    (1, 1, 9000, 64, [8999], 4321, 7, 1),
    (1, 1, 70000, 64, [69999], 30001, 1234, 77),
]


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "close", "odd"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_evict(case, dtype, kind):
    b, hk, s, d, lens, budget, recent, protect = case
    k, v, sc = inputs(b, hk, s, d, lens, dtype, 5, kind)
    n = torch.tensor(lens)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    kd, vd, sd, nd = (x.to(DEV) for x in (k, v, sc, n))
    so = budget + 3
    ko, vo = (torch.full((b, hk, so, d), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    sco = torch.full((b, hk, so), 7.0, device=DEV)
    kept = torch.zeros(b, hk, budget, dtype=torch.int32, device=DEV)
    new = K.evict_cache(kd, vd, sd, nd, budget, recent, protect, k_out=ko, v_out=vo, scores_out=sco, kept_out=kept,
                        err_flag=flag)
    assert torch.equal(new.cpu(), n.clamp_max(budget))
    assert torch.equal(kd.cpu(), k) and torch.equal(sd.cpu().view(torch.int32), sc.view(torch.int32))  # inputs unchanged
    new2 = K.evict_cache(kd, vd, sd, nd, budget, recent, protect, err_flag=flag)           # in place
    assert torch.equal(new2, new) and torch.equal(nd.cpu(), n)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    for i, m in enumerate(lens):
        for h in range(hk):
            at = O.evict(sc[i, h].tolist(), m, budget, recent, protect)
            c = len(at)
            assert kept[i, h].tolist() == at + [-1] * (budget - c)
            for got, old, tail in ((ko, k, 7.0), (vo, v, 7.0), (kd, k, None), (vd, v, None)):
                got = got[i, h].cpu()
                assert torch.equal(got[:c].view(bits), old[i, h][at].view(bits))
                # rows past the new length are left as they were
                assert torch.equal(got[c:].view(bits), (old[i, h][c:] if tail is None else torch.full_like(got[c:], tail)).view(bits))
            for got in (sco, sd):
                got = got[i, h].cpu()
                assert torch.equal(got[:c].view(torch.int32), sc[i, h][at].view(torch.int32))
                assert not got[c:].view(torch.int32).any()
    assert int(flag) == 0


def test_strided_caches_and_fp16():
    b, hk, s, d, lens = 3, 2, 90, 64, [90, 61, 20]
    k, v, sc = inputs(b, hk, s, d, lens, torch.float16, 9)
    both = torch.stack([k, v], 3).to(DEV)                                  # [B, Hk, S, 2, D]: K and V rows interleaved
    kd, vd = both[..., 0, :], both[..., 1, :]
    scd = torch.full((b, s, 2 * hk), 3.0, device=DEV).transpose(1, 2).contiguous()[:, ::2]
    scd.copy_(sc)
    n = torch.tensor(lens, device=DEV)
    out = torch.empty(3, dtype=torch.int64, device=DEV)
    assert K.evict_cache(kd, vd, scd, n, 40, 8, 2, len_out=out) is out
    for i, m in enumerate(lens):
        for h in range(hk):
            at = O.evict(sc[i, h].tolist(), m, 40, 8, 2)
            assert torch.equal(kd[i, h, :len(at)].cpu(), k[i, h][at]) and torch.equal(vd[i, h, :len(at)].cpu(), v[i, h][at])
            assert torch.equal(kd[i, h, len(at):].cpu(), k[i, h][len(at):])


def test_lengths_out_of_range_are_held_and_flagged():
    k, v, sc = inputs(2, 1, 30, 64, [30, 0], torch.bfloat16, 1)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    kd, vd, sd = (x.to(DEV) for x in (k, v, sc))
    new = K.evict_cache(kd, vd, sd, torch.tensor([31, -2], device=DEV), 10, 2, err_flag=flag)
    assert new.tolist() == [10, 0] and int(flag) == _lib.KANI_FLAG_SLOT_OOB
    at = O.evict(sc[0, 0].tolist(), 30, 10, 2, 0)
    assert torch.equal(kd[0, 0, :10].cpu(), k[0, 0][at]) and torch.equal(kd[1].cpu(), k[1])


def test_weights_then_eviction_then_attention_in_a_graph():
    """A cycle as a decode loop runs it: steps that add weights, an eviction, a step over
    what is left; captured and replayed, against the definitions."""
    g = torch.Generator().manual_seed(17)
    dt = torch.bfloat16
    b, hq, hk, d, p, s, budget = 4, 8, 4, 64, 150, 96, 48
    q = torch.randn(4, b, hq, d, generator=g).to(dt)
    k, v = torch.randn(b, hk, s, d, generator=g).to(dt), torch.randn(b, hk, s, d, generator=g).to(dt)
    pk, pv = torch.randn(hk, p, d, generator=g).to(dt), torch.randn(hk, p, d, generator=g).to(dt)
    lens = [96, 90, 48, 20]
    qd, kd, vd, pkd, pvd, n = (x.to(DEV) for x in (q, k, v, pk, pv, torch.tensor(lens)))
    scores = torch.zeros(b, hk, s, device=DEV)
    kept = torch.empty(b, hk, budget, dtype=torch.int32, device=DEV)

    def cycle():
        for i in range(3):
            K.prefix_decode_attention(qd[i], kd, vd, n, pkd, pvd, scores=scores)
        snap = scores.clone()
        n.copy_(K.evict_cache(kd, vd, scores, n, budget, 8, 4, kept_out=kept))
        return snap, K.prefix_decode_attention(qd[3], kd, vd, n, pkd, pvd)

    K.prefix_decode_attention(qd[0], kd, vd, n, pkd, pvd, scores=scores.clone())       # warm up
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        snap, out = cycle()
    gr.replay()
    torch.cuda.synchronize()
    assert n.tolist() == [48, 48, 48, 20]
    snap = snap.cpu()
    want = sum(O.prefix_decode_attention(q[i], k, v, lens, pk, pv, p, 0.125)[3] for i in range(3))
    torch.testing.assert_close(snap.double(), want, rtol=2.0 ** -15, atol=1e-12)       # see the attention tests' bounds
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    for i in range(b):
        for h in range(hk):
            at = O.evict(snap[i, h].tolist(), lens[i], budget, 8, 4)
            assert [x for x in kept[i, h].tolist() if x >= 0] == at
            k2[i, h, :len(at)], v2[i, h, :len(at)] = k[i, h][at], v[i, h][at]
            assert torch.equal(scores[i, h, :len(at)].cpu(), snap[i, h][at]) and not scores[i, h, len(at):].any()
    ref, mass, _, _ = O.prefix_decode_attention(q[3], k2, v2, n.tolist(), pk, pv, p, 0.125)
    assert ((out.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -14) * mass).all()


def test_refusals_on_the_device():
    dt = torch.bfloat16

    def z(*s, dtype=dt):
        return torch.zeros(*s, dtype=dtype, device=DEV)

    k, v, sc, n = z(2, 2, 16, 64), z(2, 2, 16, 64), z(2, 2, 16, dtype=torch.float32), torch.ones(2, dtype=torch.int64, device=DEV)
    ko, vo, so = z(2, 2, 8, 64), z(2, 2, 8, 64), z(2, 2, 8, dtype=torch.float32)

    def refused(exc, *a, **kw):
        with pytest.raises(exc):
            K.evict_cache(*a, **kw)

    refused(ValueError, k, v, sc, n, 17, 0)
    refused(ValueError, k, v, sc, n, 8, 9)
    refused(ValueError, k, v, sc, n, 8, 4, 5)
    refused(ValueError, k, v, sc, n, -1, 0)
    refused(ValueError, k, v, sc, n, 8, -1)
    refused(ValueError, k, k, sc, n, 8, 1)
    refused(ValueError, k, v[:, :, :8], sc, n, 8, 1)
    refused(TypeError, k, v.half(), sc, n, 8, 1)
    refused(ValueError, k, v, sc.half(), n, 8, 1)
    refused(ValueError, k, v, sc, n.int(), 8, 1)
    refused(ValueError, k, v, sc, n, 8, 1, k_out=ko)
    refused(ValueError, k, v, sc, n, 9, 1, k_out=ko, v_out=vo, scores_out=so)
    refused(ValueError, k, v, sc, n, 8, 1, k_out=k[:, :, :8], v_out=vo, scores_out=so)
    refused(ValueError, k, v, sc, n, 8, 1, k_out=ko, v_out=vo, scores_out=sc[:, :, :8])
    refused(ValueError, k, v, sc, n, 8, 1, k_out=ko, v_out=ko, scores_out=so)
    refused(ValueError, k, v, sc, n, 8, 1, len_out=n)
    refused(ValueError, k, v, sc, n, 8, 1, kept_out=z(2, 2, 8, dtype=torch.int64))
    refused(ValueError, k[:1].expand(2, 2, 16, 64), v[:1].expand(2, 2, 16, 64), sc, n, 8, 1)
    refused(ValueError, k.cpu(), v, sc, n, 8, 1)
    refused(ValueError, k, v, sc, n.cpu(), 8, 1)
    refused(_lib.KaniError, z(2, 2, 16, 68)[..., :64], z(2, 2, 16, 68)[..., :64], sc, n, 8, 1)
    assert K.evict_cache(k[:0], v[:0], sc[:0], n[:0], 8, 1).numel() == 0
