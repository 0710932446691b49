"""Attention behind a shared prefix on the GPU against its definition in 64 bits.

Bounds.  Inputs are exact.  A logit is an fp32 sum of D exact products, scaled once:
it is off by at most (D + 2) 2^-24 sum|q k| scale; its exponential's argument, at most
2 dot log2(e) in magnitude, is rounded to 2^-24 of it, twice, and the hardware's 2^x is
off by 2^-22 (the polynomial that replaces it for some weights by 2.7e-6 < 2^-18).  So
every weight, and their sum, is off by a factor within 1 +- r with
    r = (D + 2) 2^-24 dot + 8 dot 2^-24 + 2^-18 + N 2^-24
(the last term: sums over N rows), and the output by 2 r mass, mass = sum w |v|.  Weights
may be rounded to the storage type before they meet V: u mass more, u = eps / 2 of that
type.  The result is rounded once: u |out|.  fp16 adds half its smallest subnormal, 2^-25,
for the result and, for each weight below the normal range, 2^-25 relative to the largest
weight: N 2^-25 max|v|.
"""
from __future__ import annotations

import math

import pytest
import torch

from kani_tts_b200 import _lib
from kani_tts_b200 import fused_kernels as K
from oracle import prefix_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rel_bound(dot, d, n):
    return (d + 2) * 2.0 ** -24 * dot + 8 * dot * 2.0 ** -24 + 2.0 ** -18 + n * 2.0 ** -24


def check_out(got, ref, mass, dot, n, vmax):
    d = got.shape[-1]
    u = torch.finfo(got.dtype).eps / 2
    bound = u * ref.abs() + (u + 2 * rel_bound(dot, d, n))[..., None] * mass
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25 + n * 2.0 ** -25 * vmax
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    bad = err > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / bound.clamp_min(1e-30)).max()):.3g} bounds"


def make(shape, g, dtype, std=1.0):
    return (std * torch.randn(*shape, generator=g)).to(dtype)


def poison(t, lens):
    """NaN and infinities in the rows that nothing may read."""
    for i, n in enumerate(lens):
        t[i, :, n:] = float("nan")
        t[i, :, n + 1::2] = float("inf")
    return t


DECODE = [
    # batch, heads, kv heads, dim, prefix rows, prefix in use, slots, lengths
    (1, 16, 8, 64, 251, 251, 300, [37]),
    (1, 2, 1, 64, 0, 0, 1, [1]),
    (1, 2, 1, 64, 1, 1, 4, [0]),
    (2, 16, 8, 64, 130, 64, 70, [0, 70]),
    (3, 8, 8, 64, 64, 64, 65, [63, 64, 65]),
    (5, 8, 1, 128, 77, 70, 40, [0, 1, 16, 33, 40]),
    (4, 10, 2, 128, 200, 199, 260, [129, 0, 255, 260]),
    (7, 6, 2, 64, 513, 512, 129, [5, 0, 128, 127, 129, 1, 60]),
    (9, 14, 2, 64, 300, 300, 20, [20, 3, 0, 7, 1, 16, 17, 8, 15]),
    (40, 16, 4, 64, 700, 700, 90, [(i * 37) % 91 for i in range(40)]),
    (130, 2, 1, 64, 1025, 1000, 33, [(i * 7) % 34 for i in range(130)]),
    (3, 4, 2, 64, 33, 0, 2100, [2100, 2049, 0]),
    (2, 4, 4, 128, 9, 9, 1500, [1500, 1023]),
    (3, 8, 1, 64, 0, 0, 40000, [40000, 39999, 1]),          # logits in the workspace
    # from 128 MB of prefix rows times streams on: the prefix in a launch of its own
    (130, 16, 2, 64, 2100, 2000, 33, [(i * 7) % 34 for i in range(130)]),
    (70, 8, 2, 128, 2000, 2000, 40, [(i * 11) % 41 for i in range(70)]),
    (100, 14, 2, 64, 2700, 2689, 17, [(i * 5) % 18 for i in range(100)]),
    (8, 3, 1, 64, 70000, 69937, 200, [0, 1, 200, 64, 63, 130, 7, 0]),      # several partial results
    (300, 2, 1, 64, 1800, 0, 5, [i % 6 for i in range(300)]),              # a prefix of which nothing is used
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(map(str, c[:7])))
def test_decode(case, dtype):
    b, hq, hk, d, p, plen, s, lens = case
    g = torch.Generator().manual_seed(hash(case[:7]) % 10007)
    q, k, v = make((b, hq, d), g, dtype), make((b, hk, s, d), g, dtype), make((b, hk, s, d), g, dtype)
    pk, pv = make((hk, p, d), g, dtype), make((hk, p, d), g, dtype)
    start = torch.rand(b, hk, s, generator=g)
    ref, mass, dot, add = O.prefix_decode_attention(q, k, v, lens, pk, pv, plen, d ** -0.5)
    for t in (k, v):
        poison(t, lens)
    for t in (pk, pv):
        poison(t[None], [plen])
    n = plen + max(lens)
    args = [x.to(DEV) for x in (q, k, v, torch.tensor(lens), pk, pv)]
    used = None if plen == p else torch.tensor([plen], device=DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = K.prefix_decode_attention(*args, used, err_flag=flag)
    check_out(out, ref, mass, dot, n, 6.0)
    scores = start.to(DEV)
    out2 = K.prefix_decode_attention(*args, used, scores=scores, err_flag=flag)
    assert torch.equal(out2, K.prefix_decode_attention(*args, used, scores=scores.clone(), err_flag=flag))
    check_out(out2, ref, mass, dot, n, 6.0)
    # each weight within 2 r of its value; the running sum is rounded once more per call
    r = rel_bound(dot, d, n).view(b, hk, -1).amax(-1)[..., None]
    want = start.double() + add
    bound = 2 * r * add + 8 * 2.0 ** -24 * add + 2.0 ** -24 * want
    err = (scores.cpu().double() - want).abs()
    assert (err <= bound).all(), float((err / bound.clamp_min(1e-30)).max())
    for i, m in enumerate(lens):
        assert torch.equal(scores[i, :, m:].cpu(), start[i, :, m:])       # rows past the length: untouched
    assert int(flag) == 0


@pytest.mark.parametrize("case", DECODE[4:12] + DECODE[14:18], ids=lambda c: "-".join(map(str, c[:7])))
def test_step_launch_reads_the_newest_row_after_its_writer(case):
    """As a decode step calls it: the launch just before writes q and each stream's newest
    row (a KV write by this library), and the step's attention sees them; bit for bit the
    plain call's result, weights included."""
    b, hq, hk, d, p, plen, s, lens = case
    g = torch.Generator().manual_seed(5)
    dt = torch.bfloat16
    q, k, v, pk, pv = (make(sh, g, dt).to(DEV) for sh in ((b, hq, d), (b, hk, s, d), (b, hk, s, d), (hk, p, d), (hk, p, d)))
    used = torch.tensor([plen], device=DEV)
    n = torch.tensor(lens, device=DEV)
    slot = (n - 1).clamp_min(0)
    scores = torch.zeros(b, hk, s, device=DEV)
    for _ in range(20):
        kn, vn = (make((b, hk, 1, d), g, dt).to(DEV) for _ in range(2))
        k1, v1, s1, s2 = k.clone(), v.clone(), scores.clone(), scores.clone()
        torch.cuda.synchronize()
        K.kv_cache_write(kn, vn, k, v, slot)
        got = K.prefix_decode_attention(q, k, v, n, pk, pv, used, scores=s1, prefix_final=True)
        torch.cuda.synchronize()
        K.kv_cache_write(kn, vn, k1, v1, slot)
        torch.cuda.synchronize()
        want = K.prefix_decode_attention(q, k1, v1, n, pk, pv, used, scores=s2)
        assert torch.equal(got, want) and torch.equal(s1, s2) and torch.equal(k, k1)


def test_decode_without_prefix_is_decode_attention():
    g = torch.Generator().manual_seed(3)
    q, k, v = make((6, 16, 64), g, torch.bfloat16), make((6, 8, 200, 64), g, torch.bfloat16), make((6, 8, 200, 64), g, torch.bfloat16)
    lens = [0, 1, 64, 65, 150, 200]
    ref, mass, dot, _ = O.prefix_decode_attention(q, k, v, lens, k[0, :, :0], v[0, :, :0], 0, 0.125)
    args = [x.to(DEV) for x in (q, k, v, torch.tensor(lens))]
    check_out(K.prefix_decode_attention(*args), ref, mass, dot, 200, 6.0)
    check_out(K.decode_attention(*args), ref, mass, dot, 200, 6.0)


@pytest.mark.parametrize("scale", [0.0, 0.02, 3.0])
def test_decode_scales_and_sharp_weights(scale):
    """Uniform weights (scale 0) and a softmax that one row nearly owns; large logits."""
    g = torch.Generator().manual_seed(11)
    b, hq, hk, d, p, s = 12, 8, 4, 64, 321, 100
    q, k, v = make((b, hq, d), g, torch.bfloat16), make((b, hk, s, d), g, torch.bfloat16, 2.0), make((b, hk, s, d), g, torch.bfloat16)
    pk, pv = make((hk, p, d), g, torch.bfloat16, 2.0), make((hk, p, d), g, torch.bfloat16)
    lens = [(i * 9) % 101 for i in range(b)]
    ref, mass, dot, add = O.prefix_decode_attention(q, k, v, lens, pk, pv, p, scale)
    scores = torch.zeros(b, hk, s, device=DEV)
    out = K.prefix_decode_attention(*(x.to(DEV) for x in (q, k, v, torch.tensor(lens), pk, pv)), scale=scale, scores=scores)
    check_out(out, ref, mass, dot, p + s, 6.0)
    r = rel_bound(dot, d, p + s).view(b, hk, -1).amax(-1)[..., None]
    # weights below 2^-126 / 2^-149 may flush to zero
    assert ((scores.cpu().double() - add).abs() <= (2 * r + 8 * 2.0 ** -24) * add + 2.0 ** -120).all()


@pytest.mark.parametrize("layout", ["slot-major", "packed", "wide rows"])
def test_decode_strided_inputs(layout):
    g = torch.Generator().manual_seed(21)
    b, hq, hk, d, p, s = 5, 8, 4, 64, 150, 77
    dt = torch.bfloat16
    lens = [0, 77, 13, 64, 50]
    kv = make((2, b, hk, s, d), g, dt)
    pkv = make((2, hk, p, d), g, dt)
    q = make((b, hq, d), g, dt)
    ref, mass, dot, _ = O.prefix_decode_attention(q, kv[0], kv[1], lens, pkv[0], pkv[1], p, 0.125)
    kvd, pd, qd = kv.to(DEV), pkv.to(DEV), q.to(DEV)
    if layout == "slot-major":
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in kvd)
        pk, pv = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in pd)
        big = torch.full((b, 3, hq, d), float("nan"), dtype=dt, device=DEV)
        big[:, 1] = qd
        qd = big[:, 1:2]                                             # [B, 1, Hq, D], batch stride 3 Hq D
    elif layout == "packed":
        k, v = kvd.transpose(0, 3).contiguous().transpose(0, 3)      # K and V rows interleaved
        pk, pv = pd.transpose(0, 2).contiguous().transpose(0, 2)
        qd = qd.transpose(0, 1).contiguous().transpose(0, 1)
    else:
        wide = torch.full((2, b, hk, s, 2 * d), float("nan"), dtype=dt, device=DEV)
        wide[..., d:] = kvd
        k, v = wide[0, ..., d:], wide[1, ..., d:]
        pw = torch.full((2, 1, hk, p, d + 8), float("nan"), dtype=dt, device=DEV)
        pw[:, 0, :, :, :d] = pd
        pk, pv = pw[0, ..., :d], pw[1, ..., :d]
    out = K.prefix_decode_attention(qd, k, v, torch.tensor(lens, device=DEV), pk, pv)
    check_out(out, ref, mass, dot, p + s, 6.0)


def test_lengths_out_of_range_are_held_and_flagged():
    g = torch.Generator().manual_seed(4)
    dt = torch.bfloat16
    q, k, v = make((3, 4, 64), g, dt), make((3, 2, 20, 64), g, dt), make((3, 2, 20, 64), g, dt)
    pk, pv = make((2, 30, 64), g, dt), make((2, 30, 64), g, dt)
    ref, mass, dot, _ = O.prefix_decode_attention(q, k, v, [20, 0, 7], pk, pv, 30, 0.125)
    dev = [x.to(DEV) for x in (q, k, v)]
    pkd, pvd = pk.to(DEV), pv.to(DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = K.prefix_decode_attention(*dev, torch.tensor([21, -5, 7], device=DEV), pkd, pvd, err_flag=flag)
    check_out(out, ref, mass, dot, 50, 6.0)
    assert int(flag) == _lib.KANI_FLAG_SLOT_OOB
    flag.zero_()
    out = K.prefix_decode_attention(*dev, torch.tensor([20, 0, 7], device=DEV), pkd, pvd,
                                    torch.tensor([1 << 40], device=DEV), err_flag=flag)
    check_out(out, ref, mass, dot, 50, 6.0)
    assert int(flag) == _lib.KANI_FLAG_SLOT_OOB
    # prefill: more real tokens than cache rows; token i is then own row i
    flag.zero_()
    q4 = make((1, 5, 4, 64), g, dt)
    ref, mass, dot = O.prefix_prefill_attention(q4[:, :3], k[:1], v[:1], [3], [3], pk, pv, 30, 0.125)
    out = K.prefix_prefill_attention(q4.to(DEV), dev[1][:1], dev[2][:1], torch.tensor([3], device=DEV), pkd, pvd, err_flag=flag)
    check_out(out[:, :3], ref, mass, dot, 50, 6.0)
    assert torch.isfinite(out).all() and int(flag) == _lib.KANI_FLAG_SLOT_OOB


PREFILL = [
    # batch, tokens, heads, kv heads, dim, prefix rows, in use, slots, own lengths, real tokens
    (1, 1, 2, 1, 64, 0, 0, 1, [1], [1]),
    (1, 23, 16, 8, 64, 300, 300, 64, [23], [23]),
    (2, 64, 4, 2, 64, 64, 64, 64, [64, 40], [64, 40]),
    (3, 65, 4, 2, 64, 70, 1, 130, [65, 0, 130], [65, 0, 1]),
    (2, 129, 2, 2, 64, 0, 0, 300, [300, 129], [129, 77]),
    (1, 200, 8, 1, 128, 130, 130, 333, [333], [200]),
    (3, 50, 10, 2, 128, 65, 63, 90, [50, 90, 31], [50, 50, 31]),
    (2, 100, 6, 2, 64, 129, 129, 164, [163, 100], [99, 43]),
    (2, 40, 14, 2, 64, 20, 0, 41, [40, 41], [39, 2]),
    (1, 300, 2, 1, 64, 1000, 1000, 300, [300], [300]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", PREFILL, ids=lambda c: "-".join(map(str, c[:8])))
def test_prefill(case, dtype):
    b, t, hq, hk, d, p, plen, s, lens, qls = case
    g = torch.Generator().manual_seed(hash(case[:8]) % 10007)
    q, k, v = make((b, t, hq, d), g, dtype), make((b, hk, s, d), g, dtype), make((b, hk, s, d), g, dtype)
    pk, pv = make((hk, p, d), g, dtype), make((hk, p, d), g, dtype)
    ref, mass, dot = O.prefix_prefill_attention(q, k, v, lens, qls, pk, pv, plen, d ** -0.5)
    for x in (k, v):
        poison(x, lens)
    for x in (pk, pv):
        poison(x[None], [plen])
    for i, m in enumerate(qls):
        q[i, m:] = float("nan")
    args = [x.to(DEV) for x in (q, k, v, torch.tensor(lens), pk, pv)]
    used = None if plen == p else torch.tensor([plen], device=DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    full = all(m == t for m in qls)
    out = K.prefix_prefill_attention(*args, used, q_len=None if full else torch.tensor(qls, device=DEV), err_flag=flag)
    check_out(out, ref, mass, dot, plen + s, 6.0)
    for i, m in enumerate(qls):
        assert not out[i, m:].any()
    assert int(flag) == 0
    assert torch.equal(out, K.prefix_prefill_attention(*args, used, q_len=torch.tensor(qls, device=DEV)))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prefill_does_not_see_later_rows(bad):
    """A token's result does not depend on the rows after it, whatever they hold; a
    value that is not finite reaches the tokens that see it."""
    g = torch.Generator().manual_seed(8)
    dt = torch.bfloat16
    b, t, hq, hk, d, p = 1, 90, 4, 2, 64, 40
    q, k, v = make((b, t, hq, d), g, dt), make((b, hk, t, d), g, dt), make((b, hk, t, d), g, dt)
    pk, pv = make((hk, p, d), g, dt), make((hk, p, d), g, dt)
    first = 37
    ref, mass, dot = O.prefix_prefill_attention(q[:, :first], k, v, [first], [first], pk, pv, p, 0.125)
    v[:, :, first, 5] = bad
    v[:, :, 80, 9] = bad
    k[:, :, first:, 3] = bad if bad != bad else k[:, :, first:, 3]
    out = K.prefix_prefill_attention(*(x.to(DEV) for x in (q, k, v, torch.tensor([t]), pk, pv)))
    check_out(out[:, :first], ref, mass, dot, p + t, 6.0)
    later = out[:, first:].float()
    if bad != bad:
        assert later.isnan().all()
    else:
        assert (later[..., 5] == bad).all()
        assert (later[:, 80 - first:, :, 9] == bad).all()
        assert torch.isfinite(later[:, :80 - first, :, 9]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", ["nan", "inf", "spike", "huge spike"])
def test_one_odd_key_at_every_place(what, d):
    """A single key of the prefix at each place of a tile, seen by every query: a NaN or
    infinite one makes every result NaN (an infinite logit has no softmax), one whose logit
    exceeds the others by 60 or by hundreds of powers of two owns the result."""
    g = torch.Generator().manual_seed(77)
    dt = torch.bfloat16
    p, n = 192, 64
    q = torch.ones(n, 5, 2, d, dtype=dt)                       # a stream per place, 5 tokens each
    k, v = make((n, 1, 5, d), g, dt), make((n, 1, 5, d), g, dt)
    pk, pv = make((1, p, d), g, dt), make((1, p, d), g, dt)
    dev = [x.to(DEV) for x in (q, k, v, torch.full((n,), 5), pk, pv)]
    size = {"nan": float("nan"), "inf": float("inf"), "spike": 60 * math.log(2) / d, "huge spike": 400.0 / d}[what]
    for place in range(64, 128):
        bad = dev[4].clone()
        bad[0, place] = size
        out = K.prefix_prefill_attention(dev[0][:1], dev[1][:1], dev[2][:1], dev[3][:1], bad, dev[5], scale=1.0)
        dec = K.prefix_decode_attention(dev[0][:, 0], dev[1], dev[2], dev[3], bad.expand(1, p, d), dev[5], scale=1.0)
        if what in ("nan", "inf"):
            assert out.isnan().all() and dec.isnan().all()
        else:
            ref, mass, dot = O.prefix_prefill_attention(q[:1, :1], k[:1], v[:1], [1], [1], bad.cpu(), pv, p, 1.0)
            check_out(out[:, :1], ref, mass, dot, p + 5, 6.0)
            ref, mass, dot, _ = O.prefix_decode_attention(q[:1, 0], k[:1], v[:1], [5], bad.cpu(), pv, p, 1.0)
            check_out(dec[:1], ref, mass, dot, p + 5, 6.0)


def test_logits_that_keep_growing():
    """Each tile's logits exceed the last one's, by a little and by hundreds: the running
    maximum moves tile after tile."""
    g = torch.Generator().manual_seed(78)
    for step in (0.4, 5.0, 60.0):
        p, d, b = 700, 64, 70
        q = torch.ones(1, b, 2, d, dtype=torch.bfloat16)
        pk = (torch.arange(p).view(1, p, 1) * step / 64 / d + 0.01 * torch.randn(1, p, d, generator=g)).bfloat16()
        pv, k, v = make((1, p, d), g, torch.bfloat16), make((1, 1, b, d), g, torch.bfloat16), make((1, 1, b, d), g, torch.bfloat16)
        ref, mass, dot = O.prefix_prefill_attention(q, k, v, [b], [b], pk, pv, p, 1.0)
        out = K.prefix_prefill_attention(*(x.to(DEV) for x in (q, k, v, torch.tensor([b]), pk, pv)), scale=1.0)
        check_out(out, ref, mass, dot, p + b, 6.0)


def test_expanded_inputs():
    """Queries and caches expanded over streams or heads give what their copies give."""
    g = torch.Generator().manual_seed(79)
    dt = torch.bfloat16
    q = make((1, 3, 4, 64), g, dt).to(DEV).expand(5, 3, 4, 64)
    k, v = (make((1, 1, 40, 64), g, dt).to(DEV).expand(5, 2, 40, 64) for _ in range(2))
    pk, pv = (make((1, 200, 64), g, dt).to(DEV).expand(2, 200, 64) for _ in range(2))
    n = torch.tensor([40, 3, 17, 30, 8], device=DEV)
    a = K.prefix_prefill_attention(q, k, v, n, pk, pv)
    assert torch.equal(a, K.prefix_prefill_attention(*(x.contiguous() for x in (q, k, v, n, pk, pv))))
    a = K.prefix_decode_attention(q[:, 0], k, v, n, pk, pv)
    assert torch.equal(a, K.prefix_decode_attention(*(x.contiguous() for x in (q[:, 0], k, v, n, pk, pv))))
    with pytest.raises(_lib.KaniError):
        K.prefix_decode_attention(q[:, 0], k[:, :, :1].expand(5, 2, 40, 64), v[:, :, :1].expand(5, 2, 40, 64), n)


def test_prefill_strided_and_chunked():
    """Views of a packed QKV output and a slot-major cache; two chunks give the rows of one pass."""
    g = torch.Generator().manual_seed(31)
    dt = torch.bfloat16
    b, t, hq, hk, d, p = 2, 70, 4, 2, 64, 100
    qkv = make((b, t, (hq + 2 * hk) * d), g, dt).to(DEV)
    q = qkv[..., :hq * d].view(b, t, hq, d)
    k, v = (make((b, t, hk, d), g, dt).to(DEV).transpose(1, 2) for _ in range(2))
    pk, pv = (make((p, hk, d), g, dt).to(DEV).transpose(0, 1) for _ in range(2))
    n = torch.tensor([t, t], device=DEV)
    whole = K.prefix_prefill_attention(q, k, v, n, pk, pv)
    ref, mass, dot = O.prefix_prefill_attention(q, k, v, [t, t], [t, t], pk, pv, p, 0.125)
    check_out(whole, ref, mass, dot, p + t, 6.0)
    a = 45
    first = K.prefix_prefill_attention(q[:, :a], k, v, n - (t - a), pk, pv)
    out = torch.empty(b, t - a, hq, d, dtype=dt, device=DEV)
    second = K.prefix_prefill_attention(q[:, a:], k, v, n, pk, pv, out=out)
    assert second is out
    check_out(torch.cat([first, second], 1), ref, mass, dot, p + t, 6.0)
    # a decode step is a prefill of one token
    one = K.prefix_decode_attention(q[:, -1:], k, v, n, pk, pv)
    check_out(one, ref[:, -1], mass[:, -1], dot[:, -1], p + t, 6.0)


def test_captured_graphs_and_other_streams():
    """Two captured graphs replayed at the same time on two streams give the eager results
    for the inputs of the replay, and scores add up once per replay."""
    g = torch.Generator().manual_seed(41)
    dt = torch.bfloat16
    b, hq, hk, d, p, s = 24, 16, 8, 64, 2800, 300      # (over 128 MB: two launches)
    sets = []
    for _ in range(2):
        x = [make(sh, g, dt).to(DEV) for sh in ((b, hq, d), (b, hk, s, d), (b, hk, s, d), (hk, p, d), (hk, p, d))]
        sets.append((x, torch.randint(0, s + 1, (b,), generator=g).to(DEV), torch.zeros(b, hk, s, device=DEV)))
    t = make((b, 33, hq, d), g, dt).to(DEV)
    qlen = torch.full((b,), 33, device=DEV)

    def step(x, n, scores):
        return (K.prefix_decode_attention(x[0], x[1], x[2], n, x[3], x[4], scores=scores),
                K.prefix_prefill_attention(t, x[1], x[2], n.clamp_min(33), x[3], x[4], q_len=qlen))

    want = [step(x, n, sc.clone()) for x, n, sc in sets]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for (x, n, sc), st in zip(sets, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(x, n, sc.clone())
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            outs.append(step(x, n, sc))
        graphs.append(gr)
    torch.cuda.synchronize()
    assert all(not sc.any() for _, _, sc in sets)
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for w, o, (x, n, sc) in zip(want, outs, sets):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
        once = torch.zeros_like(sc)
        K.prefix_decode_attention(x[0], x[1], x[2], n, x[3], x[4], scores=once)
        torch.testing.assert_close(sc, 5 * once, rtol=2.0 ** -21, atol=0)   # 5 sums, each off by 2^-24
    # new lengths and inputs at the next replay
    sets[0][0][0].copy_(sets[1][0][0])
    sets[0][1].copy_(sets[1][1])
    graphs[0].replay()
    torch.cuda.synchronize()
    x, n, _ = sets[0]
    assert torch.equal(outs[0][0], K.prefix_decode_attention(x[0], x[1], x[2], n, x[3], x[4], scores=torch.zeros(b, hk, s, device=DEV)))


def test_two_streams_at_once():
    """The same call on two streams, interleaved: every result is the one alone."""
    g = torch.Generator().manual_seed(43)
    q, k, v, pk, pv = (make(sh, g, torch.bfloat16).to(DEV) for sh in ((64, 16, 64), (64, 8, 300, 64), (64, 8, 300, 64),
                                                                     (8, 2048, 64), (8, 2048, 64)))
    n = torch.randint(0, 301, (64,), generator=g).to(DEV)
    want = K.prefix_decode_attention(q, k, v, n, pk, pv)
    pre = K.prefix_prefill_attention(q[:, None].expand(64, 7, 16, 64), k, v, n.clamp_min(7), pk, pv)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(20):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append((K.prefix_decode_attention(q, k, v, n, pk, pv),
                             K.prefix_prefill_attention(q[:, None].expand(64, 7, 16, 64), k, v, n.clamp_min(7), pk, pv)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, pre) for a, b in outs)


def test_offsets_past_32_bits():
    """A cache whose last stream starts beyond 2^32 elements."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    d, s, hk = 64, 1 << 20, 2
    k = torch.empty(34, hk, s, d, dtype=torch.bfloat16, device=DEV)      # 4.6e9 elements
    v = k
    g = torch.Generator().manual_seed(2)
    rows = make((hk, 100, d), g, torch.bfloat16)
    k[33, :, :50] = rows[:, :50].to(DEV)
    k[33, :, s - 50:] = rows[:, 50:].to(DEV)
    lens = torch.zeros(34, dtype=torch.int64, device=DEV)
    lens[33] = 50
    q = make((34, 4, d), g, torch.bfloat16)
    out = K.prefix_decode_attention(q.to(DEV), k, v, lens)
    ref, mass, dot, _ = O.prefix_decode_attention(q[33:], rows[None, :, :50], rows[None, :, :50], [50], rows[:, :0], rows[:, :0], 0, 0.125)
    check_out(out[33:], ref, mass, dot, 50, 6.0)
    assert not out[:33].any()
    pre = K.prefix_prefill_attention(q[33:, None].to(DEV), k[33:], v[33:], lens[33:])
    check_out(pre[:, 0], ref, mass, dot, 50, 6.0)


def test_refusals_on_the_device():
    dt = torch.bfloat16

    def z(*s, dtype=dt):
        return torch.zeros(*s, dtype=dtype, device=DEV)

    q, k, n, pk = z(2, 4, 64), z(2, 2, 8, 64), torch.ones(2, dtype=torch.int64, device=DEV), z(2, 5, 64)
    v, pv = z(2, 2, 8, 64), z(2, 5, 64)
    K.prefix_decode_attention(q, k, v, n, pk, pv)

    def refused(exc, fn, *a, **kw):
        with pytest.raises(exc):
            fn(*a, **kw)

    dec, pre = K.prefix_decode_attention, K.prefix_prefill_attention
    refused(TypeError, dec, q.half(), k, v, n, pk, pv)
    refused(TypeError, dec, q, k, v, n, pk.half(), pv.half())
    refused(TypeError, dec, q.long(), k, v, n)
    refused(ValueError, dec, q, k, v[:, :, :7], n)
    refused(ValueError, dec, q, k, v, n.int())
    refused(ValueError, dec, q, k, v, n[:1])
    refused(ValueError, dec, q, k, v, n, pk, None)
    refused(ValueError, dec, q, k, v, n, None, None, n[:1])
    refused(ValueError, dec, q, k, v, n, pk[:1], pv[:1])
    refused(ValueError, dec, q, k, v, n, pk, pv, n)
    refused(ValueError, dec, q[:, :3], k, v, n)
    refused(ValueError, dec, q, k, v, n, scale=-1.0)
    refused(ValueError, dec, q, k, v, n, scale=math.nan)
    refused(ValueError, dec, q, k, v, n, scores=z(2, 2, 7, dtype=torch.float32))
    refused(ValueError, dec, q, k, v, n, scores=z(2, 2, 8))
    refused(ValueError, dec, q, k, v, n, scores=z(1, 2, 8, dtype=torch.float32).expand(2, 2, 8))
    refused(ValueError, dec, q, k, v, n, out=q)
    refused(ValueError, dec, q, k.cpu(), v, n)
    refused(ValueError, dec, q, k, v, n.cpu())
    refused(_lib.KaniError, dec, q.float(), k.float(), v.float(), n)
    refused(_lib.KaniError, dec, z(2, 18, 64), k, v, n)                  # 9 query heads a group
    refused(_lib.KaniError, dec, z(2, 4, 32), z(2, 2, 8, 32), z(2, 2, 8, 32), n)
    odd = z(2 * 2 * 8 * 64 + 1)[1:].view(2, 2, 8, 64)
    refused(_lib.KaniError, dec, q, odd, odd, n)                         # rows not 16-byte aligned
    refused(_lib.KaniError, dec, q, z(2, 2, 8, 68)[..., :64], z(2, 2, 8, 68)[..., :64], n)
    refused(ValueError, pre, q, k, v, n)
    q4 = z(2, 3, 4, 64)
    refused(ValueError, pre, q4, k, v, n, q_len=n[:1])
    refused(ValueError, pre, q4, k, v, n, out=z(2, 3, 4, 65)[..., :64])
    refused(ValueError, pre, q4, k, v, n, out=q4)
    # nothing to do
    assert dec(z(0, 4, 64), z(0, 2, 8, 64), z(0, 2, 8, 64), n[:0]).shape == (0, 4, 64)
    assert pre(z(2, 0, 4, 64), k, v, n).shape == (2, 0, 4, 64)
    assert not dec(q, z(2, 2, 0, 64), z(2, 2, 0, 64), n * 0).any()
