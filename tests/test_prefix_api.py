"""The shared-prefix and eviction entry points refuse bad calls before any launch (no GPU needed)."""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200 import _lib
from kani_tts_b200 import fused_kernels as K
from oracle import prefix_oracle as O

A = 0x1000          # an aligned address that no refused call may touch
DECODE = dict(dtype=1, batch=2, hq=4, hk=2, d=64, q=A, qb=256, qh=64, k=A, v=A, cb=1024, ch=512, cs=64, s=8, n=A, pk=A,
              pv=A, ph=320, ps=64, p=5, plen=0, scale=0.125, scores=0, sb=0, sh=0, out=A, ob=256, oh=64, ws=A,
              nbytes=1 << 40, err=0, stream=0)
PREFILL = dict(dtype=1, batch=2, t=3, hq=4, hk=2, d=64, q=A, qb=768, qt=256, qh=64, k=A, v=A, cb=1024, ch=512, cs=64,
               s=8, n=A, ql=0, pk=A, pv=A, ph=320, ps=64, p=5, plen=0, scale=0.125, out=A, ob=768, ot=256, oh=64, err=0,
               stream=0)
EVICT = dict(dtype=1, batch=2, hk=2, d=64, k=A, v=2 * A, cb=1024, ch=512, cs=64, s=8, sc=A, sb=16, sh=8, n=A, budget=4,
             recent=1, protect=1, ko=3 * A, vo=4 * A, cbo=512, cho=256, cso=64, so=4, sco=5 * A, sbo=8, sho=4, lo=6 * A,
             kept=0, err=0, stream=0)


def call(name, base, **change):
    return getattr(_lib.load_library(), name)(*{**base, **change}.values())


BAD, DTYPE, UNSUP = -1, -2, -3
ATTENTION = [(dict(batch=-1), BAD), (dict(hk=0), BAD), (dict(hq=5), BAD), (dict(q=0), BAD), (dict(k=0), BAD),
             (dict(n=0), BAD), (dict(pk=0), BAD), (dict(out=0), BAD), (dict(scale=-1.0), BAD),
             (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(p=-1), BAD), (dict(s=-1), BAD),
             (dict(dtype=7), DTYPE), (dict(dtype=0), UNSUP), (dict(d=32), UNSUP), (dict(hq=18), UNSUP),
             (dict(q=A + 2), UNSUP), (dict(k=A + 8), UNSUP), (dict(pv=A + 4), UNSUP), (dict(cs=65), UNSUP),
             (dict(ps=66), UNSUP), (dict(qh=60), UNSUP), (dict(oh=4), UNSUP), (dict(batch=70000), UNSUP),
             (dict(s=1 << 31), UNSUP), (dict(p=1 << 31), UNSUP)]


@pytest.mark.parametrize("change,status", ATTENTION, ids=str)
@pytest.mark.parametrize("name,base", [("kani_prefix_decode_attention", DECODE),
                                       ("kani_prefix_decode_attention_step", DECODE),
                                       ("kani_prefix_prefill_attention", PREFILL)], ids=["decode", "step", "prefill"])
def test_attention_refusals(name, base, change, status):
    assert call(name, base, **change) == status


def test_attention_without_work():
    assert call("kani_prefix_decode_attention", DECODE, batch=0) == 0
    assert call("kani_prefix_prefill_attention", PREFILL, t=0) == 0


@pytest.mark.parametrize("change,status", [
    (dict(batch=-1), BAD), (dict(budget=5), BAD), (dict(recent=4), BAD), (dict(recent=-1), BAD), (dict(protect=-1), BAD),
    (dict(recent=1 << 62, protect=1 << 62), BAD), (dict(k=0), BAD), (dict(sc=0), BAD), (dict(lo=0), BAD),
    (dict(lo=A), BAD), (dict(v=A), BAD), (dict(vo=3 * A), BAD), (dict(ko=A), BAD), (dict(sco=A), BAD),
    (dict(ko=A, vo=2 * A, sco=A), BAD),                  # in place with another row count
    (dict(dtype=9), DTYPE), (dict(d=257), UNSUP), (dict(d=60), UNSUP), (dict(cs=65), UNSUP), (dict(cso=68), UNSUP),
    (dict(k=A + 8), UNSUP), (dict(batch=70000), UNSUP), (dict(s=1 << 31), UNSUP)], ids=str)
def test_evict_refusals(change, status):
    assert call("kani_cache_evict", EVICT, **change) == status


def test_python_layer_refuses_cpu_tensors():
    q, k, n = torch.zeros(1, 2, 64).bfloat16(), torch.zeros(1, 1, 4, 64).bfloat16(), torch.ones(1, dtype=torch.int64)
    with pytest.raises(ValueError):
        K.prefix_decode_attention(q, k, k.clone(), n)
    with pytest.raises(ValueError):
        K.prefix_prefill_attention(q[:, None], k, k.clone(), n)
    with pytest.raises(ValueError):
        K.evict_cache(k, k.clone(), torch.zeros(1, 1, 4), n, 2, 1)


def test_oracle_known_answers():
    assert O.evict([5, 1, 4, 4, 9], 5, 3, 1, 0) == [0, 2, 4]               # a tie: the lower slot
    assert O.evict([5, 1, 4], 3, 3, 1, 1) == [0, 1, 2]
    assert O.evict([float("nan"), 0.0, float("-inf"), 1.0], 4, 2, 0, 0) == [1, 3]
    q = torch.ones(1, 1, 2)
    k = torch.zeros(1, 1, 3, 2)
    v = torch.tensor([[[[1.0, 2.0], [3.0, 4.0], [99.0, 99.0]]]])
    out, _, _, w = O.prefix_decode_attention(q, k, v, [2], torch.zeros(1, 2, 2), torch.ones(1, 2, 2), 2, 1.0)
    assert out[0, 0].tolist() == [1.5, 2.0] and w[0, 0].tolist() == [0.25, 0.25, 0.0]
