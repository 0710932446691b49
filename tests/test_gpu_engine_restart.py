"""One captured step for voice after voice: every start of the engine gives the tokens of an
engine captured for it alone, and leaves the results of earlier starts as they are."""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200.decode import DecodeEngine, FusedDecoder
from kani_tts_b200.model import synthetic_state_dict, tiny_config
from kani_tts_b200.sampling import SamplingParams

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("b", [1, 3, 20])
@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("budget", [None, 24])
def test_one_capture_for_every_voice(b, sampled, budget):
    cfg, max_len, n = tiny_config(), 40, 30
    sd = synthetic_state_dict(cfg, seed=6)
    g = torch.Generator().manual_seed(2)
    voices = [(torch.randint(10, cfg.vocab_size, (p,), generator=g).to(DEV),
               torch.randint(10, cfg.vocab_size, (b, t), generator=g).to(DEV)) for p, t in ((40, 7), (60, 9), (33, 1))]
    voices.append(voices[0])

    def engine():
        dec = FusedDecoder(cfg, sd, DEV, batch=b, max_len=max_len)
        dec.set_prefix(voices[0][0], capacity=60)
        return dec, DecodeEngine(dec, sampling=SamplingParams(seed=3) if sampled else None, cache_budget=budget)

    def steps(own):
        return n if budget is not None else max_len - own.shape[1]

    want = []
    for prefix, own in voices:
        dec, eng = engine()
        dec.set_prefix(prefix)
        eng.start(own, None, steps(own))
        eng.capture()
        eng.run(steps(own))
        want.append((eng.generated.clone(), eng.positions.clone(), eng.kv_len.clone(), eng.seen))
        eng.graph = None
    dec, eng = engine()
    got = []
    for i, (prefix, own) in enumerate(voices):
        dec.set_prefix(prefix)
        eng.start(own, None, steps(own))
        if i == 0:
            eng.capture()
        elif eng.generated.shape[1] > got[0].shape[1]:
            with pytest.raises(RuntimeError):
                eng.run(1)
            eng.start(own, None, got[0].shape[1])
        junk = [torch.full((b, 64), -1, device=DEV) for _ in range(8)]   # takes memory that was given back
        eng.run(4)
        eng.run(eng.generated.shape[1] - 4)
        torch.cuda.synchronize()
        assert all((j == -1).all() for j in junk)
        got.append(eng.generated)
        if eng.generated.shape == want[i][0].shape:
            assert torch.equal(eng.positions, want[i][1]) and torch.equal(eng.kv_len, want[i][2])
            if sampled:
                assert torch.equal(eng.seen, want[i][3])
    for a, (w, *_) in zip(got, want):
        assert torch.equal(a, w[:, :a.shape[1]])
    assert not torch.equal(got[0], got[1])
    assert torch.equal(got[0], got[3])
    assert int(dec.err_flag.item()) == 0
