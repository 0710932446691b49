"""A captured engine with a cache budget against the plain one, before any eviction."""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200.decode import DecodeEngine, FusedDecoder
from kani_tts_b200.model import synthetic_state_dict, tiny_config

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("with_prefix", [False, True])
@pytest.mark.parametrize("b", [1, 2, 6])
def test_tokens_before_an_eviction_are_the_plain_engines(b, with_prefix):
    """Captured steps of both are given the same tokens and generate their own.  The weights'
    accumulation takes another attention kernel, whose logits agree with the plain one's
    within 2 % of the largest logit on the tiny model (the decode tests' convention), so
    each choice is, by the plain engine's logits, the best one or within twice that of it."""
    cfg, n = tiny_config(), 24
    sd = synthetic_state_dict(cfg, seed=12)
    g = torch.Generator().manual_seed(5)
    own = torch.randint(10, cfg.vocab_size, (b, 8), generator=g).to(DEV)
    voice = torch.randint(10, cfg.vocab_size, (50,), generator=g).to(DEV)
    forced = torch.randint(10, cfg.vocab_size, (n, b, 1), generator=g).to(DEV)

    def started(budget):
        dec = FusedDecoder(cfg, sd, DEV, batch=b, max_len=40)
        if with_prefix:
            dec.set_prefix(voice)
        eng = DecodeEngine(dec, cache_budget=budget)
        eng.start(own, None, n)
        return dec, eng

    tokens = {}
    for budget in (None, 30):
        dec, eng = started(budget)
        eng.capture()
        for ids in forced:
            eng.input_ids.copy_(ids)
            eng.run(1)
        torch.cuda.synchronize()
        assert eng._filled == 8 + n and int(dec.err_flag.item()) == 0      # no eviction
        assert dec.scores is None                                          # kept for the engine's own steps alone
        if budget is not None:
            assert all((s[:, :, :8 + n] > 0).all() for s in eng.scores.values())
        tokens[budget] = dec.full_to_reduced[eng.generated]
        eng.graph = None
    dec, eng = started(None)
    clear = 0
    for i, ids in enumerate(forced):
        eng.input_ids.copy_(ids)
        conv = {j: c.clone() for j, c in dec.conv_state.items()}
        logits = dec.step(eng.input_ids, eng.positions, eng.slots, eng.kv_len)[:, 0].float()
        for j, c in conv.items():
            dec.conv_state[j].copy_(c)
        eng._step_body()
        assert torch.equal(dec.full_to_reduced[eng.generated[:, i]], tokens[None][:, i])
        slack = 2 * 0.02 * logits.abs().amax(-1)
        best = logits.topk(2, dim=-1).values
        assert (logits.gather(1, tokens[30][:, i:i + 1])[:, 0] >= best[:, 0] - slack).all()
        sure = best[:, 0] - best[:, 1] > slack
        assert torch.equal(tokens[30][sure, i], tokens[None][sure, i])
        clear += int(sure.sum())
    assert clear > 0


def test_a_capture_when_the_caches_are_full():
    """The warm-up step of a capture needs a row too: captured again with full caches, the
    engine goes on as one that was not, and no slot past the end is written."""
    cfg = tiny_config()
    sd = synthetic_state_dict(cfg, seed=9)
    own = torch.randint(10, cfg.audio_tokens_start, (2, 6), generator=torch.Generator().manual_seed(8)).to(DEV)
    results = []
    for again in (False, True):
        dec = FusedDecoder(cfg, sd, DEV, batch=2, max_len=20)
        eng = DecodeEngine(dec, cache_budget=12, cache_recent=3)
        eng.start(own, None, 40)
        eng.capture()
        eng.run(14)
        assert eng._filled == 20
        if again:
            eng.capture()
        eng.run(26)
        torch.cuda.synchronize()
        assert int(dec.err_flag.item()) == 0
        results.append((eng.generated.clone(), eng.positions.clone(), eng.kv_len.clone(),
                        *(t.clone() for t in eng.scores.values())))
        eng.graph = None
    for a, b in zip(*results):
        assert torch.equal(a, b)
