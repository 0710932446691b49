"""The decode engine behind a shared prefix and with evicting caches.

Comparisons of logits use the decode tests' convention (two bf16 paths that accumulate in
another order agree within 2 % of the largest logit on the tiny model, 5 % at full size)."""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200.decode import DecodeEngine, FusedDecoder
from kani_tts_b200.model import LFM2Config, synthetic_state_dict, tiny_config
from kani_tts_b200.sampling import SamplingParams, seen_bitmap
from oracle import prefix_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def close(got, ref, frac=0.02):
    got, ref = got.detach().float().cpu(), ref.detach().float().cpu()
    err, scale = float((got - ref).abs().max()), float(ref.abs().max())
    assert err <= frac * scale, f"max error {err} vs scale {scale}"


def prompts(cfg, b, p, t, seed):
    g = torch.Generator().manual_seed(seed)
    prefix = torch.randint(10, cfg.vocab_size, (p,), generator=g).to(DEV)      # text and audio tokens
    own = torch.randint(10, cfg.audio_tokens_start, (b, t), generator=g).to(DEV)
    return prefix, own


def feed(dec, eng, tokens):
    """Logits of steps that are given their tokens (teacher forcing), with the engine's bookkeeping."""
    out = []
    for k in range(tokens.shape[0]):
        pos = eng.base_pos + (k // dec.cfg.tokens_per_frame) * int(dec.cfg.audio_step)
        out.append(dec.step(tokens[k].view(-1, 1), pos, eng.base_slot + k, eng.base_slot + k + 1).clone())
    return out


@pytest.mark.parametrize("full,b,speaker", [(False, 1, False), (False, 3, False), (False, 2, True), (True, 1, False),
                                            (True, 8, True), (True, 40, False)])
def test_prefix_equals_the_whole_prompt(full, b, speaker):
    """Prompt = prefix + own tokens: prefill and steps behind the shared prefix give the
    logits of a decoder that has the whole prompt in every stream's cache."""
    cfg = LFM2Config() if full else tiny_config()
    sd = synthetic_state_dict(cfg, seed=5)
    p, t, frac = 70, 9, 0.05 if full else 0.02
    prefix, own = prompts(cfg, b, p, t, 3)
    spk = torch.randn(1, cfg.speaker_emb_dim, generator=torch.Generator().manual_seed(1)).to(DEV) if speaker else None
    whole = FusedDecoder(cfg, sd, DEV, batch=b, max_len=128)
    e0 = DecodeEngine(whole)
    e0.start(torch.cat([prefix.expand(b, -1), own], 1), None if spk is None else spk.expand(b, -1), 16)
    dec = FusedDecoder(cfg, sd, DEV, batch=b, max_len=32)
    rows = dec.set_prefix(prefix, speaker_emb=spk)
    assert rows == p + speaker
    eng = DecodeEngine(dec)
    eng.start(own, None, 16)
    assert torch.equal(eng.base_pos, e0.base_pos)
    assert torch.equal(eng.base_slot + rows, e0.base_slot)
    tokens = torch.randint(cfg.audio_tokens_start, cfg.vocab_size, (6, b), generator=torch.Generator().manual_seed(4)).to(DEV)
    for got, ref in zip(feed(dec, eng, tokens), feed(whole, e0, tokens)):
        close(got, ref, frac)
    for i in cfg.attn_layers:      # the same rows, in the prefix and behind it
        close(dec.prefix.k[i][0, :, :rows], whole.k_cache[i][0, :, :rows], frac)
        close(dec.k_cache[i][:, :, :t + 6], whole.k_cache[i][:, :, rows:rows + t + 6], frac)
    for i in dec.conv_state:
        close(dec.conv_state[i], whole.conv_state[i], frac)
    assert int(dec.err_flag.item()) == 0


def test_a_captured_step_serves_the_next_voice():
    """A second prefix that fits the buffers takes their place under a captured graph; one
    that does not, and a removed one, need a new capture."""
    cfg, b = tiny_config(), 2
    sd = synthetic_state_dict(cfg, seed=6)
    (pa, own), (pb, _), (pc, _) = prompts(cfg, b, 40, 7, 1), prompts(cfg, b, 55, 7, 2), prompts(cfg, b, 90, 7, 3)

    def fresh(prefix):
        d = FusedDecoder(cfg, sd, DEV, batch=b, max_len=40)
        d.set_prefix(prefix)
        e = DecodeEngine(d)
        e.start(own, None, 20)
        e.capture()
        e.run(20)
        return e.generated.clone()

    dec = FusedDecoder(cfg, sd, DEV, batch=b, max_len=40)
    dec.set_prefix(pa, capacity=60)
    eng = DecodeEngine(dec)
    eng.start(own, None, 20)
    eng.capture()
    eng.run(20)
    assert torch.equal(eng.generated, fresh(pa))
    dec.set_prefix(pb)
    eng.start(own, None, 20)
    eng.capture()                 # (the token buffer is new per start)
    eng.run(20)
    assert torch.equal(eng.generated, fresh(pb))
    dec.set_prefix(pc)
    with pytest.raises(RuntimeError):
        eng.run(1)
    dec.clear_prefix()
    with pytest.raises(RuntimeError):
        eng.run(1)
    with pytest.raises(ValueError):
        dec.set_prefix(pa[:0])
    dec.set_prefix(pa)
    with pytest.raises(ValueError):
        dec.prefill(own, torch.arange(8, device=DEV).repeat(b, 1), torch.zeros(b, cfg.speaker_emb_dim, device=DEV))


def test_replacing_the_prefix_in_place_changes_the_replay():
    """One capture, two voices: the graph reads the prefix's length and rows at the replay."""
    cfg, b = tiny_config(), 2
    sd = synthetic_state_dict(cfg, seed=6)
    (pa, own), (pb, _) = prompts(cfg, b, 40, 7, 1), prompts(cfg, b, 55, 7, 2)
    dec = FusedDecoder(cfg, sd, DEV, batch=b, max_len=40)
    dec.set_prefix(pa, capacity=60)
    eng = DecodeEngine(dec, sampling=None)
    eng.start(own, None, 4)
    eng.capture()
    for prefix in (pb, pa):
        dec.set_prefix(prefix)
        generated = eng.generated
        eng.start(own, None, 4)
        args = (eng.input_ids.clone(), eng.positions.clone(), eng.slots.clone(), eng.kv_len.clone())
        conv = {i: c.clone() for i, c in dec.conv_state.items()}
        want = dec.step_greedy(*args).clone()
        for i, c in conv.items():
            dec.conv_state[i].copy_(c)
        eng.generated = generated
        eng.run(1)
        torch.cuda.synchronize()
        assert torch.equal(eng.input_ids.view(-1), want)


@pytest.mark.parametrize("b,with_prefix", [(1, False), (3, True)])
def test_eviction_in_the_engine(b, with_prefix):
    """Generation past the cache's end: weights accumulate as the definition says, the kept
    rows are the oracle's choice from them, and lengths, slots and positions go on."""
    cfg = tiny_config()
    sd = synthetic_state_dict(cfg, seed=9)
    prefix, own = prompts(cfg, b, 30, 6, 8)
    dec = FusedDecoder(cfg, sd, DEV, batch=b, max_len=48)
    if with_prefix:
        dec.set_prefix(prefix)
    before = 30 if with_prefix else 0
    eng = DecodeEngine(dec, cache_budget=24, cache_recent=5)
    eng.start(own, None, 120)
    eng.capture()
    assert not any(t.any() for t in eng.scores.values())              # capture leaves no trace
    eng.run(42)                                                        # rows 6 .. 47: the cache is full
    torch.cuda.synchronize()
    assert eng._filled == 48
    layer = cfg.attn_layers[-1]
    # every step's weights sum to 1 over prefix and own rows: 42 steps x 2 heads a group
    total = eng.scores[layer].sum(-1)
    if with_prefix:
        assert (total < 42 * 2).all() and (total > 0).all()
    else:
        torch.testing.assert_close(total, torch.full_like(total, 84.0), rtol=2.0 ** -16, atol=0)
    k, v = dec.k_cache[layer].clone(), dec.v_cache[layer].clone()
    sc = {i: t.cpu().clone() for i, t in eng.scores.items()}
    pos = eng.positions.clone()
    eng._evict()
    torch.cuda.synchronize()
    assert eng._filled == 24 and torch.equal(eng.positions, pos)
    assert (eng.slots == 24).all() and (eng.kv_len == 25).all()
    for i in range(b):
        for h in range(cfg.num_key_value_heads):
            at = O.evict(sc[layer][i, h].tolist(), 48, 24, 5, 6)
            assert torch.equal(dec.k_cache[layer][i, h, :24], k[i, h][at])
            assert torch.equal(dec.v_cache[layer][i, h, :24], v[i, h][at])
            assert torch.equal(eng.scores[layer][i, h, :24].cpu(), sc[layer][i, h][at])
            assert not eng.scores[layer][i, h, 24:].any()
    eng.run(78)                                                        # three more evictions
    torch.cuda.synchronize()
    assert int(eng.step_idx) == 120 and int(dec.err_flag.item()) == 0
    assert 24 < eng._filled <= 48 and (eng.kv_len == eng._filled + 1).all()
    tpf = cfg.tokens_per_frame
    assert (eng.positions == before + 6 + 120 // tpf).all()
    tok = eng.generated
    assert ((tok >= cfg.audio_tokens_start) | (tok == cfg.eos_token_id)).all()


def test_an_engine_that_never_fills_its_cache_generates_as_before():
    """With a budget but no eviction yet, greedy tokens equal those of the plain engine
    wherever the plain engine's choice is clear (the weights' accumulation changes the
    attention kernel, not its result beyond rounding)."""
    cfg = tiny_config()
    sd = synthetic_state_dict(cfg, seed=12)
    _, own = prompts(cfg, 2, 1, 8, 5)
    a, c = FusedDecoder(cfg, sd, DEV, batch=2, max_len=40), FusedDecoder(cfg, sd, DEV, batch=2, max_len=40)
    ea, ec = DecodeEngine(a), DecodeEngine(c, cache_budget=30)
    ea.start(own, None, 16)
    ec.start(own, None, 16)
    c.scores = ec.scores
    tokens = torch.randint(cfg.audio_tokens_start, cfg.vocab_size, (8, 2), generator=torch.Generator().manual_seed(4)).to(DEV)
    for got, ref in zip(feed(c, ec, tokens), feed(a, ea, tokens)):
        close(got, ref)
    c.scores = None


def test_sampling_history_holds_the_prefix():
    cfg = tiny_config()
    sd = synthetic_state_dict(cfg, seed=13)
    prefix, own = prompts(cfg, 2, 30, 6, 6)
    dec = FusedDecoder(cfg, sd, DEV, batch=2, max_len=40)
    dec.set_prefix(prefix)
    eng = DecodeEngine(dec, sampling=SamplingParams(seed=3))
    eng.start(own, None, 8)
    seen = seen_bitmap(torch.cat([prefix.expand(2, -1), own], 1), dec.num_reduced, dec.full_to_reduced, device=DEV)
    assert torch.equal(eng.seen & seen, seen)
    eng.capture()
    eng.run(8)
    torch.cuda.synchronize()
    assert int(eng.step_idx) == 8 and int(dec.err_flag.item()) == 0


def test_engine_refusals():
    cfg = tiny_config()
    dec = FusedDecoder(cfg, synthetic_state_dict(cfg, seed=1), DEV, batch=1, max_len=32)
    for kw in (dict(cache_budget=32), dict(cache_budget=0), dict(cache_recent=4), dict(cache_budget=8, cache_recent=9),
               dict(cache_budget=8, keep_mask=True)):
        with pytest.raises(ValueError):
            DecodeEngine(dec, **kw)
    own = torch.randint(10, 500, (1, 12), device=DEV)
    with pytest.raises(ValueError):
        DecodeEngine(dec, cache_budget=14, cache_recent=4).start(own, None, 100)
    with pytest.raises(ValueError):
        DecodeEngine(dec).start(own, None, 100)
