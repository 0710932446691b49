"""Starting a captured decode engine again: what the captured step reads and writes has to
outlive the start that it was captured after (no GPU needed).

A CUDA graph keeps addresses, not tensors.  The stand-in graph here keeps weak references
to the tensors that the captured step's last launches were given and runs those launches
at a replay, so a buffer that nothing else holds any more shows as a dead reference.
"""
from __future__ import annotations

import contextlib
import gc
import weakref

import pytest
import torch

from kani_tts_b200 import decode
from kani_tts_b200.decode import DecodeEngine
from kani_tts_b200.model import tiny_config
from kani_tts_b200.sampling import SamplingParams, seen_bitmap

V = 40


class Decoder:
    """The parts of FusedDecoder that the engine touches; its logits name the token `step`."""

    def __init__(self, b, max_len=64):
        self.cfg, self.batch, self.max_len, self.device = tiny_config(), b, max_len, torch.device("cpu")
        self.conv_state, self.k_cache, self.prefix, self.scores = {}, {}, None, None
        self.fused_greedy_head, self.fused_head = False, None
        self.head = torch.zeros(V, 4)
        self.reduced_to_full = torch.arange(V) + 600
        self.full_to_reduced = torch.full((700,), -1)
        self.full_to_reduced[600:600 + V] = torch.arange(V)
        self.next = 0

    def new_scores(self):
        return {}

    def _logits(self):
        self.next = (self.next + 1) % V
        return torch.nn.functional.one_hot(torch.full((self.batch, 1), self.next), V).float()

    def prefill(self, input_ids, positions, speaker_emb=None):
        return self._logits()

    def step(self, *args):
        return self._logits()


class Graph:
    def __init__(self):
        self.launches = []

    def replay(self):
        for fn, args in self.launches:
            args = [a() for a in args]
            assert all(a is not None for a in args), "a captured launch uses memory that was given back"
            fn(*args)


@pytest.fixture
def engine_on_cpu(monkeypatch):
    recording = []

    def launch(fn, *args):
        if recording:
            # (of a view its tensor; all of them are views of the same shape)
            recording[0].launches.append((fn, [weakref.ref(a if a._base is None else a._base) for a in args]))
        else:
            fn(*args)

    def advance(token, input_ids, generated, step):
        generated[:, int(step)] = token
        input_ids.copy_(token.view(-1, 1))
        step += 1

    def sample(seen, out, step):
        out.copy_(seen[:, 0].long() * 1000 + int(step))     # says which history it was given
        seen[:, 0] += 1

    monkeypatch.setattr(decode, "decode_advance", lambda token, ids, gen, step, *a, **kw: launch(advance, token, ids, gen, step))
    monkeypatch.setattr(decode, "sample_tokens", lambda logits, seen, out, step, **kw: launch(sample, seen, out, step))

    class Stream:
        def wait_stream(self, other):
            pass

    @contextlib.contextmanager
    def graph(g):
        recording.append(g)
        yield
        recording.pop()

    monkeypatch.setattr(torch.cuda, "Stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", graph)

    def make(b, sampling=None, **kw):
        eng = DecodeEngine(Decoder(b), sampling=sampling, **kw)
        if sampling is None:      # greedy tokens pass through a static buffer too, each one more than the last
            def next_token(logits):
                launch(lambda out, ids: out.copy_(ids.view(-1) + 1), eng.next_tok, eng.input_ids)
                return eng.next_tok
            eng._next_token = next_token
        return eng

    return make


def prompt(b, t, first):
    return torch.full((b, t), first)


def test_a_second_start_is_served_by_the_captured_step(engine_on_cpu):
    eng = engine_on_cpu(2)
    eng.start(prompt(2, 5, 20), None, 6)
    eng.capture()
    eng.input_ids.fill_(100)
    eng.run(6)
    assert eng.generated.tolist() == [[101, 102, 103, 104, 105, 106]] * 2
    eng.start(prompt(2, 7, 30), None, 6)
    gc.collect()
    eng.input_ids.fill_(200)
    eng.run(2)
    eng.run(3)
    assert eng.generated.tolist() == [[201, 202, 203, 204, 205, 0]] * 2


def test_results_of_an_earlier_start_stay(engine_on_cpu):
    eng = engine_on_cpu(1)
    results = []
    for first in (100, 200, 300):
        eng.start(prompt(1, 5, 20), None, 4)
        if not results:
            eng.capture()
        eng.input_ids.fill_(first)
        eng.run(4)
        results.append(eng.generated)
    assert [r.tolist() for r in results] == [[[f + 1, f + 2, f + 3, f + 4]] for f in (100, 200, 300)]


def test_the_sampler_of_a_second_start_knows_its_history(engine_on_cpu):
    eng = engine_on_cpu(1, sampling=SamplingParams())
    eng.start(prompt(1, 5, 603), None, 4)
    eng.capture()
    eng.run(1)
    eng.start(prompt(1, 5, 605), None, 4)
    gc.collect()
    # reduced token 5 is in the new prompt; the prefill's own sample was the first step
    seen = seen_bitmap(prompt(1, 5, 605), V, eng.dec.full_to_reduced)
    assert int(eng.seen[0, 0]) == int(seen[0, 0]) + 1
    eng.run(1)
    assert eng.generated[0, 0] == (int(seen[0, 0]) + 1) * 1000 + 1


def test_other_numbers_of_new_tokens(engine_on_cpu):
    eng = engine_on_cpu(1)
    eng.start(prompt(1, 5, 20), None, 8)
    with pytest.raises(RuntimeError):
        eng.run(1)                              # nothing captured yet
    eng.capture()
    eng.start(prompt(1, 5, 20), None, 3)        # fewer: the captured step serves them
    eng.input_ids.fill_(100)
    eng.run(5)
    assert eng.generated.tolist() == [[101, 102, 103]]
    eng.start(prompt(1, 5, 20), None, 9)        # more than it was captured for
    with pytest.raises(RuntimeError):
        eng.run(1)
    eng.capture()
    eng.input_ids.fill_(100)
    eng.run(9)
    assert eng.generated.tolist() == [list(range(101, 110))]


def test_eager_steps_and_replays_go_on_from_one_another(engine_on_cpu):
    eng = engine_on_cpu(1)
    eng.start(prompt(1, 5, 20), None, 5)
    eng.capture()
    eng.input_ids.fill_(100)
    eng._step_body()
    eng.run(2)
    eng._step_body()
    assert eng.generated.tolist() == [[101, 102, 103, 104, 0]]
