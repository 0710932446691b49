"""What set_prefix refuses before it touches a buffer (no GPU needed)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from kani_tts_b200.decode import FusedDecoder
from kani_tts_b200.model import tiny_config


class Pass(Exception):
    """The prompt pass was reached."""


def decoder():
    def prompt_pass(*args, **kw):
        raise Pass

    cfg = tiny_config()
    return SimpleNamespace(cfg=cfg, device=torch.device("cpu"), dtype=torch.bfloat16, hk=1, d=64, k_cache={}, v_cache={},
                           conv_state={}, prefix=None, _prompt_pass=prompt_pass)


@pytest.mark.parametrize("shape", [(9,), (1, 9)])
def test_one_sequence_is_taken(shape):
    with pytest.raises(Pass):
        FusedDecoder.set_prefix(decoder(), torch.ones(shape, dtype=torch.long))


@pytest.mark.parametrize("shape", [(2, 9), (1, 2, 9), (1, 1, 9), ()])
def test_several_sequences_are_not_run_together(shape):
    """One prefix serves all streams: a batch of prompts is not their concatenation."""
    with pytest.raises(ValueError):
        FusedDecoder.set_prefix(decoder(), torch.ones(shape, dtype=torch.long))


@pytest.mark.parametrize("speaker", [False, True])
def test_positions_of_another_length_are_refused(speaker):
    """Before the pass: it fills the buffers of a prefix that may be in use layer by layer."""
    spk = torch.zeros(1, 32) if speaker else None
    for n in (8, 10, 11):
        if n == 9 + speaker:
            continue
        with pytest.raises(ValueError):
            FusedDecoder.set_prefix(decoder(), torch.ones(9, dtype=torch.long), torch.arange(n).view(1, n), spk)
    with pytest.raises(Pass):
        FusedDecoder.set_prefix(decoder(), torch.ones(9, dtype=torch.long), torch.arange(9 + speaker).view(1, -1), spk)
