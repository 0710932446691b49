"""What a decode engine with a cache budget accepts (no GPU needed)."""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200.decode import DecodeEngine
from test_engine_restart import Decoder


@pytest.mark.parametrize("recent", [None, 0, 3])
def test_the_budget_has_room_behind_the_prompt(recent):
    """A prompt is never cut, so one that takes the whole budget would cost every
    generated row at every eviction."""
    eng = DecodeEngine(Decoder(2), cache_budget=10, cache_recent=recent)
    for rows in range(10 - max(recent or 0, 1) + 1, 13):
        with pytest.raises(ValueError):
            eng.start(torch.zeros(2, rows, dtype=torch.long), None, 100)
    for rows in range(1, 10 - max(recent or 0, 1) + 1):
        eng.start(torch.zeros(2, rows, dtype=torch.long), None, 100)
