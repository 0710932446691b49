"""Outputs that share memory with themselves or with one another are refused before any
launch (no GPU needed: the checks look at shapes, strides and addresses alone)."""
from __future__ import annotations

import pytest
import torch

from kani_tts_b200 import fused_kernels as K


@pytest.mark.parametrize("shape,strides,fine", [
    ((2, 3, 5, 8), (120, 40, 8, 1), True),
    ((2, 3, 5, 8), (120, 8, 24, 1), True),          # slot-major
    ((2, 3, 5, 8), (240, 80, 16, 1), True),         # K and V rows interleaved
    ((2, 3, 5, 8), (0, 40, 8, 1), False),           # expanded
    ((1, 3, 5, 8), (0, 40, 8, 1), True),            # (a stride that is never followed)
    ((2, 3, 5, 8), (120, 40, 4, 1), False),         # windows that overlap
    ((2, 3, 5, 8), (120, 24, 8, 1), False),
    ((2, 3, 0, 8), (0, 0, 0, 1), True),             # nothing in it
])
def test_elements_of_an_output_lie_apart(shape, strides, fine):
    t = torch.zeros(1000).as_strided(shape, strides)
    if fine:
        K._refuse_shared(t, "out")
    else:
        with pytest.raises(ValueError):
            K._refuse_shared(t, "out")


def test_keys_and_values_lie_apart():
    a = torch.zeros(2, 3, 6, 2, 8)
    K._refuse_shared_rows(a[..., 0, :], a[..., 1, :])                       # interleaved rows
    K._refuse_shared_rows(a[:, :, :, 1, :], a[:, :, :, 0, :])
    K._refuse_shared_rows(torch.zeros(2, 3, 6, 8), torch.zeros(2, 3, 6, 8))
    b = torch.zeros(2, 2, 3, 6, 8)
    K._refuse_shared_rows(b[0], b[1])
    K._refuse_shared_rows(b[:, 0], b[:, 1])
    K._refuse_shared_rows(b[:, :, :, :3].flatten(0, 1), b[:, :, :, 3:].flatten(0, 1))
    c = torch.zeros(2, 3, 7, 8)
    for x, y in ((c, c), (c[:, :, :-1], c[:, :, 1:]), (c[..., :6], c[..., 2:]), (c[:, :2], c[:, 1:])):
        with pytest.raises(ValueError):
            K._refuse_shared_rows(x, y)
    K._refuse_shared_rows(c[:, :, :0], c[:, :, :0])                         # nothing in them


def test_lengths_and_kept_slots_lie_apart_from_the_other_outputs():
    a, b, c = torch.zeros(16), torch.zeros(16), torch.zeros(16)
    outs, ins = ((a, "a"), (a[4:], "a4")), ((b, "b"), (None, "none"))       # (outs among themselves: not looked at)
    K._refuse_overlap(outs, ins, ((c[:8], "c0"), (None, "none"), (c[8:], "c8")))
    for then in (((b[3:4], "x"),), ((a[15:], "x"),), ((c[:9], "x"), (c[8:], "y"))):
        with pytest.raises(ValueError):
            K._refuse_overlap(outs, ins, then)
    with pytest.raises(ValueError):
        K._refuse_overlap(((b[:1], "x"),), ins)
