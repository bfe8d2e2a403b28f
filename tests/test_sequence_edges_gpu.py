"""Calls of the sequence operators that the documentation allows and that go wrong most easily: slots without states, offsets of which some are
bad, rows that overlap."""
import numpy as np
import pytest
import torch

import acrotensor_b200 as ab
import sequence_reference as ref
from acrotensor_b200 import _lib
from acrotensor_b200._lib import lib
from test_sequence_gpu import Problem, scratch_for, status_ok, stream, within, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f32", "f64"])
@pytest.mark.parametrize("lengths,packed", [([70, 40, 130], True), ([150] * 3, False), ([2100, 900, 1500], True)])
def test_slots_without_states_only_say_which_sequences_are_there(kind, lengths, packed):
    p = Problem(kind, lengths, packed, 2, 1, 32, 32, states=False)
    expect, _ = p.forward(final=False)
    out = p.blank(2, 32)
    ab.linear_attention(out, p.q, p.k, p.v, p.g, scale=p.scale, offsets=p.offsets, slots=torch.tensor([2 ** 31 - 1, -1, 0], dtype=torch.int32, device="cuda"),
                        scratch=scratch_for(ab.linear_attention_scratch_bytes(p.q, p.k, p.v, p.offsets)), stream=stream())
    status_ok()
    for i in (0, 2):
        assert torch.equal(p.of(out, i), p.of(expect, i))
    assert bool((p.of(out, 1) == -7.0).all())
    p.untouched(out)
