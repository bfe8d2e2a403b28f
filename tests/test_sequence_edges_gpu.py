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


def owned(offsets, rows):
    """(sequence, begin, end) of the sequences that no bad entry starts or ends: below zero, behind the rows or lower than one in front."""
    found, highest = [], -2 ** 63
    for n, (b, e) in enumerate(zip(offsets, offsets[1:])):
        if 0 <= b <= e <= rows and b >= highest:
            found.append((n, b, e))
        highest = max(highest, b)
    return found


OFFSETS = [(90, [0, 5000], 0), (90, [-5, 60], 0), (90, [60, 30], 0), (3000, [0, 5000], 0), (90, [0, 50, 20, 90], 1), (90, [-40, 30, 60, 90], 2), (90, [0, 30, 60, 5000], 2), (90, [2 ** 40, 30, -2 ** 60, 2 ** 62], 0),
           (90, [0, 5000, 10, 5000], 0), (90, [5, 40, 40, 80, 70, 90], 3), (3000, [0, 1300, 900, 3000], 1), (3000, [0, 700, 2 ** 40, 2000, 3000], 1),
           (3000, [100, 2900, 2900, 2950, -1, 3000], 3), (3000, list(range(1500)) + [0] + list(range(1501, 2001)) + [1700] + list(range(2002, 3001)), 2996)]


@pytest.mark.parametrize("kind", ["bf16", "f32", "f64"])
@pytest.mark.parametrize("rows,offsets,count", OFFSETS, ids=lambda x: str(x)[:30])
def test_sequences_at_bad_offsets_are_left_alone(kind, rows, offsets, count):
    """Their rows, their states and the rows between them; the others get what they get without them."""
    n, d = len(offsets) - 1, 16
    good = owned(offsets, rows)
    assert len(good) == count
    p = Problem(kind, [rows] + [0] * (n - 1), True, 2, 1, d, d, spare=0)
    p.offsets = torch.tensor(offsets, device="cuda")
    out, end = p.forward()
    assert lib().acro_b200_device_status() == _lib.EINVAL
    grads = p.backward()
    assert lib().acro_b200_device_status() == _lib.EINVAL
    left, gone = torch.ones(rows, dtype=torch.bool, device="cuda"), [i for i in range(n) if i not in {s for s, _, _ in good}]
    for s, b, e in good:
        left[b:e] = False
    for x in (out,) + grads[:3]:
        assert bool((x[left] == -7.0).all())
    for x in (end, grads[3]):
        assert bool((x[gone] == -7.0).all())
    # one after the other, as many as there are different kinds of
    for s, b, e in good[:3] + good[-3:] + [g for g in good if g[0] in (1498, 1501, 1502, 1999, 2000, 2002, 2003)]:
        one = Problem(kind, [e - b], True, 2, 1, d, d, spare=0)
        one.q, one.k, one.v, one.dout = (x[b:e] for x in (p.q, p.k, p.v, p.dout))
        one.initial, one.dfinal = p.initial[s:s + 1], p.dfinal[s:s + 1]
        one.check_forward(out[b:e], end[s:s + 1])
        one.check_backward(*[x[b:e] for x in grads[:3]], grads[3][s:s + 1])


def engine_calls(te, bad):
    """(name, call of a result, the result's shape) of the engine's methods; with `bad` they are refused by the kernel layer: too many columns a
    head, a negative eps, rows too wide to be overwritten."""
    T, H, d = 5, 2, 257 if bad else 8
    rng = np.random.default_rng(0)
    t = lambda *s: ab.Tensor(s, hdata=rng.standard_normal(s))
    yield "out", lambda r: te.LinearAttention(r, t(T, H, d), t(T, H, d), t(T, H, d), t(H), 1.0, None, None), (T, H, d)
    yield "final", lambda r: te.LinearAttention(t(T, H, d), t(T, H, d), t(T, H, d), t(T, H, d), t(H), 1.0, None, r), (H, d, d)
    yield "step", lambda r: te.LinearAttentionStep(r, t(T, H, d, d), t(T, H, d), t(T, H, d), t(T, H, d), t(H), t(T, H, d, d), 1.0), (T, H, d)
    yield "dq", lambda r: te.LinearAttentionBackward(r, t(T, H, d), t(T, H, d), t(T, H, d), t(T, H, d), t(T, H, d), t(T, H, d), t(H), 1.0), (T, H, d)
    if bad:
        yield "norm", lambda r: te.LayerNorm(r, t(T, 9), eps=-1.0), (T, 9)
        y = t(2, 9000)
        yield "dweight", lambda r: te.LayerNormBackward(y, r, None, y, t(2, 9000), t(2), t(2)), (9000,)
    else:
        yield "norm", lambda r: te.LayerNorm(r, t(T, 9)), (T, 9)
        yield "dweight", lambda r: te.LayerNormBackward(t(T, 9), r, None, t(T, 9), t(T, 9), t(T), t(T)), (9,)


def test_engine_leaves_results_of_refused_calls_where_they_are():
    te = ab.TensorEngine("Cuda")
    for name, call, shape in engine_calls(te, True):
        result = ab.Tensor(shape, hdata=np.full(shape, 5.0))
        with pytest.raises(ab.AcroError):
            call(result)
        assert not result.IsOnGPU(), name
        result.MoveFromGPU()
        assert (result.numpy() == 5.0).all(), name
    status_ok()


def test_engine_keeps_the_rest_of_a_tensor_whose_part_is_written():
    te = ab.TensorEngine("Cuda")
    for name, call, shape in engine_calls(te, False):
        whole = ab.Tensor((3,) + shape, hdata=np.full((3,) + shape, 5.0))
        call(ab.SliceTensor(whole, 1))
        assert whole.IsOnGPU()
        whole.MoveFromGPU()
        assert (whole.numpy()[[0, 2]] == 5.0).all() and not (whole.numpy()[1] == 5.0).any(), name
    status_ok()
