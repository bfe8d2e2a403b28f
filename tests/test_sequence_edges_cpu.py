"""What the sequence operators refuse without a GPU, beyond types and shapes: results whose rows overlap."""
import pytest

import acrotensor_b200 as ab
from acrotensor_b200 import _lib
from acrotensor_b200._lib import LinearAttentionDesc, TokenArray, lib

D = 16      # columns of every head below; addresses are never followed


def desc(sequences=2, tokens=3):
    return LinearAttentionDesc(type=2, q_heads=4, kv_heads=4, dk=D, dv=D, sequences=sequences, tokens=tokens, scale=1.0)


def rows(at, strides):
    return TokenArray(4096 * (at + 1), *strides)


#: sequence, token and head strides of 2 sequences of 3 tokens of 4 heads: rows that share entries, and rows that do not
OVERLAP = [(12 * D, D, D), (12 * D, 4 * D - 1, D), (12 * D - 8, 4 * D, D), (D, D, 6 * D), (3 * D, D, 3 * D), (6 * D, 4 * D, D), (2 ** 62, 2 ** 61, 2 ** 61)]
APART = [(12 * D, 4 * D, D), (12 * D, D, 3 * D), (D, 8 * D, 2 * D), (4 * D, 8 * D, D), (2 ** 62, 2 ** 60, 2 ** 40), (100 * D, 6 * D, D + 8)]


def forward(out, packed=None):
    plain = (12 * D, 4 * D, D)
    lib().acro_b200_linear_attention(desc(), rows(0, plain), rows(1, plain), rows(2, plain), rows(3, out), 1 << 20, packed, None, None, None, 2, None, 0, None)
    return lib().acro_b200_last_error()


def backward(which, strides):
    plain = (12 * D, 4 * D, D)
    arrays = [rows(i, strides if i == which else plain) for i in range(7)]
    lib().acro_b200_linear_attention_backward(desc(), *arrays[:4], 1 << 20, None, None, None, *arrays[4:], None, None, 0, None)
    return lib().acro_b200_last_error()


@pytest.mark.parametrize("strides", OVERLAP)
def test_results_whose_rows_overlap_are_refused(strides):
    assert b"out has rows that overlap" in forward(strides)
    for i, name in ((4, b"dq"), (5, b"dk"), (6, b"dv")):
        assert name + b" has rows that overlap" in backward(i, strides)


@pytest.mark.parametrize("strides", APART)
def test_results_whose_rows_are_apart_are_not(strides):
    """These addresses are no device's, which is looked at last."""
    assert b"not memory of the current device" in forward(strides)
    for i in range(7):
        assert b"not memory of the current device" in backward(i, strides)


def test_overlap_of_packed_rows_and_of_a_step():
    # the distance of sequences is not used when they are packed, that of tokens not in a step
    assert b"out has rows that overlap" in forward((0, D, D), packed=8192)
    assert b"not memory of the current device" in forward((0, 4 * D, D), packed=8192)
    step = desc(sequences=3, tokens=1)
    for strides, word in (((D, 0, D), b"out has rows that overlap"), ((4 * D, 0, D), b"not memory"), ((D, 0, 3 * D), b"not memory")):
        arrays = [rows(i, (4 * D, 4 * D, D)) for i in range(3)] + [rows(3, strides)]
        assert lib().acro_b200_linear_attention_step(step, *arrays, 1 << 20, 1 << 21, 1 << 21, None, 3, None) == _lib.EINVAL
        assert word in lib().acro_b200_last_error()


def test_engine_refuses_a_row_cut_over_the_ranks():
    """A rank has a part of the row, and no mean or variance of it."""
    te, stats = ab.TensorEngine("Cuda"), ab.Tensor(1)
    x = ab.Tensor(8)
    x.SetSharded(True)
    for call in (lambda: te.LayerNorm(ab.Tensor(8), x), lambda: te.LayerNormBackward(ab.Tensor(8), None, None, ab.Tensor(8), x, stats, stats)):
        with pytest.raises(ab.AcroError, match="sharded over its entries"):
            call()


STATE = 4 * D * D * 4       # bytes of one sequence's (request's) state


@pytest.mark.parametrize("shift", [1, STATE // 4, 2 * STATE // 4 - 1])
def test_states_that_overlap_without_being_the_same_are_refused(shift):
    """Sequence 0 would write what sequence 1 starts from."""
    plain = (12 * D, 4 * D, D)
    at, log_decay = 1 << 30, 1 << 20
    for other, word in ((at + 4 * shift, b"overlap"), (at - 4 * shift, b"overlap"), (at + 2 * STATE, b"not memory"), (at - 2 * STATE, b"not memory"),
                        (at, b"not memory")):
        assert lib().acro_b200_linear_attention(desc(), *[rows(i, plain) for i in range(4)], log_decay, None, at, other, None, 2, None, 0, None) == _lib.EINVAL
        assert word in lib().acro_b200_last_error()
        assert lib().acro_b200_linear_attention_step(desc(tokens=1), *[rows(i, plain) for i in range(4)], log_decay, at, other, None, 2, None) == _lib.EINVAL
        assert word in lib().acro_b200_last_error()
        for states in ((at, None, other), (None, at, other)):
            initial, d_final, d_initial = states
            assert lib().acro_b200_linear_attention_backward(desc(), *[rows(i, plain) for i in range(4)], log_decay, None, initial, d_final,
                                                             *[rows(i, plain) for i in range(4, 7)], d_initial, None, 0, None) == _lib.EINVAL
            assert (b"not memory" in lib().acro_b200_last_error()) == (abs(other - at) == 2 * STATE)


def test_statistics_in_one_place_are_refused():
    at = [4096 * (i + 1) for i in range(5)]
    call = lambda mean, rstd: lib().acro_b200_layer_norm(2, at[0], 8, at[1], at[2], at[3], 8, mean, rstd, 3, 8, 1e-5, None)
    assert call(at[4], at[4]) == _lib.EINVAL and b"same place" in lib().acro_b200_last_error()
    for mean, rstd in ((None, None), (at[4], None), (None, at[4]), (at[4], at[4] + 64)):
        assert call(mean, rstd) == _lib.EINVAL and b"memory of the current device" in lib().acro_b200_last_error()
