"""The sequence operators without a GPU: what their calls refuse before anything is launched, the scratch they ask for, and the 64-bit
reference of the GPU tests against differences."""
import ctypes

import numpy as np
import pytest
import torch

import acrotensor_b200 as ab
import sequence_reference as ref
from acrotensor_b200 import _lib
from acrotensor_b200._lib import LinearAttentionDesc, lib


def arrays(lead=(2, 5), heads=4, kv=2, dk=8, dv=16, dtype=torch.bfloat16, states=2):
    a = {"q": torch.zeros(lead + (heads, dk), dtype=dtype), "k": torch.zeros(lead + (kv, dk), dtype=dtype),
         "v": torch.zeros(lead + (kv, dv), dtype=dtype), "out": torch.zeros(lead + (heads, dv), dtype=dtype)}
    sums = torch.float64 if dtype == torch.float64 else torch.float32
    a["g"], a["s"] = torch.zeros(heads, dtype=sums), torch.zeros(states, heads, dk, dv, dtype=sums)
    return a


def forward(a, **kw):
    ab.linear_attention(kw.pop("out", a["out"]), a["q"], a["k"], a["v"], a["g"], **kw)


@pytest.mark.parametrize("change", [
    lambda a: a.update(q=a["q"].to(torch.int32)), lambda a: a.update(k=a["k"].float()), lambda a: a.update(out=a["out"].float()),
    lambda a: a.update(k=a["k"][:, :4]), lambda a: a.update(v=a["v"][..., :1, :]), lambda a: a.update(q=a["q"][0]),
    lambda a: a.update(out=a["out"][..., :8]), lambda a: a.update(g=a["g"][:2]), lambda a: a.update(g=a["g"].double()),
    lambda a: a.update(q=torch.zeros(2, 5, 8, 4, dtype=torch.bfloat16).transpose(2, 3)), lambda a: a.update(k=a["k"][..., :7])])
def test_forward_refuses_arrays(change):
    a = arrays()
    change(a)
    with pytest.raises((ValueError, ab.AcroError)):
        forward(a)


@pytest.mark.parametrize("kw", [
    {"initial_state": torch.zeros(2, 4, 8, 15)}, {"initial_state": torch.zeros(3, 4, 8, 16)}, {"final_state": torch.zeros(2, 4, 8, 16, dtype=torch.float64)},
    {"final_state": torch.zeros(2, 4, 16, 8).transpose(2, 3)}, {"slots": torch.zeros(2, dtype=torch.int64)}, {"slots": torch.zeros(3, dtype=torch.int32)},
    {"scale": float("nan")}, {"scale": float("inf")}])
def test_forward_refuses_states(kw):
    with pytest.raises((ValueError, ab.AcroError)):
        forward(arrays(), **kw)


def test_packed_refuses():
    a = arrays(lead=(7,))
    for offsets in (torch.zeros(3, dtype=torch.int32), torch.zeros((3, 1), dtype=torch.int64), torch.zeros(0, dtype=torch.int64)):
        with pytest.raises(ValueError):
            forward(a, offsets=offsets)
    with pytest.raises(ValueError):
        forward(arrays(), offsets=torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("field,value", [("q_heads", 3), ("q_heads", 0), ("kv_heads", 0), ("dk", 0), ("dk", 257), ("dv", -1), ("dv", 300), ("type", 4),
                                         ("type", -1), ("sequences", -1), ("tokens", -1)])
def test_descriptor_refusals(field, value):
    good = dict(type=2, q_heads=4, kv_heads=2, dk=8, dv=16, sequences=2, tokens=5, scale=1.0)
    desc = LinearAttentionDesc(**{**good, field: value})
    none = [None] * 4
    assert lib().acro_b200_linear_attention(desc, *none, None, None, None, None, None, 2, None, 0, None) == _lib.EINVAL
    assert lib().acro_b200_last_error()
    assert lib().acro_b200_linear_attention_scratch_bytes(desc, 0) == 0
    assert lib().acro_b200_linear_attention_backward_scratch_bytes(desc, 1) == 0


def test_null_arrays_and_descriptor():
    assert lib().acro_b200_linear_attention(None, None, None, None, None, None, None, None, None, None, 0, None, 0, None) == _lib.EINVAL
    desc = LinearAttentionDesc(type=2, q_heads=4, kv_heads=2, dk=8, dv=16, sequences=2, tokens=5, scale=1.0)
    assert lib().acro_b200_linear_attention(desc, None, None, None, None, None, None, None, None, None, 2, None, 0, None) == _lib.EINVAL
    assert lib().acro_b200_linear_attention_step(desc, None, None, None, None, None, None, None, None, 2, None) == _lib.EINVAL     # tokens is not 1
    desc.tokens = 1
    assert lib().acro_b200_linear_attention_step(desc, None, None, None, None, None, None, None, None, 2, None) == _lib.EINVAL
    desc.sequences = 0
    assert lib().acro_b200_linear_attention_step(desc, None, None, None, None, None, None, None, None, 0, None) == _lib.OK
    assert lib().acro_b200_linear_attention(desc, None, None, None, None, None, None, None, None, None, 0, None, 0, None) == _lib.OK


def test_host_memory_is_refused():
    """No device here, or memory that is not a device's: an error, not a launch."""
    with pytest.raises(ab.AcroError):
        forward(arrays())
    x = torch.zeros(3, 8)
    with pytest.raises(ab.AcroError):
        ab.layer_norm(x.clone(), x)


def test_scratch_grows_with_segments_and_shared_heads():
    a = arrays(lead=(1, 64), heads=4, kv=4)
    assert ab.linear_attention_scratch_bytes(a["q"], a["k"], a["v"]) == 0                   # one segment
    b = arrays(lead=(1, 65536), heads=1, kv=1)
    assert ab.linear_attention_scratch_bytes(b["q"], b["k"], b["v"]) >= 2 * 8 * 16 * 4      # a state per segment
    assert ab.linear_attention_backward_scratch_bytes(b["q"], b["k"], b["v"]) > ab.linear_attention_scratch_bytes(b["q"], b["k"], b["v"])
    c = arrays(lead=(1, 64), heads=4, kv=2)
    assert ab.linear_attention_backward_scratch_bytes(c["q"], c["k"], c["v"]) >= 64 * 4 * (8 + 16) * 4
    with pytest.raises(ValueError):
        ab.linear_attention(b["out"], b["q"], b["k"], b["v"], b["g"])                        # no scratch given


def test_scratch_does_not_grow_with_the_number_of_packed_sequences():
    few, many = torch.zeros(3, dtype=torch.int64), torch.zeros(5001, dtype=torch.int64)
    for dtype in (torch.bfloat16, torch.float32, torch.float64):
        a = arrays(lead=(65536,), heads=2, kv=2, dtype=dtype)
        for bytes_of in (ab.linear_attention_scratch_bytes, ab.linear_attention_backward_scratch_bytes):
            assert 0 < bytes_of(a["q"], a["k"], a["v"], many) == bytes_of(a["q"], a["k"], a["v"], few)


def test_sizes_that_no_memory_holds_are_refused():
    """Sizes whose scratch would pass 64 bits: an error, not a small scratch."""
    for sequences, tokens, packed in ((1, 2 ** 62, 0), (2 ** 62, 1, 1), (2 ** 40, 2 ** 40, 0), (3, 2 ** 39, 1)):
        desc = LinearAttentionDesc(type=1, q_heads=4, kv_heads=2, dk=8, dv=16, sequences=sequences, tokens=tokens, scale=1.0)
        assert lib().acro_b200_linear_attention_scratch_bytes(desc, packed) == 0
        assert lib().acro_b200_linear_attention(desc, *[None] * 4, None, None, None, None, None, sequences, None, 0, None) == _lib.EINVAL
        assert b"2^40 rows" in lib().acro_b200_last_error()


def between_elements(call, count):
    """Addresses (never followed: this memory is no device's) of which one at a time is off its elements by a byte."""
    for bad in range(count):
        at = [4096 * (i + 1) + (i == bad) for i in range(count)]
        assert call(at) == _lib.EINVAL and b"aligned to its elements" in lib().acro_b200_last_error(), bad


def test_pointers_between_elements_are_refused():
    """They would fault on the device."""
    desc = LinearAttentionDesc(type=2, q_heads=1, kv_heads=1, dk=16, dv=16, sequences=1, tokens=1, scale=1.0)
    rows = lambda at: [_lib.TokenArray(a, 16, 16, 16) for a in at]
    between_elements(lambda at: lib().acro_b200_linear_attention(desc, *rows(at[:4]), *at[4:9], 1, None, 0, None), 9)
    between_elements(lambda at: lib().acro_b200_linear_attention_step(desc, *rows(at[:4]), *at[4:8], 1, None), 8)
    between_elements(lambda at: lib().acro_b200_linear_attention_backward(desc, *rows(at[:4]), *at[4:8], *rows(at[8:11]), at[11], None, 0, None), 12)
    between_elements(lambda at: lib().acro_b200_layer_norm(2, at[0], 8, at[1], at[2], at[3], 8, at[4], at[5], 3, 8, 1e-5, None), 6)
    between_elements(lambda at: lib().acro_b200_layer_norm_backward(2, at[0], 8, at[1], 8, *at[2:6], 8, at[6], at[7], 3, 8, None, 0, None), 8)


def test_two_results_in_one_place_are_refused():
    """And a step's result in the place of an operand that other heads still read.  (Addresses that are never followed.)"""
    desc = LinearAttentionDesc(type=2, q_heads=1, kv_heads=1, dk=16, dv=16, sequences=1, tokens=1, scale=1.0)
    rows = [_lib.TokenArray(4096 * (i + 1), 16, 16, 16) for i in range(4)]
    for operand in rows[:3]:
        assert lib().acro_b200_linear_attention_step(desc, *rows[:3], operand, *[1 << 20] * 3, None, 1, None) == _lib.EINVAL
    at = [4096 * (i + 1) for i in range(6)]
    assert lib().acro_b200_layer_norm_backward(2, at[0], 8, at[1], 8, *at[2:6], 8, 1 << 20, 1 << 20, 3, 8, None, 0, None) == _lib.EINVAL
    assert b"same place" in lib().acro_b200_last_error()


@pytest.mark.parametrize("kw", [
    {"weight": torch.zeros(7)}, {"weight": torch.zeros(8, dtype=torch.float64)}, {"bias": torch.zeros(16)[::2]}, {"mean": torch.zeros(2)},
    {"mean": torch.zeros(3, dtype=torch.float64)}, {"out": torch.zeros(3, 7)}, {"out": torch.zeros(3, 8, dtype=torch.float16)}, {"eps": -1.0},
    {"eps": float("nan")}, {"out": torch.zeros(8, 3).t()}])
def test_norm_refuses(kw):
    x = torch.zeros(3, 8)
    with pytest.raises((ValueError, ab.AcroError)):
        ab.layer_norm(kw.pop("out", torch.zeros(3, 8)), x, **kw)


def test_norm_refuses_uneven_rows_and_bad_sizes():
    x = torch.zeros(4, 6, 8)[:, :3]
    with pytest.raises(ValueError):
        ab.layer_norm(torch.zeros(4, 3, 8), x)
    null = None
    assert lib().acro_b200_layer_norm(2, null, 8, null, null, null, 8, null, null, 3, 0, 1e-5, null) == _lib.EINVAL
    assert lib().acro_b200_layer_norm(7, null, 8, null, null, null, 8, null, null, 3, 8, 1e-5, null) == _lib.EINVAL
    assert lib().acro_b200_layer_norm(2, null, 8, null, null, null, 8, null, null, -1, 8, 1e-5, null) == _lib.EINVAL
    assert lib().acro_b200_layer_norm(2, null, 8, null, null, null, 8, null, null, 0, 8, 1e-5, null) == _lib.OK
    assert lib().acro_b200_layer_norm_backward_scratch_bytes(2, 0, 8) == 0
    assert lib().acro_b200_layer_norm_backward_scratch_bytes(2, 100, 8) >= 2 * 8 * 4


def test_engine_checks_dims_before_the_device():
    te = ab.TensorEngine("Cuda")
    q, k, v, g = ab.Tensor(5, 4, 8), ab.Tensor(5, 2, 8), ab.Tensor(5, 2, 16), ab.Tensor(4)
    out = ab.Tensor(5, 4, 16)
    for bad in ((ab.Tensor(5, 4, 8), q, k, v, g), (out, q, ab.Tensor(6, 2, 8), v, g), (out, q, k, v, ab.Tensor(3)), (out, ab.Tensor(4, 8), k, v, g)):
        with pytest.raises(ab.AcroError) as e:
            te.LinearAttention(*bad, 1.0)
        assert e.value.status == _lib.EINVAL
    with pytest.raises(ab.AcroError):
        te.LayerNorm(ab.Tensor(3, 7), ab.Tensor(3, 8))
    with pytest.raises(ab.AcroError):
        te.LayerNorm(ab.Tensor(3, 8), ab.Tensor(3, 8), ab.Tensor(7))
    lib().acro_engine_layer_norm.restype = ctypes.c_int
    assert lib().acro_engine_layer_norm(None, None, None, None, None, 1e-5, None, None) == _lib.EINVAL


def test_reference_gradient_against_differences():
    rng = np.random.default_rng(3)
    T, H, kv, dk, dv = 4, 2, 1, 3, 2
    q, k, v = rng.standard_normal((T, H, dk)), rng.standard_normal((T, kv, dk)), rng.standard_normal((T, kv, dv))
    s, g = rng.standard_normal((H, dk, dv)), np.array([-0.3, -1.1])
    do, ds = rng.standard_normal((T, H, dv)), rng.standard_normal((H, dk, dv))

    def loss(q, k, v, s):
        out, final = ref.attention(q, k, v, g, 0.7, s)
        return (out * do).sum() + (final * ds).sum()

    grads = ref.attention_backward(q, k, v, g, 0.7, s, do, ds)
    for n, grad in enumerate(grads):
        for i in np.ndindex(grad.shape):
            a, b = [x.copy() for x in (q, k, v, s)], [x.copy() for x in (q, k, v, s)]
            a[n][i] += 1e-5
            b[n][i] -= 1e-5
            assert abs((loss(*a) - loss(*b)) / 2e-5 - grad[i]) < 1e-8
