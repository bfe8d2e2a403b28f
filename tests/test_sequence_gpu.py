"""The sequence operators on the GPU against the 64-bit reference (sequence_reference.py, which derives the tolerances): types, head layouts,
lengths, strides, states, slots, packed sequences, rows that no sequence owns, non-finite values beside finite ones, streams and graphs."""
import numpy as np
import pytest
import torch

import acrotensor_b200 as ab
import sequence_reference as ref
from acrotensor_b200 import _lib
from acrotensor_b200._lib import lib

pytestmark = pytest.mark.gpu

DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def sums_of(kind):
    return torch.float64 if kind == "f64" else torch.float32


def scratch_for(n):
    # poisoned: nothing may be read before it is written
    return torch.full((max(n, 8) // 8 + 1,), float("nan"), dtype=torch.float64, device="cuda")


def wide(x):
    return x.detach().cpu().double().numpy()


class Problem:
    """Inputs of one call, rows of all sequences one behind the other with spare rows in front (packed only) and behind."""

    def __init__(self, kind, lengths, packed, heads, kv, dk, dv, states=True, seed=0, decay=None, fused=False, spare=3, lead=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.kind, self.lengths, self.packed, self.heads, self.kv, self.dk, self.dv = kind, lengths, packed, heads, kv, dk, dv
        dt, sums = DTYPES[kind], sums_of(kind)
        n = len(lengths)
        shape = (lead + sum(lengths) + spare,) if packed else (n, lengths[0])

        def rows(h, c):
            return torch.randn(shape + (h, c), generator=g, device="cuda").to(dt)

        if fused:       # one buffer of q, k and v columns beside one another: strides that are not the heads' own
            total = heads * dk + kv * dk + kv * dv + 8
            buf = torch.randn(shape + (total,), generator=g, device="cuda").to(dt)
            cut = [0, heads * dk, heads * dk + kv * dk, heads * dk + kv * dk + kv * dv]
            self.q = buf[..., cut[0]:cut[1]].unflatten(-1, (heads, dk))
            self.k = buf[..., cut[1]:cut[2]].unflatten(-1, (kv, dk))
            self.v = buf[..., cut[2]:cut[3]].unflatten(-1, (kv, dv))
        else:
            self.q, self.k, self.v = rows(heads, dk), rows(kv, dk), rows(kv, dv)
        self.dout = rows(heads, dv)
        if decay is None:
            decay = -torch.exp2(-torch.linspace(0, 9, heads, dtype=torch.float64))
        self.g = torch.as_tensor(decay, dtype=torch.float64).to(sums).cuda()
        self.scale = dk ** -0.5
        state = (n, heads, dk, dv)
        self.initial = torch.randn(state, generator=g, device="cuda").to(sums) if states else None
        self.dfinal = torch.randn(state, generator=g, device="cuda").to(sums) if states else None
        self.starts = [lead + sum(lengths[:i]) for i in range(n)]
        self.offsets = torch.tensor(self.starts + [lead + sum(lengths)], dtype=torch.int64, device="cuda") if packed else None
        self.spare_rows = [] if not packed else list(range(lead)) + list(range(lead + sum(lengths), shape[0]))
        if packed:      # what no sequence owns must not be read
            for x in (self.q, self.k, self.v, self.dout):
                x[self.spare_rows] = float("nan")

    def of(self, x, i):
        return x[self.starts[i]:self.starts[i] + self.lengths[i]] if self.packed else x[i]

    def blank(self, h, c):
        return torch.full(tuple(self.q.shape[:-2]) + (h, c), -7.0, dtype=DTYPES[self.kind], device="cuda")

    def forward(self, final=True, scratch=None):
        out = self.blank(self.heads, self.dv)
        end = torch.full((len(self.lengths), self.heads, self.dk, self.dv), -7.0, dtype=sums_of(self.kind), device="cuda") if final else None
        if scratch is None:
            scratch = scratch_for(ab.linear_attention_scratch_bytes(self.q, self.k, self.v, self.offsets))
        ab.linear_attention(out, self.q, self.k, self.v, self.g, scale=self.scale, offsets=self.offsets, initial_state=self.initial, final_state=end,
                            scratch=scratch, stream=stream())
        return out, end

    def backward(self, dinitial=True):
        dq, dk, dv = self.blank(self.heads, self.dk), self.blank(self.kv, self.dk), self.blank(self.kv, self.dv)
        first = torch.full((len(self.lengths), self.heads, self.dk, self.dv), -7.0, dtype=sums_of(self.kind), device="cuda") if dinitial else None
        scratch = scratch_for(ab.linear_attention_backward_scratch_bytes(self.q, self.k, self.v, self.offsets))
        ab.linear_attention_backward(dq, dk, dv, self.dout, self.q, self.k, self.v, self.g, scale=self.scale, offsets=self.offsets,
                                     initial_state=self.initial, d_final_state=self.dfinal, d_initial_state=first, scratch=scratch, stream=stream())
        return dq, dk, dv, first

    def state(self, x, i):
        return None if x is None else wide(x[i])

    def check_forward(self, out, end, rows=None):
        g = wide(self.g)
        for i, T in enumerate(self.lengths):
            a = [wide(self.of(x, i)) for x in (self.q, self.k, self.v)]
            s = self.state(self.initial, i)
            exact, final = ref.attention(*a, g, self.scale, s)
            mag, fmag = ref.attention(*[np.abs(x) for x in a], g, self.scale, None if s is None else np.abs(s))
            within(wide(self.of(out, i)), exact, ref.attention_tolerance(self.kind, exact, mag, T, self.dk), ("out", i))
            if end is not None:
                within(wide(end[i]), final, ref.attention_tolerance(state_kind(self.kind), final, fmag, T, 1, rounded=False), ("final", i))
        self.untouched(out)

    def untouched(self, *arrays):
        for x in arrays:
            if self.packed and self.spare_rows:
                assert bool((x[self.spare_rows] == -7.0).all())

    def check_backward(self, dq, dk, dv, first):
        g = wide(self.g)
        for i, T in enumerate(self.lengths):
            a = [wide(self.of(x, i)) for x in (self.q, self.k, self.v)]
            do, s, e = wide(self.of(self.dout, i)), self.state(self.initial, i), self.state(self.dfinal, i)
            exact = ref.attention_backward(*a, g, self.scale, s, do, e)
            mag = ref.attention_backward(*[np.abs(x) for x in a], g, self.scale, *[None if x is None else np.abs(x) for x in (s, do, e)])
            columns = max(self.dk, self.dv) + self.heads // self.kv
            for name, got, x, m in zip(("dq", "dk", "dv"), (dq, dk, dv), exact, mag):
                within(wide(self.of(got, i)), x, ref.attention_tolerance(self.kind, x, m, T, columns), (name, i))
            if first is not None:
                within(wide(first[i]), exact[3], ref.attention_tolerance(state_kind(self.kind), exact[3], mag[3], T, 1, rounded=False), ("first", i))
        self.untouched(dq, dk, dv)


def state_kind(kind):
    """States are sums in 32 (64) bits: no operand of theirs loses bits."""
    return "f64" if kind == "f64" else "f32x"


ref.HALF_STEP["f32x"], ref.SUM_HALF_STEP["f32x"], ref.SPLIT["f32x"] = 2.0 ** -24, 2.0 ** -24, 2.0 ** -23


def within(got, exact, tolerance, what):
    assert got.shape == exact.shape
    bad = ~(np.abs(got - exact) <= tolerance)
    assert not bad.any(), "%s: %d of %d entries, worst %.3g times the tolerance" % (
        what, bad.sum(), bad.size, np.nanmax(np.abs(got - exact) / tolerance))


def status_ok():
    assert lib().acro_b200_device_status() == _lib.OK, lib().acro_b200_last_error()


SHAPES = [  # lengths, packed, heads, kv_heads, dk, dv, fused
    ([1], False, 1, 1, 1, 1, False), ([1, 1], False, 2, 1, 64, 64, False), ([64], False, 2, 2, 64, 64, False), ([65, 65], False, 4, 2, 32, 16, True),
    ([0, 5, 0, 130, 1, 64, 63], True, 2, 1, 128, 128, False), ([200], True, 3, 3, 80, 48, True), ([33, 97], True, 6, 2, 72, 128, False),
    ([129, 40], True, 2, 2, 7, 13, False), ([70], False, 1, 1, 256, 256, False), ([150], True, 2, 1, 129, 250, False), ([0, 0], True, 1, 1, 16, 16, False),
    ([191, 2, 128], True, 4, 4, 64, 128, True), ([300], False, 2, 1, 96, 33, False)]


@pytest.mark.parametrize("kind", ["bf16", "f32", "f16", "f64"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[0])) + "x%dx%dx%dx%d" % s[2:6])
def test_forward(kind, shape):
    lengths, packed, heads, kv, dk, dv, fused = shape
    for states in (True, False):
        p = Problem(kind, lengths, packed, heads, kv, dk, dv, states=states, fused=fused, seed=len(lengths) + dk, lead=4 if packed else 0)
        p.check_forward(*p.forward(final=True))
    status_ok()


@pytest.mark.parametrize("kind", ["bf16", "f32", "f16", "f64"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[0])) + "x%dx%dx%dx%d" % s[2:6])
def test_backward(kind, shape):
    lengths, packed, heads, kv, dk, dv, fused = shape
    for states in (True, False):
        p = Problem(kind, lengths, packed, heads, kv, dk, dv, states=states, fused=fused, seed=len(lengths) + dv, lead=4 if packed else 0)
        p.check_backward(*p.backward())
    status_ok()


@pytest.mark.parametrize("kind,dk", [("bf16", 64), ("bf16", 128), ("bf16", 48), ("f32", 64), ("f64", 16), ("f16", 20)])
def test_long_sequences_are_cut_and_joined(kind, dk):
    """Few heads: segments beside one another, the same result as one after the other."""
    for lengths, packed in (([2500], False), ([700, 0, 1900, 3], True)):
        p = Problem(kind, lengths, packed, 2, 1, dk, dk, decay=[-1 / 64, -1 / 900])
        assert ab.linear_attention_scratch_bytes(p.q, p.k, p.v, p.offsets) > 0
        p.check_forward(*p.forward())
        p.check_backward(*p.backward())
    status_ok()


@pytest.mark.parametrize("kind,dk,dv", [("bf16", 64, 64), ("bf16", 128, 128), ("f32", 40, 24)])
def test_decays_at_their_ends(kind, dk, dv):
    """No decay at all, complete decay, and decays whose powers leave the type's range within a chunk."""
    p = Problem(kind, [260, 70], True, 6, 6, dk, dv, decay=[0.0, float("-inf"), -300.0, -5.0, -1e-7, -0.7])
    p.check_forward(*p.forward())
    p.check_backward(*p.backward())


@pytest.mark.parametrize("kind,d", [("bf16", 64), ("bf16", 128), ("bf16", 33), ("f32", 64), ("f64", 16)])
def test_later_and_other_tokens_do_not_reach_a_row(kind, d):
    """Infinities and NaN of a later token, or of another sequence, meet weights of zero: they must not become NaN."""
    p = Problem(kind, [100, 150, 90], True, 2, 2, d, d)
    clean, _ = p.forward()
    clean_grads = p.backward()
    bad = p.starts[1] + 77
    for x in (p.q, p.k, p.v, p.dout):
        x[bad] = float("nan")
        x[bad, :, 1] = float("inf")
    out, end = p.forward()
    assert torch.equal(out[:bad], clean[:bad]) and torch.equal(out[p.starts[2]:], clean[p.starts[2]:])
    assert bool(torch.isnan(out[bad:p.starts[2]].float()).any(-1).all())
    assert bool(torch.isfinite(end[0]).all()) and bool(torch.isfinite(end[2]).all()) and not bool(torch.isfinite(end[1]).all())
    dq, dk, dv, first = p.backward()
    for got, was in ((dk, clean_grads[1]), (dv, clean_grads[2])):
        assert torch.equal(got[bad + 1:], was[bad + 1:]) and torch.equal(got[:p.starts[1]], was[:p.starts[1]])
    assert torch.equal(dq[:bad], clean_grads[0][:bad]) and torch.equal(dq[p.starts[2]:], clean_grads[0][p.starts[2]:])
    assert torch.equal(first[0], clean_grads[3][0]) and torch.equal(first[2], clean_grads[3][2])


@pytest.mark.parametrize("kind,d", [("bf16", 128), ("f32", 64)])
def test_same_bits_on_every_run(kind, d):
    p = Problem(kind, [900, 300], True, 4, 2, d, d)
    a, b = p.forward() + p.backward(), p.forward() + p.backward()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", ["bf16", "f32", "f16", "f64"])
@pytest.mark.parametrize("n,heads,kv,dk,dv", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (5, 2, 2, 128, 128), (2, 6, 3, 72, 33), (4, 2, 1, 256, 250), (9, 1, 1, 7, 256)])
def test_step(kind, n, heads, kv, dk, dv):
    p = Problem(kind, [1] * n, False, heads, kv, dk, dv, seed=dk)
    out, state = torch.zeros((n, heads, dv), dtype=DTYPES[kind], device="cuda"), torch.empty_like(p.initial)
    ab.linear_attention_step(out, state, p.q[:, 0], p.k[:, 0], p.v[:, 0], p.g, p.initial, scale=p.scale, stream=stream())
    p.check_forward(out[:, None], state)
    # in place
    again, mine = torch.zeros_like(out), p.initial.clone()
    ab.linear_attention_step(again, mine, p.q[:, 0], p.k[:, 0], p.v[:, 0], p.g, mine, scale=p.scale, stream=stream())
    assert torch.equal(again, out) and torch.equal(mine, state)
    status_ok()


def test_slots_of_a_step():
    """Permuted slots, requests that are not there, and slots out of range or used twice: skipped and reported, nothing else touched."""
    n, states, h, d = 6, 9, 2, 64
    p = Problem("bf16", [1] * n, False, h, h, d, d)
    cache = torch.randn(states, h, d, d, device="cuda")

    def run(slots):
        mine, out = cache.clone(), torch.full((n, h, d), -7.0, dtype=torch.bfloat16, device="cuda")
        ab.linear_attention_step(out, mine, p.q[:, 0], p.k[:, 0], p.v[:, 0], p.g, mine, scale=p.scale,
                                 slots=torch.tensor(slots, dtype=torch.int32, device="cuda"), stream=stream())
        return out, mine

    def check(slots, live):
        out, mine = run(slots)
        touched = {slots[r] for r in live}
        for r in range(n):
            if r in live:
                q, k, v = (wide(x[r]) for x in (p.q, p.k, p.v))
                exact, final = ref.attention(q, k, v, wide(p.g), p.scale, wide(cache[slots[r]]))
                assert np.allclose(wide(out[r]), exact[0], rtol=2.0 ** -8, atol=1e-4) and np.allclose(wide(mine[slots[r]]), final, rtol=1e-6, atol=1e-6)
            else:
                assert bool((out[r] == -7.0).all())
        for s in set(range(states)) - touched:
            assert torch.equal(mine[s], cache[s])

    check([8, 0, 3, 2, 7, 1], range(6))
    check([8, -1, 3, -5, 7, 1], [0, 2, 4, 5])
    status_ok()
    check([4, 9, 3, 2 ** 31 - 1, 7, 1], [0, 2, 4, 5])
    assert lib().acro_b200_device_status() == _lib.EINVAL
    check([4, 0, 4, 2, 0, 4], [0, 1, 3])
    assert lib().acro_b200_device_status() == _lib.EINVAL
    status_ok()         # reported once


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_slots_of_a_prompt(kind):
    for lengths, packed, heads in (([70, 0, 130, 12], True, 3), ([2100, 900, 5, 0], True, 1), ([1500] * 4, False, 1)):
        p = Problem(kind, lengths, packed, heads, heads, 64, 64, spare=2)
        cache = torch.randn(7, heads, 64, 64, device="cuda")
        slots = [5, 2, 9, 5]        # the third is out of range, the fourth has the first's
        mine, out = cache.clone(), p.blank(heads, 64)
        ab.linear_attention(out, p.q, p.k, p.v, p.g, scale=p.scale, offsets=p.offsets, initial_state=mine, final_state=mine,
                            slots=torch.tensor(slots, dtype=torch.int32, device="cuda"),
                            scratch=scratch_for(ab.linear_attention_scratch_bytes(p.q, p.k, p.v, p.offsets)), stream=stream())
        assert lib().acro_b200_device_status() == _lib.EINVAL
        p.initial = cache[[5, 2, 0, 0]]
        expect, final = p.forward()
        for i in (0, 1):
            assert torch.equal(p.of(out, i), p.of(expect, i)) and torch.equal(mine[slots[i]], final[i])
        for i in (2, 3):
            assert bool((p.of(out, i) == -7.0).all())
        for s in (0, 1, 3, 4, 6):
            assert torch.equal(mine[s], cache[s])


def test_offsets_that_make_no_sense_touch_nothing_else():
    """Decreasing offsets and offsets outside the rows are cut back to the rows and reported."""
    for offsets in ([0, 50, 20, 90], [-40, 30, 60, 90], [0, 30, 60, 5000], [2 ** 40, 30, -2 ** 60, 2 ** 62]):
        p = Problem("bf16", [30, 30, 30], True, 2, 1, 64, 64)
        guard = torch.full((64, 2, 64), -7.0, dtype=torch.bfloat16, device="cuda")
        whole = torch.full((p.q.shape[0] + 128, 2, 64), -7.0, dtype=torch.bfloat16, device="cuda")
        out = whole[64:64 + p.q.shape[0]]
        ab.linear_attention(out, p.q, p.k, p.v, p.g, offsets=torch.tensor(offsets, device="cuda"), stream=stream(),
                            scratch=scratch_for(ab.linear_attention_scratch_bytes(p.q, p.k, p.v, p.offsets)))
        assert lib().acro_b200_device_status() == _lib.EINVAL
        assert torch.equal(whole[:64], guard) and torch.equal(whole[-64:], guard)


@pytest.mark.parametrize("kind,d", [("bf16", 64), ("f32", 48), ("f64", 32)])
def test_prompt_then_tokens(kind, d):
    """A prompt in two parts and then single tokens, through a cache with slots, against the whole sequence at once."""
    T, first, steps, h, kv = 150, 77, 9, 4, 2
    p = Problem(kind, [T], False, h, kv, d, d, states=False)
    exact, _ = ref.attention(*[wide(x[0]) for x in (p.q, p.k, p.v)], wide(p.g), p.scale, None)
    mag, _ = ref.attention(*[np.abs(wide(x[0])) for x in (p.q, p.k, p.v)], wide(p.g), p.scale, None)
    cache = torch.zeros(3, h, d, d, dtype=sums_of(kind), device="cuda")
    slot = torch.tensor([2], dtype=torch.int32, device="cuda")
    out = p.blank(h, d)
    for a, b in ((0, first), (first, T - steps)):
        ab.linear_attention(out[:, a:b], p.q[:, a:b], p.k[:, a:b], p.v[:, a:b], p.g, scale=p.scale, initial_state=cache, final_state=cache, slots=slot,
                            scratch=scratch_for(ab.linear_attention_scratch_bytes(p.q, p.k, p.v)), stream=stream())
    for t in range(T - steps, T):
        ab.linear_attention_step(out[:, t], cache, p.q[:, t], p.k[:, t], p.v[:, t], p.g, cache, scale=p.scale, slots=slot, stream=stream())
    within(wide(out[0]), exact, ref.attention_tolerance(kind, exact, mag, T, d), "out")
    status_ok()


def test_gradient_against_differences():
    p = Problem("f64", [6, 70], True, 2, 1, 5, 4)
    grads = p.backward()

    def loss():
        out, end = p.forward()
        rows = [i for i in range(out.shape[0]) if i not in p.spare_rows]
        return float((out[rows] * p.dout[rows]).sum() + (end * p.dfinal).sum())

    rng = np.random.default_rng(0)
    for x, grad in zip((p.q, p.k, p.v, p.initial), grads):
        flat, rows = x.view(-1), grad.reshape(-1)
        per_row = flat.numel() // x.shape[0]
        live = [i for i in range(flat.numel()) if x is p.initial or i // per_row not in p.spare_rows]
        for i in rng.choice(live, 6):
            was = float(flat[i])
            flat[i] = was + 1e-4
            up = loss()
            flat[i] = was - 1e-4
            down = loss()
            flat[i] = was
            # the loss is of second degree in each entry at most: the difference is exact up to rounding
            assert abs((up - down) / 2e-4 - float(rows[i])) < 1e-7


def test_captured_calls_replay_on_new_inputs():
    """Prompt, gradient, step and norms in one graph on a stream of its own; two graphs with a scratch of their own each."""
    made = []
    for seed in (1, 2):
        p = Problem("bf16", [1300, 40], True, 2, 1, 64, 64, seed=seed)
        x = torch.randn(50, 256, device="cuda")
        bufs = {"out": p.blank(2, 64), "end": torch.empty(2, 2, 64, 64, device="cuda"), "dq": p.blank(2, 64), "dk": p.blank(1, 64), "dv": p.blank(1, 64),
                "first": torch.empty(2, 2, 64, 64, device="cuda"), "y": torch.empty_like(x), "mean": torch.empty(50, device="cuda"),
                "rstd": torch.empty(50, device="cuda"), "dx": torch.empty_like(x), "dw": torch.empty(256, device="cuda"), "db": torch.empty(256, device="cuda"),
                "so": torch.empty(2, 2, 64, dtype=torch.bfloat16, device="cuda"), "ss": torch.empty(2, 2, 64, 64, device="cuda")}
        scratch = [scratch_for(n) for n in (ab.linear_attention_scratch_bytes(p.q, p.k, p.v, p.offsets),
                                            ab.linear_attention_backward_scratch_bytes(p.q, p.k, p.v, p.offsets), ab.layer_norm_backward_scratch_bytes(x))]

        def calls(b=bufs, p=p, x=x, scratch=scratch):
            s = stream()
            ab.linear_attention(b["out"], p.q, p.k, p.v, p.g, p.scale, p.offsets, p.initial, b["end"], scratch=scratch[0], stream=s)
            ab.linear_attention_backward(b["dq"], b["dk"], b["dv"], p.dout, p.q, p.k, p.v, p.g, p.scale, p.offsets, p.initial, p.dfinal, b["first"],
                                         scratch=scratch[1], stream=s)
            ab.linear_attention_step(b["so"], b["ss"], p.q[:2], p.k[:2], p.v[:2], p.g, b["end"], p.scale, stream=s)
            ab.layer_norm(b["y"], x, mean=b["mean"], rstd=b["rstd"], stream=s)
            ab.layer_norm_backward(b["dx"], b["dw"], b["db"], b["y"], x, b["mean"], b["rstd"], scratch=scratch[2], stream=s)

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            calls()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                calls()
        made.append((graph, p, x, bufs, calls))
    for graph, p, x, bufs, calls in made:
        new = Problem("bf16", [1300, 40], True, 2, 1, 64, 64, seed=9)
        for a, b in zip((p.q, p.k, p.v, p.dout, p.initial, p.dfinal), (new.q, new.k, new.v, new.dout, new.initial, new.dfinal)):
            a.copy_(b)
        x.copy_(torch.randn_like(x))
        for b in bufs.values():
            b.fill_(-7.0)
    torch.cuda.synchronize()
    for graph, *_ in made:
        graph.replay()
    torch.cuda.synchronize()
    for graph, p, x, bufs, calls in made:
        got = {k: v.clone() for k, v in bufs.items()}
        p.check_forward(got["out"], got["end"])
        p.check_backward(got["dq"], got["dk"], got["dv"], got["first"])
        for b in bufs.values():
            b.fill_(-7.0)
        calls()
        assert all(torch.equal(got[k], bufs[k]) for k in bufs)
    status_ok()


def test_calls_on_two_streams_at_once():
    ps = [Problem("bf16", [2600], False, 1, 1, 128, 128, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    results = [None, None]
    for _ in range(3):
        for i, (p, s) in enumerate(zip(ps, streams)):
            with torch.cuda.stream(s):
                results[i] = p.forward() + p.backward()
    torch.cuda.synchronize()
    for p, r in zip(ps, results):
        p.check_forward(*r[:2])
        p.check_backward(*r[2:])


def test_the_threads_stream_is_the_default():
    p = Problem("f32", [70], False, 1, 1, 16, 16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = p.blank(1, 16)
    s.wait_stream(torch.cuda.current_stream())
    ab.set_stream(s.cuda_stream)
    try:
        ab.linear_attention(out, p.q, p.k, p.v, p.g, scale=p.scale, initial_state=p.initial)
        s.synchronize()
    finally:
        ab.set_stream(0)
    p.check_forward(out, None)


def test_operands_that_would_be_overwritten_are_refused():
    p = Problem("bf16", [70], False, 1, 1, 64, 64)
    for to in (p.q, p.k, p.v):
        with pytest.raises(ab.AcroError):
            ab.linear_attention(to, p.q, p.k, p.v, p.g, stream=stream())
    outs = [p.blank(1, 64) for _ in range(3)]
    for i, x in enumerate((p.q, p.k, p.dout)):
        bad = list(outs)
        bad[i] = x
        with pytest.raises(ab.AcroError):
            ab.linear_attention_backward(*bad, p.dout, p.q, p.k, p.v, p.g, stream=stream())
    with pytest.raises(ab.AcroError):
        ab.linear_attention_backward(*outs, p.dout, p.q, p.k, p.v, p.g, d_final_state=p.dfinal, d_initial_state=p.dfinal, stream=stream())
    long = Problem("bf16", [5000], False, 1, 1, 64, 64)
    with pytest.raises(ValueError):
        ab.linear_attention(long.blank(1, 64), long.q, long.k, long.v, long.g, stream=stream())
    with pytest.raises(ab.AcroError):
        ab.linear_attention(long.blank(1, 64), long.q, long.k, long.v, long.g, scratch=torch.empty(64, device="cuda"), stream=stream())
    with pytest.raises(ab.AcroError):       # host memory
        ab.linear_attention(torch.empty(1, 70, 1, 64, dtype=torch.bfloat16), p.q, p.k, p.v, p.g, stream=stream())
    with pytest.raises(ab.AcroError):
        ab.linear_attention_backward(outs[0], outs[0], outs[1], p.dout, p.q, p.k, p.v, p.g, stream=stream())


def test_host_memory_is_refused_wherever_it_stands():
    """Every pointer that a kernel would follow: an error, not a launch."""
    p = Problem("f32", [40, 30], True, 2, 2, 16, 16)
    out, host = p.blank(2, 16), lambda x: x.cpu()
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(log_decay=p.g, offsets=p.offsets, initial_state=p.initial, final_state=p.initial.clone(), slots=slots)
    for name in good:
        with pytest.raises(ab.AcroError):
            ab.linear_attention(out, p.q, p.k, p.v, **{**good, name: host(good[name])}, stream=stream())
    q, k, v, o = p.q[:2], p.k[:2], p.v[:2], out[:2]
    good = dict(state_out=p.initial.clone(), q=q, k=k, v=v, log_decay=p.g, state_in=p.initial, slots=slots)
    for name in good:
        with pytest.raises(ab.AcroError):
            ab.linear_attention_step(o, **{**good, name: host(good[name])}, stream=stream())
    good = dict(log_decay=p.g, offsets=p.offsets, initial_state=p.initial, d_final_state=p.dfinal, d_initial_state=torch.empty_like(p.dfinal))
    outs = [p.blank(2, 16) for _ in range(3)]
    for name in good:
        with pytest.raises(ab.AcroError):
            ab.linear_attention_backward(*outs, p.dout, p.q, p.k, p.v, **{**good, name: host(good[name])}, stream=stream())
    x, w, r = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda"), torch.ones(4, device="cuda")
    good = dict(out=torch.empty_like(x), x=x, weight=w, bias=w, mean=r, rstd=r)
    for name in good:
        with pytest.raises(ab.AcroError):
            ab.layer_norm(**{**good, name: host(good[name])}, stream=stream())
    good = dict(dx=torch.empty_like(x), dweight=w, dbias=w.clone(), dout=x, x=x, mean=r, rstd=r, weight=w,
                scratch=scratch_for(ab.layer_norm_backward_scratch_bytes(x)))
    for name in good:
        with pytest.raises(ab.AcroError):
            ab.layer_norm_backward(**{**good, name: host(good[name])}, stream=stream())
    status_ok()


@pytest.mark.parametrize("kind", ["bf16", "f32", "f64"])
def test_nothing_at_all(kind):
    """No sequences, no rows, no tokens: states pass through, gradients of states too."""
    p = Problem(kind, [0, 0, 0], True, 2, 1, 16, 8, spare=0)
    assert p.q.numel() == 0
    out, end = p.forward()
    assert torch.equal(end, p.initial)
    assert torch.equal(p.backward()[3], p.dfinal)
    e = torch.empty(2, 0, 2, 16, dtype=DTYPES[kind], device="cuda")
    final = torch.empty_like(p.initial[:2])
    ab.linear_attention(e[..., :8], e, e[:, :, :1], e[:, :, :1, :8], p.g, initial_state=p.initial[:2], final_state=final, stream=stream())
    assert torch.equal(final, p.initial[:2])
    n = torch.empty(0, 5, 2, 16, dtype=DTYPES[kind], device="cuda")
    ab.linear_attention(n, n, n, n, p.g, stream=stream())
    status_ok()


@pytest.mark.parametrize("kind", ["bf16", "f32", "f16"])
def test_arrays_off_their_boundaries(kind):
    """Rows that start off the 16-byte boundaries which copies like best, head strides longer than the head, tokens behind heads."""
    dt = DTYPES[kind]
    for d, pad, offset in ((64, 1, 0), (64, 0, 3), (40, 3, 1), (128, 8, 8)):
        p = Problem(kind, [150, 140], True, 2, 2, d, d, seed=pad + offset)
        for name in ("q", "k", "v", "dout"):
            x = getattr(p, name)
            rows, h = x.shape[0], x.shape[1]
            buf = torch.full((h, rows * (d + pad) + offset + 8), float("nan"), dtype=dt, device="cuda")
            view = buf[:, offset:offset + rows * (d + pad)].unflatten(1, (rows, d + pad))[..., :d].transpose(0, 1)
            view.copy_(x)
            setattr(p, name, view)
        p.check_forward(*p.forward())
        p.check_backward(*p.backward())
    status_ok()


@pytest.mark.parametrize("kind", ["bf16", "f32", "f64"])
def test_more_sequences_than_threads(kind):
    """Thousands of sequences, most of them a few tokens or none, long ones among them."""
    lengths = [i % 4 for i in range(1500)] + [700] + [i % 3 for i in range(900)] + [1300, 1]
    p = Problem(kind, lengths, True, 1, 1, 16, 16, decay=[-1 / 50])
    out, end = p.forward()
    grads = p.backward()
    keep = [0, 1, 2, 3, 799, 801, 1499, 1500, 1501, 2398, 2399, 2400, 2401]
    for i in keep:
        one = Problem(kind, [lengths[i]], True, 1, 1, 16, 16, decay=[-1 / 50])
        for name in ("q", "k", "v", "dout"):
            x = p.of(getattr(p, name), i)
            setattr(one, name, torch.cat([x, torch.full((3,) + tuple(x.shape[1:]), float("nan"), dtype=x.dtype, device="cuda")]))
        one.initial, one.dfinal = p.initial[i:i + 1], p.dfinal[i:i + 1]
        pad = lambda x: torch.cat([p.of(x, i), torch.full((3,) + tuple(x.shape[1:]), -7.0, dtype=x.dtype, device="cuda")])
        one.check_forward(pad(out), end[i:i + 1])
        one.check_backward(*[pad(x) for x in grads[:3]], grads[3][i:i + 1])
    p.untouched(out, *grads[:3])
    status_ok()


@pytest.mark.parametrize("kind", ["bf16", "f32", "f64"])
def test_many_sequences_are_cut(kind):
    """Packed sequences that are all longer than a segment, or end anywhere inside one, with short ones between them."""
    lengths = [513, 1, 1025, 0, 700, 512, 1537, 3, 1024, 640, 0, 129, 2049, 511, 515, 520, 1400, 64, 999, 1281]
    p = Problem(kind, lengths, True, 1, 1, 16, 16, decay=[-1 / 300])
    p.check_forward(*p.forward())
    p.check_backward(*p.backward())
    status_ok()


def test_a_scale_that_changes_in_place():
    """A scale given as an array is taken at its value of each call."""
    p = Problem("f32", [9], False, 1, 1, 16, 16)
    scale, outs = torch.tensor(1.0), []
    for value in (1.0, 2.0):
        scale.fill_(value)
        outs.append(p.blank(1, 16))
        ab.linear_attention(outs[-1], p.q, p.k, p.v, p.g, scale=scale, initial_state=p.initial, stream=stream())
    assert torch.equal(outs[1], 2 * outs[0])


def test_offsets_beyond_31_bits():
    """A cache of more than 2^31 entries, and arrays of more than 2^31 elements of which one sequence at the end is used."""
    count, d = 140000, 128
    cache = torch.empty(count, 1, d, d, device="cuda")
    p = Problem("bf16", [1, 1], False, 1, 1, d, d)
    slots = [count - 1, 131072]
    cache[slots] = p.initial
    out = torch.zeros(2, 1, d, dtype=torch.bfloat16, device="cuda")
    ab.linear_attention_step(out, cache, p.q[:, 0], p.k[:, 0], p.v[:, 0], p.g, cache, scale=p.scale,
                             slots=torch.tensor(slots, dtype=torch.int32, device="cuda"), stream=stream())
    p.check_forward(out[:, None], cache[slots])
    del cache
    rows, heads, tokens = 70000, 256, 130
    big = Problem("bf16", [tokens], True, heads, heads, d, d, states=False, spare=0)
    wide_rows = {n: torch.empty(rows, heads, d, dtype=torch.bfloat16, device="cuda") for n in ("q", "k", "v", "out")}
    for n in ("q", "k", "v"):
        wide_rows[n][-tokens:] = getattr(big, n)
    offsets = torch.tensor([rows - tokens, rows], device="cuda")
    q, k, v, out = (wide_rows[n] for n in ("q", "k", "v", "out"))
    ab.linear_attention(out, q, k, v, big.g, scale=big.scale, offsets=offsets, scratch=scratch_for(ab.linear_attention_scratch_bytes(q, k, v, offsets)),
                        stream=stream())
    expect, _ = big.forward()
    assert torch.equal(out[-tokens:], expect)
    status_ok()


# ---------------------------------------------------------------- layer norm

NORM_SHAPES = [(1, 1), (3, 7), (5, 32), (2, 33), (300, 64), (1, 4096), (9, 1001), (4, 4096), (17, 4104), (3, 8192), (2, 16384), (2, 16385), (3, 40000), (700, 250)]


def norm_case(kind, rows, width, seed=0, pad=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[kind]
    x = (torch.randn(rows, width + pad, generator=g, device="cuda") * 2 + torch.randn(rows, 1, generator=g, device="cuda") * 30).to(dt)[:, :width]
    w, b = (torch.randn(width, generator=g, device="cuda").to(dt) for _ in range(2))
    dy = torch.randn(rows, width + 2 * pad, generator=g, device="cuda").to(dt)[:, :width]
    return x, w, b, dy


def norm_errors(kind, x, width):
    """Error of the centred entries relative to 1 (the size of xhat): the mean is a sum of `width` terms in the type of sums, added in at most
    width/32 + 40 steps on any path, each half a step of the sum of magnitudes; so is the mean square."""
    u, n = ref.SUM_HALF_STEP[kind], min(width, width / 32 + 48)
    mean_abs = np.abs(x).mean(1, keepdims=True)
    var = x.var(1, keepdims=True)
    rstd = 1 / np.sqrt(var + 1e-5)
    return u * (n + 4) * mean_abs, u * (n + 4) * (1 + 2 * mean_abs * rstd) + 8 * u, rstd


@pytest.mark.parametrize("kind", ["bf16", "f32", "f16", "f64"])
@pytest.mark.parametrize("rows,width", NORM_SHAPES)
def test_norm(kind, rows, width):
    for pad, affine in ((0, True), (3, False), (8, True)):
        x, w, b, _ = norm_case(kind, rows, width, seed=width, pad=pad)
        sums = sums_of(kind)
        out, mean, rstd = torch.full((rows, width), -7.0, dtype=x.dtype, device="cuda"), torch.empty(rows, dtype=sums, device="cuda"), torch.empty(rows, dtype=sums, device="cuda")
        ab.layer_norm(out, x, w if affine else None, b if affine else None, eps=1e-5, mean=mean, rstd=rstd, stream=stream())
        X = wide(x)
        exact, m, r = ref.norm(X, wide(w) if affine else None, wide(b) if affine else None, 1e-5)
        dm, dr, rs = norm_errors(kind, X, width)
        within(wide(mean), m, dm[:, 0], "mean")
        within(wide(rstd), r, (dr * rs)[:, 0], "rstd")
        W = np.abs(wide(w)) if affine else 1.0
        xhat = np.abs(X - m[:, None]) * rs
        tol = ref.HALF_STEP[kind] * np.abs(exact) + W * (dm * rs + dr * xhat) + 8 * ref.SUM_HALF_STEP[kind] * (np.abs(exact) + W * xhat) + 2.0 ** -25
        within(wide(out), exact, tol if kind != "f64" else tol - 2.0 ** -25 + 1e-300, "out")
        # in place
        ab.layer_norm(x, x, w if affine else None, b if affine else None, eps=1e-5, stream=stream())
        assert torch.equal(x, out)


@pytest.mark.parametrize("kind", ["bf16", "f32", "f16", "f64"])
@pytest.mark.parametrize("rows,width", NORM_SHAPES + [(5000, 40), (2000, 1024)])
def test_norm_backward(kind, rows, width):
    for pad, affine in ((0, True), (3, False), (8, True)):
        x, w, _, dy = norm_case(kind, rows, width, seed=rows + width, pad=pad)
        sums = sums_of(kind)
        X, D = wide(x), wide(dy)
        _, m, r = ref.norm(X, None, None, 1e-5)
        mean, rstd = torch.tensor(m).to(sums).cuda(), torch.tensor(r).to(sums).cuda()
        dx = torch.full((rows, width), -7.0, dtype=x.dtype, device="cuda")
        dw, db = torch.full((width,), -7.0, dtype=sums, device="cuda"), torch.full((width,), -7.0, dtype=sums, device="cuda")
        scratch = scratch_for(ab.layer_norm_backward_scratch_bytes(x))
        args = (dy, x, mean, rstd, w if affine else None)
        ab.layer_norm_backward(dx, dw, db, *args, scratch=scratch, stream=stream())
        m, r = wide(mean), wide(rstd)
        W = wide(w) if affine else None
        exact = ref.norm_backward(D, X, m, r, W)
        # magnitudes of the terms; xhat itself is off by a half step of x rstd and mean rstd
        u = ref.SUM_HALF_STEP[kind]
        xmag = (np.abs(X) + np.abs(m)[:, None]) * r[:, None]
        gmag = np.abs(D) * (1 if W is None else np.abs(W))
        n = min(width, width / 32 + 48) + 16
        mag = r[:, None] * (gmag + gmag.mean(1, keepdims=True) + xmag * (gmag * xmag).mean(1, keepdims=True))
        within(wide(dx), exact[0], ref.HALF_STEP[kind] * np.abs(exact[0]) + 1.01 * n * u * mag + (2.0 ** -25 if kind == "f16" else 1e-300), "dx")
        steps = min(rows, rows / 64 + 80) + 8 if width <= 16384 else rows + 8
        within(wide(dw), exact[1], 1.01 * u * (steps * (np.abs(D) * xmag).sum(0)) + 1e-300, "dweight")
        within(wide(db), exact[2], 1.01 * u * (steps * np.abs(D).sum(0)) + 1e-300, "dbias")
        # the same bits again, the parts alone, in place
        dx2, dw2 = torch.empty_like(dx), torch.empty_like(dw)
        ab.layer_norm_backward(dx2, dw2, None, *args, scratch=scratch, stream=stream())
        assert torch.equal(dx2, dx) and torch.equal(dw2, dw)
        ab.layer_norm_backward(dy, None, None, *args, stream=stream())
        assert torch.equal(dy, dx)


def test_norm_rows_keep_to_themselves():
    """A row of NaN, one of infinities, a constant one (variance zero) beside ordinary ones; no rows at all."""
    for width in (48, 1024, 20000):
        x = torch.randn(6, width, device="cuda")
        clean = torch.empty_like(x)
        ab.layer_norm(clean, x, stream=stream())
        x[1], x[3], x[4] = float("nan"), float("inf"), 2.5
        out = torch.empty_like(x)
        ab.layer_norm(out, x, stream=stream())
        assert torch.equal(out[[0, 2, 5]], clean[[0, 2, 5]]) and bool((out[4] == 0).all()) and bool(torch.isnan(out[[1, 3]]).all())
    e = torch.empty(0, 48, device="cuda")
    ab.layer_norm(e, e, stream=stream())
    dw, db = torch.ones(48, device="cuda"), torch.ones(48, device="cuda")
    ab.layer_norm_backward(e, dw, db, e, e, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"), stream=stream())
    assert bool((dw == 0).all()) and bool((db == 0).all())
    wide_rows = torch.randn(2, 20000, device="cuda")
    stats = torch.ones(2, device="cuda")
    w = torch.empty(20000, device="cuda")
    with pytest.raises(ab.AcroError):       # the column sums would read what the rows overwrote
        ab.layer_norm_backward(wide_rows, w, None, wide_rows, wide_rows, stats, stats, stream=stream(),
                               scratch=scratch_for(ab.layer_norm_backward_scratch_bytes(wide_rows)))


# ---------------------------------------------------------------- through the engine, and together

def test_engine_on_tensors():
    """acro::TensorEngine's methods on fp64 tensors, one sequence and several."""
    rng = np.random.default_rng(5)
    te = ab.TensorEngine("Cuda")
    H, kv, dk, dv = 4, 2, 8, 12
    for lead in ((), (3,)):
        n, T = (lead[0] if lead else 1), 1400
        host = {"q": rng.standard_normal(lead + (T, H, dk)), "k": rng.standard_normal(lead + (T, kv, dk)), "v": rng.standard_normal(lead + (T, kv, dv)),
                "do": rng.standard_normal(lead + (T, H, dv)), "g": -np.array([1e-3, 0.01, 0.2, 1.0]), "s": rng.standard_normal(lead + (H, dk, dv)),
                "ds": rng.standard_normal(lead + (H, dk, dv))}
        t = {k: ab.Tensor(x.shape, hdata=x) for k, x in host.items()}
        out, fin = ab.Tensor(*lead, T, H, dv), ab.Tensor(*lead, H, dk, dv)
        te.LinearAttention(out, t["q"], t["k"], t["v"], t["g"], 0.3, t["s"], fin)
        gr = [ab.Tensor(*x.shape) for x in (t["q"], t["k"], t["v"], t["s"])]
        te.LinearAttentionBackward(gr[0], gr[1], gr[2], t["do"], t["q"], t["k"], t["v"], t["g"], 0.3, t["s"], t["ds"], gr[3])
        for x in [out, fin] + gr:
            x.MoveFromGPU()
        for i in range(n):
            pick = (lambda x: x[i]) if lead else (lambda x: x)
            a = [pick(host[k]) for k in ("q", "k", "v")]
            exact = ref.attention(*a, host["g"], 0.3, pick(host["s"])) + ref.attention_backward(*a, host["g"], 0.3, pick(host["s"]), pick(host["do"]), pick(host["ds"]))
            for got, e in zip([out, fin] + gr, exact):
                assert np.allclose(pick(got.numpy()), e, rtol=1e-11, atol=1e-10)
    step_out, state = ab.Tensor(3, H, dv), ab.Tensor(3, H, dk, dv)
    q1, k1, v1 = (np.ascontiguousarray(host[k][:, 0]) for k in ("q", "k", "v"))
    ts = [ab.Tensor(x.shape, hdata=x) for x in (q1, k1, v1)]
    te.LinearAttentionStep(step_out, state, *ts, t["g"], t["s"], 0.3)
    step_out.MoveFromGPU()
    for i in range(3):
        e, _ = ref.attention(q1[i][None], k1[i][None], v1[i][None], host["g"], 0.3, host["s"][i])
        assert np.allclose(step_out.numpy()[i], e[0], rtol=1e-12, atol=1e-12)


def test_engine_norm_and_its_rank_sum():
    rng = np.random.default_rng(6)
    x, w, b, dy = rng.standard_normal((4, 9, 50)), rng.standard_normal(50), rng.standard_normal(50), rng.standard_normal((4, 9, 50))
    te = ab.TensorEngine("Cuda")
    te.SetPeerGroup(ab.PeerGroup(1, 0))         # a sharded batch over one rank: the sum over the ranks is its own
    X, W, B, D = (ab.Tensor(a.shape, hdata=a) for a in (x, w, b, dy))
    X.SetSharded(True)
    Y, M, R, dX, dW, dB = ab.Tensor(4, 9, 50), ab.Tensor(36), ab.Tensor(36), ab.Tensor(4, 9, 50), ab.Tensor(50), ab.Tensor(50)
    te.LayerNorm(Y, X, W, B, 1e-5, M, R)
    te.LayerNormBackward(dX, dW, dB, D, X, M, R, W)
    for t in (Y, M, R, dX, dW, dB):
        t.MoveFromGPU()
    y, m, r = ref.norm(x.reshape(36, 50), w, b, 1e-5)
    gx, gw, gb = ref.norm_backward(dy.reshape(36, 50), x.reshape(36, 50), m, r, w)
    for got, e in ((Y, y), (M, m), (R, r), (dX, gx), (dW, gw), (dB, gb)):
        assert np.allclose(got.numpy().reshape(e.shape), e, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("kind", ["f64", "f32", "bf16"])
def test_a_layer_and_its_gradient(kind):
    """norm -> projections -> linear attention -> norm over each head -> loss, as a layer uses them, against autograd of the formulas in 64 bits."""
    n, T, width, h, kv, d = 2, 90, 64, 4, 2, 16
    torch.manual_seed(0)
    dt, sums = DTYPES[kind], sums_of(kind)
    x = torch.randn(n, T, width, device="cuda").to(dt)
    w1, w2 = (1 + 0.1 * torch.randn(c, device="cuda").to(dt) for c in (width, d))
    proj = [(torch.randn(width, m * d, device="cuda") / 8).to(dt) for m in (h, kv, kv)]
    g = -torch.tensor([1.0, 0.3, 0.05, 0.01], dtype=sums, device="cuda")
    dy = torch.randn(n, T, h, d, device="cuda").to(dt)
    s = stream()
    # forward
    y1, m1, r1 = torch.empty_like(x), torch.empty(n, T, dtype=sums, device="cuda"), torch.empty(n, T, dtype=sums, device="cuda")
    ab.layer_norm(y1, x, w1, mean=m1, rstd=r1, stream=s)
    q, k, v = ((y1 @ p).unflatten(-1, (m, d)) for p, m in zip(proj, (h, kv, kv)))
    o = torch.empty_like(dy)
    ab.linear_attention(o, q, k, v, g, scale=0.25, stream=s)
    y2, m2, r2 = torch.empty_like(o), torch.empty(n, T, h, dtype=sums, device="cuda"), torch.empty(n, T, h, dtype=sums, device="cuda")
    ab.layer_norm(y2, o, w2, mean=m2, rstd=r2, stream=s)
    # backward
    do, dw2, dw1, dx = torch.empty_like(o), torch.empty(d, dtype=sums, device="cuda"), torch.empty(width, dtype=sums, device="cuda"), torch.empty_like(x)
    ab.layer_norm_backward(do, dw2, None, dy, o, m2, r2, w2, scratch=scratch_for(ab.layer_norm_backward_scratch_bytes(o)), stream=s)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    ab.linear_attention_backward(dq, dk, dv, do, q, k, v, g, scale=0.25, scratch=scratch_for(ab.linear_attention_backward_scratch_bytes(q, k, v)), stream=s)
    dy1 = sum(t.flatten(2).double() @ p.double().t() for t, p in zip((dq, dk, dv), proj)).to(dt)
    ab.layer_norm_backward(dx, dw1, None, dy1, x, m1, r1, w1, scratch=scratch_for(ab.layer_norm_backward_scratch_bytes(x)), stream=s)
    # the formulas in 64 bits
    X, W1, W2 = (t.cpu().double().requires_grad_() for t in (x, w1, w2))
    P, lam = [p.cpu().double() for p in proj], torch.exp(g.cpu().double())

    def norm64(a, w):
        c = a - a.mean(-1, keepdim=True)
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w

    Y1 = norm64(X, W1)
    Q, K, V = ((Y1 @ p).unflatten(-1, (m, d)) for p, m in zip(P, (h, kv, kv)))
    K, V = K.repeat_interleave(h // kv, 2), V.repeat_interleave(h // kv, 2)
    t = torch.arange(T, dtype=torch.float64)
    gap = t[:, None] - t[None, :]
    decay = torch.where(gap >= 0, lam[:, None, None] ** gap.clamp(min=0), 0.0)
    O = 0.25 * torch.einsum("nhts,nshd->nthd", torch.einsum("nthd,nshd->nhts", Q, K) * decay, V)
    Y2 = norm64(O, W2)
    Y2.backward(dy.cpu().double())
    # six roundings to the element type lie between the input and the gradient; each reaches it through sums of independent terms
    limit = {"f64": 1e-11, "f32": 2e-5, "bf16": 6 * 2.0 ** -8}[kind]
    for got, want in ((y2, Y2), (dx, X.grad), (dw1, W1.grad), (dw2, W2.grad)):
        got, want = got.cpu().double(), want.detach()
        assert float((got - want).norm() / want.norm()) < limit
    status_ok()
