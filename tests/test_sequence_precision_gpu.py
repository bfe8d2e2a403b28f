"""How many bits of its operands linear attention keeps: sums whose large terms cancel exactly, so that what is left is the operands' last bits.

Every case is built so that fp32 arithmetic gives the result exactly.  A sum on the tensor cores is aligned to its largest term (below 4 here)
and each of its few terms that are not zero may lose less than a step 2^-22 there; four such steps are allowed, and the rounding of the result
to its type."""
import pytest
import torch

import acrotensor_b200 as ab
import sequence_reference as ref
from acrotensor_b200 import _lib
from acrotensor_b200._lib import lib
from test_sequence_gpu import DTYPES, scratch_for, stream, sums_of

pytestmark = pytest.mark.gpu

T = 130             # tokens: two whole chunks and two more, and enough for every type to take the tensor cores
STEPS = 4 * 2.0 ** -22


def zeros(kind, heads, columns, tokens=T):
    return torch.zeros(1, tokens, heads, columns, dtype=DTYPES[kind], device="cuda")


def forward(kind, q, k, v, state=None):
    heads = q.shape[2]
    out = torch.full_like(v, -7.0)
    ab.linear_attention(out, q, k, v, torch.zeros(heads, dtype=sums_of(kind), device="cuda"), initial_state=state, stream=stream(),
                        scratch=scratch_for(ab.linear_attention_scratch_bytes(q, k, v)))
    assert lib().acro_b200_device_status() == _lib.OK
    return out[0].double()


def near(kind, got, want):
    want = torch.as_tensor(want, dtype=torch.float64, device="cuda").expand_as(got)
    assert bool(((got - want).abs() <= STEPS + ref.HALF_STEP[kind] * want.abs()).all()), float((got - want).abs().max())


def last_bits(n, seed):
    """n values of 24 bits in 1 .. 2, and the same without their last 8."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = 1 + torch.randint(0, 2 ** 23, (n,), generator=g, device="cuda").double() * 2.0 ** -23
    return x, torch.floor(x * 2 ** 15) / 2 ** 15


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_a_state_enters_its_product_whole(kind, d):
    x, y = last_bits(d, d)
    state = torch.zeros(1, 1, d, d, device="cuda")
    state[0, 0, 0], state[0, 0, 1] = x.float(), -y.float()
    q = zeros(kind, 1, d)
    q[..., :2] = 1
    near(kind, forward(kind, q, zeros(kind, 1, d), zeros(kind, 1, d), state)[:, 0], x - y)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_scores_enter_their_product_whole(kind, d):
    """Scores of 1 + 2^-9 + 2^-17 and 1 + 2^-9, of tokens whose values are 1 and -1; and the same backward in time."""
    few, more, bits = torch.tensor([1.0, 1, 0]), torch.tensor([1.0, 1, 1]), torch.tensor([1.0, 2.0 ** -9, 2.0 ** -17])
    q, k, v = zeros(kind, 1, d), zeros(kind, 1, d), zeros(kind, 1, d)
    q[..., :3] = bits
    k[0, 0, 0, :3], k[0, 1, 0, :3] = more, few
    v[0, 0], v[0, 1] = 1, -1
    near(kind, forward(kind, q, k, v)[1:, 0], 2.0 ** -17)
    q, k, do = zeros(kind, 1, d), zeros(kind, 1, d), zeros(kind, 1, d)
    k[..., :3] = bits
    q[0, -1, 0, :3], q[0, -2, 0, :3] = more, few
    do[0, -1], do[0, -2] = 1, -1
    dq, dk, dv = (torch.full_like(x, -7.0) for x in (q, k, v))
    ab.linear_attention_backward(dq, dk, dv, do, q, k, v, torch.zeros(1, device="cuda"), stream=stream(),
                                 scratch=scratch_for(ab.linear_attention_backward_scratch_bytes(q, k, v)))
    near(kind, dv[0, :-1, 0].double(), 2.0 ** -17)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_second_parts_are_multiplied_with_each_other(kind, d):
    """The square of 1 + 3 2^-10 less its first two terms: queries by keys, and scores (and keys) by values."""
    x, y = 1 + 3 * 2.0 ** -10, 6 * 2.0 ** -10
    q, k, v = zeros(kind, 1, d), zeros(kind, 1, d), zeros(kind, 1, d)
    q[..., :3] = torch.tensor([x, 1, 1])
    k[0, 0, 0, 0] = x
    k[0, 1, 0, 1:3] = torch.tensor([1, y])
    v[0, 0], v[0, 1] = 1, -1
    near(kind, forward(kind, q, k, v)[1:, 0], 9 * 2.0 ** -20)
    q[..., :3] = torch.tensor([1.0, 1, 0])
    k[0, :2, 0, :3] = torch.tensor([[x, 0, 0], [0, 1, 0]])
    v[0, 0], v[0, 1] = x, -(1 + y)
    near(kind, forward(kind, q, k, v)[1:, 0], 9 * 2.0 ** -20)


@pytest.mark.parametrize("of", ["q", "k", "v"])
@pytest.mark.parametrize("d", [64, 128])
def test_single_precision_keeps_its_last_bits(of, d):
    """x - y, the last 8 of 24 bits, by way of queries, keys or values, a head for each pair."""
    heads = 32
    x, y = (a.float() for a in last_bits(heads, d))
    q, k, v = (zeros("f32", heads, d) for _ in range(3))
    q[..., :2] = 1
    k[0, 0, :, 0], k[0, 1, :, 1] = 1, 1
    v[0, 0], v[0, 1] = 1, -1
    if of == "q":
        q[0, :, :, 0], q[0, :, :, 1] = x, y
    if of == "k":
        k[0, 0, :, 0], k[0, 1, :, 1] = x, y
    if of == "v":
        v[0, 0], v[0, 1] = x[:, None], -y[:, None]
    near("f32", forward("f32", q, k, v)[1:], (x.double() - y.double())[:, None])


@pytest.mark.parametrize("kind,of", [("f32", "q"), ("f32", "k"), ("f32", "v"), ("f32", "state"), ("bf16", "state"), ("f32", "score"), ("bf16", "score")])
@pytest.mark.parametrize("d", [64, 128])
def test_values_above_the_largest_bf16_stay_finite(kind, of, d):
    """3.4e38 is an fp32 value beyond the numbers of bf16: as an operand, as a state and as a score.  One term an entry: 16 roundings at most."""
    most, little = 3.4e38, 2.0 ** -20
    q, k, v, state = zeros(kind, 1, d), zeros(kind, 1, d), zeros(kind, 1, d), torch.zeros(1, 1, d, d, device="cuda")
    q[..., 0], k[0, 5, 0, 0], v[0, 5] = 1, 1, 1
    if of == "q":
        q[..., 0], v[0, 5] = most, little
    if of == "k":
        k[0, 5, 0, 0], v[0, 5] = most, little
    if of == "v":
        v[0, 5], k[0, 5, 0, 0] = most, little
    if of == "state":
        state[..., 1, :], q[..., 1] = most, little
    if of == "score":       # (2 - 2^-8) 2^127
        q[..., 0], q[..., 1] = 1.9921875 * 2.0 ** 64, 2.0 ** 60
        k[0, 5, 0, 0], k[0, 5, 0, 1], v[0, 5] = 2.0 ** 63, 2.0 ** 59, little
    exact, _ = ref.attention(*[x[0].double().cpu().numpy() for x in (q, k, v)], torch.zeros(1).numpy(), 1.0, state[0].double().cpu().numpy())
    exact = torch.as_tensor(exact, device="cuda")
    got = forward(kind, q, k, v, state)
    assert bool(((got - exact).abs() <= (ref.HALF_STEP[kind] + 16 * 2.0 ** -24) * exact.abs()).all())


@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_values_above_the_largest_bf16_stay_finite(d):
    q, k, v, do = (zeros("f32", 1, d) for _ in range(4))
    q[0, 7, 0, 0], k[..., 0], do[0, 7] = 1, 2.0 ** -20, 3.4e38
    dq, dk, dv = (torch.full_like(x, -7.0) for x in (q, k, v))
    ab.linear_attention_backward(dq, dk, dv, do, q, k, v, torch.zeros(1, device="cuda"), stream=stream(),
                                 scratch=scratch_for(ab.linear_attention_backward_scratch_bytes(q, k, v)))
    want = 2.0 ** -20 * float(torch.tensor(3.4e38))
    assert bool(((dv[0, :8].double() - want).abs() <= 16 * 2.0 ** -24 * want).all()) and bool((dv[0, 8:] == 0).all())
    assert bool((dq == 0).all()) and bool((dk == 0).all())
