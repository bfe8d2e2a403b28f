"""What the sequence operators cost: linear attention with a decay for each head (prompt, single token, gradient) and layer norm
(forward, gradient), each over the sizes that a layer meets in training and serving.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges, ``prepare(case, seed)`` makes what a program has in hand
before the call, ``run(state)`` makes one pass, ``work(case)`` says what the pass cannot do without and ``exact(case, seed)`` gives the
result in 64 bits.  With ``own`` false ``run`` computes the operators from elementary torch operations; with ``own`` true it calls the
library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "f64": 8}
EPS = 1e-5
CHUNK = 128
SPARE_ROWS = 5          # rows behind the last packed sequence, which no operator touches


def listed():
    return [
        # One request generates one token: the smallest call, pure latency.
        {"name": "step_one", "op": "step", "dtype": "bf16", "requests": 1, "heads": 8, "kv_heads": 8, "dk": 64, "dv": 64},
        # A full serving batch generates one token each; the states are in the order of their slots, the requests are not.
        {"name": "step_batch", "op": "step", "dtype": "bf16", "requests": 192, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128},
        # A short prompt of one request.
        {"name": "prompt_short", "op": "forward", "dtype": "bf16", "lengths": "37", "packed": False, "states": True, "heads": 8, "kv_heads": 8,
         "dk": 64, "dv": 64},
        # Prompts of many requests packed one behind the other, some of them continued from a state, one of them empty.
        {"name": "prompt_packed", "op": "forward", "dtype": "bf16", "lengths": "1 4003 129 0 2048 64 777 3001 1500 517", "packed": True,
         "states": True, "heads": 16, "kv_heads": 4, "dk": 128, "dv": 128},
        # One very long document: few rows of work beside one another, a long axis.
        {"name": "prompt_long", "op": "forward", "dtype": "bf16", "lengths": "65536", "packed": False, "states": True, "heads": 8, "kv_heads": 8,
         "dk": 128, "dv": 128},
        # A training batch in 32 bits.
        {"name": "train_forward_f32", "op": "forward", "dtype": "f32", "lengths": "1024 1024 1024 1024", "packed": False, "states": False, "heads": 12,
         "kv_heads": 12, "dk": 64, "dv": 64},
        # The gradient of a training batch.
        {"name": "train_backward", "op": "backward", "dtype": "bf16", "lengths": "4096 4096 4096 4096", "packed": False, "states": False, "heads": 32,
         "kv_heads": 32, "dk": 64, "dv": 64},
        # The gradient of packed sequences with shared key and value heads and states, in 32 bits and odd head sizes.
        {"name": "packed_backward_f32", "op": "backward", "dtype": "f32", "lengths": "311 1 700 1037", "packed": True, "states": True, "heads": 12,
         "kv_heads": 4, "dk": 72, "dv": 80},
        # The norm of the few rows of a decoding step.
        {"name": "norm_few_rows", "op": "norm", "dtype": "f16", "rows": 3, "width": 4096},
        # The norm in front of a layer in training.
        {"name": "norm_forward", "op": "norm", "dtype": "bf16", "rows": 16384, "width": 4096},
        # Its gradient, with the reduction of the weight's and the bias's over all rows.
        {"name": "norm_backward", "op": "norm_backward", "dtype": "bf16", "rows": 16384, "width": 4096},
        # The same for an odd width in 32 bits.
        {"name": "norm_backward_odd", "op": "norm_backward", "dtype": "f32", "rows": 4999, "width": 1001},
    ]


def _lengths(case):
    return [int(x) for x in case["lengths"].split()]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    return kv * rng.choice([1, 1, 2, 3, 4]), kv


def _head_size(rng):
    return rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, rng.randrange(9, 129)])


def draw(rng):
    op = rng.choice(["step", "forward", "forward", "backward", "norm", "norm_backward"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32", "f64"])
    case = {"op": op, "dtype": dtype}
    if op in ("norm", "norm_backward"):
        width = _spread(rng, 32, 16384)
        case.update(rows=_spread(rng, 1, min(16384 * 4096 * 2 // (width * BYTES[dtype]), 100000)), width=width)
        return case
    heads, kv_heads = _heads(rng)
    dk = _head_size(rng)
    dv = dk if rng.random() < 0.6 else _head_size(rng)
    case.update(heads=heads, kv_heads=kv_heads, dk=dk, dv=dv)
    if op == "step":
        case["requests"] = _spread(rng, 1, 256)
        return case
    # tokens x heads are bounded so that no drawn case costs more than the largest listed one; the types without a narrow format cost more
    budget = 65536 * 8 * 128 // (heads * max(dk, dv))
    budget = budget // {"bf16": 2, "f16": 6, "f32": 6, "f64": 16}[dtype] // (3 if op == "backward" else 1)
    total = _spread(rng, 1, max(2, min(65536, budget)))
    packed = rng.random() < 0.6
    if packed:
        n = rng.choice([1, 2, 3, 5, 9, 17])
        cuts = sorted(rng.randrange(0, total + 1) for _ in range(n - 1))
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    else:
        n = rng.choice([1, 2, 3, 4, 8])
        lengths = [max(1, total // n)] * n
    case.update(lengths=" ".join(map(str, lengths)), packed=packed, states=rng.random() < 0.6)
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, factor=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * factor).to(DTYPES[dtype])


def _aux(dtype):
    """The type of states, decays and row statistics."""
    return torch.float64 if dtype == "f64" else torch.float32


def prepare(case, seed):
    g = _generator(seed)
    dtype, op = case["dtype"], case["op"]
    aux = _aux(dtype)
    s = {"case": case}
    if op in ("norm", "norm_backward"):
        rows, width = case["rows"], case["width"]
        s["x"] = _normal(g, (rows, width), dtype, 1.5) + torch.randn((rows, 1), generator=g, device="cuda").to(DTYPES[dtype])
        s["weight"] = (1 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(DTYPES[dtype])
        s["bias"] = _normal(g, (width,), dtype, 0.1)
        s["mean"], s["rstd"] = torch.empty(rows, dtype=aux, device="cuda"), torch.empty(rows, dtype=aux, device="cuda")
        s["out"] = torch.empty_like(s["x"])
        if op == "norm_backward":
            x64 = s["x"].to(torch.float64)
            s["mean"] = x64.mean(1).to(aux)
            s["rstd"] = torch.rsqrt(x64.var(1, unbiased=False) + EPS).to(aux)
            s["dout"] = _normal(g, (rows, width), dtype)
            s["dweight"], s["dbias"] = (torch.empty(width, dtype=aux, device="cuda") for _ in range(2))
        return s
    heads, kv_heads, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    # decays of 1 - 2^-2 ... 1 - 2^-12 over the heads: from a few tokens' memory to thousands
    exponent = torch.linspace(2, 12, heads, dtype=torch.float64)
    s["log_decay"] = torch.log1p(-torch.exp2(-exponent)).to(aux).cuda()
    s["scale"] = dk ** -0.5
    if op == "step":
        n = case["requests"]
        lead = (n,)
    else:
        lengths = _lengths(case)
        n = len(lengths)
        lead = (sum(lengths) + SPARE_ROWS,) if case["packed"] else (n, lengths[0])
    s["q"] = _normal(g, lead + (heads, dk), dtype)
    s["k"] = _normal(g, lead + (kv_heads, dk), dtype)
    s["v"] = _normal(g, lead + (kv_heads, dv), dtype)
    s["out"] = torch.zeros(lead + (heads, dv), dtype=DTYPES[dtype], device="cuda")
    if op == "step":
        s["state"] = torch.randn((n, heads, dk, dv), generator=g, device="cuda", dtype=aux)
        s["state_out"] = torch.empty_like(s["state"])
        s["slots"] = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        return s
    s["offsets"] = None
    if case["packed"]:
        ends = torch.tensor([0] + lengths).cumsum(0)
        s["offsets"] = ends.cuda()
    s["initial"] = s["final"] = s["d_final"] = s["d_initial"] = None
    if case["states"]:
        s["initial"] = torch.randn((n, heads, dk, dv), generator=g, device="cuda", dtype=aux)
        s["final"] = torch.empty_like(s["initial"])
    if op == "backward":
        s["dout"] = _normal(g, lead + (heads, dv), dtype)
        for name in ("q", "k", "v"):
            s["d" + name] = torch.zeros_like(s[name])
        if case["states"]:
            s["d_final"] = torch.randn((n, heads, dk, dv), generator=g, device="cuda", dtype=aux)
            s["d_initial"] = torch.empty_like(s["initial"])
    if case["packed"]:
        # what the sequences' rows are, for the plain form: row of (sequence, token), and whether there is one
        longest = max(1, max(lengths))
        t = torch.arange(longest)
        s["valid"] = (t[None, :] < torch.tensor(lengths)[:, None]).cuda()
        s["rows"] = (ends[:-1, None] + t[None, :]).clamp(max=lead[0] - 1).cuda()
    s["lengths"] = torch.tensor(lengths, dtype=torch.float64).cuda()
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_backward":
        return _plain_norm_backward(state)
    if op == "step":
        return _plain_step(state)
    return _plain_forward(state) if op == "forward" else _plain_backward(state)


# ---------------------------------------------------------------- the library's calls

def _run_own(s, op):
    import acrotensor_b200 as ab
    stream = torch.cuda.current_stream().cuda_stream
    if op == "norm":
        ab.layer_norm(s["out"], s["x"], s["weight"], s["bias"], eps=EPS, mean=s["mean"], rstd=s["rstd"], stream=stream)
        return {"out": s["out"], "mean": s["mean"], "rstd": s["rstd"]}
    if op == "norm_backward":
        scratch = torch.empty(ab.layer_norm_backward_scratch_bytes(s["x"]), dtype=torch.uint8, device="cuda")
        ab.layer_norm_backward(s["out"], s["dweight"], s["dbias"], s["dout"], s["x"], s["mean"], s["rstd"], s["weight"], scratch=scratch, stream=stream)
        return {"dx": s["out"], "dweight": s["dweight"], "dbias": s["dbias"]}
    if op == "step":
        ab.linear_attention_step(s["out"], s["state_out"], s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"], slots=s["slots"],
                                 stream=stream)
        return {"out": s["out"], "state": s["state_out"]}
    if op == "forward":
        scratch = torch.empty(ab.linear_attention_scratch_bytes(s["q"], s["k"], s["v"], s["offsets"]), dtype=torch.uint8, device="cuda")
        ab.linear_attention(s["out"], s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], offsets=s["offsets"], initial_state=s["initial"],
                            final_state=s["final"], scratch=scratch, stream=stream)
        return {"out": s["out"]} if s["final"] is None else {"out": s["out"], "final": s["final"]}
    scratch = torch.empty(ab.linear_attention_backward_scratch_bytes(s["q"], s["k"], s["v"], s["offsets"]), dtype=torch.uint8, device="cuda")
    ab.linear_attention_backward(s["dq"], s["dk"], s["dv"], s["dout"], s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], offsets=s["offsets"],
                                 initial_state=s["initial"], d_final_state=s["d_final"], d_initial_state=s["d_initial"], scratch=scratch,
                                 stream=stream)
    out = {"dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}
    return out if s["d_initial"] is None else {**out, "d_initial": s["d_initial"]}


# ---------------------------------------------------------------- the plain forms

def _plain_norm(s):
    x, aux = s["x"], s["mean"].dtype
    w = x.to(aux)
    mean = w.mean(1, keepdim=True)
    c = w - mean
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)
    y = c * rstd * s["weight"].to(aux) + s["bias"].to(aux)
    return {"out": y.to(x.dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _plain_norm_backward(s):
    x, aux = s["x"], s["mean"].dtype
    xhat = (x.to(aux) - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["dout"].to(aux)
    g = dy * s["weight"].to(aux)
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return {"dx": dx.to(x.dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}


def _plain_step(s):
    aux, group = s["state"].dtype, s["case"]["heads"] // s["case"]["kv_heads"]
    slots = s["slots"].long()
    k, v = (s[n].to(aux).repeat_interleave(group, 1) for n in ("k", "v"))
    new = torch.exp(s["log_decay"])[:, None, None] * s["state"][slots] + k[..., :, None] * v[..., None, :]
    out = s["scale"] * torch.matmul(s["q"].to(aux)[..., None, :], new)[..., 0, :]
    s["state_out"][slots] = new
    return {"out": out.to(s["q"].dtype), "state": s["state_out"]}


def _spread_out(s, x, aux):
    """[sequences, heads, chunks, CHUNK, d] in the computing type, zeros behind each sequence's end."""
    x = x.to(aux)
    if s["case"]["packed"]:
        x = torch.where(s["valid"][:, :, None, None], x[s["rows"]], 0)
    x = x.transpose(1, 2)
    pad = -x.shape[2] % CHUNK
    x = torch.nn.functional.pad(x, (0, 0, 0, pad))
    return x.unflatten(2, (-1, CHUNK))


def _gather_in(s, x, like):
    """The reverse, rounded once: rows of ``like``'s layout, zeros where no sequence has a row."""
    x = x.flatten(2, 3).transpose(1, 2)
    if not s["case"]["packed"]:
        return x[:, :like.shape[1]].to(like.dtype)
    out = torch.zeros(like.shape, dtype=like.dtype, device=like.device)
    out[s["rows"][s["valid"]]] = x[:, :s["valid"].shape[1]][s["valid"]].to(like.dtype)
    return out


def _powers(s, exponent, aux):
    """exp(exponent * log_decay) over the heads: exponent in 64 bits, [heads, ...] or [sequences, heads, ...]; 0 for negative exponents."""
    g = s["log_decay"].to(torch.float64).reshape((-1,) + (1,) * (exponent.dim() - 1))
    return torch.where(exponent >= 0, torch.exp(exponent.clamp(min=0) * g), 0).to(aux)


def _causal(s, q, k, v, initial, reverse, aux, extra=1.0):
    """sum over the earlier tokens, this one included, of lam^distance (q.k) v, and the state's part, all of it without the scale.
    Chunks beside one another; ``reverse`` looks at the later tokens instead.  The state's first weight is lam^extra."""
    heads = q.shape[1]
    i = torch.arange(CHUNK, device="cuda", dtype=torch.float64)
    c = torch.arange(q.shape[2], device="cuda", dtype=torch.float64)
    one = torch.ones((heads, 1, 1), device="cuda", dtype=torch.float64)
    near = (i[:, None] - i[None, :]) * one
    far = (c[:, None] - 1 - c[None, :]) * CHUNK * one
    if reverse:
        near, far = near.transpose(1, 2), far.transpose(1, 2)
    left = (i if reverse else CHUNK - 1 - i) * one[:, 0]
    come = (CHUNK - i if reverse else i + 1) * one[:, 0]
    scores = torch.matmul(q, k.transpose(-1, -2)) * _powers(s, near, aux)[None, :, None]
    local = torch.matmul((k * _powers(s, left, aux)[None, :, None, :, None]).transpose(-1, -2), v)
    start = torch.matmul(_powers(s, far, aux)[None], local.flatten(3)).unflatten(3, local.shape[3:])
    out = torch.matmul(scores, v) + torch.matmul(q * _powers(s, come, aux)[None, :, None, :, None], start)
    if initial is not None:
        t = (c[:, None] * CHUNK + i[None, :])
        t = (s["lengths"][:, None, None, None] - 1 - t if reverse else t[None, None]) * one[None] + extra
        weight = _powers2(s, t, aux)
        out = out + torch.matmul(q * weight[..., None], initial[:, :, None])
    return out


def _powers2(s, exponent, aux):
    """The same for [sequences, heads, ...]."""
    g = s["log_decay"].to(torch.float64)[None, :, None, None]
    return torch.where(exponent >= 0, torch.exp(exponent.clamp(min=0) * g), 0).to(aux)


def _end_state(s, k, v, initial, reverse, aux):
    """sum over a sequence's tokens of lam^(tokens behind it) k v^T (``reverse``: tokens before it and itself), and what is left of ``initial``."""
    i = torch.arange(k.shape[2] * CHUNK, device="cuda", dtype=torch.float64)
    n = s["lengths"][:, None]
    behind = (i[None, :] + 1) * torch.ones_like(n) if reverse else n - 1 - i[None, :]
    behind = behind[:, None, None, :].expand(-1, k.shape[1], 1, -1)
    weight = _powers2(s, behind, aux)[:, :, 0]
    state = torch.matmul((k.flatten(2, 3) * weight[..., None]).transpose(-1, -2), v.flatten(2, 3))
    if initial is not None:
        state = state + _powers2(s, n[:, None, None, :].expand(-1, k.shape[1], -1, -1), aux) * initial
    return state


def _plain_forward(s):
    aux, group = _aux(s["case"]["dtype"]), s["case"]["heads"] // s["case"]["kv_heads"]
    q = _spread_out(s, s["q"], aux)
    k, v = (_spread_out(s, s[n], aux).repeat_interleave(group, 1) for n in ("k", "v"))
    out = {"out": _gather_in(s, s["scale"] * _causal(s, q, k, v, s["initial"], False, aux), s["out"])}
    if s["final"] is not None:
        out["final"] = _end_state(s, k, v, s["initial"], False, aux)
    return out


def _plain_backward(s):
    aux, group = _aux(s["case"]["dtype"]), s["case"]["heads"] // s["case"]["kv_heads"]
    q, do = (_spread_out(s, s[n], aux) for n in ("q", "dout"))
    k, v = (_spread_out(s, s[n], aux).repeat_interleave(group, 1) for n in ("k", "v"))
    turned = None if s["initial"] is None else s["initial"].transpose(-1, -2)
    dfinal = None if s["d_final"] is None else s["d_final"] / s["scale"]
    dturned = None if dfinal is None else dfinal.transpose(-1, -2)
    dq = s["scale"] * _causal(s, do, v, k, turned, False, aux)
    dk = s["scale"] * _causal(s, v, do, q, dturned, True, aux, 0.0)
    dv = s["scale"] * _causal(s, k, q, do, dfinal, True, aux, 0.0)
    if group > 1:
        dk, dv = (x.unflatten(1, (-1, group)).sum(2) for x in (dk, dv))
    out = {"dq": _gather_in(s, dq, s["dq"]), "dk": _gather_in(s, dk, s["dk"]), "dv": _gather_in(s, dv, s["dv"])}
    if s["d_initial"] is not None:
        out["d_initial"] = s["scale"] * _end_state(s, q, do, dfinal, True, aux)
    return out


# ---------------------------------------------------------------- what cannot be done without

def work(case):
    e, op = BYTES[case["dtype"]], case["op"]
    a = 8 if case["dtype"] == "f64" else 4
    if op == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": 2 * n * e + 2 * case["width"] * e + 2 * case["rows"] * a, "flops": 8 * n}
    if op == "norm_backward":
        n = case["rows"] * case["width"]
        return {"bytes": 3 * n * e + case["width"] * (e + 2 * a) + 2 * case["rows"] * a, "flops": 13 * n}
    heads, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    qs, ks, vs, os = heads * dk * e, kv * dk * e, kv * dv * e, heads * dv * e
    state = heads * dk * dv * a
    if op == "step":
        n = case["requests"]
        return {"bytes": n * (qs + ks + vs + os + 2 * state + 4) + heads * a, "flops": 5 * n * heads * dk * dv}
    n = sum(_lengths(case))
    states = len(_lengths(case)) * state if case["states"] else 0
    if op == "forward":
        return {"bytes": n * (qs + ks + vs + os) + 2 * states, "flops": 4 * n * heads * dk * dv}
    return {"bytes": n * (2 * qs + 2 * ks + 2 * vs + os) + 3 * states, "flops": 10 * n * heads * dk * dv}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], torch.float64
    if op in ("norm", "norm_backward"):
        x = s["x"].to(d)
        if op == "norm":
            mean, var = x.mean(1), x.var(1, unbiased=False)
            rstd = 1 / torch.sqrt(var + EPS)
            return {"out": (x - mean[:, None]) * rstd[:, None] * s["weight"].to(d) + s["bias"].to(d), "mean": mean, "rstd": rstd}
        leaf, weight, bias = (t.to(d).requires_grad_() for t in (s["x"], s["weight"], s["bias"]))
        # the statistics are inputs here: the gradient through them is written out
        mean, rstd = s["mean"].to(d)[:, None], s["rstd"].to(d)[:, None]
        g = s["dout"].to(d) * weight.detach()
        xhat = (x - mean) * rstd
        width = case["width"]
        dx = (width * g - g.sum(1, keepdim=True) - xhat * (g * xhat).sum(1, keepdim=True)) * rstd / width
        ((leaf.detach() - mean) * rstd * weight + bias).backward(s["dout"].to(d))
        return {"dx": dx, "dweight": weight.grad, "dbias": bias.grad}
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    lam = torch.exp(s["log_decay"].to(d))[:, None, None]
    q, k, v = s["q"].to(d), s["k"].to(d).repeat_interleave(group, -2), s["v"].to(d).repeat_interleave(group, -2)
    scale = s["scale"]
    if op == "step":
        state = torch.empty(s["state"].shape, dtype=d, device="cuda")
        out = torch.empty(s["out"].shape, dtype=d, device="cuda")
        for r, slot in enumerate(s["slots"].tolist()):
            state[slot] = lam * s["state"][slot].to(d) + torch.einsum("ha,hb->hab", k[r], v[r])
            out[r] = scale * torch.einsum("ha,hab->hb", q[r], state[slot])
        return {"out": out, "state": state}
    lengths = _lengths(case)
    n = len(lengths)
    starts = [sum(lengths[:i]) for i in range(n)]

    def of(x, i):
        return x[starts[i]:starts[i] + lengths[i]] if case["packed"] else x[i]

    if not case["packed"]:
        groups = [list(range(n))]          # equal lengths go together
    else:
        groups = [[i] for i in range(n)]
    if sum(max(lengths[i] for i in g) for g in groups) * (2 if op == "backward" else 1) > 140000:
        return None

    def walk(order, a, b, c, state, first):
        """state <- lam state + b c^T (``first``: lam skipped at the first token); rows a . state."""
        rows = torch.empty(a.shape[:-1] + (c.shape[-1],), dtype=d, device="cuda")
        for t in order:
            if not (first and t == order[0]):
                state = lam * state
            state = state + b[:, t, :, :, None] * c[:, t, :, None, :]
            rows[:, t] = torch.matmul(a[:, t, :, None, :], state)[..., 0, :]
        return rows, state

    def zero(g):
        return torch.zeros((len(g), heads, case["dk"], case["dv"]), dtype=d, device="cuda")

    if op == "forward":
        out = torch.zeros(s["out"].shape, dtype=d, device="cuda")
        final = torch.zeros((n, heads, case["dk"], case["dv"]), dtype=d, device="cuda")
        for g in groups:
            a, b, c = (torch.stack([of(x, i) for i in g]) for x in (q, k, v))
            state = zero(g) if s["initial"] is None else s["initial"][g].to(d)
            rows, state = walk(range(a.shape[1]), a, b, c, state, False)
            for j, i in enumerate(g):
                of(out, i)[:] = scale * rows[j]
                final[i] = state[j]
        return {"out": out} if s["final"] is None else {"out": out, "final": final}
    dq, dk, dv = (torch.zeros(x.shape, dtype=d, device="cuda") for x in (q, k, v))
    first_grad = torch.zeros((n, heads, case["dk"], case["dv"]), dtype=d, device="cuda")
    do = s["dout"].to(d)
    for g in groups:
        a, b, c, e = (torch.stack([of(x, i) for i in g]) for x in (q, k, v, do))
        state = zero(g) if s["initial"] is None else s["initial"][g].to(d)
        back = zero(g) if s["d_final"] is None else s["d_final"][g].to(d)
        tokens = a.shape[1]
        rows_q = torch.empty_like(a)
        for t in range(tokens):
            state = lam * state + b[:, t, :, :, None] * c[:, t, :, None, :]
            rows_q[:, t] = scale * torch.matmul(state, e[:, t, :, :, None])[..., 0]
        rows_k, rows_v = torch.empty_like(b), torch.empty_like(c)
        for t in range(tokens - 1, -1, -1):
            back = back + scale * a[:, t, :, :, None] * e[:, t, :, None, :]
            rows_k[:, t] = torch.matmul(back, c[:, t, :, :, None])[..., 0]
            rows_v[:, t] = torch.matmul(b[:, t, :, None, :], back)[..., 0, :]
            back = lam * back
        for j, i in enumerate(g):
            of(dq, i)[:], of(dk, i)[:], of(dv, i)[:] = rows_q[j], rows_k[j], rows_v[j]
            first_grad[i] = back[j]
    dk, dv = (x.unflatten(-2, (-1, group)).sum(-2) for x in (dk, dv))
    out = {"dq": dq, "dk": dk, "dv": dv}
    return out if s["d_initial"] is None else {**out, "d_initial": first_grad}
