"""Linear attention with a decay for each head and layer norm in 64 bits, token by token and row by row: what the kernels are held
against.  Every function also returns the sum of the magnitudes of an entry's terms, the scale rounding errors are measured by."""
import numpy as np

#: half a step of each element type relative to the value (the error of one rounding)
HALF_STEP = {"f64": 2.0 ** -53, "f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
#: the same for the type of sums
SUM_HALF_STEP = {"f64": 2.0 ** -53, "f32": 2.0 ** -24, "bf16": 2.0 ** -24, "f16": 2.0 ** -24}
#: relative error of a product on the tensor cores: both of its operands may be a sum of two bf16 parts (8 bits each, so 2^-18 of the operand is lost)
SPLIT = {"f64": 0.0, "f32": 2.0 ** -17, "bf16": 2.0 ** -17, "f16": 2.0 ** -17}


def attention(q, k, v, log_decay, scale, state):
    """One sequence: q [T, H, dk], k, v [T, Hkv, ...], state [H, dk, dv] or None -> out, final state."""
    T, H, dk = q.shape
    group, dv = H // k.shape[1], v.shape[2]
    k, v = np.repeat(k, group, 1), np.repeat(v, group, 1)
    lam = np.exp(log_decay)[:, None, None]
    S = np.zeros((H, dk, dv)) if state is None else state.copy()
    out = np.zeros((T, H, dv))
    for t in range(T):
        S = lam * S + k[t][:, :, None] * v[t][:, None, :]
        out[t] = scale * np.einsum("ha,hab->hb", q[t], S)
    return out, S


def attention_backward(q, k, v, log_decay, scale, state, dout, dfinal):
    """-> dq, dk, dv, gradient of the initial state."""
    T, H, dk = q.shape
    group, dv = H // k.shape[1], v.shape[2]
    kk, vv = np.repeat(k, group, 1), np.repeat(v, group, 1)
    lam = np.exp(log_decay)[:, None, None]
    S = np.zeros((H, dk, dv)) if state is None else state.copy()
    G = np.zeros((H, dk, dv)) if dfinal is None else dfinal.copy()
    dq, gk, gv = np.zeros(q.shape), np.zeros(kk.shape), np.zeros(vv.shape)
    for t in range(T):
        S = lam * S + kk[t][:, :, None] * vv[t][:, None, :]
        dq[t] = scale * np.einsum("hab,hb->ha", S, dout[t])
    for t in reversed(range(T)):
        G = G + scale * q[t][:, :, None] * dout[t][:, None, :]
        gk[t] = np.einsum("hab,hb->ha", G, vv[t])
        gv[t] = np.einsum("hab,ha->hb", G, kk[t])
        G = lam * G
    return dq, gk.reshape(T, H // group, group, dk).sum(2), gv.reshape(T, H // group, group, dv).sum(2), G


def attention_tolerance(kind, exact, magnitude, tokens, columns, rounded=True):
    """|computed - exact| of an output of either function.

    An entry is a sum over the columns of products of sums over the tokens (or the other way round): at most columns + tokens + 16
    roundings of the type of sums lie between an operand and the result (16: the powers of the decay, scales and partial sums that
    are joined), each of them half a step of the magnitude; a product on the tensor cores loses SPLIT of it in either of two products;
    an output in the element type is rounded once.  Below the normal numbers of 32 bits (2^-126) nothing is relative any more: a term such as
    exp(-300) k v is 5e-131 here and zero there, so each of the terms may be off by 2^-126."""
    return ((HALF_STEP[kind] * np.abs(exact) if rounded else 0.0)
            + 1.01 * (SUM_HALF_STEP[kind] * (columns + tokens + 16) + 2 * SPLIT[kind]) * magnitude
            + (1e-300 if kind == "f64" else 2.0 ** -126 * (columns + tokens + 16))
            + (2.0 ** -25 if rounded and kind == "f16" else 0.0))      # half a step of the smallest half-precision numbers


def norm(x, weight, bias, eps):
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    y = (x - mean) * rstd
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y, mean[..., 0], rstd[..., 0]


def norm_backward(dy, x, mean, rstd, weight):
    xhat = (x - mean[:, None]) * rstd[:, None]
    g = dy if weight is None else dy * weight
    dx = rstd[:, None] * (g - g.mean(1, keepdims=True) - xhat * (g * xhat).mean(1, keepdims=True))
    return dx, (dy * xhat).sum(0), dy.sum(0)
