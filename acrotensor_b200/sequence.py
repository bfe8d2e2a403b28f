"""Sequence operators on device arrays: linear attention with a decay for each head and layer norm, with their gradients.

Arrays are objects with ``data_ptr()``, ``shape``, ``stride()`` (in elements) and ``dtype`` on the current CUDA device, for example torch
CUDA tensors; outputs come first and are the caller's, as everywhere in this library.  Element types: float64, float32, bfloat16,
float16.  Sums, states, decays and row statistics are float32 (float64 for float64 data).  ``stream`` is an integer cudaStream_t; None
means the calling thread's stream (:func:`acrotensor_b200.set_stream`, else the legacy default stream), which is NOT a stream that
another library has made current.  Nothing here synchronises; every call may be captured into a CUDA graph.  Bad arguments raise
AcroError or ValueError before anything is launched; bad entries of ``offsets`` and ``slots``, which only the device reads, are skipped
and reported by ``acro_b200_device_status()``.

The formulas stand in include/acro_b200.h; acro::TensorEngine has the same operators for fp64 tensors (``TensorEngine.LinearAttention``).
"""
import threading

from ._lib import LinearAttentionDesc, TokenArray, check, lib

_TYPES = {"float64": 0, "float32": 1, "bfloat16": 2, "float16": 3}
_type_of_dtype = {}         # dtype object -> (type code, name of the type of sums)


def _type(x, name):
    """Type code of an array's elements and the name of their type of sums."""
    found = _type_of_dtype.get(x.dtype)
    if found is None:
        text = str(x.dtype).rsplit(".", 1)[-1]
        if text not in _TYPES:
            raise ValueError("%s has elements of type %s; float64, float32, bfloat16 and float16 are supported" % (name, text))
        found = _type_of_dtype[x.dtype] = (_TYPES[text], "float64" if text == "float64" else "float32", text)
    return found


def _same_type(like, **arrays):
    for name, x in arrays.items():
        if x is not None and x.dtype != like:
            raise ValueError("%s has elements of type %s, not %s" % (name, x.dtype, like))


def _of_type(text, **arrays):
    for name, x in arrays.items():
        if x is not None and str(x.dtype).rsplit(".", 1)[-1] != text:
            raise ValueError("%s has elements of type %s, not %s" % (name, x.dtype, text))


def _shape(name, x, shape):
    if tuple(x.shape) != shape:
        raise ValueError("%s has the shape %s, not %s" % (name, tuple(x.shape), shape))


def _contiguous(name, x):
    if x is None:
        return
    expect = 1
    for n, s in zip(reversed(tuple(x.shape)), reversed(tuple(x.stride()))):
        if n != 1 and s != expect:
            raise ValueError("%s is not contiguous" % name)
        expect *= n


def _pointer(x):
    return None if x is None else x.data_ptr()


def _stream(stream):
    return lib().acro_b200_get_stream() if stream is None else stream


def _rows(name, x, lead):
    """The C view of an array [(sequences,) tokens, heads, columns] or, for a step, [requests, heads, columns]."""
    stride = x.stride()
    if x.shape[-1] > 1 and stride[-1] != 1:
        raise ValueError("the columns of %s are not contiguous" % name)
    if lead == 2:
        return TokenArray(x.data_ptr(), stride[0], stride[1], stride[2])
    return TokenArray(x.data_ptr(), stride[0], stride[0], stride[1])


def _scratch(scratch, need):
    if not need:
        return None, 0
    if scratch is None:
        raise ValueError("this call needs %d bytes of scratch" % need)
    n = scratch.element_size()
    if len(scratch.shape) != 1 or (scratch.shape[0] > 1 and scratch.stride()[0] != 1):
        _contiguous("scratch", scratch)
    for d in scratch.shape:
        n *= d
    return scratch.data_ptr(), n


class _Plan:
    """What a call's shapes, strides and types come to, checked: everything but the addresses.  Kept per thread, since a call fills the
    addresses in."""
    __slots__ = ("desc", "rows", "count", "need", "extra")


_local = threading.local()
_PLANS = 1024               # kept per thread


def _known(key):
    plans = getattr(_local, "plans", None)
    if plans is None:
        plans = _local.plans = {}
    return plans.get(key)


def _keep(key, desc, rows, count=0, need=0, extra=None):
    plan = _Plan()
    plan.desc, plan.rows, plan.count, plan.need, plan.extra = desc, rows, count, need, extra
    if len(_local.plans) >= _PLANS:
        _local.plans.clear()
    _local.plans[key] = plan
    return plan


def _form(x):
    return None if x is None else (x.shape, x.stride(), x.dtype)


def _attention_desc(q, k, v, scale, offsets, step=False):
    code = _type(q, "q")[0]
    _same_type(q.dtype, k=k, v=v)
    lead = 1 if step or offsets is not None else 2
    if len(q.shape) != lead + 2 or len(k.shape) != lead + 2 or len(v.shape) != lead + 2:
        raise ValueError("q, k and v have %d dims: %s" % (lead + 2, "[requests, heads, columns]" if step else
                                                          "[rows, heads, columns] with offsets, else [sequences, tokens, heads, columns]"))
    if tuple(k.shape[:lead]) != tuple(q.shape[:lead]) or tuple(v.shape[:lead + 1]) != tuple(k.shape[:lead + 1]) or k.shape[-1] != q.shape[-1]:
        raise ValueError("mismatched shapes of q %s, k %s and v %s" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if step:
        sequences, tokens = q.shape[0], 1
    elif offsets is None:
        sequences, tokens = q.shape[0], q.shape[1]
    else:
        _of_type("int64", offsets=offsets)
        _contiguous("offsets", offsets)
        if len(offsets.shape) != 1 or offsets.shape[0] < 1:
            raise ValueError("offsets is not an array of sequences + 1 row numbers")
        sequences, tokens = offsets.shape[0] - 1, q.shape[0]
    return LinearAttentionDesc(code, q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1], 0, sequences, tokens, float(scale)), lead


def _check_states(desc, sums, log_decay, slots, **states):
    _of_type(sums, log_decay=log_decay, **states)
    _shape("log_decay", log_decay, (desc.q_heads,))
    _contiguous("log_decay", log_decay)
    count = desc.sequences
    if slots is not None:
        _of_type("int32", slots=slots)
        _shape("slots", slots, (desc.sequences,))
        _contiguous("slots", slots)
        count = next((x.shape[0] for x in states.values() if x is not None), 0)
    for name, x in states.items():
        if x is not None:
            _shape(name, x, (count, desc.q_heads, desc.dk, desc.dv))
            _contiguous(name, x)
    return count


def linear_attention_scratch_bytes(q, k, v, offsets=None):
    """Bytes of scratch :func:`linear_attention` needs for arrays of these shapes."""
    key = (5, _form(q), _form(k), _form(v), _form(offsets))
    plan = _known(key)
    if plan is None:
        desc, _ = _attention_desc(q, k, v, 1.0, offsets)
        plan = _keep(key, None, None, need=lib().acro_b200_linear_attention_scratch_bytes(desc, offsets is not None))
    return plan.need


def linear_attention(out, q, k, v, log_decay, scale=1.0, offsets=None, initial_state=None, final_state=None, slots=None, scratch=None, stream=None):
    """``S_t = exp(log_decay[head]) S_(t-1) + k_t v_t^T,  out_t = scale q_t^T S_t`` per sequence and query head.

    q, k [sequences, tokens, heads, dk], v, out [..., dv]; or, with ``offsets`` (int64, sequences + 1 row numbers), [rows, heads, columns] with
    sequence n in the rows offsets[n] .. offsets[n+1]-1.  k and v may have fewer heads (a divisor of q's).  States are
    [sequences, heads, dk, dv]; with ``slots`` (int32 per sequence, negative: not there) [any number, heads, dk, dv].  Slots without states
    only say which sequences are there.  ``final_state`` may be ``initial_state``.  ``scratch``: any contiguous array of :func:`linear_attention_scratch_bytes` bytes."""
    scale = float(scale)
    key = (0, scale, _form(q), _form(k), _form(v), _form(out), _form(log_decay), _form(offsets), _form(initial_state), _form(final_state), _form(slots))
    plan = _known(key)
    if plan is None:
        desc, lead = _attention_desc(q, k, v, scale, offsets)
        _same_type(q.dtype, out=out)
        _shape("out", out, tuple(q.shape[:-1]) + (desc.dv,))
        count = _check_states(desc, _type(q, "q")[1], log_decay, slots, initial_state=initial_state, final_state=final_state)
        need = lib().acro_b200_linear_attention_scratch_bytes(desc, offsets is not None)
        plan = _keep(key, desc, tuple(_rows(n, x, lead) for n, x in (("q", q), ("k", k), ("v", v), ("out", out))), count, need)
    rq, rk, rv, ro = plan.rows
    rq.data, rk.data, rv.data, ro.data = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    at, have = _scratch(scratch, plan.need)
    check(lib().acro_b200_linear_attention(plan.desc, rq, rk, rv, ro, log_decay.data_ptr(), _pointer(offsets), _pointer(initial_state),
                                           _pointer(final_state), _pointer(slots), plan.count, at, have, _stream(stream)))


def linear_attention_step(out, state_out, q, k, v, log_decay, state_in, scale=1.0, slots=None, stream=None):
    """One token of each request: ``state_out[slot] = exp(log_decay) state_in[slot] + k v^T,  out = scale q^T state_out[slot]``.

    q, k [requests, heads, dk], v, out [requests, heads, dv]; states [requests, heads, dk, dv], or with ``slots`` (int32 per request,
    negative: not there) [any number, heads, dk, dv].  ``state_out`` may be ``state_in``."""
    scale = float(scale)
    key = (1, scale, _form(q), _form(k), _form(v), _form(out), _form(log_decay), _form(state_in), _form(state_out), _form(slots))
    plan = _known(key)
    if plan is None:
        desc, lead = _attention_desc(q, k, v, scale, None, step=True)
        _same_type(q.dtype, out=out)
        _shape("out", out, (desc.sequences, desc.q_heads, desc.dv))
        if state_in is None or state_out is None:
            raise ValueError("a step needs states")
        count = _check_states(desc, _type(q, "q")[1], log_decay, slots, state_in=state_in, state_out=state_out)
        plan = _keep(key, desc, tuple(_rows(n, x, lead) for n, x in (("q", q), ("k", k), ("v", v), ("out", out))), count)
    rq, rk, rv, ro = plan.rows
    rq.data, rk.data, rv.data, ro.data = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    check(lib().acro_b200_linear_attention_step(plan.desc, rq, rk, rv, ro, log_decay.data_ptr(), state_in.data_ptr(), state_out.data_ptr(),
                                                _pointer(slots), plan.count, _stream(stream)))


def linear_attention_backward_scratch_bytes(q, k, v, offsets=None):
    """Bytes of scratch :func:`linear_attention_backward` needs for arrays of these shapes."""
    key = (6, _form(q), _form(k), _form(v), _form(offsets))
    plan = _known(key)
    if plan is None:
        desc, _ = _attention_desc(q, k, v, 1.0, offsets)
        plan = _keep(key, None, None, need=lib().acro_b200_linear_attention_backward_scratch_bytes(desc, offsets is not None))
    return plan.need


def linear_attention_backward(dq, dk, dv, dout, q, k, v, log_decay, scale=1.0, offsets=None, initial_state=None, d_final_state=None,
                              d_initial_state=None, scratch=None, stream=None):
    """Gradients of :func:`linear_attention` for ``dout`` (and ``d_final_state``) with respect to q, k, v (and the initial state).  The
    decays are constants of the layer and get none.  Shapes as there; states [sequences, heads, dk, dv]."""
    scale = float(scale)
    key = (2, scale, _form(q), _form(k), _form(v), _form(dout), _form(dq), _form(dk), _form(dv), _form(log_decay), _form(offsets), _form(initial_state),
           _form(d_final_state), _form(d_initial_state))
    plan = _known(key)
    if plan is None:
        desc, lead = _attention_desc(q, k, v, scale, offsets)
        _same_type(q.dtype, dout=dout, dq=dq, dk=dk, dv=dv)
        _shape("dout", dout, tuple(q.shape[:-1]) + (desc.dv,))
        for name, x, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
            _shape(name, x, tuple(like.shape))
        _check_states(desc, _type(q, "q")[1], log_decay, None, initial_state=initial_state, d_final_state=d_final_state,
                      d_initial_state=d_initial_state)
        need = lib().acro_b200_linear_attention_backward_scratch_bytes(desc, offsets is not None)
        arrays = (("q", q), ("k", k), ("v", v), ("dout", dout), ("dq", dq), ("dk", dk), ("dv", dv))
        plan = _keep(key, desc, tuple(_rows(n, x, lead) for n, x in arrays), 0, need)
    rows = plan.rows
    for r, x in zip(rows, (q, k, v, dout, dq, dk, dv)):
        r.data = x.data_ptr()
    at, have = _scratch(scratch, plan.need)
    check(lib().acro_b200_linear_attention_backward(
        plan.desc, rows[0], rows[1], rows[2], rows[3], log_decay.data_ptr(), _pointer(offsets), _pointer(initial_state), _pointer(d_final_state),
        rows[4], rows[5], rows[6], _pointer(d_initial_state), at, have, _stream(stream)))


def _matrix(name, x):
    """(rows, width, row stride) of an array whose leading dims run through evenly spaced rows."""
    if len(x.shape) < 1:
        raise ValueError("%s has no dims" % name)
    shape, stride = tuple(x.shape), tuple(x.stride())
    width = shape[-1]
    if width > 1 and stride[-1] != 1:
        raise ValueError("the rows of %s are not contiguous" % name)
    rows, step = 1, None
    for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if n != 1 and rows != 0:
            if step is None:
                step = s
            elif s != step * rows:
                raise ValueError("the rows of %s are not evenly spaced" % name)
        rows *= n
    return rows, width, (width if step is None else step)


def layer_norm(out, x, weight=None, bias=None, eps=1e-5, mean=None, rstd=None, stream=None):
    """``out = (x - mean) rstd weight + bias`` over the last dim of x, rstd = 1 / sqrt(variance + eps).  weight and bias (both may be None)
    are of x's type; mean and rstd (if given) receive the row statistics, as the gradient wants them.  ``out`` may be ``x``."""
    key = (3, _form(x), _form(out), _form(weight), _form(bias), _form(mean), _form(rstd))
    plan = _known(key)
    if plan is None:
        code, sums, _ = _type(x, "x")
        _same_type(x.dtype, out=out, weight=weight, bias=bias)
        _shape("out", out, tuple(x.shape))
        rows, width, x_stride = _matrix("x", x)
        y_stride = _matrix("out", out)[2]
        _row_arrays(rows, sums, mean=mean, rstd=rstd)
        _column_arrays(width, weight=weight, bias=bias)
        plan = _keep(key, None, None, extra=(code, x_stride, y_stride, rows, width))
    code, x_stride, y_stride, rows, width = plan.extra
    check(lib().acro_b200_layer_norm(code, x.data_ptr(), x_stride, _pointer(weight), _pointer(bias), out.data_ptr(), y_stride, _pointer(mean),
                                     _pointer(rstd), rows, width, eps, _stream(stream)))


def _row_arrays(rows, sums, **arrays):
    _of_type(sums, **arrays)
    for name, a in arrays.items():
        if a is not None:
            n = 1
            for d in a.shape:
                n *= d
            if n != rows:
                raise ValueError("%s has %d entries for %d rows" % (name, n, rows))
            _contiguous(name, a)


def _column_arrays(width, **arrays):
    for name, a in arrays.items():
        if a is not None:
            _shape(name, a, (width,))
            _contiguous(name, a)


def layer_norm_backward_scratch_bytes(x):
    """Bytes of scratch :func:`layer_norm_backward` needs for an array of this shape."""
    key = (7, _form(x))
    plan = _known(key)
    if plan is None:
        rows, width, _ = _matrix("x", x)
        plan = _keep(key, None, None, need=lib().acro_b200_layer_norm_backward_scratch_bytes(_type(x, "x")[0], rows, width))
    return plan.need


def layer_norm_backward(dx, dweight, dbias, dout, x, mean, rstd, weight=None, scratch=None, stream=None):
    """Gradients of :func:`layer_norm`: dx, and (unless None) dweight and dbias, the sums over all rows, in the type of sums.  mean and
    rstd are the forward pass's.  ``scratch`` is needed for dweight and dbias only.  ``dx`` may be ``dout`` or ``x``."""
    key = (4, _form(x), _form(dx), _form(dout), _form(mean), _form(rstd), _form(weight), _form(dweight), _form(dbias))
    plan = _known(key)
    if plan is None:
        code, sums, _ = _type(x, "x")
        _same_type(x.dtype, dx=dx, dout=dout, weight=weight)
        _shape("dx", dx, tuple(x.shape))
        _shape("dout", dout, tuple(x.shape))
        rows, width, x_stride = _matrix("x", x)
        if mean is None or rstd is None:
            raise ValueError("the gradient needs the mean and rstd of the forward pass")
        _row_arrays(rows, sums, mean=mean, rstd=rstd)
        _of_type(sums, dweight=dweight, dbias=dbias)
        _column_arrays(width, weight=weight, dweight=dweight, dbias=dbias)
        need = 0 if dweight is None and dbias is None else lib().acro_b200_layer_norm_backward_scratch_bytes(code, rows, width)
        plan = _keep(key, None, None, need=need, extra=(code, x_stride, _matrix("dout", dout)[2], _matrix("dx", dx)[2], rows, width))
    code, x_stride, dy_stride, dx_stride, rows, width = plan.extra
    at, have = _scratch(scratch, plan.need)
    check(lib().acro_b200_layer_norm_backward(code, dout.data_ptr(), dy_stride, x.data_ptr(), x_stride, _pointer(weight), mean.data_ptr(),
                                              rstd.data_ptr(), dx.data_ptr(), dx_stride, _pointer(dweight), _pointer(dbias), rows, width, at, have,
                                              _stream(stream)))
