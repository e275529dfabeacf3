"""Linear attention with a decay for each head (no reference counterpart; kernels in
``csrc/linear_attention.cu``): a sequence mixer whose state is one matrix per sequence
and head.

    S_t = exp(log_decay) S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t

``q`` and ``k`` are (batch, time, heads * dk), ``v`` (batch, time, heads * dv), with any
strides whose channels are dense (column slices of a projection are read in place), and
``log_decay`` (heads), the logarithms of the heads' decays, at most 0; it is a constant of
the model and receives no gradient.  ``reset`` (batch, time), u32, marks positions where a
new document starts: the state before such a position is zero, so documents packed into
one row do not see each other, not even their NaN.  Heads have up to 256 channels.

Operands enter the products as pairs of half-precision numbers, 22 bits of each row (and of the
state) relative to its length: results are good to about 6e-7 of their terms.  Rows that are not
0 but shorter than 2^-60, or longer than 2^63, sizes 2^110 apart within 64 positions, an infinity or
a NaN, and heads of more than 128 channels are worked through position by position, which takes
longer.
"""

from ._common import F, check, compact, empty, finite32, ptr_or_none
from .utils import mark_written

_MOST = 256


def _typed(what, **tensors):
    for name, t in tensors.items():
        if t is not None and t.type != ("u32" if name == "reset" else "f32"):
            raise TypeError(f"{what} expects {'u32' if name == 'reset' else 'f32'} {name}, got "
                            f"{t.type!r}")


def _inner_dense(t):
    """``t`` when its rows are dense (any other strides: a column slice of a projection's
    output is read in place), else a dense copy."""
    return t if t.shape[-1] <= 1 or t.stride[-1] == 1 and min(t.stride) >= 0 else compact(t)


def _heads(what, q, k, v, log_decay, rank):
    """(H, dk, dv) of operands of the given rank that fit together."""
    names = "(batch, time, channels)" if rank == 3 else "(batch, channels)"
    for name, t in (("q", q), ("k", k), ("v", v)):
        if len(t.shape) != rank:
            raise ValueError(f"{what} expects {name} {names}, got {tuple(t.shape)}")
        if tuple(t.shape[:-1]) != tuple(q.shape[:-1]):
            raise ValueError(f"{what}: {name} {tuple(t.shape)} does not match q {tuple(q.shape)}")
    if tuple(k.shape) != tuple(q.shape):
        raise ValueError(f"{what}: k {tuple(k.shape)} is not like q {tuple(q.shape)}")
    if len(log_decay.shape) != 1 or log_decay.shape[0] < 1:
        raise ValueError(f"{what} expects one log_decay a head, got {tuple(log_decay.shape)}")
    H = log_decay.shape[0]
    if q.shape[-1] % H or v.shape[-1] % H:
        raise ValueError(f"{what}: {q.shape[-1]} and {v.shape[-1]} channels cannot be split over "
                         f"{H} heads")
    dk, dv = q.shape[-1] // H, v.shape[-1] // H
    if dk > _MOST or dv > _MOST:
        raise ValueError(f"{what}: heads of {dk} and {dv} channels, {_MOST} at most")
    return H, dk, dv


def _operands(what, q, k, v, log_decay, h0, reset, scale):
    _typed(what, q=q, k=k, v=v, log_decay=log_decay, h0=h0, reset=reset)
    H, dk, dv = _heads(what, q, k, v, log_decay, 3)
    B, T, _ = q.shape
    if h0 is not None and tuple(h0.shape) != (B, H, dk, dv):
        raise ValueError(f"{what}: h0 {tuple(h0.shape)} is not {(B, H, dk, dv)}")
    if reset is not None and tuple(reset.shape) != (B, T):
        raise ValueError(f"{what}: reset {tuple(reset.shape)} is not {(B, T)}")
    scale = float(scale)
    if not finite32(scale):
        raise ValueError(f"{what}: the scale must be finite in 32 bits, got {scale}")
    given = [None if t is None else compact(t) for t in (log_decay, h0, reset)]
    return (*(_inner_dense(t) for t in (q, k, v)), *given, scale, B, T, H, dk, dv)


def linear_attention(q, k, v, log_decay, h0=None, reset=None, scale=1.0):
    """``(o, last)``: the outputs (batch, time, heads * dv) and the state after the last
    position (batch, heads, dk, dv), which a following call or ``linear_attention_step``
    continues from.  ``h0`` is the state before position 0 (zero when omitted)."""
    q, k, v, log_decay, h0, reset, scale, B, T, H, dk, dv = _operands(
        "linear_attention", q, k, v, log_decay, h0, reset, scale)
    o = empty((B, T, H * dv))
    last = empty((B, H, dk, dv))
    check(F.wxx_linear_attention(o.buffer.ptr, last.buffer.ptr, q.ptr, q.stride[0], q.stride[1],
                                 k.ptr, k.stride[0], k.stride[1], v.ptr, v.stride[0], v.stride[1],
                                 log_decay.ptr, ptr_or_none(h0), ptr_or_none(reset), B, T, H, dk,
                                 dv, scale), "linear_attention")
    return o, last


def linear_attention_backward(grad, q, k, v, log_decay, h0=None, reset=None, grad_last=None,
                              scale=1.0):
    """``(dq, dk, dv, dh0)`` from the gradient ``grad`` of the outputs and, when given,
    ``grad_last`` of the last state.  ``dh0`` is None without ``h0``."""
    what = "linear_attention_backward"
    q, k, v, log_decay, h0, reset, scale, B, T, H, dk, dv = _operands(
        what, q, k, v, log_decay, h0, reset, scale)
    _typed(what, grad=grad, grad_last=grad_last)
    for name, t, shape in (("grad", grad, (B, T, H * dv)),
                           ("grad_last", grad_last, (B, H, dk, dv))):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f"{what}: {name} {tuple(t.shape)} is not {shape}")
    grad = compact(grad)
    grad_last = None if grad_last is None else compact(grad_last)
    dq, dkey, dvalue = empty((B, T, H * dk)), empty((B, T, H * dk)), empty((B, T, H * dv))
    dh0 = None if h0 is None else empty((B, H, dk, dv))
    check(F.wxx_linear_attention_backward(
        dq.buffer.ptr, dkey.buffer.ptr, dvalue.buffer.ptr, ptr_or_none(dh0), grad.ptr,
        ptr_or_none(grad_last), q.ptr, q.stride[0], q.stride[1], k.ptr, k.stride[0], k.stride[1],
        v.ptr, v.stride[0], v.stride[1], log_decay.ptr, ptr_or_none(h0), ptr_or_none(reset), B, T,
        H, dk, dv, scale), what)
    return dq, dkey, dvalue, dh0


def linear_attention_step(q, k, v, log_decay, state, scale=1.0):
    """One position per sequence: ``state`` (batch, heads, dk, dv) becomes
    ``exp(log_decay) state + k v^T`` in place, and the outputs (batch, heads * dv) are
    returned; ``q``, ``k`` (batch, heads * dk), ``v`` (batch, heads * dv)."""
    what = "linear_attention_step"
    _typed(what, q=q, k=k, v=v, log_decay=log_decay, state=state)
    H, dk, dv = _heads(what, q, k, v, log_decay, 2)
    B = q.shape[0]
    if tuple(state.shape) != (B, H, dk, dv):
        raise ValueError(f"{what}: state {tuple(state.shape)} is not {(B, H, dk, dv)}")
    if not state.is_dense():
        raise ValueError(f"{what}: the state is updated in place and must be dense")
    scale = float(scale)
    if not finite32(scale):
        raise ValueError(f"{what}: the scale must be finite in 32 bits, got {scale}")
    q, k, v, log_decay = (_inner_dense(t) for t in (q, k, v, log_decay))
    o = empty((B, H * dv))
    check(F.wxx_linear_attention_step(o.buffer.ptr, state.ptr, q.ptr, q.stride[0], k.ptr,
                                      k.stride[0], v.ptr, v.stride[0], log_decay.ptr, B, H, dk, dv,
                                      scale), what)
    mark_written(state)
    return o
