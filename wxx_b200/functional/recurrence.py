"""The gated linear recurrence: a sequence mixer whose state is one vector per
sequence (no reference counterpart; kernels in ``csrc/recurrence.cu``).

    a_t = sigmoid(gate_t)        h_t = a_t h_{t-1} + (1 - a_t) x_t

``x`` is (batch, time, channels) and ``gate`` (batch, time, heads), the heads
dividing the channels: a head's gate serves its channels / heads neighbouring
channels (heads = channels: a gate per channel).  ``reset`` (batch, time),
u32, marks positions where a new document starts: the state before such a
position is zero, so documents packed into one row do not see each other, not
even their NaN.  Behind an infinite ``x`` a document's states are infinite as
the formula has it, or NaN once the product of the gates since is too small
for f32.
"""

from ._common import F, check, compact, empty, ptr_or_none
from .utils import mark_written


def _typed(name, t, dtype):
    if t.type != dtype:
        raise TypeError(f"gated_recurrence expects {dtype} {name}, got {t.type!r}")


def _inner_dense(t):
    """``t`` when its rows are dense (any other strides: a column slice of a
    projection's output is read in place), else a dense copy."""
    return t if t.shape[-1] <= 1 or t.stride[-1] == 1 and min(t.stride) >= 0 else compact(t)


def _operands(x, gate, h0, reset):
    if x.type != "f32" or gate.type != "f32":
        _typed("x", x, "f32")
        _typed("gate", gate, "f32")
    if len(x.shape) != 3 or len(gate.shape) != 3:
        raise ValueError(f"gated_recurrence expects x (batch, time, channels) and gate (batch, "
                         f"time, heads), got {tuple(x.shape)} and {tuple(gate.shape)}")
    B, T, D = x.shape
    H = gate.shape[2]
    if gate.shape[0] != B or gate.shape[1] != T:
        raise ValueError(f"gated_recurrence: gate {tuple(gate.shape)} does not match x "
                         f"{tuple(x.shape)}")
    if D and (H < 1 or D % H):
        raise ValueError(f"gated_recurrence: {D} channels cannot be split over {H} gates")
    if h0 is not None:
        _typed("h0", h0, "f32")
        if tuple(h0.shape) != (B, D):
            raise ValueError(f"gated_recurrence: h0 {tuple(h0.shape)} is not {(B, D)}")
        h0 = compact(h0)
    if reset is not None:
        _typed("reset", reset, "u32")
        if tuple(reset.shape) != (B, T):
            raise ValueError(f"gated_recurrence: reset {tuple(reset.shape)} is not {(B, T)}")
        reset = compact(reset)
    return _inner_dense(x), _inner_dense(gate), h0, reset, B, T, D, H


def gated_recurrence(x, gate, h0=None, reset=None):
    """``(h, h_last)``: the states (batch, time, channels) and the state after
    the last position (batch, channels), which a following call or
    ``gated_recurrence_step`` continues from.  ``h0`` (batch, channels) is the
    state before position 0 (zero when omitted)."""
    x, gate, h0, reset, B, T, D, H = _operands(x, gate, h0, reset)
    h = empty((B, T, D))
    last = empty((B, D))
    check(F.wxx_gated_recurrence(h.buffer.ptr, last.buffer.ptr, x.ptr, x.stride[0], x.stride[1],
                                 gate.ptr, gate.stride[0], gate.stride[1], ptr_or_none(h0),
                                 ptr_or_none(reset), B, T, D, H), "gated_recurrence")
    return h, last


def gated_recurrence_backward(grad, x, gate, h, h0=None, reset=None, grad_last=None):
    """``(dx, dgate, dh0)`` from the gradient ``grad`` of the states and, when
    given, ``grad_last`` of ``h_last``; ``h`` is the forward's first result.
    ``dh0`` is None without ``h0``.  A gate shared by a head's channels
    receives the sum over them."""
    x, gate, h0, reset, B, T, D, H = _operands(x, gate, h0, reset)
    for name, t, shape in (("grad", grad, (B, T, D)), ("h", h, (B, T, D)),
                           ("grad_last", grad_last, (B, D))):
        if t is None and name == "grad_last":
            continue
        _typed(name, t, "f32")
        if tuple(t.shape) != shape:
            raise ValueError(f"gated_recurrence_backward: {name} {tuple(t.shape)} is not {shape}")
    grad, h = compact(grad), compact(h)
    grad_last = None if grad_last is None else compact(grad_last)
    dx = empty((B, T, D))
    dgate = empty((B, T, H))
    dh0 = None if h0 is None else empty((B, D))
    check(F.wxx_gated_recurrence_backward(
        dx.buffer.ptr, dgate.buffer.ptr, ptr_or_none(dh0), grad.ptr, ptr_or_none(grad_last), x.ptr,
        x.stride[0], x.stride[1], gate.ptr, gate.stride[0], gate.stride[1], h.ptr, ptr_or_none(h0),
        ptr_or_none(reset), B, T, D, H), "gated_recurrence_backward")
    return dx, dgate, dh0


def gated_recurrence_step(x, gate, state):
    """One position per sequence: ``state`` (batch, channels) becomes
    ``a state + (1 - a) x`` in place and is returned; ``x`` (batch, channels),
    ``gate`` (batch, heads)."""
    for name, t in (("x", x), ("gate", gate), ("state", state)):
        _typed(name, t, "f32")
        if len(t.shape) != 2:
            raise ValueError(f"gated_recurrence_step expects x (batch, channels), gate (batch, "
                             f"heads) and state (batch, channels), got {name} {tuple(t.shape)}")
    B, D = x.shape
    H = gate.shape[1]
    if gate.shape[0] != B or tuple(state.shape) != (B, D):
        raise ValueError(f"gated_recurrence_step: gate {tuple(gate.shape)} and state "
                         f"{tuple(state.shape)} do not match x {tuple(x.shape)}")
    if D and (H < 1 or D % H):
        raise ValueError(f"gated_recurrence_step: {D} channels cannot be split over {H} gates")
    if not state.is_dense():
        raise ValueError("gated_recurrence_step: the state is updated in place and must be dense")
    x, gate = _inner_dense(x), _inner_dense(gate)
    check(F.wxx_gated_recurrence_step(state.ptr, x.ptr, x.stride[0], gate.ptr, gate.stride[0], B,
                                      D, H), "gated_recurrence_step")
    mark_written(state)
    return state
