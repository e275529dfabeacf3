"""Group norm over trailing channels with an activation (no reference counterpart;
kernels in ``csrc/group_norm.cu``).

``x`` is (samples, ..., channels): every sample's groups of neighbouring channels are
normalised over all its positions, ``z = (x - mean) / sqrt(var + eps)``, ``n = gamma z +
beta``.  The result is ``act(n)``, or with a gate ``n act(gate)``.  Tokens that are
normalised each by itself are samples: ``x.reshape((batch * time, channels))``.
Numbers of up to 2^126 in size, whose squares 32 bits do not hold, are normalised as any other;
a NaN or an infinity makes its group's results NaN.
"""

import math

from ._common import F, check, compact, empty, empty_group, finite32, ptr_or_none

_SMALL = 1 << 20
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _operands(what, x, groups, gamma, beta, activation, gate):
    for name, t in (("x", x), ("gamma", gamma), ("beta", beta), ("gate", gate)):
        if t is not None and t.type != "f32":
            raise TypeError(f"{what} expects f32 {name}, got {t.type!r}")
    if len(x.shape) < 2:
        raise ValueError(f"{what} expects (samples, ..., channels), got {tuple(x.shape)}")
    C, groups = x.shape[-1], int(groups)
    if groups < 1 or C % groups:
        raise ValueError(f"{what}: {C} channels cannot be split over {groups} groups")
    for name, t in (("gamma", gamma), ("beta", beta)):
        if t is not None and tuple(t.shape) != (C,):
            raise ValueError(f"{what}: {name} {tuple(t.shape)} is not {(C,)}")
    if gate is not None and tuple(gate.shape) != tuple(x.shape):
        raise ValueError(f"{what}: gate {tuple(gate.shape)} does not match x {tuple(x.shape)}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: activation must be None, 'relu', 'silu' or 'gelu', got "
                         f"{activation!r}")
    given = [None if t is None else compact(t) for t in (x, gamma, beta, gate)]
    return (*given, groups, _ACTIVATIONS[activation], x.shape[0], math.prod(x.shape[1:-1]), C)


def group_norm(x, groups, gamma=None, beta=None, activation=None, gate=None, eps=1e-5):
    """``(y, mean, inv)``: the result like ``x``, and the groups' means and 1 / sqrt(var + eps)
    (samples, groups), which the backward takes.  ``gamma`` and ``beta`` (channels) default
    to 1 and 0; ``activation`` (None, ``"relu"``, ``"silu"`` or ``"gelu"``, the tanh form) is
    the result's, or with ``gate`` (like ``x``) the gate's, which multiplies the result.  Up to
    2^20 numbers share one allocation with their statistics, which is kept while any of the three
    is."""
    x, gamma, beta, gate, groups, code, N, S, C = _operands("group_norm", x, groups, gamma, beta,
                                                            activation, gate)
    if not (2.0 ** -149 <= eps and finite32(eps)):
        raise ValueError(f"group_norm: eps must be positive, got {eps}")
    # A small call takes as long as its host work: one allocation (14.7 -> 12 us).  A large
    # result must not be kept by the statistics.
    stats = (((N, groups), "f32"), ((N, groups), "f32"))
    if N * S * C <= _SMALL:
        y, mean, inv = empty_group((x.shape, "f32"), *stats)
    else:
        y, (mean, inv) = empty(x.shape), empty_group(*stats)
    check(F.wxx_group_norm(y.ptr, mean.ptr, inv.ptr, x.ptr, ptr_or_none(gate),
                           ptr_or_none(gamma), ptr_or_none(beta), N, S, C, groups, code,
                           float(eps)), "group_norm")
    return y, mean, inv


def group_norm_backward(grad, x, mean, inv, groups, gamma=None, beta=None, activation=None,
                        gate=None):
    """``(dx, dgamma, dbeta, dgate)`` from the gradient ``grad`` of ``group_norm``'s result,
    its inputs and its ``mean`` and ``inv``; ``dgate`` is None without a gate.  ``dgamma`` and
    ``dbeta`` are summed over samples and positions in a fixed order."""
    x, gamma, beta, gate, groups, code, N, S, C = _operands("group_norm_backward", x, groups,
                                                            gamma, beta, activation, gate)
    for name, t, shape in (("grad", grad, tuple(x.shape)), ("mean", mean, (N, groups)),
                           ("inv", inv, (N, groups))):
        if t.type != "f32":
            raise TypeError(f"group_norm_backward expects f32 {name}, got {t.type!r}")
        if tuple(t.shape) != shape:
            raise ValueError(f"group_norm_backward: {name} {tuple(t.shape)} is not {shape}")
    grad, mean, inv = compact(grad), compact(mean), compact(inv)
    dx = empty(x.shape)
    dgate = None if gate is None else empty(x.shape)
    dgamma, dbeta = empty_group(((C,), "f32"), ((C,), "f32"))
    check(F.wxx_group_norm_backward(dx.buffer.ptr, dgamma.ptr, dbeta.ptr, ptr_or_none(dgate),
                                    grad.ptr, x.ptr, ptr_or_none(gate), ptr_or_none(gamma),
                                    ptr_or_none(beta), mean.ptr, inv.ptr, N, S, C, groups, code),
          "group_norm_backward")
    return dx, dgamma, dbeta, dgate
