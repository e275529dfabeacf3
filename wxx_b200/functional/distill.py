"""Distillation from a teacher's top logits (no reference counterpart; kernels
in ``csrc/distill.cu``).

Per row, with p the softmax of the teacher's stored logits over temperature
and q the softmax of the student's logits over temperature,

    loss = temperature^2 sum_k p_k (log p_k - log q_{id_k})

A stored logit of -inf is an absent entry, so rows may hold fewer than K; a row
with none has loss 0 and gradient 0.
"""

import math

from ._common import F, check, compact, empty, empty_group

_MAX_STORED = 1024


def _refuse(what, logits, top_logits, top_ids):
    """The message for operands that do not fit together."""
    for name, t, dtype in (("logits", logits, "f32"), ("top_logits", top_logits, "f32"),
                           ("top_ids", top_ids, "u32")):
        if t.type != dtype:
            raise TypeError(f"{what} expects {dtype} {name}, got {t.type!r}")
        if len(t.shape) != 2:
            raise ValueError(f"{what} expects a matrix of {name}, got {tuple(t.shape)}")
    raise ValueError(f"{what}: top_logits {tuple(top_logits.shape)} and top_ids "
                     f"{tuple(top_ids.shape)} do not match logits {tuple(logits.shape)}")


def _operands(what, logits, top_logits, top_ids, temperature):
    if (logits.type != "f32" or top_logits.type != "f32" or top_ids.type != "u32"
            or len(logits.shape) != 2 or len(top_logits.shape) != 2
            or top_ids.shape != top_logits.shape or top_logits.shape[0] != logits.shape[0]):
        _refuse(what, logits, top_logits, top_ids)
    N, V = logits.shape
    K = top_logits.shape[1]
    if V < 1 or not 1 <= K <= _MAX_STORED:
        raise ValueError(f"{what}: needs at least one logit and 1 to {_MAX_STORED} stored ones, "
                         f"got {V} and {K}")
    temperature = float(temperature)
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"{what}: the temperature must be positive, got {temperature}")
    if logits.stride[1] != 1 or logits.stride[0] < V:
        logits = compact(logits)
    return logits, compact(top_logits), compact(top_ids), temperature, N, V, K


def distill_loss(logits, top_logits, top_ids, temperature=1.0):
    """``(loss, stats)``: the loss (N, 1) of every row of the student's
    ``logits`` (N, V) against the teacher's stored ``top_logits`` (N, K) of the
    ids ``top_ids`` (N, K) u32, and the row statistics (N, 4) that
    ``distill_loss_backward`` takes.  An id outside [0, V) sets the device
    error word and counts as absent."""
    z, t, ids, tau, N, V, K = _operands("distill_loss", logits, top_logits, top_ids, temperature)
    stats, loss = empty_group(((N, 4), "f32"), ((N, 1), "f32"))
    check(F.wxx_distill_loss(loss.ptr, stats.ptr, z.ptr, z.stride[0], t.ptr, ids.ptr,
                             N, V, K, tau), "distill_loss")
    return loss, stats


def distill_loss_backward(grad, logits, top_logits, top_ids, stats, temperature=1.0):
    """The gradient (N, V) of the logits from the gradient ``grad`` (N, 1) of the
    losses: ``grad temperature (q_j - sum of p_k over id_k = j)``."""
    z, t, ids, tau, N, V, K = _operands("distill_loss_backward", logits, top_logits, top_ids,
                                        temperature)
    for name, v, shape in (("grad", grad, (N, 1)), ("stats", stats, (N, 4))):
        if v.type != "f32":
            raise TypeError(f"distill_loss_backward expects f32 {name}, got {v.type!r}")
        if tuple(v.shape) != shape:
            raise ValueError(f"distill_loss_backward: {name} {tuple(v.shape)} is not {shape}")
    grad, stats = compact(grad), compact(stats)
    dz = empty((N, V))
    check(F.wxx_distill_backward(dz.buffer.ptr, grad.ptr, z.ptr, z.stride[0], t.ptr, ids.ptr,
                                 stats.ptr, N, V, K, tau), "distill_loss_backward")
    return dz
