"""Selection over logits: top-k and the steps of beam search (no reference
counterpart; kernels in ``csrc/select.cu``).

Values are compared as numbers and equal values ordered by the lower id, so
the results are the same on every run.
"""

import ctypes

from .. import validation
from ._common import F, check, compact, empty_group, ptr_or_none
from .utils import mark_written

_MAX_TOPK = 256
_MAX_BEAMS = 16


def topk(x, k):
    """``(values, ids)`` of the ``k`` largest entries along the last axis, in
    descending order; ids are u32.  NaN counts as larger than every number."""
    if x.type != "f32":
        raise TypeError(f"topk expects f32, got {x.type!r}")
    if not x.shape:
        raise ValueError("topk expects at least one axis")
    if isinstance(k, bool) or not isinstance(k, int):
        raise TypeError(f"k must be an int, got {type(k).__name__}")
    V = x.shape[-1]
    if not 1 <= k <= min(V, _MAX_TOPK):
        raise ValueError(f"topk: k = {k} outside [1, {min(V, _MAX_TOPK)}] for {V} entries")
    if not (len(x.shape) == 2 and x.stride[1] == 1 and x.stride[0] >= V):
        x = compact(x)
    lead = list(x.shape[:-1])
    N = validation.numel(lead)
    values, ids = empty_group((lead + [k], "f32"), (lead + [k], "u32"))
    check(F.wxx_topk(values.ptr, ids.ptr, x.ptr,
                     x.stride[0] if len(lead) == 1 else V, N, V, k), "topk")
    return values, ids


def beam_select(logits, scores, finished=None, stop_token=None):
    """One selection step of beam search.

    ``scores`` (batch, beams) are the beams' summed log-probabilities and
    ``logits`` (batch * beams, vocab) their next-token logits, the beams of an
    item in neighbouring rows.  Every beam proposes its best ``beams`` tokens
    with ``score + log softmax(logits)[token]``; the best ``beams`` proposals
    of an item are kept, equal scores by the lower beam, then the better
    logit.  With ``finished`` (batch, beams) u32 and ``stop_token``, a
    finished beam proposes only the stop token at its present score.  A beam
    without probabilities (NaN or +inf in its logits, or nothing but -inf)
    proposes at -inf.

    Returns ``(scores, parents, tokens, finished)``, each (batch, beams), best
    first: ``parents`` (u32) is the beam within the item that the proposal
    continues; ``finished`` is None without a stop token."""
    for name, t, dtype in (("logits", logits, "f32"), ("scores", scores, "f32"),
                           ("finished", finished, "u32")):
        if t is not None and t.type != dtype:
            raise TypeError(f"beam_select expects {dtype} {name}, got {t.type!r}")
    if len(scores.shape) != 2 or len(logits.shape) != 2:
        raise ValueError(f"beam_select expects logits (batch * beams, vocab) and scores (batch, "
                         f"beams), got {tuple(logits.shape)} and {tuple(scores.shape)}")
    B, W = scores.shape
    V = logits.shape[1]
    if not 1 <= W <= _MAX_BEAMS:
        raise ValueError(f"beam_select: {W} beams outside [1, {_MAX_BEAMS}]")
    if logits.shape[0] != B * W or V < 1:
        raise ValueError(f"beam_select: logits {tuple(logits.shape)} do not match scores "
                         f"{(B, W)}")
    if (finished is None) != (stop_token is None):
        raise ValueError("beam_select: finished and stop_token go together")
    if finished is not None:
        if tuple(finished.shape) != (B, W):
            raise ValueError(f"beam_select: finished {tuple(finished.shape)} is not {(B, W)}")
        if not 0 <= int(stop_token) < V:
            raise ValueError(f"beam_select: stop_token {stop_token} outside [0, {V})")
        finished = compact(finished)
    scores = compact(scores)
    if logits.stride[1] != 1 or logits.stride[0] < V:
        logits = compact(logits)
    whole = ((B, W), "u32")
    new_scores, parents, tokens, *more = empty_group(
        ((B, W), "f32"), whole, whole, *([] if finished is None else [whole]))
    new_finished = more[0] if more else None
    check(F.wxx_beam_select(new_scores.ptr, parents.ptr, tokens.ptr,
                            ptr_or_none(new_finished), logits.ptr, logits.stride[0], scores.ptr,
                            ptr_or_none(finished), B, W, V, int(stop_token or 0)), "beam_select")
    return new_scores, parents, tokens, new_finished


def beam_reorder(states, parents, cur_len=None):
    """Moves the rows of every tensor of ``states`` in place: row
    ``b * beams + w`` takes what row ``b * beams + parents[b, w]`` had.

    ``states`` are dense tensors of one axis 0 of batch * beams rows, of any
    type.  With ``cur_len`` (a u32 tensor of one element, read on the device)
    axis 1 of every state counts positions and only the first ``cur_len``
    move: a K/V cache's empty tail stays untouched.  A parent outside
    [0, beams) sets the device error word and leaves its row."""
    states = list(states)
    if parents.type != "u32":
        raise TypeError(f"beam_reorder expects u32 parents, got {parents.type!r}")
    if len(parents.shape) != 2 or not 1 <= parents.shape[1] <= _MAX_BEAMS:
        raise ValueError(f"beam_reorder expects parents (batch, beams) of 1 to {_MAX_BEAMS} "
                         f"beams, got {tuple(parents.shape)}")
    B, W = parents.shape
    if cur_len is not None and (cur_len.type != "u32" or validation.numel(cur_len.shape) != 1):
        raise TypeError("beam_reorder expects cur_len as a u32 tensor of one element")
    n = len(states)
    ptrs = (ctypes.c_void_p * max(n, 1))()
    rows = (ctypes.c_int64 * max(n, 1))()
    units = (ctypes.c_int64 * max(n, 1))()
    for i, t in enumerate(states):
        if len(t.shape) < (1 if cur_len is None else 2) or t.shape[0] != B * W:
            raise ValueError(f"beam_reorder: state {i} of shape {tuple(t.shape)} does not have "
                             f"{B * W} rows" + ("" if cur_len is None else " of positions"))
        if not t.is_dense():
            raise ValueError(f"beam_reorder: state {i} is moved in place and must be dense")
        words = t.itemsize() // 4
        ptrs[i] = t.ptr
        rows[i] = words * validation.numel(t.shape[1:])
        units[i] = 0 if cur_len is None else words * validation.numel(t.shape[2:])
    order = sorted(range(n), key=lambda i: ptrs[i] or 0)
    for i, j in zip(order, order[1:]):
        # each would move rows that the other is moving
        if rows[i] and rows[j] and (ptrs[i] or 0) + 4 * B * W * rows[i] > (ptrs[j] or 0):
            raise ValueError(f"beam_reorder: states {i} and {j} overlap in memory")
    parents = compact(parents)
    check(F.wxx_beam_reorder(n, ptrs, rows, units, parents.ptr, B, W, ptr_or_none(cur_len)),
          "beam_reorder")
    for t in states:
        mark_written(t)
    return states


def beam_append(ids, tokens, cur_len):
    """Writes the chosen tokens behind the beams' ids: ``ids[r, cur_len] =
    tokens[r]`` for the rows of ``ids`` (rows, most) u32, ``tokens`` of as many
    u32 elements, then ``cur_len`` (a u32 tensor of one element) grows by one,
    all on the device.  A full ``ids`` is left and sets the device error word."""
    for name, t in (("ids", ids), ("tokens", tokens), ("cur_len", cur_len)):
        if t.type != "u32":
            raise TypeError(f"beam_append expects u32 {name}, got {t.type!r}")
    if len(ids.shape) != 2 or ids.stride[1] != 1 or ids.stride[0] < ids.shape[1]:
        raise ValueError("beam_append: ids are written in place and must be rows of neighbouring "
                         f"elements, got shape {tuple(ids.shape)} stride {tuple(ids.stride)}")
    if validation.numel(tokens.shape) != ids.shape[0] or validation.numel(cur_len.shape) != 1:
        raise ValueError(f"beam_append: {tuple(tokens.shape)} tokens and cur_len "
                         f"{tuple(cur_len.shape)} for {ids.shape[0]} rows")
    tokens = compact(tokens)
    check(F.wxx_beam_append(ids.ptr, ids.stride[0], ids.shape[0], tokens.ptr, cur_len.ptr,
                            ids.shape[1]), "beam_append")
    mark_written(ids)
    mark_written(cur_len)
    return ids
