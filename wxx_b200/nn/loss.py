"""Losses (interface: src/wxx/nn/loss.py): called as ``loss(prediction, truth)``
and returning a scalar tensor whose ``backward()`` trains the model."""

import math

from .. import autograd


class loss:
    """Base of the losses."""

    def __call__(self, *args, **kwargs):
        raise NotImplementedError


def _over_rows(rows, mask):
    """The mean of the rows' losses (N, 1), or their mean weighted by ``mask``."""
    if mask is None:
        return rows.mean()
    n = rows.shape[0]
    if math.prod(mask.shape) != n:
        raise ValueError(f"mask must contain one value per prediction row; got "
                         f"{math.prod(mask.shape)} values for {n} rows")
    weights = mask.reshape((n, 1))
    return (rows * weights).sum() / weights.sum()


class CCELoss(loss):
    """Mean softmax cross-entropy of (B, K) logits against (B,) u32 targets
    (``CrossEntropyLoss`` per row, then the mean).  With ``mask`` (B values)
    the rows are weighted and the sum is divided by ``mask.sum()``."""

    def __call__(self, prediction, truth, mask=None):
        rows = autograd.CrossEntropyLoss(prediction).forward(prediction, truth)
        return _over_rows(rows, mask)


class DistillLoss(loss):
    """Mean over rows of ``temperature^2 KL(teacher || student)`` for (N, V)
    student logits against a teacher's stored top logits (N, K) and their ids
    (N, K) u32 (``functional.distill_loss``; the teacher's come from
    ``functional.topk``).  ``mask`` as for ``CCELoss``."""

    def __init__(self, temperature=1.0):
        self.temperature = float(temperature)

    def __call__(self, prediction, top_logits, top_ids, mask=None):
        rows = autograd.DistillLoss(prediction).forward(prediction, top_logits, top_ids,
                                                        self.temperature)
        return _over_rows(rows, mask)


class MAELoss(loss):
    """Mean absolute error."""

    def __call__(self, prediction, truth):
        return (truth - prediction).abs().mean()
