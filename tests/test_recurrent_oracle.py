"""CPU tests of the 64-bit restatements of the recurrence, distillation, top-k
and beam-search operators (gradients against central differences), and the
operators' argument checks, which raise before any device work."""

import numpy as np
import pytest

from oracle import recurrent


def differences(f, v, eps=1e-5):
    g = np.zeros_like(v)
    for i in np.ndindex(v.shape):
        up, down = v.copy(), v.copy()
        up[i] += eps
        down[i] -= eps
        g[i] = (f(up) - f(down)) / (2 * eps)
    return g


@pytest.mark.parametrize("heads", [6, 2])
@pytest.mark.parametrize("with_reset", [False, True])
def test_recurrence_gradients_against_differences(heads, with_reset):
    rng = np.random.default_rng(0)
    B, T, D = 2, 5, 6
    x, g = rng.standard_normal((B, T, D)), rng.standard_normal((B, T, heads))
    h0, dh = rng.standard_normal((B, D)), rng.standard_normal((B, T, D))
    dlast = rng.standard_normal((B, D))
    reset = None
    if with_reset:
        reset = np.zeros((B, T), np.uint32)
        reset[0, 0] = reset[1, 2] = reset[1, 3] = 1

    def value(x, g, h0):
        h, last = recurrent.recurrence(x, g, h0, reset)
        return (h * dh).sum() + (last * dlast).sum()

    dx, dg, dh0 = recurrent.recurrence_backward(dh, x, g, h0, reset, dlast)
    # second-order differences at 1e-5: truncation 1e-10, rounding 1e-16 / 1e-5
    assert np.abs(dx - differences(lambda v: value(v, g, h0), x)).max() < 1e-8
    assert np.abs(dg - differences(lambda v: value(x, v, h0), g)).max() < 1e-8
    assert np.abs(dh0 - differences(lambda v: value(x, g, v), h0)).max() < 1e-8


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_distill_gradient_against_differences(tau):
    rng = np.random.default_rng(1)
    N, V, K = 4, 9, 5
    z, top = rng.standard_normal((N, V)), rng.standard_normal((N, K))
    ids = np.stack([rng.permutation(V)[:K] for _ in range(N)])
    top[1, 3:] = -np.inf
    top[2] = -np.inf
    ids[3, 1] = ids[3, 0]                    # an id stored twice
    grad = rng.standard_normal((N, 1))
    d = recurrent.distill_backward(grad, z, top, ids, tau)
    ref = differences(lambda v: (recurrent.distill(v, top, ids, tau)[0] * grad).sum(), z)
    assert np.abs(d - ref).max() < 1e-8
    assert not d[2].any()


def test_distill_is_zero_for_the_same_distribution():
    rng = np.random.default_rng(2)
    z = rng.standard_normal((3, 7))
    ids = np.tile(np.arange(7), (3, 1))
    loss, _, _ = recurrent.distill(z, z + 4.0, ids, 1.5)
    assert np.abs(loss).max() < 1e-14


def test_beam_select_equals_search_over_all_sequences():
    """Two steps with as many beams as tokens keep the best pairs of tokens."""
    rng = np.random.default_rng(3)
    W = V = 4
    first, second = rng.standard_normal((1, V)), rng.standard_normal((V, V))

    def logp(r):
        return r - np.log(np.exp(r).sum(-1, keepdims=True))

    start = np.full((1, W), -np.inf)
    start[0, 0] = 0.0
    s, p, t, _ = recurrent.beam_select(np.repeat(first, W, 0), start)
    assert not p.any()
    s2, p2, t2, _ = recurrent.beam_select(second[t[0]], s)
    pairs = logp(first)[0][:, None] + logp(second)
    best = np.sort(pairs.reshape(-1))[::-1][:W]
    assert np.allclose(s2[0], best, atol=1e-12)
    assert np.allclose(pairs[t[0][p2[0]], t2[0]], best, atol=1e-12)


def test_beam_select_finished_and_empty_rows():
    z = np.zeros((3, 5))
    z[1] = -np.inf
    s, p, t, f = recurrent.beam_select(z, np.array([[-1.0, -2.0, -0.5]]), np.array([[0, 0, 1]]), 2)
    assert p[0, 0] == 2 and t[0, 0] == 2 and s[0, 0] == -0.5 and f[0, 0] == 1
    assert list(p[0, 1:]) == [0, 0] and list(t[0, 1:]) == [0, 1]


class _Fake:
    """A tensor's metadata without a device."""

    def __init__(self, shape, dtype="f32", stride=None):
        from wxx_b200 import validation

        self.shape, self.type = list(shape), dtype
        self.stride = stride or validation.contiguous_strides(self.shape)
        self.offset, self.ptr = 0, 0

    def is_dense(self):
        from wxx_b200 import validation

        return validation.is_contiguous_layout(self.shape, self.stride)

    def itemsize(self):
        return 4


def test_refusals():
    import wxx_b200.functional as F

    f, u = _Fake, lambda *s: _Fake(s, "u32")
    x = f((2, 5, 6))
    for args, err in [((u(2, 5, 6), x), TypeError),
                      ((x, f((2, 5, 4))), ValueError),             # 6 channels, 4 gates
                      ((x, f((2, 4, 6))), ValueError),
                      ((f((5, 6)), f((5, 6))), ValueError),
                      ((x, x, f((2, 5))), ValueError),
                      ((x, x, None, f((2, 5))), TypeError),
                      ((x, x, None, u(2, 4)), ValueError)]:
        with pytest.raises(err):
            F.gated_recurrence(*args)
    with pytest.raises(ValueError):
        F.gated_recurrence_backward(f((2, 5, 5)), x, x, x)
    with pytest.raises(ValueError):
        F.gated_recurrence_backward(x, x, x, f((2, 4, 6)))
    with pytest.raises(ValueError):
        F.gated_recurrence_step(f((2, 6)), f((2, 6)), f((2, 6), stride=(12, 1)))
    with pytest.raises(ValueError):
        F.gated_recurrence_step(f((2, 6)), f((2, 6)), f((3, 6)))

    z, t, i = f((4, 9)), f((4, 3)), u(4, 3)
    for args, err in [((z, t, f((4, 3))), TypeError), ((z, t, u(4, 2)), ValueError),
                      ((z, f((3, 3)), u(3, 3)), ValueError), ((z, t, i, 0.0), ValueError),
                      ((z, t, i, float("inf")), ValueError), ((z, t, i, float("nan")), ValueError),
                      ((f((4, 0)), t, i), ValueError), ((z, f((4, 0)), u(4, 0)), ValueError),
                      ((z, f((4, 1025)), u(4, 1025)), ValueError)]:
        with pytest.raises(err):
            F.distill_loss(*args)
    with pytest.raises(ValueError):
        F.distill_loss_backward(f((4,)), z, t, i, f((4, 2)))

    for k, err in [(0, ValueError), (10, ValueError), (2.0, TypeError), (True, TypeError)]:
        with pytest.raises(err):
            F.topk(z, k)
    with pytest.raises(ValueError):
        F.topk(f((2, 1000)), 257)
    with pytest.raises(TypeError):
        F.topk(i, 1)

    s = f((2, 2))
    for args, err in [((f((3, 9)), s), ValueError), ((z, f((1, 17))), ValueError),
                      ((z, s, u(2, 2)), ValueError), ((z, s, None, 1), ValueError),
                      ((z, s, u(2, 2), 9), ValueError), ((z, s, s, 1), TypeError),
                      ((z, s, u(2, 3), 1), ValueError), ((z, u(2, 2)), TypeError)]:
        with pytest.raises(err):
            F.beam_select(*args)
    p = u(2, 2)
    for args, err in [(([f((4, 3))], s), TypeError), (([f((3, 3))], p), ValueError),
                      (([f((4, 3), stride=(6, 1))], p), ValueError),
                      (([f((4,))], p, u(1)), ValueError), (([f((4, 3))], p, f((1,))), TypeError),
                      (([f((4, 3))], p, u(2)), TypeError)]:
        with pytest.raises(err):
            F.beam_reorder(*args)
    a = f((4, 3))
    with pytest.raises(ValueError, match="overlap"):
        F.beam_reorder([a, a], p)
