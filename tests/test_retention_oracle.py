"""CPU tests of the 64-bit restatements of rotary positions, linear attention and the group norm
(gradients against central differences, the chunked form against the recurrence), of the rotary
frequencies, and of the operators' argument checks, which raise before any device work."""

import math

import numpy as np
import pytest

from oracle import retention


def differences(f, v, eps=1e-5):
    g = np.zeros_like(v)
    for i in np.ndindex(v.shape):
        up, down = v.copy(), v.copy()
        up[i] += eps
        down[i] -= eps
        g[i] = (f(up) - f(down)) / (2 * eps)
    return g


@pytest.mark.parametrize("with_reset", [False, True])
def test_linear_attention_gradients_against_differences(with_reset):
    rng = np.random.default_rng(0)
    B, T, H, dk, dv = 2, 5, 2, 3, 2
    q, k = rng.standard_normal((B, T, H * dk)), rng.standard_normal((B, T, H * dk))
    v, do = rng.standard_normal((B, T, H * dv)), rng.standard_normal((B, T, H * dv))
    h0, dlast = rng.standard_normal((B, H, dk, dv)), rng.standard_normal((B, H, dk, dv))
    ld = np.array([-0.3, 0.0])
    reset = None
    if with_reset:
        reset = np.zeros((B, T), np.uint32)
        reset[0, 0] = reset[1, 2] = reset[1, 3] = 1

    def value(q, k, v, h0):
        o, last = retention.linear_attention(q, k, v, ld, h0, reset, 0.7)
        return (o * do).sum() + (last * dlast).sum()

    got = retention.linear_attention_backward(do, q, k, v, ld, h0, reset, dlast, 0.7)
    # second-order differences at 1e-5: truncation 1e-10, rounding 1e-16 / 1e-5
    for i, g in enumerate(got):
        args = [q, k, v, h0]
        ref = differences(lambda t: value(*args[:i], t, *args[i + 1:]), args[i])
        assert np.abs(g - ref).max() < 1e-8, i


def test_linear_attention_is_the_masked_product():
    """o_t = scale sum_s exp((t - s) log_decay) (q_t . k_s) v_s over the document so far."""
    rng = np.random.default_rng(1)
    T, ld = 9, -0.2
    q, k, v = (rng.standard_normal((1, T, 4)) for _ in range(3))
    reset = np.zeros((1, T), np.uint32)
    reset[0, 4] = 1
    o, _ = retention.linear_attention(q, k, v, np.array([ld]), None, reset, 0.5)
    t, s = np.mgrid[:T, :T]
    w = np.where((s <= t) & ((s >= 4) == (t >= 4)), np.exp((t - s) * ld), 0.0)
    assert np.abs(o[0] - 0.5 * (w * (q[0] @ k[0].T)) @ v[0]).max() < 1e-13


@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_group_norm_gradients_against_differences(activation, gated):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((2, 3, 6))
    gate = rng.standard_normal(x.shape) if gated else None
    gamma, beta = rng.standard_normal(6), rng.standard_normal(6)
    dy = rng.standard_normal(x.shape)

    def value(x, gamma, beta, gate):
        return (retention.group_norm(x, 2, gamma, beta, activation, gate)[0] * dy).sum()

    args = [x, gamma, beta] + ([gate] if gated else [])
    got = retention.group_norm_backward(dy, x, 2, gamma, beta, activation, gate)
    for i, a in enumerate(args):
        def of(t):
            given = [x, gamma, beta, gate]
            given[i] = t
            return value(*given)
        assert np.abs(got[i] - differences(of, a)).max() < 1e-7, i


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_keeps_lengths_and_distances(layout):
    rng = np.random.default_rng(3)
    f = 10000.0 ** (-np.arange(4) / 4)
    q, k = rng.standard_normal((1, 6, 10)), rng.standard_normal((1, 6, 10))
    at = np.array([[0, 5, 7, 100, 3, 3]])
    a, b = (retention.rotary(t, 1, f, 1.0, at, 0, layout) for t in (q, k))
    assert np.allclose(np.linalg.norm(a, axis=-1), np.linalg.norm(q, axis=-1), rtol=1e-14)
    assert np.array_equal(a[..., 8:], q[..., 8:])
    c, d = (retention.rotary(t, 1, f, 1.0, at, 1000, layout) for t in (q, k))
    assert np.allclose(a[0] @ b[0].T, c[0] @ d[0].T, atol=1e-11)


def test_frequencies():
    import wxx_b200.functional as F

    plain = F.rotary_frequencies(8)
    assert plain.dim == 8 and plain.gain == 1.0
    assert np.allclose(plain.frequencies, 10000.0 ** (-np.arange(4) / 4), rtol=1e-15)
    assert np.allclose(F.rotary_frequencies(8, scaling="linear", factor=4.0).frequencies,
                       np.array(plain.frequencies) / 4, rtol=1e-15)
    ntk = F.rotary_frequencies(8, scaling="ntk", factor=4.0).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain.frequencies[-1] / 4, rel_tol=1e-12)
    yarn = F.rotary_frequencies(8, scaling="yarn", factor=4.0, original_length=64)
    assert math.isclose(yarn.gain, 0.1 * math.log(4.0) + 1)
    assert yarn.frequencies[-1] == plain.frequencies[-1] / 4          # turns 0.01 times over 64
    assert plain.frequencies[0] / 4 < yarn.frequencies[0] < plain.frequencies[0]
    assert F.rotary_frequencies(2, scaling="ntk", factor=2.0).frequencies == (1.0,)
    for bad in [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=514),
                dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, base=float("nan")),
                dict(rotary_dim=8, scaling="yarn"), dict(rotary_dim=8, scaling="cubic"),
                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, factor=float("inf"))]:
        with pytest.raises(ValueError):
            F.rotary_frequencies(**bad)
    with pytest.raises(ValueError):
        F.RotaryFrequencies([])
    with pytest.raises(ValueError):
        F.RotaryFrequencies([1.0, float("nan")])
    with pytest.raises(ValueError):
        F.RotaryFrequencies([1.0], float("inf"))


class _Fake:
    """Shape and type of a tensor, for the checks that come before device work."""

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

    f, u = lambda *s: _Fake(s), lambda *s: _Fake(s, "u32")  # noqa: E731
    x, fr = f(2, 3, 16), F.rotary_frequencies(8)
    for args, err in [((u(2, 3, 16), 2, fr), TypeError), ((f(2, 16), 2, fr), ValueError),
                      ((x, 2, (1.0,)), TypeError), ((x, 3, fr), ValueError),
                      ((x, 0, fr), ValueError), ((x, 4, fr), ValueError),
                      ((x, 2, fr, f(3)), TypeError), ((x, 2, fr, u(2)), ValueError),
                      ((x, 2, fr, u(3, 2)), ValueError), ((x, 2, fr, None, -1), ValueError),
                      ((x, 2, fr, None, 1 << 32), ValueError),
                      ((x, 2, fr, None, 0, "both"), ValueError)]:
        for call in (F.rotary, F.rotary_backward):
            with pytest.raises(err):
                call(*args)

    q, v, d = f(2, 3, 8), f(2, 3, 12), f(2)
    bad = [((u(2, 3, 8), q, v, d), TypeError), ((q, u(2, 3, 8), v, d), TypeError),
           ((q, q, v, u(2)), TypeError), ((q, f(2, 4, 8), v, d), ValueError),
           ((q, f(2, 3, 6), v, d), ValueError), ((q, q, f(2, 3, 13), d), ValueError),
           ((q, q, v, f(3)), ValueError), ((q, q, v, f(2, 1)), ValueError),
           ((q, q, v, f(0)), ValueError), ((f(2, 8), f(2, 8), f(2, 12), d), ValueError),
           ((q, q, v, d, f(2, 2, 4, 5)), ValueError), ((q, q, v, d, u(2, 2, 4, 6)), TypeError),
           ((q, q, v, d, None, u(3, 2)), ValueError), ((q, q, v, d, None, f(2, 3)), TypeError),
           ((f(1, 1, 514), f(1, 1, 514), f(1, 1, 2), d), ValueError),
           ((f(1, 1, 2), f(1, 1, 2), f(1, 1, 514), d), ValueError),
           ((q, q, v, d, None, None), ValueError, float("nan")),
           ((q, q, v, d, None, None), ValueError, float("inf"))]
    for args, err, *scale in bad:
        kw = {"scale": scale[0]} if scale else {}
        with pytest.raises(err):
            F.linear_attention(*args, **kw)
        with pytest.raises(err):
            F.linear_attention_backward(v, *args, **kw)
    for grad, last, err in [(f(2, 3, 8), None, ValueError), (u(2, 3, 12), None, TypeError),
                            (v, f(2, 2, 6, 4), ValueError), (v, u(2, 2, 4, 6), TypeError)]:
        with pytest.raises(err):
            F.linear_attention_backward(grad, q, q, v, d, None, None, last)
    q, v, s = f(2, 8), f(2, 12), f(2, 2, 4, 6)
    for args, err in [((q, q, v, d, f(2, 2, 6, 4)), ValueError), ((q, q, v, d, u(2, 2, 4, 6)), TypeError),
                      ((q, q, v, d, _Fake((2, 2, 4, 6), stride=[96, 24, 6, 1])), ValueError),
                      ((q, f(3, 8), v, d, s), ValueError), ((q, q, f(2, 13), d, s), ValueError),
                      ((f(2, 1, 8), q, v, d, s), ValueError),
                      ((q, q, v, d, s, float("inf")), ValueError)]:
        with pytest.raises(err):
            F.linear_attention_step(*args)

    x = f(4, 5, 6)
    for args, err in [((u(4, 6), 2), TypeError), ((f(6), 2), ValueError), ((x, 4), ValueError),
                      ((x, 0), ValueError), ((x, 2, f(4)), ValueError), ((x, 2, u(6)), TypeError),
                      ((x, 2, None, f(5)), ValueError), ((x, 2, None, None, "tanh"), ValueError),
                      ((x, 2, None, None, None, f(4, 6)), ValueError),
                      ((x, 2, None, None, None, u(4, 5, 6)), TypeError),
                      ((x, 2, None, None, None, None, 0.0), ValueError),
                      ((x, 2, None, None, None, None, float("nan")), ValueError)]:
        with pytest.raises(err):
            F.group_norm(*args)
    m = f(4, 2)
    for args, err in [((f(4, 5, 5), x, m, m, 2), ValueError), ((x, x, f(4, 3), m, 2), ValueError),
                      ((x, x, m, f(5, 2), 2), ValueError), ((x, x, u(4, 2), m, 2), TypeError),
                      ((u(4, 5, 6), x, m, m, 2), TypeError), ((x, x, m, m, 4), ValueError)]:
        with pytest.raises(err):
            F.group_norm_backward(*args)


def test_linear_attention_a_chunk_at_a_time(rng):
    """The form for long rows against the one that goes position by position."""
    B, T, H, dk, dv = 2, 300, 3, 4, 6
    q, k = (rng.standard_normal((B, T, H * dk)) for _ in range(2))
    v, do = (rng.standard_normal((B, T, H * dv)) for _ in range(2))
    h0, dlast = (rng.standard_normal((B, H, dk, dv)) for _ in range(2))
    decay = np.array([-0.5, -0.01, 0.0])
    got = retention.linear_attention_long(do, q, k, v, decay, h0, dlast)
    want = (retention.linear_attention(q, k, v, decay, h0)
            + retention.linear_attention_backward(do, q, k, v, decay, h0, None, dlast))
    for a, b in zip(got, want):
        assert a.shape == b.shape
        assert np.abs(a - b).max() < 1e-11 * np.abs(b).max()


def test_numbers_that_32_bits_do_not_hold_are_refused():
    """The kernels take them in 32 bits, where 1e39 is infinite and 1e-50 is 0."""
    import wxx_b200.functional as F

    f = lambda *s: _Fake(s)  # noqa: E731
    for call in (lambda v: F.RotaryFrequencies((1.0,), v),
                 lambda v: F.linear_attention(f(2, 3, 8), f(2, 3, 8), f(2, 3, 12), f(2), scale=v),
                 lambda v: F.linear_attention_backward(f(2, 3, 12), f(2, 3, 8), f(2, 3, 8), f(2, 3, 12),
                                                       f(2), scale=v),
                 lambda v: F.linear_attention_step(f(2, 8), f(2, 8), f(2, 12), f(2), f(2, 2, 4, 6), v),
                 lambda v: F.group_norm(f(4, 6), 2, eps=v)):
        with pytest.raises(ValueError):
            call(1e39)
    with pytest.raises(ValueError):
        F.group_norm(f(4, 6), 2, eps=1e-50)
