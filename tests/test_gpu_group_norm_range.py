"""Group norm of numbers whose squares, or whose sums, are out of 32 bits' range."""

import numpy as np
import pytest

from oracle import retention

pytestmark = pytest.mark.gpu


def _F():
    import wxx_b200 as wxx

    return wxx.functional


def up(a, dtype=np.float32):
    return None if a is None else _F().from_numpy(np.asarray(a), dtype=dtype)


@pytest.mark.parametrize("size", [2.0 ** 62, 2.0 ** 90, 2.0 ** 124])
@pytest.mark.parametrize("shape,G", [((5, 64), 1), ((40, 1024), 16), ((3, 100), 5), ((1, 5000), 1),
                                     ((33, 2048), 2), ((3, 16, 16, 64), 32), ((2, 1000, 8), 8),
                                     ((2, 33, 700), 7), ((1, 3000, 260), 4), ((9, 3, 12), 4)])
def test_large_numbers(shape, G, size, rng):
    """The result and the gradients are those of the same numbers at an ordinary size: with u =
    2^-24, z is off by 64 u (1 + R) (1 + |z|), R = max |x| inv, as for any input."""
    F = _F()
    x = (rng.uniform(-1, 1, shape) * 2 + 0.5).astype(np.float32)
    some = x.copy()
    some[0] *= np.float32(size)                     # samples of an ordinary size beside it
    C = shape[-1]
    gamma, beta = ((1 + 0.3 * rng.standard_normal(C)).astype(np.float32) for _ in range(2))
    gate, dy = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    args = (up(gamma), up(beta), "silu", up(gate))
    y, mean, inv = F.group_norm(up(some), G, *args)
    ry, rmean, rinv = retention.group_norm(some.astype(np.float64), G, gamma, beta, "silu", gate)
    z, R = 4.0, 5.0                                 # of uniform numbers
    off = 64 * 2.0 ** -24 * (1 + R) * (1 + z) * 2
    assert np.abs(y.numpy() - ry).max() < 2 * off * np.abs(gate).max()
    wide = np.abs(some).reshape(shape[0], -1).max(-1)[:, None]
    assert (np.abs(mean.numpy() - rmean) < 64 * 2.0 ** -24 * wide).all()
    assert (np.abs(inv.numpy() - rinv) < 64 * 2.0 ** -24 * (1 + R) ** 2 * rinv).all()
    grads = F.group_norm_backward(up(dy), up(some), mean, inv, G, *args)
    refs = retention.group_norm_backward(dy, some.astype(np.float64), G, gamma, beta, "silu", gate)
    for got, ref in zip(grads, refs):
        got = got.numpy().astype(np.float64)
        assert np.isfinite(got).all()
        parts = [(got, ref)] if got.ndim == 1 else [(got[:1], ref[:1]), (got[1:], ref[1:])]
        for a, b in parts:                          # the large sample's dx by itself
            assert np.linalg.norm(a - b) <= 4e-6 * np.linalg.norm(b)


@pytest.mark.parametrize("shape,G", [((4, 64), 2), ((2, 2048), 1), ((2, 50, 16), 4), ((2, 40, 700), 7)])
def test_a_large_group_beside_others(shape, G, rng):
    """One group of a sample large, or with an infinity: the others to the bit as without it."""
    F = _F()
    x = rng.standard_normal(shape).astype(np.float32)
    per = shape[-1] // G
    good = F.group_norm(up(x), G)[0].numpy()
    for value in (3e30, np.inf, np.nan):
        big = x.copy()
        big[1, ..., 1] = value
        y, mean, inv = (t.numpy() for t in F.group_norm(up(big), G))
        own = np.zeros(shape, bool)
        own[1, ..., :per] = True
        assert np.array_equal(y[~own], good[~own])
        assert np.isfinite(y[own]).all() == np.isfinite(value)
        if np.isfinite(value):
            ref = retention.group_norm(big.astype(np.float64), G)[0]
            assert np.abs(y - ref)[own].max() < 1e-4 * np.abs(ref).max()
