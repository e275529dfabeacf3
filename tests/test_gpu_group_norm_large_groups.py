"""Group norm of groups of more numbers than a block's registers take."""

import numpy as np
import pytest

from oracle import retention

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _F():
    import wxx_b200 as wxx

    return wxx.functional


def up(a):
    return _F().from_numpy(a)


@pytest.mark.parametrize("offset", [0.0, 5.0, -50.0])
@pytest.mark.parametrize("shape,G", [((184, 2305), 1), ((26, 23628), 12), ((600, 1700), 1),
                                     ((1, 100000), 2), ((4, 5001, 6), 2), ((1, 70000, 8), 8),
                                     ((2, 4096, 512), 32), ((3, 64, 64, 36), 3)])
def test_numbers_away_from_zero(shape, G, offset, rng):
    """Means are joined as distances from one of them, so with R = |mean| inv the mean is off by its
    own rounding, u / 2 of it, and z by (R / 2 + a few) u: (R + 16) u in the 2-norm."""
    F = _F()
    x = (rng.standard_normal(shape) + offset).astype(np.float32)
    C = shape[-1]
    gamma = (1 + 0.3 * rng.standard_normal(C)).astype(np.float32)
    dy = rng.standard_normal(shape).astype(np.float32)
    y, mean, inv = F.group_norm(up(x), G, up(gamma))
    ry, rmean, rinv = retention.group_norm(x, G, gamma)
    R = np.abs(rmean * rinv).max()
    assert np.abs(mean.numpy() - rmean).max() <= (R + 4) * U / rinv.min()
    assert np.abs(inv.numpy() / rinv - 1).max() < 16 * U
    assert np.linalg.norm(y.numpy() - ry) <= (R + 16) * U * np.linalg.norm(ry)
    grads = F.group_norm_backward(up(dy), up(x), mean, inv, G, up(gamma))[:3]
    refs = retention.group_norm_backward(dy, x, G, gamma)[:3]
    # dx through z twice; the channels' sums in 32 bits
    for got, ref in zip(grads, refs):
        assert np.linalg.norm(got.numpy() - ref) <= (2 * R + 64) * U * np.linalg.norm(ref)
