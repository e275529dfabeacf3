"""Group norm with an activation on the GPU against its 64-bit restatement.

Tolerances.  With u = 2^-24 and R = max |x| inv the statistics are off by a few u of the
values they are made from (the sums run over threads, each of at most 64 roundings and
mostly far fewer), so z = (x - mean) inv is off by at most 64 u (1 + R) (1 + |z|); the
activations and their slopes are good to a few u and change by at most 2 per unit.  The
gradients are made of u = gamma dn and z by means over a group.
"""

import numpy as np
import pytest

from oracle import retention

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _F():
    import wxx_b200 as wxx

    return wxx.functional


def up(a, dtype=np.float32):
    return None if a is None else _F().from_numpy(np.asarray(a), dtype=dtype)


def inputs(rng, shape, affine, gated, offset=0.5):
    x = (rng.standard_normal(shape) * 2 + offset).astype(np.float32)
    C = shape[-1]
    gamma = (1 + 0.3 * rng.standard_normal(C)).astype(np.float32) if affine else None
    beta = (0.3 * rng.standard_normal(C)).astype(np.float32) if affine else None
    gate = (2 * rng.standard_normal(shape)).astype(np.float32) if gated else None
    return x, gamma, beta, gate


def near(got, ref, bound, norm=4e-6):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape and np.isfinite(got).all()
    assert np.abs(got - ref).max(initial=0) <= bound, (np.abs(got - ref).max(), bound)
    if norm is not None:
        assert np.linalg.norm(got - ref) <= norm * np.linalg.norm(ref) + 1e-30


def check(rng, shape, G, activation, affine, gated, offset=0.5, norm=4e-6):
    F = _F()
    x, gamma, beta, gate = inputs(rng, shape, affine, gated, offset)
    args = [up(gamma), up(beta), activation, up(gate)]
    y, mean, inv = F.group_norm(up(x), G, *args)
    ry, rmean, rinv = retention.group_norm(x, G, gamma, beta, activation, gate)
    z = (x.reshape(shape[0], -1, G, shape[-1] // G) - rmean[:, None, :, None]) * rinv[:, None, :, None]
    Z, R = np.abs(z).max(initial=0), np.abs(x).max(initial=0) * rinv.max(initial=0)
    ga = 1 if gamma is None else np.abs(gamma).max()
    off = 64 * U * (1 + R) * (1 + Z) * (ga + 1)
    A = 1 if gate is None else np.abs(gate).max()
    near(y.numpy(), ry, 2 * A * off, norm)
    near(mean.numpy(), rmean, 64 * U * np.abs(x).max(initial=0), None)
    near(inv.numpy(), rinv, 64 * U * (1 + R) ** 2 * rinv.max(initial=0), None)

    dy = rng.standard_normal(shape).astype(np.float32)
    dx, dgamma, dbeta, dgate = F.group_norm_backward(up(dy), up(x), mean, inv, G, *args)
    rdx, rdgamma, rdbeta, rdgate = retention.group_norm_backward(dy, x, G, gamma, beta, activation, gate)
    D = np.abs(dy).max(initial=0) * A * 2
    near(dx.numpy(), rdx, 8 * off * D * ga * (1 + Z) ** 2 * rinv.max(initial=0), norm)
    rows = x.size / shape[-1]
    # sums over `rows` places in a fixed order, each off by what dn and z are
    near(dgamma.numpy(), rdgamma, 4 * off * D * (1 + Z) * rows, None)
    near(dbeta.numpy(), rdbeta, 4 * off * D * rows, None)
    for got, ref in ((dgamma, rdgamma), (dbeta, rdbeta)):
        assert np.linalg.norm(got.numpy() - ref) <= 1e-5 * (np.linalg.norm(ref) + np.sqrt(rows * ref.size) * D * off * 1e5)
    if gate is None:
        assert dgate is None
    else:
        near(dgate.numpy(), rdgate, 4 * off * D, norm)


SHAPES = [
    # shape, groups
    ((1, 8), 1), ((3, 16), 2), ((5, 64), 1), ((33, 1024), 16), ((2, 100), 5), ((70, 36), 3),
    ((4, 330), 10), ((2, 2048), 2), ((1, 5000), 1), ((9, 3, 12), 4), ((2, 7, 9, 30), 3),
    ((3, 16, 16, 64), 32), ((2, 1000, 8), 8), ((1, 4097, 6), 2), ((2, 5, 320), 1), ((65, 2, 40), 5),
    ((2, 33, 700), 7), ((1, 3000, 260), 4), ((300, 128), 2), ((40, 96), 1),
]


@pytest.mark.parametrize("shape,G", SHAPES)
@pytest.mark.parametrize("activation,gated", [(None, False), ("silu", False), ("silu", True),
                                              ("gelu", True)])
def test_forward_and_backward(shape, G, activation, gated, rng):
    check(rng, shape, G, activation, True, gated)


@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape,G", [((13, 64), 4), ((3, 21, 24), 2)])
def test_activations_without_affine(shape, G, activation, gated, rng):
    # relu's slope jumps at 0: none of these results lies within its rounding of it
    check(rng, shape, G, activation, False, gated)


@pytest.mark.parametrize("shape,G", [((4, 1024), 16), ((2, 500, 32), 8)])
def test_values_far_from_zero(shape, G, rng):
    """mean 1000 standard deviations away: the sums of squares must not cancel.  z is good to u
    R, so the 2-norm is compared with that."""
    check(rng, shape, G, "silu", True, False, offset=2000.0, norm=64 * U * 1000)


def test_constant_groups(rng):
    """No variance: z is 0, y = act(beta), and the gradient stays finite."""
    F = _F()
    x = np.full((3, 5, 8), 7.25, np.float32)
    beta = rng.standard_normal(8).astype(np.float32)
    y, mean, inv = F.group_norm(up(x), 2, None, up(beta), "silu")
    assert np.abs(y.numpy() - retention.act(beta.astype(np.float64), "silu")).max() < 1e-6
    assert np.array_equal(mean.numpy(), np.full((3, 2), 7.25, np.float32))
    assert np.abs(inv.numpy() - 1e5 ** 0.5).max() < 1e-4
    dx = F.group_norm_backward(up(np.ones_like(x)), up(x), mean, inv, 2, None, up(beta), "silu")[0]
    assert np.isfinite(dx.numpy()).all()


def test_groups_and_samples_do_not_meet(rng):
    F = _F()
    for shape in ((4, 64), (3, 50, 16)):
        x = rng.standard_normal(shape).astype(np.float32)
        bad = x.copy()
        bad[(1,) * (len(shape) - 1) + (5,)] = np.nan        # sample 1, group 1 of channels 4..7
        good, got = (F.group_norm(up(t), shape[-1] // 4, activation="gelu")[0].numpy() for t in (x, bad))
        hit = np.zeros(shape, bool)
        hit[1, ..., 4:8] = True
        assert np.array_equal(np.isnan(got), hit)
        assert np.array_equal(got[~hit], good[~hit])


def test_activations_far_out(rng):
    """Saturated gates: silu and gelu of +-100 are 100 and 0, with slopes 1 and 0."""
    F = _F()
    x = rng.standard_normal((2, 32)).astype(np.float32)
    n = F.group_norm(up(x), 1)[0].numpy()
    dy = rng.standard_normal((2, 32)).astype(np.float32)
    for name in ("silu", "gelu"):
        for v in (100.0, -100.0):
            gate = np.full((2, 32), v, np.float32)
            y, mean, inv = F.group_norm(up(x), 1, None, None, name, up(gate))
            assert np.abs(y.numpy() - n * max(v, 0)).max() < 1e-4
            dgate = F.group_norm_backward(up(dy), up(x), mean, inv, 1, None, None, name, up(gate))[3]
            assert np.abs(dgate.numpy() - dy * n * (v > 0)).max() < 1e-5


def test_views_and_unaligned_memory(rng):
    F = _F()
    wide = rng.standard_normal((6, 5, 70)).astype(np.float32)
    t = up(wide)
    for view, host in ((t[..., 3:35], wide[..., 3:35]), (t[1:], wide[1:]), (t[:, 2], wide[:, 2])):
        c = host.shape[-1]
        got = F.group_norm(view[..., :c // 4 * 4], 4, activation="silu")[0].numpy()
        ref = retention.group_norm(host[..., :c // 4 * 4], 4, activation="silu")[0]
        near(got, ref, 1e-5)
    flat = up(rng.standard_normal(1 + 8 * 64).astype(np.float32))
    odd = flat.narrow(0, 1, 8 * 64)                 # 4 bytes off a 16-byte boundary
    view = type(flat)((8, 64), buffer=odd.buffer, offset=odd.offset)
    near(F.group_norm(view, 4)[0].numpy(), retention.group_norm(view.numpy(), 4)[0], 1e-5)


def test_gradient_against_differences(rng):
    """The kernels' own forward, differenced at 2^-7: truncation is 2e-5 of the third
    derivative, rounding u / 2^-7 of the sum's terms."""
    F = _F()
    x, gamma, beta, gate = inputs(rng, (2, 3, 8), True, True)
    dy = rng.standard_normal(x.shape).astype(np.float32)
    given = {"x": x, "gamma": gamma, "beta": beta, "gate": gate}

    def value(x, gamma, beta, gate):
        y = F.group_norm(up(x), 2, up(gamma), up(beta), "silu", up(gate))[0].numpy()
        return (y.astype(np.float64) * dy).sum()

    _, mean, inv = F.group_norm(up(x), 2, up(gamma), up(beta), "silu", up(gate))
    grads = F.group_norm_backward(up(dy), up(x), mean, inv, 2, up(gamma), up(beta), "silu", up(gate))
    h = 2.0 ** -7
    for name, got in zip(("x", "gamma", "beta", "gate"), grads):
        got = got.numpy()
        for i in np.ndindex(got.shape):
            a, b = given[name].copy(), given[name].copy()
            a[i] += h
            b[i] -= h
            d = (value(**{**given, name: a}) - value(**{**given, name: b})) / (2 * h)
            assert abs(d - got[i]) < 1e-3 * max(1, np.abs(got).max())


def test_empty_and_captured(rng):
    import wxx_b200 as wxx

    F = _F()
    e = up(np.zeros((0, 8), np.float32))
    y, mean, inv = F.group_norm(e, 2)
    assert y.shape == [0, 8] and mean.shape == [0, 2]
    dx, dgamma, dbeta, _ = F.group_norm_backward(e, e, mean, inv, 2)
    assert dx.shape == [0, 8] and not dgamma.numpy().any() and not dbeta.numpy().any()
    x, gamma, beta, gate = inputs(rng, (6, 64), True, True)
    t = up(x)
    g = wxx.graph.capture(lambda: F.group_norm(t, 4, up_gamma, up_beta, "silu", up_gate)[0]) \
        if (up_gamma := up(gamma)) and (up_beta := up(beta)) and (up_gate := up(gate)) else None
    for k in (1.0, -3.0):
        F.assign(t, up(k * x))
        near(g.replay().numpy(), retention.group_norm(k * x, 4, gamma, beta, "silu", gate)[0], 1e-4)
    g.close()


def test_more_than_32_bits_of_numbers(rng):
    """Tokens and maps of more than 2^31 numbers, and more threads' places than 32 bits count:
    zeros, whose result is beta, but for a few rows."""
    import wxx_b200 as wxx

    F = _F()
    for shape, G, per in [((2100003, 1024), 16, 64), ((131100, 128, 128), 8, 16),
                          (((1 << 25) + 5, 144), 16, 9)]:
        x = wxx.Tensor(shape, value=0.0)
        N, C = shape[0], shape[-1]
        assert N * np.prod(shape[1:]) > 2 ** 31
        rows = [0, N // 2, N // 2 + 1, N - 1]
        some = rng.standard_normal((4, *shape[1:])).astype(np.float32)
        for i, r in enumerate(rows):
            F.assign(x.narrow(0, r, 1), up(some[i:i + 1]))
        gamma, beta = (rng.standard_normal(C).astype(np.float32) for _ in range(2))
        y, mean, inv = F.group_norm(x, G, up(gamma), up(beta))
        ref, rmean, _ = retention.group_norm(some, G, gamma, beta)
        for i, r in enumerate(rows):
            near(y.narrow(0, r, 1).numpy()[0], ref[i], 1e-5)
            near(mean.narrow(0, r, 1).numpy()[0], rmean[i], 1e-5, None)
        for r in (1, N // 4, N // 2 + 2, 3 * (N // 4), N - 2):
            got = y.narrow(0, r, 1).numpy()[0]
            assert np.array_equal(got, np.broadcast_to(beta, got.shape))
        del x, y, mean, inv


def test_refusals():
    F = _F()
    x = up(np.zeros((4, 6), np.float32))
    z = lambda *s: up(np.zeros(s, np.float32))  # noqa: E731
    with pytest.raises(ValueError):
        F.group_norm(x, 4)
    with pytest.raises(ValueError):
        F.group_norm(x, 0)
    with pytest.raises(ValueError):
        F.group_norm(z(6), 2)
    with pytest.raises(ValueError):
        F.group_norm(x, 2, z(4))
    with pytest.raises(ValueError):
        F.group_norm(x, 2, activation="tanh")
    with pytest.raises(ValueError):
        F.group_norm(x, 2, gate=z(4, 5))
    with pytest.raises(ValueError):
        F.group_norm(x, 2, eps=0.0)
    with pytest.raises(TypeError):
        F.group_norm(up(np.zeros((4, 6)), np.uint32), 2)
    with pytest.raises(ValueError):
        F.group_norm_backward(x, x, z(4, 3), z(4, 2), 2)
