"""Rotary positions on the GPU against their 64-bit restatement.

Tolerances.  With u = 2^-24 a turned channel is a c - b s in two products and a sum (3 u of
|a| + |b|) with c and s rounded twice, once from the angle and once from the factor, and
the angle's rest rounded to u / 4 of a quarter turn: 8 u (|a| + |b|) m in all.  An angle of
position p is made in 64 bits from a frequency rounded there: p 2^-50 more.
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


def check(got, x, heads, f, positions, offset, layout, back):
    ref = retention.rotary(x, heads, f.frequencies, f.gain, positions, offset, layout, back)
    far = float(max(0 if positions is None else positions.max(), x.shape[1]) + offset)
    d = x.shape[2] // heads
    size = np.abs(np.asarray(x, np.float64)).reshape(*x.shape[:2], heads, d)
    size = 2 * size.max(-1, keepdims=True) * np.ones(d)
    bound = (8 * U + far * 2.0 ** -50) * f.gain * size.reshape(x.shape)
    assert got.shape == ref.shape
    assert (np.abs(got - ref) <= bound).all(), np.abs(got - ref).max()
    rest = got.reshape(*x.shape[:2], heads, d)[..., f.dim:]      # copied, bit by bit
    assert np.array_equal(rest, x.reshape(*x.shape[:2], heads, d)[..., f.dim:])


SHAPES = [
    # B, T, heads, head dim, turned
    (1, 1, 1, 2, 2), (2, 3, 1, 5, 4), (3, 17, 4, 64, 64), (2, 33, 3, 50, 24), (1, 130, 8, 32, 32),
    (4, 7, 2, 80, 32), (2, 65, 5, 10, 6), (1, 1000, 1, 128, 128), (32, 1, 16, 64, 64),
    (2, 9, 1, 512, 512), (1, 5, 33, 7, 2), (2, 2050, 2, 24, 8), (1, 2, 300, 16, 16),
]


@pytest.mark.parametrize("B,T,H,d,r", SHAPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("where", ["counted", "row", "rows"])
def test_forward_and_backward(B, T, H, d, r, layout, where, rng):
    F = _F()
    x = rng.standard_normal((B, T, H * d)).astype(np.float32)
    f = F.rotary_frequencies(r, scaling="yarn", factor=8.0, original_length=100)
    positions, offset = None, 0
    if where == "counted":
        offset = 12345
    elif where == "row":
        positions = rng.integers(0, 1 << 20, T).astype(np.uint32)
    else:
        positions = rng.integers(0, 1 << 32, (B, T), dtype=np.uint64).astype(np.uint32)
        positions[0, 0] = (1 << 32) - 1
    p = up(positions, np.uint32)
    check(F.rotary(up(x), H, f, p, offset, layout).numpy(), x, H, f, positions, offset, layout, False)
    check(F.rotary_backward(up(x), H, f, p, offset, layout).numpy(), x, H, f, positions, offset,
          layout, True)


def test_strided_rows_and_unaligned_views(rng):
    """Column slices of a wider tensor at any offset, a batch read twice, a row repeated."""
    F = _F()
    B, T, H, d = 3, 11, 2, 24
    wide = rng.standard_normal((B, T, 160)).astype(np.float32)
    t, f = up(wide), F.rotary_frequencies(16)
    for at in (0, 1, 2, 4, 7, 48):
        got = F.rotary(t[..., at:at + H * d], H, f).numpy()
        check(got, wide[..., at:at + H * d], H, f, None, 0, "half", False)
        same = F.rotary(up(wide[..., at:at + H * d]), H, f).numpy()
        assert np.array_equal(got, same)
    got = F.rotary(t[::2, 1::3, 8:8 + H * d], H, f, layout="interleaved").numpy()
    check(got, wide[::2, 1::3, 8:8 + H * d], H, f, None, 0, "interleaved", False)
    got = F.rotary(t.permute(1, 0, 2)[..., :H * d], H, f).numpy()
    check(got, wide.transpose(1, 0, 2)[..., :H * d], H, f, None, 0, "half", False)


def test_gradient_against_differences(rng):
    """The map is linear: differences over any step are exact up to rounding."""
    F = _F()
    f = F.rotary_frequencies(6, scaling="linear", factor=2.0)
    x, dy = (rng.standard_normal((1, 4, 16)).astype(np.float32) for _ in range(2))
    dx = F.rotary_backward(up(dy), 2, f, offset=5).numpy()

    def value(v):
        return (F.rotary(up(v), 2, f, offset=5).numpy().astype(np.float64) * dy).sum()

    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += 1
        b[i] -= 1
        assert abs((value(a) - value(b)) / 2 - dx[i]) < 64 * U * np.abs(dy).sum()


def test_products_depend_on_distance(rng):
    """What the map is for: q . k of one pair of vectors is the same at any two positions
    the same distance apart.  Bound: two roundings of 8 u each side, 64 products."""
    F = _F()
    f = F.rotary_frequencies(64)
    q, k = (rng.standard_normal((1, 1, 64)).astype(np.float32) for _ in range(2))
    def at(v, p):
        return F.rotary(up(v), 1, f, offset=p).numpy().astype(np.float64).reshape(-1)
    near = at(q, 17) @ at(k, 5)
    for p in (0, 1000, 1 << 20):
        size = np.abs(q).max() * np.abs(k).max() * 4
        assert abs(at(q, 12 + p) @ at(k, p) - near) < 64 * (16 * U + (p + 17) * 2.0 ** -50) * size


def test_scaled_frequencies():
    F = _F()
    i = np.arange(16)
    plain = 10000.0 ** (-2 * i / 32)
    assert np.allclose(F.rotary_frequencies(32).frequencies, plain, rtol=1e-14)
    assert np.allclose(F.rotary_frequencies(32, scaling="linear", factor=4).frequencies, plain / 4,
                       rtol=1e-14)
    ntk = F.rotary_frequencies(32, scaling="ntk", factor=4).frequencies
    assert ntk[0] == 1 and np.isclose(ntk[-1], plain[-1] / 4, rtol=1e-12)
    yarn = F.rotary_frequencies(32, scaling="yarn", factor=4, original_length=1000)
    turns = 1000 * plain / (2 * np.pi)
    f = np.asarray(yarn.frequencies)
    assert np.allclose(f[turns >= 32], plain[turns >= 32], rtol=1e-14)
    assert np.allclose(f[turns <= 1], plain[turns <= 1] / 4, rtol=1e-14)
    assert np.isclose(yarn.gain, 1 + 0.1 * np.log(4))


def test_non_finite_channels_stay_in_their_pairs(rng):
    F = _F()
    x = rng.standard_normal((2, 5, 24)).astype(np.float32)
    bad = x.copy()
    bad[0, 2, 3], bad[1, 4, 23] = np.nan, np.inf
    f = F.rotary_frequencies(8)
    good, got = F.rotary(up(x), 2, f).numpy(), F.rotary(up(bad), 2, f).numpy()
    differ = ~((good == got) | (np.isnan(good) & np.isnan(got)))
    assert set(map(tuple, np.argwhere(differ))) == {(0, 2, 3), (0, 2, 7), (1, 4, 23)}


def test_empty_and_captured(rng):
    import wxx_b200 as wxx

    F = _F()
    f = F.rotary_frequencies(8)
    assert F.rotary(up(np.zeros((0, 3, 16), np.float32)), 2, f).shape == [0, 3, 16]
    assert F.rotary(up(np.zeros((2, 0, 16), np.float32)), 2, f).shape == [2, 0, 16]
    x = rng.standard_normal((4, 1, 16)).astype(np.float32)
    t, p = up(x), up(np.zeros((4, 1)), np.uint32)
    g = wxx.graph.capture(lambda: F.rotary(t, 2, f, p))
    for n in (3, 99999):
        F.assign(p, up(np.full((4, 1), n), np.uint32))
        check(g.replay().numpy(), x, 2, f, np.full((4, 1), n), 0, "half", False)
    g.close()


def test_refusals():
    F = _F()
    x, f = up(np.zeros((2, 3, 16), np.float32)), F.rotary_frequencies(8)
    with pytest.raises(ValueError):
        F.rotary(up(np.zeros((2, 16), np.float32)), 2, f)
    with pytest.raises(ValueError):
        F.rotary(x, 3, f)
    with pytest.raises(ValueError):
        F.rotary(x, 4, f)                       # 8 channels to turn in heads of 4
    with pytest.raises(ValueError):
        F.rotary(x, 2, f, layout="both")
    with pytest.raises(ValueError):
        F.rotary(x, 2, f, up(np.zeros((3, 2)), np.uint32))
    with pytest.raises(ValueError):
        F.rotary(x, 2, f, offset=-1)
    with pytest.raises(TypeError):
        F.rotary(x, 2, f, up(np.zeros(3, np.float32)))
    with pytest.raises(TypeError):
        F.rotary(up(np.zeros((2, 3, 16)), np.uint32), 2, f)
    with pytest.raises(TypeError):
        F.rotary(x, 2, [1.0, 0.5])
