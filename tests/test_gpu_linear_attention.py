"""Linear attention with a decay for each head on the GPU against its 64-bit restatement.

Tolerances.  With u = 2^-24: an output is a sum of terms lambda^(i - j) x_ip y_jp z_jr.  Every
factor reaches a product with 2^-22 of its row's largest entry lost at most (two halves of
11 bits), products and sums of up to L = min(T, 1 / (1 - lambda)) positions and dk channels
are rounded once each, and a power lambda^n as a rounded exponent's exponential is off by n
|log lambda| u: over the terms that matter (lambda^n >= 2^-24) 17 u.  So a sum is off by at
most (3 * 2^-22 + (64 + 8 sqrt(L) + dk) u) M, with M the sum of the terms' largest possible
sizes, which a sweep over the rows' largest entries gives.  The roundings are independent:
in the 2-norm 4e-6 = 64 u of the result covers sqrt(L) u for every L here.
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


def decays(H, low=3, high=10):
    """log decays of memories of 2^low to 2^high positions"""
    return np.log1p(-1 / 2.0 ** np.linspace(low, high, H)).astype(np.float32)


def inputs(rng, B, T, H, dk, dv, with_h0, with_reset):
    q, k = (rng.standard_normal((B, T, H * dk)).astype(np.float32) for _ in range(2))
    v = rng.standard_normal((B, T, H * dv)).astype(np.float32)
    h0 = rng.standard_normal((B, H, dk, dv)).astype(np.float32) if with_h0 else None
    reset = None
    if with_reset:
        reset = (rng.random((B, T)) < 0.02).astype(np.uint32) * 9     # any non-zero value
        if T:
            reset[0, 0] = 1
        if T > 70:
            reset[B - 1, 63:66] = 1                # at the edge of a chunk, one after the other
    return q, k, v, h0, reset


def largest(t, H):
    """every head's entries replaced by its row's largest size"""
    t = np.abs(np.asarray(t, np.float64)).reshape(*t.shape[:-1], H, -1)
    return np.broadcast_to(t.max(-1, keepdims=True) if t.size else t, t.shape).reshape(
        *t.shape[:-2], -1)


def room(decay, T, d):
    L = min(max(T, 1), 1 / max(1e-9, (1 - np.exp(np.float64(decay.max())))))
    return 3 * 2.0 ** -22 + (64 + 8 * np.sqrt(L) + d) * U


def close(got, ref, bound, norm=4e-6):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape
    if ref.size == 0:
        return
    assert np.isfinite(got).all()
    # a number below the smallest of 32 bits, 2^-149, is rounded to it or to 0
    assert (np.abs(got - ref) <= bound + 2.0 ** -149).all(), (np.abs(got - ref) / bound).max()
    least = 2.0 ** -149 * np.sqrt(ref.size)
    assert np.linalg.norm(got - ref) <= norm * np.linalg.norm(ref) + least, \
        np.linalg.norm(got - ref) / np.linalg.norm(ref)


def check(rng, B, T, H, dk, dv, with_h0, with_reset, decay=None, scale=0.3):
    F = _F()
    q, k, v, h0, reset = inputs(rng, B, T, H, dk, dv, with_h0, with_reset)
    decay = decays(H) if decay is None else decay
    args = [up(t) for t in (q, k, v, decay, h0)] + [up(reset, np.uint32)]
    o, last = F.linear_attention(*args, scale=scale)
    ro, rlast = retention.linear_attention(q, k, v, decay, h0, reset, scale)
    top = [largest(t, H) for t in (q, k, v)]
    th0 = None if h0 is None else np.abs(h0).max() * np.ones(h0.shape)
    mo, mlast = retention.linear_attention(*top, decay, th0, reset, scale)
    c = room(decay, T, dk)
    close(o.numpy(), ro, c * mo)
    close(last.numpy(), rlast, c * mlast)

    do = rng.standard_normal((B, T, H * dv)).astype(np.float32)
    dlast = rng.standard_normal((B, H, dk, dv)).astype(np.float32) if with_h0 else None
    grads = F.linear_attention_backward(up(do), *args, up(dlast), scale=scale)
    refs = retention.linear_attention_backward(do, q, k, v, decay, h0, reset, dlast, scale)
    tlast = None if dlast is None else np.abs(dlast).max() * np.ones(dlast.shape)
    tops = retention.linear_attention_backward(largest(do, H), *top, decay, th0, reset, tlast, scale)
    for got, ref, size in zip(grads[:3], refs, tops):
        close(got.numpy(), ref, room(decay, T, max(dk, dv)) * size)
    if h0 is None:
        assert grads[3] is None
    else:
        close(grads[3].numpy(), refs[3], room(decay, T, dk) * tops[3])


SHAPES = [
    # B, T, H, dk, dv
    (1, 1, 1, 1, 1), (2, 1, 3, 5, 2), (1, 2, 2, 32, 32), (3, 7, 2, 33, 31), (2, 63, 2, 64, 64),
    (2, 64, 1, 64, 32), (1, 65, 4, 32, 64), (2, 127, 2, 40, 72), (1, 128, 3, 64, 64),
    (2, 129, 1, 128, 64), (1, 200, 2, 64, 128), (1, 300, 5, 16, 24), (2, 257, 2, 100, 36),
    (1, 150, 1, 256, 33), (1, 140, 1, 31, 256), (4, 500, 2, 32, 32), (1, 3000, 1, 64, 64),
    (1, 5000, 2, 32, 32), (9, 320, 8, 64, 64), (2, 77, 3, 130, 130),
]


@pytest.mark.parametrize("B,T,H,dk,dv", SHAPES)
@pytest.mark.parametrize("h0,reset", [(False, False), (True, True)])
def test_forward_and_backward(B, T, H, dk, dv, h0, reset, rng):
    check(rng, B, T, H, dk, dv, h0, reset)


@pytest.mark.parametrize("B,T,H,dk,dv", [(24, 130, 16, 64, 64), (8, 200, 16, 64, 64),
                                         (24, 70, 16, 63, 62), (10, 90, 32, 64, 40)])
def test_more_rows_than_fit_at_a_time(B, T, H, dk, dv, rng):
    """Hundreds of sequences and heads: three blocks on an SM, with the operands in place
    (forward from 300 rows on, backward, whose passes run side by side, from 100)."""
    check(rng, B, T, H, dk, dv, True, True)


def test_non_finite_values_among_many_rows(rng):
    F = _F()
    B, T, H, d = 24, 150, 16, 64
    q, k, v, h0, reset = inputs(rng, B, T, H, d, d, True, True)

    def run(k):
        o, last = F.linear_attention(up(q), up(k), up(v), up(decays(H)), up(h0), up(reset, np.uint32))
        return o.numpy().reshape(B, T, H, d), last.numpy()

    good, good_last = run(k)
    bad = k.copy()
    bad[7, 80, 3 * d + 5] = np.nan                  # head 3
    got, last = run(bad)
    hit = ~np.isfinite(got)
    behind = np.flatnonzero(reset[7, 81:])
    end = 81 + behind[0] if behind.size else T
    want = np.zeros_like(hit)
    want[7, 80:end, 3] = True
    assert np.array_equal(hit, want)
    others = np.ones((B, H), bool)
    others[7, 3] = False
    assert np.array_equal(got.transpose(0, 2, 1, 3)[others], good.transpose(0, 2, 1, 3)[others])
    assert np.array_equal(last[others], good_last[others])


def test_operands_and_states_past_32_bits(rng):
    """Sequences more than 2^31 numbers apart in one buffer, and states of more than 2^31
    numbers; rows behind the last sequence stay as they were."""
    import wxx_b200 as wxx

    F = _F()
    T, H, d = 70, 2, 32
    far = wxx.Tensor._empty([2, 1 << 21, 1100])             # 18 GB, only a corner is used
    corner = far.narrow(1, 0, T).narrow(2, 8, 3 * H * d)
    x = rng.standard_normal((2, T, 3 * H * d)).astype(np.float32)
    F.assign(corner, up(x))
    q, k, v = (corner.narrow(2, i * H * d, H * d) for i in range(3))
    assert q.stride[0] > 2 ** 31
    n = [np.ascontiguousarray(x[:, :, i * H * d:(i + 1) * H * d]) for i in range(3)]
    for a, b in zip(F.linear_attention(q, k, v, up(decays(H))),
                    F.linear_attention(*(up(t) for t in n), up(decays(H)))):
        assert np.array_equal(a.numpy(), b.numpy())
    f = F.rotary_frequencies(d)
    assert np.array_equal(F.rotary(q, H, f).numpy(), F.rotary(up(n[0]), H, f).numpy())
    del far, corner, q, k, v
    B, d = 33000, 256
    state = wxx.Tensor((B + 1, 1, d, d), value=0.25)
    qkv = rng.standard_normal((3, B, d)).astype(np.float32)
    o = F.linear_attention_step(*(up(t) for t in qkv), up(np.float32([-0.5])), state.narrow(0, 0, B))
    for b in (0, B - 1):
        ref = np.float64(np.exp(np.float64(-0.5))) * 0.25 + np.outer(qkv[1, b], qkv[2, b].astype(np.float64))
        got = state.narrow(0, b, 1).numpy().reshape(d, d)
        assert np.abs(got - ref).max() < 4 * U * np.abs(ref).max()
        out = qkv[0, b] @ ref
        assert np.abs(o.narrow(0, b, 1).numpy() - out).max() < (4 + d) * U * (
            np.abs(qkv[0, b]) @ np.abs(ref)).max()
    assert (state.narrow(0, B, 1).numpy() == 0.25).all()


@pytest.mark.parametrize("value", [0.0, -1e-6, -0.7, -20.0, -200.0, -np.inf])
def test_extreme_decays(value, rng):
    """No decay, almost none, and decays that forget everything: at 0 the state is a plain
    sum, at -inf every position sees itself alone."""
    check(rng, 2, 150, 2, 32, 32, True, False, np.full(2, value, np.float32))


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 32), (40, 72), (5, 3)])
def test_strided_operands(dk, dv, rng):
    """Column slices of one projection, at even and odd offsets, and a transposed batch."""
    F = _F()
    B, T, H = 3, 100, 2
    width = H * (2 * dk + dv)
    wide = rng.standard_normal((B, T, width + 8)).astype(np.float32)
    t, decay = up(wide), up(decays(H))
    for at in (0, 1, 4):
        cols = [slice(at, at + H * dk), slice(at + H * dk, at + 2 * H * dk),
                slice(at + 2 * H * dk, at + width)]
        a = F.linear_attention(*(t[..., c] for c in cols), decay)
        b = F.linear_attention(*(up(wide[..., c]) for c in cols), decay)
        # a path without the copy engine may be taken: the same to a rounding
        for x, y in zip(a, b):
            x, y = x.numpy(), y.numpy()
            assert np.abs(x - y).max() <= 2.0 ** -20 * np.abs(y).max()
    turned = t.permute(1, 0, 2)
    a = F.linear_attention(*(turned[..., c] for c in cols), decay)[0].numpy()
    b = F.linear_attention(*(up(wide.transpose(1, 0, 2)[..., c]) for c in cols), decay)[0].numpy()
    assert np.abs(a - b).max() <= 2.0 ** -20 * np.abs(b).max()


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 32), (12, 20)])
def test_calls_that_carry_the_state_on(dk, dv, rng):
    """A sequence in pieces, then token by token, against the whole."""
    F = _F()
    B, T, H = 2, 400, 3
    q, k, v, h0, _ = inputs(rng, B, T, H, dk, dv, True, False)
    decay = decays(H)
    ro, rlast = retention.linear_attention(q, k, v, decay, h0)
    size = np.abs(ro).max()
    state, at = up(h0), 0
    for n in (1, 63, 130, 200):
        part = [up(t[:, at:at + n]) for t in (q, k, v)]
        o, state = F.linear_attention(*part, up(decay), state)
        assert np.abs(o.numpy() - ro[:, at:at + n]).max() < 2e-6 * size
        at += n
    for t in range(at, T):
        o = F.linear_attention_step(*(up(a[:, t]) for a in (q, k, v)), up(decay), state)
        assert np.abs(o.numpy() - ro[:, t]).max() < 2e-6 * size
    assert np.abs(state.numpy() - rlast).max() < 2e-6 * np.abs(rlast).max()


@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (32, 16, 64, 64), (3, 5, 40, 72), (2, 2, 7, 33),
                                       (1, 3, 256, 256), (70, 2, 32, 32), (2, 1, 100, 130)])
def test_step(B, H, dk, dv, rng):
    """A position: a product, a sum and a product with q over dk channels.  (4 + dk) u of the
    terms' sizes."""
    F = _F()
    wide = rng.standard_normal((B, H * (2 * dk + dv) + 5)).astype(np.float32)
    state = rng.standard_normal((B, H, dk, dv)).astype(np.float32)
    t, s, decay = up(wide), up(state), decays(H)
    a, b, c = H * dk, 2 * H * dk, H * (2 * dk + dv)
    o = F.linear_attention_step(t[:, :a], t[:, a:b], t[:, b:c], up(decay), s, scale=0.5)
    args = [wide[:, None, :a], wide[:, None, a:b], wide[:, None, b:c]]
    ro, rlast = retention.linear_attention(*args, decay, state, None, 0.5)
    mo, mlast = retention.linear_attention(*map(np.abs, args), decay, np.abs(state), None, 0.5)
    assert (np.abs(o.numpy() - ro[:, 0]) <= (4 + dk) * U * mo[:, 0]).all()
    assert (np.abs(s.numpy() - rlast) <= 4 * U * mlast).all()


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 32), (24, 10), (128, 64)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_non_finite_values_stay_where_the_formula_has_them(dk, dv, bad, rng):
    """A NaN or an infinity reaches its own and later positions of its document and head, no
    earlier one, no other document, head or row; in v only its own column."""
    F = _F()
    B, T, H = 2, 300, 2
    q, k, v, h0, _ = inputs(rng, B, T, H, dk, dv, True, False)
    decay = decays(H)
    reset = np.zeros((B, T), np.uint32)
    reset[:, 200] = 1
    where = 100

    def run(q, k, v):
        o, last = F.linear_attention(up(q), up(k), up(v), up(decay), up(h0), up(reset, np.uint32))
        return o.numpy().reshape(B, T, H, dv), last.numpy()

    good, good_last = run(q, k, v)
    for name in ("q", "k", "v"):
        a = {"q": q.copy(), "k": k.copy(), "v": v.copy()}
        a[name][0, where, 3] = bad               # head 0, channel 3
        got, last = run(**a)
        with np.errstate(invalid="ignore"):
            ref = retention.linear_attention(a["q"], a["k"], a["v"], decay, h0, reset)[0]
        ref = ref.reshape(B, T, H, dv)
        hit = ~np.isfinite(got)
        assert np.array_equal(hit, ~np.isfinite(ref))
        # the other row and head to the bit; the document behind shares a chunk with the bad
        # one, which may be added in another order: each within its room of the exact state,
        # (3 * 2^-22 + (64 + 8 sqrt(1024)) u) of its terms, below 2e-6 of the largest state
        assert np.array_equal(last[1], good_last[1]) and np.array_equal(last[0, 1], good_last[0, 1])
        assert np.abs(last - good_last).max() < 2e-6 * np.abs(good_last).max()
        size = np.abs(good).max()
        assert np.abs(np.where(hit, 0, got) - np.where(hit, 0, good)).max() < 2e-6 * size
        if name == "q":
            assert hit.sum() == dv


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 32), (9, 17)])
def test_a_state_that_is_not_finite(dk, dv, rng):
    """h0 with a NaN in one entry: only outputs of its column until the next document."""
    F = _F()
    B, T, H = 1, 200, 2
    q, k, v, h0, _ = inputs(rng, B, T, H, dk, dv, True, False)
    reset = np.zeros((B, T), np.uint32)
    reset[0, 130] = 1
    h0[0, 1, 2, 4 % dv] = np.nan
    o, last = F.linear_attention(up(q), up(k), up(v), up(decays(H)), up(h0), up(reset, np.uint32))
    hit = np.isnan(o.numpy().reshape(B, T, H, dv))
    want = np.zeros_like(hit)
    want[0, :130, 1, 4 % dv] = True
    assert np.array_equal(hit, want)
    assert np.isfinite(last.numpy()).all()


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 32)])
def test_sizes_far_apart(dk, dv, rng):
    """Rows from 1e-18 to 1e18: every output is as good as its own terms allow."""
    F = _F()
    B, T, H = 1, 200, 2
    q, k, v, h0, _ = inputs(rng, B, T, H, dk, dv, True, False)
    for t in (q, k, v):
        t *= (10.0 ** rng.uniform(-12, 12, (B, T, 1))).astype(np.float32)
    decay = decays(H)
    o, last = F.linear_attention(up(q), up(k), up(v), up(decay), up(h0))
    ro, rlast = retention.linear_attention(q, k, v, decay, h0)
    top = [largest(t, H) for t in (q, k, v)]
    mo, mlast = retention.linear_attention(*top, decay, np.abs(h0).max() * np.ones(h0.shape))
    c = room(decay, T, dk)
    close(o.numpy(), ro, c * mo)
    close(last.numpy(), rlast, c * mlast)


def test_gradient_against_differences(rng):
    """The kernels' own forward, differenced; it is linear in each operand."""
    F = _F()
    B, T, H, dk, dv = 1, 5, 2, 3, 2
    q, k, v, h0, _ = inputs(rng, B, T, H, dk, dv, True, False)
    do = rng.standard_normal((B, T, H * dv)).astype(np.float32)
    dlast = rng.standard_normal((B, H, dk, dv)).astype(np.float32)
    decay = up(decays(H, 1, 2))
    given = {"q": q, "k": k, "v": v, "h0": h0}

    def value(**a):
        o, last = F.linear_attention(up(a["q"]), up(a["k"]), up(a["v"]), decay, up(a["h0"]), scale=0.7)
        return ((o.numpy().astype(np.float64) * do).sum()
                + (last.numpy().astype(np.float64) * dlast).sum())

    grads = F.linear_attention_backward(up(do), up(q), up(k), up(v), decay, up(h0), None, up(dlast),
                                        scale=0.7)
    for name, got in zip(("q", "k", "v", "h0"), grads):
        got, ref = got.numpy(), np.zeros(given[name].shape)
        for i in np.ndindex(ref.shape):
            a, b = given[name].copy(), given[name].copy()
            a[i] += 1
            b[i] -= 1
            ref[i] = (value(**{**given, name: a}) - value(**{**given, name: b})) / 2
        assert np.abs(got - ref).max() < 1e-4 * max(1, np.abs(ref).max())


def test_empty_sizes(rng):
    F = _F()
    decay = up(decays(2))
    z = lambda *s: up(np.zeros(s, np.float32))  # noqa: E731
    h0 = rng.standard_normal((3, 2, 4, 6)).astype(np.float32)
    o, last = F.linear_attention(z(3, 0, 8), z(3, 0, 8), z(3, 0, 12), decay, up(h0))
    assert o.shape == [3, 0, 12] and np.array_equal(last.numpy(), h0)
    o, last = F.linear_attention(z(3, 0, 8), z(3, 0, 8), z(3, 0, 12), decay)
    assert not last.numpy().any()
    grads = F.linear_attention_backward(z(3, 0, 12), z(3, 0, 8), z(3, 0, 8), z(3, 0, 12), decay,
                                        up(h0), None, up(h0))
    assert np.array_equal(grads[3].numpy(), h0)
    o, last = F.linear_attention(z(0, 5, 8), z(0, 5, 8), z(0, 5, 12), decay)
    assert o.shape == [0, 5, 12] and last.shape == [0, 2, 4, 6]
    assert not F.linear_attention(z(1, 5, 0), z(1, 5, 0), z(1, 5, 12), decay)[0].numpy().any()
    assert F.linear_attention_step(z(0, 8), z(0, 8), z(0, 12), decay, z(0, 2, 4, 6)).shape == [0, 12]


def test_captured_graphs_beside_each_other(rng):
    """Two recorded calls and a direct one, replayed in turns on other inputs."""
    import wxx_b200 as wxx

    F = _F()
    B, T, H, d = 2, 700, 2, 64
    decay = up(decays(H))
    sets = [inputs(rng, B, T, H, d, d, False, False)[:3] for _ in range(3)]
    bufs = [[up(t) for t in sets[0]] for _ in range(2)]
    graphs = [wxx.graph.capture(lambda b=b: F.linear_attention(*b, decay)) for b in bufs]
    want = [F.linear_attention(*(up(t) for t in s), decay)[0].numpy() for s in sets]
    for i, j in ((1, 2), (2, 0), (0, 1)):
        for b, s in zip(bufs, (i, j)):
            for x, y in zip(b, sets[s]):
                F.assign(x, up(y))
        a = graphs[0].replay()[0]
        c = F.linear_attention(*bufs[1], decay)[0]
        e = graphs[1].replay()[0]
        assert np.array_equal(a.numpy(), want[i])
        assert np.array_equal(c.numpy(), want[j]) and np.array_equal(e.numpy(), want[j])
    for g in graphs:
        g.close()


def test_refusals():
    F = _F()
    z = lambda *s: up(np.zeros(s, np.float32))  # noqa: E731
    q, v, d = z(2, 3, 8), z(2, 3, 12), z(2)
    with pytest.raises(ValueError):
        F.linear_attention(q, z(2, 4, 8), v, d)
    with pytest.raises(ValueError):
        F.linear_attention(q, z(2, 3, 6), v, d)
    with pytest.raises(ValueError):
        F.linear_attention(q, q, z(2, 3, 13), d)
    with pytest.raises(ValueError):
        F.linear_attention(z(2, 8), z(2, 8), z(2, 12), d)
    with pytest.raises(ValueError):
        F.linear_attention(q, q, v, d, z(2, 2, 4, 5))
    with pytest.raises(ValueError):
        F.linear_attention(q, q, v, d, None, up(np.zeros((3, 2)), np.uint32))
    with pytest.raises(ValueError):
        F.linear_attention(z(1, 1, 514), z(1, 1, 514), z(1, 1, 2), d)        # heads of 257
    with pytest.raises(ValueError):
        F.linear_attention(q, q, v, d, scale=float("nan"))
    with pytest.raises(TypeError):
        F.linear_attention(q, q, v, d, None, z(2, 3))
    with pytest.raises(TypeError):
        F.linear_attention(up(np.zeros((2, 3, 8)), np.uint32), q, v, d)
    with pytest.raises(ValueError):
        F.linear_attention_backward(z(2, 3, 8), q, q, v, d)
    with pytest.raises(ValueError):
        F.linear_attention_step(z(2, 8), z(2, 8), z(2, 12), d, z(2, 2, 6, 4))
    with pytest.raises(ValueError):
        F.linear_attention_step(z(2, 8), z(2, 8), z(2, 12), d, z(2, 2, 6, 4).transpose(2, 3))
