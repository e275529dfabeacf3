"""Top-k and beam search's steps on the GPU against their restatements: values,
ids, parents and moved states exactly; summed log-probabilities to
u (16 R + 64) with u = 2^-24 and R the largest magnitude that a score is summed
from (the rounding of the shift, the log of the sum and the two additions)."""

import numpy as np
import pytest

from oracle import recurrent

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _F():
    import wxx_b200 as wxx

    return wxx.functional


def up(a, dtype=np.float32):
    return None if a is None else _F().from_numpy(np.asarray(a), dtype=dtype)


def check_topk(x, k):
    values, ids = _F().topk(up(x), k)
    rv, ri = recurrent.topk(x, k)
    assert ids.type == "u32" and np.array_equal(ids.numpy().astype(np.int64), ri)
    assert np.array_equal(values.numpy(), rv, equal_nan=True)


@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (3, 2, 2), (5, 31, 4), (2, 33, 33), (4, 255, 255),
                                   (4, 256, 256), (3, 1000, 256), (64, 1024, 32), (7, 1021, 17),
                                   (2, 4099, 100), (3, 50304, 64), (2, 50303, 256), (1, 131073, 1),
                                   (150, 5000, 8), (2, 300000, 128), (600, 129, 16)])
def test_topk_random(N, V, K, rng):
    check_topk(rng.standard_normal((N, V)).astype(np.float32), K)


@pytest.mark.parametrize("V,K", [(40, 7), (1024, 64), (9000, 256), (50304, 100)])
def test_topk_ties_and_order(V, K, rng):
    """Few distinct values, one value, sorted rows, and rows whose large values
    sit close together: the lower id wins every tie."""
    rows = [rng.integers(0, 5, V).astype(np.float32), np.full(V, 3.5, np.float32),
            np.arange(V, dtype=np.float32), np.arange(V, dtype=np.float32)[::-1],
            np.full(V, -np.inf, np.float32), np.zeros(V, np.float32),
            np.where(np.arange(V) < V // 3, 10 + rng.random(V), 0).astype(np.float32),
            np.where(np.arange(V) % 7 == 3, 10 + rng.random(V), rng.random(V)).astype(np.float32),
            np.where(np.arange(V) // 64 % 3 == 1, 5.0, 1.0).astype(np.float32)]
    rows[5][1::2] = -0.0                     # equal to 0
    check_topk(np.stack(rows), K)


def test_topk_crowded_lanes(rng):
    """All large values where one thread, warp or stretch of the row finds them."""
    V, K = 50304, 256
    rows = []
    at = np.arange(V)
    for period in (4, 32, 128, 256, 512, 1024, 2048, 4096):
        for width in (1, 4, 32, 128):
            if width < period:
                rows.append(np.where(at % period < width, 100 + rng.random(V), rng.random(V)))
    x = np.stack(rows).astype(np.float32)
    for k in (1, 31, 64, K):
        check_topk(x, k)


@pytest.mark.parametrize("V", [1, 31, 32, 33, 200, 256, 257, 511, 513, 1000, 1024, 1025, 2047, 2048,
                               2049])
def test_topk_short_rows(V, rng):
    """Rows about the lengths where the kernel changes: random, of few values (more
    equal entries than are looked at together), one lane's entries above all others,
    infinities and NaN, falling and rising; every number of rows of a block."""
    at = np.arange(V)
    few = rng.integers(0, 3, V)
    odd = rng.standard_normal(V)
    odd[rng.integers(0, V, 5)] = [np.nan, np.inf, -np.inf, 0.0, -0.0]
    rows = [rng.standard_normal(V), few, np.where(few == 2, rng.random(V) + 2, few),
            np.where(at % 32 == 5, 10 + rng.random(V), rng.random(V)), odd, at, -at, np.zeros(V),
            np.full(V, -np.inf), np.full(V, np.nan), np.where(at < V // 2, -np.inf, odd)]
    x = np.stack(rows).astype(np.float32)
    for k in (1, 7, 31, 32, 33, 63, 65, 128, 129, 160, 256):
        if k <= V:
            check_topk(x, k)
            check_topk(x[:2], k)
    check_topk(rng.standard_normal((601, V)).astype(np.float32), min(V, 40))


def test_topk_foreign_values(rng):
    x = rng.standard_normal((6, 777)).astype(np.float32)
    x[0, [5, 700]] = np.nan
    x[1, [9, 11]] = np.inf
    x[2] = np.nan
    x[3, 3:] = -np.inf
    x[4] = np.finfo(np.float32).min
    x[5, 100] = -np.float32(np.nan)
    for k in (1, 2, 40, 256):
        check_topk(x, k)


def test_topk_shapes(rng):
    F = _F()
    x = rng.standard_normal((2, 3, 90)).astype(np.float32)
    v, i = F.topk(up(x), 5)
    rv, ri = recurrent.topk(x.reshape(6, 90), 5)
    assert v.shape == [2, 3, 5] and np.array_equal(i.numpy().reshape(6, 5), ri)
    v, i = F.topk(up(x[0, 0]), 5)
    assert v.shape == [5] and np.array_equal(v.numpy(), rv[0])
    wide = up(rng.standard_normal((4, 100)))
    v, i = F.topk(wide[:, 3:90], 6)
    rv, ri = recurrent.topk(wide.numpy()[:, 3:90], 6)
    assert np.array_equal(i.numpy(), ri) and np.array_equal(v.numpy(), rv)
    v, i = F.topk(up(x).transpose(1, 2), 2)
    rv, ri = recurrent.topk(x.transpose(0, 2, 1).reshape(-1, 3), 2)
    assert np.array_equal(i.numpy().reshape(-1, 2), ri)
    assert F.topk(up(np.zeros((0, 9))), 3)[0].shape == [0, 3]


def test_topk_offsets_past_32_bits(rng):
    """43000 x 50304 entries (2^31 of them, 8.7 GB): rows of one value, and the last."""
    F = _F()
    import wxx_b200 as wxx

    N, V, n = 43000, 50304, 2
    x = rng.standard_normal((n, V)).astype(np.float32)
    big = wxx.Tensor((N, V), value=-1.5)
    F.assign(big.narrow(0, N - n, n), up(x))
    values, ids = F.topk(big, 3)
    rv, ri = recurrent.topk(x, 3)
    assert np.array_equal(ids.numpy()[N - n:], ri) and np.array_equal(values.numpy()[N - n:], rv)
    assert np.array_equal(ids.numpy()[:N - n], np.tile([0, 1, 2], (N - n, 1)))
    assert wxx.backend.device_status() == 0


def test_reorder_offsets_past_32_bits(rng):
    """States of 3 x 1.5 GB rows: the last words of the last beam."""
    F = _F()
    import wxx_b200 as wxx

    row = 400_000_000
    t = wxx.Tensor((3, row), value=0.0)
    for w in range(3):
        F.assign(t.narrow(0, w, 1), float(w + 1))
        F.assign(t.narrow(0, w, 1).narrow(1, row - 5, 5), float(10 * (w + 1)))
    F.beam_reorder([t], up([[2, 2, 0]], np.uint32))
    for w, p in enumerate((2, 2, 0)):
        assert np.all(t.narrow(0, w, 1).narrow(1, row - 9, 4).numpy() == p + 1)
        assert np.all(t.narrow(0, w, 1).narrow(1, row - 5, 5).numpy() == 10 * (p + 1))
    assert wxx.backend.device_status() == 0


def beams(rng, B, W, V, done):
    z = (rng.standard_normal((B * W, V)) * 3).astype(np.float32)
    s = (-10 - 2 * rng.random((B, W))).astype(np.float32)
    return z, s, ((rng.random((B, W)) < 0.3).astype(np.uint32) * 5 if done else None)


def apart(z, s, f, stop, W, bound):
    """Whether the proposals around the cut are apart by more than rounding."""
    many = recurrent.beam_select(z, s, f, stop)
    wide = np.sort(many[0], -1)
    return (np.diff(wide, axis=-1) > 4 * bound).all()


@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 1, 50), (2, 2, 2), (1, 4, 1024), (3, 5, 77),
                                   (2, 8, 50304), (4, 16, 1000), (1, 16, 50303), (1, 3, 131072),
                                   (40, 4, 33), (2, 12, 9)])
@pytest.mark.parametrize("done", [False, True])
def test_beam_select(B, W, V, done, rng):
    F = _F()
    stop = V - 1 if done else None
    bound = U * (16 * 40 + 64)
    for _ in range(20):
        z, s, f = beams(rng, B, W, V, done)
        if apart(z, s, f, stop, W, bound):
            break
    got = F.beam_select(up(z), up(s), up(f, np.uint32), stop)
    ref = recurrent.beam_select(z, s, f, stop)
    fine = np.isfinite(ref[0])
    assert np.array_equal(np.isfinite(got[0].numpy()), fine)
    assert np.abs(got[0].numpy() - ref[0])[fine].max() <= bound
    assert np.array_equal(got[1].numpy(), ref[1]) and np.array_equal(got[2].numpy(), ref[2])
    if done:
        assert np.array_equal(got[3].numpy(), ref[3])
    else:
        assert got[3] is None


def test_beam_select_ties_and_masks(rng):
    """Equal scores go to the lower beam and the lower token; beams without
    probabilities, the first step's single live beam, fewer tokens than beams."""
    F = _F()
    W, V = 4, 300
    z = np.zeros((5 * W, V), np.float32)
    s = np.full((5, W), -1.0, np.float32)
    z[W] = -np.inf                           # item 1: a beam with nothing allowed,
    z[W + 1, 7] = np.nan                     # one with a NaN,
    z[W + 2, 7] = np.inf                     # one with an infinity
    z[W + 3, 5:] = np.finfo(np.float32).min
    s[2, 1:] = -np.inf                       # item 2: the first step
    s[3] = -np.inf                           # item 3: nothing alive
    s[4, 2] = np.nan                         # item 4: a beam without a score
    got = F.beam_select(up(z), up(s))
    ref = recurrent.beam_select(z, s)
    for a, b in zip(got[1:3], ref[1:3]):
        assert np.array_equal(a.numpy(), b)
    fine = np.isfinite(ref[0])
    assert np.array_equal(np.isfinite(got[0].numpy()), fine)
    assert np.abs(got[0].numpy()[fine] - ref[0][fine]).max() <= U * 300
    assert (got[0].numpy()[~fine] == -np.inf).all()


def test_beam_select_strided_logits_and_empty_batch(rng):
    F = _F()
    z, s, f = beams(rng, 2, 4, 100, True)
    wide = np.full((8, 112), 50.0, np.float32)
    wide[:, 5:105] = z
    a = F.beam_select(up(wide)[:, 5:105], up(s), up(f, np.uint32), 3)
    b = F.beam_select(up(z), up(s), up(f, np.uint32), 3)
    for u, v in zip(a[1:], b[1:]):
        assert np.array_equal(u.numpy(), v.numpy())
    assert F.beam_select(up(z[:0]), up(s[:0]))[0].shape == [0, 4]


@pytest.mark.parametrize("B,W,shape", [(1, 1, (3,)), (2, 4, (256,)), (3, 5, (7,)), (1, 16, (33,)),
                                       (2, 8, (20, 64)), (4, 3, (5, 9)), (1, 2, (1, 1)),
                                       (2, 12, (300, 128)), (2, 7, ())])
def test_beam_reorder(B, W, shape, rng):
    F = _F()
    R = B * W
    states = [rng.standard_normal((R,) + shape).astype(np.float32) for _ in range(3)]
    ids = rng.integers(0, 2 ** 32, (R,) + shape, dtype=np.uint32)
    z = (rng.standard_normal((R,) + shape) + 1j * rng.standard_normal((R,) + shape)).astype(np.complex64)
    for parents in (rng.integers(0, W, (B, W)), np.zeros((B, W)), np.tile(np.arange(W), (B, 1)),
                    np.tile(np.arange(W)[::-1], (B, 1)), np.tile(np.roll(np.arange(W), 1), (B, 1))):
        parents = parents.astype(np.uint32)
        t = [up(v) for v in states] + [up(ids, np.uint32), F.from_numpy_complex(z)]
        out = F.beam_reorder(t, up(parents, np.uint32))
        for a, b in zip(out, states + [ids, z]):
            assert np.array_equal(a.numpy(), recurrent.beam_reorder(b, parents))


@pytest.mark.parametrize("used", [0, 1, 13, 64, 100])
def test_beam_reorder_of_a_cache(used, rng):
    F = _F()
    B, W, P = 2, 4, 64
    parents = rng.integers(0, W, (B, W)).astype(np.uint32)
    caches = [rng.standard_normal((B * W, P, c)).astype(np.float32) for c in (32, 9)]
    caches.append(rng.standard_normal((B * W, P)).astype(np.float32))
    t = [up(c) for c in caches]
    version = t[0].buffer.version
    F.beam_reorder(t, up(parents, np.uint32), up([used], np.uint32))
    for a, b in zip(t, caches):
        assert np.array_equal(a.numpy(), recurrent.beam_reorder(b, parents, used))
    assert t[0].buffer.version > version


def test_beam_reorder_views_and_many_states(rng):
    """States inside one buffer at odd offsets, and more than one launch takes."""
    F = _F()
    B, W = 1, 3
    base = rng.standard_normal(1 + 140 * 3 * 11).astype(np.float32)
    t = up(base)
    parents = np.array([[2, 0, 0]], np.uint32)
    views = [t.narrow(0, 1 + 33 * i, 33).reshape((3, 11)) for i in range(140)]
    F.beam_reorder(views, up(parents, np.uint32))
    ref = base.copy()
    for i in range(140):
        v = ref[1 + 33 * i:34 + 33 * i].reshape(3, 11)
        v[:] = v[[2, 0, 0]]
    assert np.array_equal(t.numpy(), ref)


def test_beam_reorder_bad_parent(rng):
    F = _F()
    import wxx_b200 as wxx

    v = rng.standard_normal((4, 50)).astype(np.float32)
    t = up(v)
    F.beam_reorder([t], up([[1, 7, 0, 3]], np.uint32))
    assert wxx.backend.device_status() == 2
    assert np.array_equal(t.numpy(), v[[1, 1, 0, 3]])


@pytest.mark.parametrize("W", [1, 3, 5, 7, 9, 15])
def test_beam_reorder_parent_just_outside(W, rng):
    """A parent of beams or a little more leaves its row as it was: the next item's
    rows, or what lies behind the last one's, are not read."""
    F = _F()
    import wxx_b200 as wxx

    v = rng.standard_normal((2 * W, 20)).astype(np.float32)
    for bad in (W, 16):
        parents = np.tile(np.arange(W)[::-1], (2, 1)).astype(np.uint32)
        parents[0, 0] = parents[1, W // 2] = bad
        t = up(v)
        F.beam_reorder([t], up(parents, np.uint32))
        assert wxx.backend.device_status() == 2
        kept = np.where(parents < W, parents, np.arange(W, dtype=np.uint32))
        assert np.array_equal(t.numpy(), recurrent.beam_reorder(v, kept))


def test_steps_in_a_graph(rng):
    F = _F()
    import wxx_b200 as wxx

    z, s, f = beams(rng, 2, 4, 500, True)
    state = rng.standard_normal((8, 30)).astype(np.float32)
    tz, ts, tf, st = up(z), up(s), up(f, np.uint32), up(state)

    def step():
        picked = F.beam_select(tz, ts, tf, 3)
        F.beam_reorder([st], picked[1])
        return picked

    g = wxx.graph.capture(step)
    F.assign(st, up(state))
    out = g.replay()
    ref = recurrent.beam_select(z, s, f, 3)
    assert np.array_equal(out[1].numpy(), ref[1]) and np.array_equal(out[2].numpy(), ref[2])
    assert np.array_equal(st.numpy(), recurrent.beam_reorder(state, ref[1]))
    g.close()
    assert wxx.backend.device_status() == 0
