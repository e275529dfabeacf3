"""The gated linear recurrence on the GPU against its 64-bit restatement.

Tolerances.  With u = 2^-24 a step h + z (x - h) rounds x - h, the gate's z
(a few u of itself; 32 u allows for a short exponential) and the result, so it
adds at most u (64 z + 4) M with M the largest |x| or |h0|; an error decays by
a = 1 - z a step, so it is multiplied by at most L = min(T, 1 / smallest z).
That gives u M (64 + 8 L), the 8 also covering the products of a that join
pieces of a row.  The gradients obey the same recursion with the largest total
gradient G in the place of M.  In the 2-norm independent roundings grow with
the root of L: 4 sqrt(L) u < 1e-5 for every L here.
"""

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


def close(got, ref, bound):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape
    if ref.size == 0:
        return
    assert np.isfinite(got).all()
    assert np.abs(got - ref).max() <= bound, (np.abs(got - ref).max(), bound)
    norm = np.linalg.norm(ref)
    assert np.linalg.norm(got - ref) <= 1e-5 * norm or norm < bound


def inputs(rng, B, T, D, H, with_h0, with_reset):
    x = rng.standard_normal((B, T, D)).astype(np.float32)
    gate = np.clip(rng.standard_normal((B, T, H)) * 1.5 + 2, -6, 6).astype(np.float32)
    h0 = rng.standard_normal((B, D)).astype(np.float32) if with_h0 else None
    reset = None
    if with_reset:
        reset = (rng.random((B, T)) < 0.02).astype(np.uint32) * 7     # any non-zero value
        if T:
            reset[0, 0] = 1
    return x, gate, h0, reset


def reach(gate, T):
    z = 1 / (1 + np.exp(np.asarray(gate, np.float64)))
    return min(max(T, 1), 1 / z.min()) if z.size else 1.0, z


SHAPES = [
    # B, T, D, H
    (1, 1, 1, 1), (2, 1, 5, 5), (1, 2, 3, 1), (3, 7, 33, 33), (2, 16, 32, 32), (2, 17, 64, 2),
    (1, 127, 40, 8), (2, 128, 31, 31), (1, 129, 96, 3), (4, 255, 30, 6), (1, 1000, 250, 250),
    (2, 300, 70, 7), (1, 513, 256, 4), (1, 200, 192, 1), (3, 4097, 34, 17), (1, 20000, 32, 32),
    (5, 640, 128, 128), (1, 9000, 65, 13), (2, 2048, 160, 5), (16, 130, 4, 4),
    (2, 150, 300, 1), (1, 140, 514, 2), (1, 33, 8192, 1),
]


@pytest.mark.parametrize("B,T,D,H", SHAPES)
@pytest.mark.parametrize("h0,reset", [(False, False), (True, True)])
def test_forward_and_backward(B, T, D, H, h0, reset, rng):
    F = _F()
    x, gate, h0, reset = inputs(rng, B, T, D, H, h0, reset)
    L, z = reach(gate, T)
    M = max(np.abs(x).max(), 0 if h0 is None else np.abs(h0).max())
    tx, tg, th0, tr = up(x), up(gate), up(h0), up(reset, np.uint32)
    h, last = F.gated_recurrence(tx, tg, th0, tr)
    rh, rlast = recurrent.recurrence(x, gate, h0, reset)
    bound = U * M * (64 + 8 * L)
    close(h.numpy(), rh, bound)
    assert np.array_equal(last.numpy(), h.numpy()[:, -1])

    dh = rng.standard_normal((B, T, D)).astype(np.float32)
    dlast = rng.standard_normal((B, D)).astype(np.float32) if h0 is not None else None
    dx, dg, dh0 = F.gated_recurrence_backward(up(dh), tx, tg, h, th0, tr, up(dlast))
    rdx, rdg, rdh0 = recurrent.recurrence_backward(dh, x, gate, h0, reset, dlast)
    G = np.abs(rdx / np.repeat(z, D // H, -1)).max()
    bound = U * G * (64 + 8 * L)
    close(dx.numpy(), rdx, bound)
    close(dg.numpy(), rdg, bound * 2 * max(M, 1) * (D // H))
    if h0 is None:
        assert dh0 is None
    else:
        close(dh0.numpy(), rdh0, bound)


# enough tiles for two channels a lane: even and odd widths, gates of 1, 2, 3, 25 and 64
# channels, rows of more than 128 tiles, a last block with one channel or none whole
MANY = [(8, 2100, 190, 190), (4, 4097, 131, 131), (7, 3001, 128, 64), (3, 17000, 66, 22),
        (17, 1025, 100, 4), (6, 3100, 192, 3), (40, 900, 65, 65), (38, 129, 256, 256)]


@pytest.mark.parametrize("B,T,D,H", MANY)
@pytest.mark.parametrize("h0,reset", [(False, False), (True, True)])
def test_many_tiles(B, T, D, H, h0, reset, rng):
    test_forward_and_backward(B, T, D, H, h0, reset, rng)


def test_many_tiles_strided(rng):
    """Column slices at odd and even offsets, and an odd number of channels."""
    F = _F()
    B, T, D = 9, 1500, 102
    both = rng.standard_normal((B, T, 3 * D)).astype(np.float32)
    t = up(both)
    for a, b, n in ((0, 2 * D, D), (1, 2 * D, D), (2, D + 1, D - 1), (4, 2 * D, D - 2)):
        x, gate = t[..., a:a + n], t[..., b:b + n]
        h, last = F.gated_recurrence(x, gate)
        same, same_last = F.gated_recurrence(up(both[..., a:a + n]), up(both[..., b:b + n]))
        assert np.array_equal(h.numpy(), same.numpy())
        assert np.array_equal(last.numpy(), same_last.numpy())
        assert np.array_equal(last.numpy(), h.numpy()[:, -1])


def test_gradient_against_differences(rng):
    """The kernels' own forward, differenced: the loss is linear in x and h0, so a
    wide step loses nothing there; in the gate the truncation is step^2 / 6 of the
    third derivative (below 1/2 a step)."""
    F = _F()
    B, T, D, H = 1, 6, 4, 2
    x, gate, h0, _ = inputs(rng, B, T, D, H, True, False)
    dh = rng.standard_normal((B, T, D)).astype(np.float32)

    def value(x, gate, h0):
        h = F.gated_recurrence(up(x), up(gate), up(h0))[0].numpy()
        return (h.astype(np.float64) * dh).sum()

    h, _ = F.gated_recurrence(up(x), up(gate), up(h0))
    got = F.gated_recurrence_backward(up(dh), up(x), up(gate), h, up(h0))
    step = 2.0 ** -4
    M, W = max(np.abs(x).max(), np.abs(h0).max()) + step, np.abs(dh).sum()
    for k, v in enumerate((x, gate, h0)):
        ref = np.zeros(v.shape)
        for i in np.ndindex(v.shape):
            at = [x.copy(), gate.copy(), h0.copy()]
            at[k][i] += step
            hi = value(*at)
            at[k][i] -= 2 * step
            ref[i] = (hi - value(*at)) / (2 * step)
        rounding = U * M * W * (64 + 8 * T) / step
        truncation = step ** 2 / 6 * 0.5 * M * W if k == 1 else 0.0
        assert np.abs(got[k].numpy() - ref).max() <= rounding + truncation


def test_step_continues_the_scan(rng):
    F = _F()
    B, T, D, H = 3, 70, 48, 6
    x, gate, h0, _ = inputs(rng, B, T, D, H, True, False)
    L, _ = reach(gate, T)
    bound = U * max(np.abs(x).max(), np.abs(h0).max()) * (64 + 8 * L)
    ref, _ = recurrent.recurrence(x, gate, h0)
    _, state = F.gated_recurrence(up(x[:, :50]), up(gate[:, :50]), up(h0))
    version = state.buffer.version
    for t in range(50, T):
        out = F.gated_recurrence_step(up(x[:, t]), up(gate[:, t]), state)
        assert out is state
        close(state.numpy(), ref[:, t], bound)
    assert state.buffer.version > version


@pytest.mark.parametrize("B,D,H", [(1, 1, 1), (3, 5, 5), (2, 1024, 16), (257, 36, 12), (64, 4096, 4096)])
def test_step_sizes(B, D, H, rng):
    F = _F()
    x, gate, h0, _ = inputs(rng, B, 1, D, H, True, False)
    state = up(h0)
    F.gated_recurrence_step(up(x[:, 0]), up(gate[:, 0]), state)
    ref, _ = recurrent.recurrence(x, gate, h0)
    close(state.numpy(), ref[:, 0], U * max(np.abs(x).max(), np.abs(h0).max()) * 72)


def test_strided_operands(rng):
    """x and the gate as column slices of one projection, time-major storage,
    a broadcast gate (time stride 0) and an offset base."""
    F = _F()
    B, T, D = 2, 150, 24
    both = rng.standard_normal((B, T, 3 * D)).astype(np.float32)
    t = up(both)
    x, gate = t[..., 1:1 + D], t[..., 2 * D:]
    h, last = F.gated_recurrence(x, gate)
    same, same_last = F.gated_recurrence(up(both[..., 1:1 + D]), up(both[..., 2 * D:]))
    assert np.array_equal(h.numpy(), same.numpy())
    assert np.array_equal(last.numpy(), same_last.numpy())
    dh = up(rng.standard_normal((B, T, D)))
    got = F.gated_recurrence_backward(dh, x, gate, h)
    ref = F.gated_recurrence_backward(dh, up(both[..., 1:1 + D]), up(both[..., 2 * D:]), same)
    for a, b in zip(got[:2], ref[:2]):
        assert np.array_equal(a.numpy(), b.numpy())
    # (T, B, D) storage read as (B, T, D), and x with a strided last axis (copied)
    tm = up(np.ascontiguousarray(both[..., :D].transpose(1, 0, 2)))
    a = F.gated_recurrence(tm.permute(1, 0, 2), gate)[0].numpy()
    assert np.array_equal(a, F.gated_recurrence(up(both[..., :D]), gate)[0].numpy())
    a = F.gated_recurrence(t[..., 0:2 * D:2], gate)[0].numpy()
    assert np.array_equal(a, F.gated_recurrence(up(both[..., 0:2 * D:2]), gate)[0].numpy())


def test_saturated_gates_and_foreign_values(rng):
    """Gates of +-inf keep or replace the state exactly; NaN and infinities of one
    document or channel do not reach another."""
    F = _F()
    B, T, D = 1, 400, 37
    x, gate, h0, _ = inputs(rng, B, T, D, D, True, False)
    gate[0, :, 0], gate[0, :, 1] = np.inf, -np.inf
    gate[0, :, 2], gate[0, :, 3] = 200.0, -200.0
    h = F.gated_recurrence(up(x), up(gate), up(h0))[0].numpy()
    assert (h[0, :, 0] == h0[0, 0]).all() and np.array_equal(h[0, :, 1], x[0, :, 1])
    assert (h[0, :, 2] == h0[0, 2]).all() and np.array_equal(h[0, :, 3], x[0, :, 3])

    x, gate, h0, _ = inputs(rng, B, T, D, D, True, False)
    clean = x.copy()
    reset = np.zeros((B, T), np.uint32)
    reset[0, [150, 320]] = 1
    x[0, 100, 5] = np.nan
    x[0, 200, 6] = np.inf
    h, last = F.gated_recurrence(up(x), up(gate), up(h0), up(reset, np.uint32))
    ref, _ = F.gated_recurrence(up(clean), up(gate), up(h0), up(reset, np.uint32))
    h, ref = h.numpy(), ref.numpy()
    assert np.isnan(h[0, 100:150, 5]).all() and not np.isfinite(h[0, 200:320, 6]).any()
    h[0, 100:150, 5], h[0, 200:320, 6] = ref[0, 100:150, 5], ref[0, 200:320, 6]
    assert np.array_equal(h, ref)
    assert np.isfinite(last.numpy()).all()
    # backwards: a NaN gradient stays within its document and channel
    dh = rng.standard_normal((B, T, D)).astype(np.float32)
    th = F.gated_recurrence(up(clean), up(gate), up(h0), up(reset, np.uint32))[0]
    ref = [v.numpy() for v in F.gated_recurrence_backward(up(dh), up(clean), up(gate), th, up(h0),
                                                          up(reset, np.uint32))]
    dh[0, 200, 9] = np.nan
    got = [v.numpy() for v in F.gated_recurrence_backward(up(dh), up(clean), up(gate), th, up(h0),
                                                          up(reset, np.uint32))]
    for a, b in zip(got[:2], ref[:2]):
        assert np.isnan(a[0, 150:201, 9]).all()
        a[0, 150:201, 9] = b[0, 150:201, 9]
        assert np.array_equal(a, b)
    assert np.array_equal(got[2], ref[2])


def test_infinities_and_the_largest_numbers(rng):
    """An infinite x makes the states infinite from its position on, as the formula
    has it (gates of 0 to 4: no product of 128 weights is zero); opposite infinities
    meet in NaN; opposite numbers near the largest stay finite."""
    F = _F()
    B, T, D = 1, 300, 40
    x = rng.standard_normal((B, T, D)).astype(np.float32)
    gate = (rng.random((B, T, D)) * 4).astype(np.float32)
    gate[0, :, 8:12] *= -1
    for c in range(16):
        x[0, 37 + 16 * c, c] = np.inf if c % 2 else -np.inf
    x[0, 250, 3] = -np.inf
    x[0, :, 16:24] = np.where(rng.random((T, 8)) < 0.5, -3e38, 3e38)
    gate[0, :, 20:24] *= -1
    with np.errstate(invalid="ignore"):
        ref = recurrent.recurrence(x, gate)[0]
    h, last = F.gated_recurrence(up(x), up(gate))
    h, last = h.numpy(), last.numpy()
    far = ~np.isfinite(ref)
    assert far[0, -1, :16].all() and np.isnan(ref[0, -1, 3])
    bound = U * (64 + 8 * reach(gate, T)[0])
    state, steps = up(np.zeros((B, D))), np.empty_like(h)
    for t in range(T):
        steps[:, t] = F.gated_recurrence_step(up(x[:, t]), up(gate[:, t]), state).numpy()
    for got in (h, steps):
        # states 128 positions and more behind an infinity, negative gates: products of
        # their weights may be zero, so infinite or NaN
        near = np.ones(got.shape, bool)
        near[0, :, 8:12] = np.arange(T)[:, None] < 37 + 16 * np.arange(8, 12) + 1
        assert np.array_equal(got[far & near], ref[far & near].astype(np.float32), equal_nan=True)
        assert not np.isfinite(got[far]).any()
        largest = np.broadcast_to(np.where(np.arange(D) // 8 == 2, 3e38, 5.0), got.shape)
        assert (np.abs(got[~far] - ref[~far]) <= bound * largest[~far]).all()
    assert np.array_equal(last, h[:, -1], equal_nan=True)


@pytest.mark.parametrize("B,T,D", [(2, 0, 5), (0, 4, 5), (2, 3, 0)])
def test_empty(B, T, D, rng):
    F = _F()
    H = max(D, 1)
    x, gate = np.zeros((B, T, D), np.float32), np.zeros((B, T, H if D else 0), np.float32)
    h0 = rng.standard_normal((B, D)).astype(np.float32)
    h, last = F.gated_recurrence(up(x), up(gate), up(h0))
    assert h.shape == [B, T, D]
    dx, dg, dh0 = F.gated_recurrence_backward(up(x), up(x), up(gate), h, up(h0), None, up(h0))
    if T == 0:
        assert np.array_equal(last.numpy(), h0) and np.array_equal(dh0.numpy(), h0)
        assert not F.gated_recurrence(up(x), up(gate))[1].numpy().any()


def test_same_bits_every_time(rng):
    """The join of a row's pieces has one order, whatever runs first."""
    F = _F()
    x, gate, h0, reset = inputs(rng, 2, 9000, 96, 3, True, True)
    dh = up(rng.standard_normal(x.shape))
    t = up(x), up(gate), up(h0), up(reset, np.uint32)
    first = None
    for _ in range(5):
        h, last = F.gated_recurrence(*t)
        out = [h, last, *F.gated_recurrence_backward(dh, t[0], t[1], h, t[2], t[3])]
        out = [v.numpy() for v in out]
        if first is None:
            first = out
        for a, b in zip(first, out):
            assert np.array_equal(a, b)


def test_scans_of_all_sizes_one_after_another(rng):
    """What one call leaves in the scan's scratch means nothing to the next, larger or
    smaller, forward or backward, recorded or not."""
    F = _F()
    import wxx_b200 as wxx

    sizes = [(1, 300, 40), (2, 20000, 32), (1, 129, 33), (3, 4100, 70), (1, 300, 40), (6, 2050, 256)]
    t = [tuple(up(v) for v in inputs(rng, B, T, D, D, True, True)[:3]) for B, T, D in sizes]

    def one(k):
        h, last = F.gated_recurrence(*t[k])
        return [h, last, *F.gated_recurrence_backward(t[k][0], t[k][0], t[k][1], h, t[k][2])]

    ref = [[v.numpy() for v in one(k)] for k in range(len(sizes))]
    graphs = [wxx.graph.capture(one, k) for k in (3, 1)]
    for _ in range(3):
        for k in rng.permutation(len(sizes)):
            out = one(int(k))
            graphs[0].replay()
            graphs[1].replay()
            for a, b in zip(out, ref[k]):
                assert np.array_equal(a.numpy(), b)
    for g, k in zip(graphs, (3, 1)):
        for a, b in zip(g.output, ref[k]):
            assert np.array_equal(a.numpy(), b)
        g.close()
    assert wxx.backend.device_status() == 0


def test_scans_of_two_host_threads(rng):
    """Two host threads on the library's stream, each asking for more scratch than the
    other has had so far: neither's is freed under it."""
    import threading

    F = _F()
    sizes = [(1, 300 + 700 * k, 32) for k in range(12)]
    x = rng.standard_normal((1, 9000, 32)).astype(np.float32)
    gate = (rng.standard_normal((1, 9000, 32)) + 2).astype(np.float32)
    want = F.gated_recurrence(up(x), up(gate))[0].numpy()
    wrong = []

    def scans(order):
        try:
            for B, T, D in order:
                h = F.gated_recurrence(up(x[:, :T]), up(gate[:, :T]))[0].numpy()
                if not np.array_equal(h, want[:, :T]):
                    wrong.append(T)
        except Exception as e:              # handed to the test's own thread
            wrong.append(e)

    threads = [threading.Thread(target=scans, args=(o,)) for o in (sizes[::2] * 2, sizes[1::2] * 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_on_another_stream(rng):
    """The library stream changed between calls: each stream has its own scratch."""
    import torch

    F = _F()
    import wxx_b200 as wxx
    from wxx_b200.backend.lib import F as C, check

    x, gate, h0, _ = inputs(rng, 2, 5000, 64, 64, True, False)
    a = up(x), up(gate), up(h0)
    ref = F.gated_recurrence(*a)[0].numpy()
    streams = [torch.cuda.Stream() for _ in range(2)]
    try:
        for k in range(6):
            check(C.wxx_sync())
            check(C.wxx_set_stream(streams[k % 2].cuda_stream))
            h = F.gated_recurrence(*a)[0]
            assert np.array_equal(h.numpy(), ref)
            del h
            check(C.wxx_sync())
    finally:
        check(C.wxx_set_stream(None))
    assert np.array_equal(F.gated_recurrence(*a)[0].numpy(), ref)
    assert wxx.backend.device_status() == 0


def test_offsets_past_32_bits():
    """A sequence batch whose last rows lie past 2^32 bytes and 2^31 elements."""
    F = _F()
    import wxx_b200 as wxx

    B, T, D = 3, 24000, 32768
    x = wxx.Tensor((1, T, D), value=0.5)
    gate = wxx.Tensor((1, T, 1), value=1.0)
    # stride 0 over the batch: only the output is large (9.4 GB)
    xb = wxx.Tensor((B, T, D), buffer=x.buffer, stride=(0, D, 1))
    gb = wxx.Tensor((B, T, 1), buffer=gate.buffer, stride=(0, 1, 1))
    h, last = F.gated_recurrence(xb, gb)
    a = 1 / (1 + np.exp(-1.0))
    tail = h[B - 1, T - 3:].numpy()
    assert np.abs(tail - 0.5).max() < 1e-6 and np.abs(last.numpy() - 0.5).max() < 1e-6
    head = h[B - 1, :3, ::4096].numpy()
    ref = 0.5 * (1 - a ** np.arange(1, 4))[:, None]
    assert np.abs(head - ref).max() < 1e-6


def test_recorded_in_a_graph(rng):
    F = _F()
    import wxx_b200 as wxx

    x, gate, h0, reset = inputs(rng, 2, 1500, 40, 40, True, True)
    t = up(x), up(gate), up(h0), up(reset, np.uint32)
    dh = up(rng.standard_normal(x.shape))

    def step():
        h, last = F.gated_recurrence(*t)
        return (h, last, *F.gated_recurrence_backward(dh, t[0], t[1], h, t[2], t[3]))

    ref = [v.numpy() for v in step()]
    g = wxx.graph.capture(step)
    for _ in range(3):
        out = g.replay()
    for a, b in zip(out, ref):
        assert np.array_equal(a.numpy(), b)
    x2 = rng.standard_normal(x.shape).astype(np.float32)
    F.assign(t[0], up(x2))
    out = [v.numpy() for v in g.replay()]
    for a, b in zip(out, step()):
        assert np.array_equal(a, b.numpy())
    g.close()
    assert wxx.backend.device_status() == 0


def test_autograd(rng):
    import wxx_b200 as wxx
    from wxx_b200 import autograd

    B, T, D, H = 2, 40, 12, 3
    x, gate, h0, _ = inputs(rng, B, T, D, H, True, False)
    w = rng.standard_normal((B, T, D)).astype(np.float32)
    leaves = [wxx.Parameter(up(v)) for v in (x, gate, h0)]
    h = autograd.gated_recurrence(*leaves).forward(*leaves)
    (h * up(w)).sum().backward()
    ref = recurrent.recurrence_backward(w, x, gate, h0)
    L, z = reach(gate, T)
    G = np.abs(ref[0] / np.repeat(z, D // H, -1)).max()
    bound = U * G * (64 + 8 * L)
    for leaf, r, k in zip(leaves, ref, (1, 2 * max(1, np.abs(x).max()) * (D // H), 1)):
        close(leaf.grad.numpy(), r, bound * k)


# gates about the places where exp(-gate), 1 + exp(-gate) and its reciprocal leave
# the normal numbers, and far beyond
FAR = [1, 20, 60, 86, 87.3, 87.4, 87.6, 88, 88.5, 88.7, 88.8, 89, 103, 104, 110, 200, 1e30, 3e38,
       np.inf]


def amplified(a):
    """How many unit errors, one a position, a state holds at most: e = a e + 1."""
    e, out = np.zeros(a[:, 0].shape), np.empty_like(a)
    for t in range(a.shape[1]):
        e = a[:, t] * e + 1
        out[:, t] = e
    return out


def far_gates(rng, T, per, mixed):
    """A head for each of the far gates and its opposite, (mixed) also gates that jump
    between them and moderate ones; a gate serves ``per`` channels."""
    values = np.array(FAR + [-v for v in FAR], np.float32)
    gate = np.broadcast_to(values, (1, T, values.size))
    if mixed:
        gate = np.concatenate([rng.choice(values, gate.shape),
                               rng.uniform(-110, 110, gate.shape).astype(np.float32)], -1)
    x = rng.standard_normal((1, T, gate.shape[-1] * per)).astype(np.float32)
    h0 = rng.standard_normal((1, gate.shape[-1] * per)).astype(np.float32)
    a = recurrent._sigmoid(np.repeat(gate.astype(np.float64), per, -1))
    return x, np.ascontiguousarray(gate), h0, a


@pytest.mark.parametrize("per", [1, 8, 25, 32, 64])
@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("mixed", [False, True])
def test_gates_far_from_zero(T, per, mixed, rng):
    """Forward, one position at a time and backward agree with the 64-bit form for
    every gate.  The bound is that of the tolerances above, entry by entry, with the
    errors' own amplification in the place of L."""
    F = _F()
    x, gate, h0, a = far_gates(rng, T, per, mixed)
    M = max(np.abs(x).max(), np.abs(h0).max())
    ref, _ = recurrent.recurrence(x, gate, h0)
    ahead = amplified(a)
    tx, tg, th0 = up(x), up(gate), up(h0)
    h, last = F.gated_recurrence(tx, tg, th0)
    assert (np.abs(h.numpy() - ref) <= U * M * (64 + 8 * ahead)).all()
    assert np.array_equal(last.numpy(), h.numpy()[:, -1])
    state = up(h0)
    for t in range(min(T, 40)):
        F.gated_recurrence_step(up(x[:, t]), up(gate[:, t]), state)
        assert (np.abs(state.numpy() - ref[:, t]) <= U * M * (64 + 8 * ahead[:, t])).all()

    dh = rng.standard_normal(x.shape).astype(np.float32)
    dlast = rng.standard_normal(h0.shape).astype(np.float32)
    got = [v.numpy() for v in F.gated_recurrence_backward(up(dh), tx, tg, h, th0, None, up(dlast))]
    dx, dg, dh0 = recurrent.recurrence_backward(dh, x, gate, h0, None, dlast)
    # the gradient reaching a position: through the weights behind it
    behind = np.ones_like(a)
    behind[:, :-1] = a[:, 1:]
    back = amplified(behind[:, ::-1])[:, ::-1]
    G = max(np.abs(dh).max(), np.abs(dlast).max()) * back.max((0, 1))
    bound = U * G * (64 + 8 * back)
    assert (np.abs(got[0] - dx) <= bound).all()
    assert (np.abs(got[2] - dh0) <= bound[:, 0]).all()
    over = (bound + U * G * (64 + 8 * ahead)) * 2 * max(M, 1)
    assert (np.abs(got[1] - dg) <= over.reshape(1, T, -1, per).sum(-1)).all()


@pytest.mark.parametrize("per", [8, 25, 32, 64])
def test_foreign_values_of_shared_gates(per, rng):
    """A NaN gate makes its own head's states NaN up to the next document, an infinite x
    its own channel's infinite or NaN; everything else keeps its bits."""
    F = _F()
    B, T, H = 2, 300, 5
    D = per * H
    x, gate, h0, _ = inputs(rng, B, T, D, H, True, False)
    reset = np.zeros((B, T), np.uint32)
    reset[:, 150] = 1
    tr = up(reset, np.uint32)
    ref = F.gated_recurrence(up(x), up(gate), up(h0), tr)[0].numpy()
    gate[0, 100, 1] = np.nan
    x[1, 60, 2 * per] = np.inf
    x[1, 200, 3 * per + 1] = -np.inf
    h, last = F.gated_recurrence(up(x), up(gate), up(h0), tr)
    h = h.numpy()
    assert np.array_equal(last.numpy(), h[:, -1], equal_nan=True)
    assert np.isnan(h[0, 100:150, per:2 * per]).all()
    assert not np.isfinite(h[1, 60:150, 2 * per]).any()
    assert not np.isfinite(h[1, 200:, 3 * per + 1]).any()
    h[0, 100:150, per:2 * per] = ref[0, 100:150, per:2 * per]
    h[1, 60:150, 2 * per] = ref[1, 60:150, 2 * per]
    h[1, 200:, 3 * per + 1] = ref[1, 200:, 3 * per + 1]
    assert np.array_equal(h, ref)


@pytest.mark.parametrize("per", [1, 4, 25, 32, 64])
@pytest.mark.parametrize("T", [1, 16, 40, 300])
def test_gradient_of_the_last_state_alone(T, per, rng):
    """With no other gradient everything is what the weights hand back from the last
    position, so the error is relative, entry by entry: a weight is good to 40 u of
    itself (gates to -30), a product of T of them and the roundings between to u (42 T +
    64).  dgate also takes the forward's error of h.  1e-36: products that have left
    the normal numbers."""
    F = _F()
    gate = np.linspace(-30, 6, 37, dtype=np.float32)
    H = gate.size
    gate = np.ascontiguousarray(np.broadcast_to(gate, (2, T, H)))
    x = rng.standard_normal((2, T, H * per)).astype(np.float32)
    h0 = rng.standard_normal((2, H * per)).astype(np.float32)
    dlast = (rng.uniform(0.5, 2, h0.shape) * rng.choice([-1, 1], h0.shape)).astype(np.float32)
    zero = np.zeros_like(x)
    h, _ = F.gated_recurrence(up(x), up(gate), up(h0))
    got = F.gated_recurrence_backward(up(zero), up(x), up(gate), h, up(h0), None, up(dlast))
    dx, dg, dh0 = recurrent.recurrence_backward(zero, x, gate, h0, None, dlast)
    rel = U * (42 * T + 64)
    assert (np.abs(got[0].numpy() - dx) <= rel * np.abs(dx) + 1e-36).all()
    assert (np.abs(got[2].numpy() - dh0) <= rel * np.abs(dh0) + 1e-36).all()
    wide = np.repeat(gate.astype(np.float64), per, -1)
    a, z = recurrent._sigmoid(wide), recurrent._sigmoid(-wide)
    before = np.concatenate([h0[:, None], recurrent.recurrence(x, gate, h0)[0][:, :-1]], 1)
    M = max(np.abs(x).max(), np.abs(h0).max())
    terms = np.abs(dx) * a * ((rel + 90 * U) * (np.abs(before) + np.abs(x))
                              + U * M * (64 + 8 * np.minimum(T, 1 / z)))
    assert (np.abs(got[1].numpy() - dg) <= terms.reshape(2, T, H, per).sum(-1) + 1e-36).all()


@pytest.mark.parametrize("per", [1, 8, 32])
def test_weights_to_their_last_bits(per, rng):
    """One position from a state of 0 or 1 shows the smaller weight, its gradients both.
    Relative, at every gate: 4 u for the exponential, 2 u for the reciprocal, a rounding
    (u) each for the exponential's correction, its product, 1 + e, e a and the result
    are 11 u; dgate has both weights."""
    F = _F()
    gate = np.linspace(-86, 86, 4001, dtype=np.float32)
    H = gate.size
    g = up(gate.reshape(1, 1, H))
    a, z = recurrent._sigmoid(gate.astype(np.float64)), recurrent._sigmoid(-gate.astype(np.float64))
    one, zero = np.ones((1, 1, H * per)), np.zeros((1, 1, H * per))

    def near(got, ref, units):
        got = got.numpy().astype(np.float64).reshape(H, -1)
        off = np.abs(got / ref[:, None] - 1).max() / U
        assert off <= units, off

    for value, start, weight, use in ((one, zero, z, gate >= 0), (zero, one, a, gate < 0)):
        h, _ = F.gated_recurrence(up(value), g, up(start[:, 0]))
        state = up(start[:, 0])
        F.gated_recurrence_step(up(value[:, 0]), up(gate.reshape(1, H)), state)
        for got in (h, state):
            smaller = np.where(use, weight, 1.0)
            off = np.abs(got.numpy().reshape(H, per) / smaller[:, None] - 1)[use].max() / U
            assert off <= 12, off
    h, _ = F.gated_recurrence(up(zero), g, up(one[:, 0]))
    dx, dg, dh0 = F.gated_recurrence_backward(up(one), up(zero), g, h, up(one[:, 0]))
    near(dx, z, 13)
    near(dh0, a, 13)
    near(dg, a * z * per, 26 + 8)


def test_gates_without_channels():
    """Gates of no channels receive the sum over none: zero, not what the memory held."""
    F = _F()
    for _ in range(4):
        used = up(np.full((2, 3, 5), 7.0))
        del used
        x, gate = up(np.zeros((2, 3, 0))), up(np.zeros((2, 3, 5)))
        h, _ = F.gated_recurrence(x, gate)
        dx, dg, dh0 = F.gated_recurrence_backward(x, x, gate, h)
        assert dx.shape == [2, 3, 0] and dh0 is None
        assert np.array_equal(dg.numpy(), np.zeros((2, 3, 5)))


# both sides of the rules that choose a kernel: 23 and 24 blocks of 32 channels (groups of
# 32 or 8 tiles), 99 partial sums of a gate and 100 and more (a thread or a warp adds them),
# from single channels and from blocks of 32
SIDES = [(1, 700, 736, 736), (1, 700, 737, 737), (1, 1100, 736, 23), (4, 1100, 192, 6),
         (1, 150, 99, 1), (1, 150, 202, 2), (3, 70, 300, 3), (1, 150, 255, 1), (2, 140, 1000, 1),
         (1, 40, 3168, 1), (1, 40, 3200, 1), (1, 40, 8160, 1)]


@pytest.mark.parametrize("B,T,D,H", SIDES)
def test_both_sides_of_the_rules(B, T, D, H, rng):
    test_forward_and_backward(B, T, D, H, True, True, rng)
