"""Distillation from a teacher's top logits on the GPU against its 64-bit
restatement.

Tolerances.  With u = 2^-24 and R the largest |z - max z| / tau (or |t - max t|
/ tau of a stored logit), an exponential's argument carries u R and the
exponential itself a few u, so p and q are good to u (8 R + 32) of themselves,
sums of V positive terms adding a few u (they are joined in a tree).  The loss
is tau^2 sum p (log p - log q): each log is a difference of numbers up to
R + log V, so it is off by u (8 R + 32 + 2 log V) in all.
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
    return _F().from_numpy(np.asarray(a), dtype=dtype)


def problem(rng, N, V, K, ragged):
    z = (rng.standard_normal((N, V)) * 2.5).astype(np.float32)
    teacher = z + rng.standard_normal((N, V)).astype(np.float32)
    ids = np.argsort(-teacher, -1, kind="stable")[:, :K].astype(np.uint32)
    top = np.take_along_axis(teacher, ids.astype(np.int64), 1)
    if ragged:
        keep = rng.integers(0, K + 1, size=(N, 1))
        keep[0] = 0
        top = np.where(np.arange(K) < keep, top, -np.inf).astype(np.float32)
    return z, top, ids


def bounds(z, top, tau):
    z, t = z.astype(np.float64), top.astype(np.float64)
    R = (z.max(-1) - z.min(-1)).max() / tau
    rows = np.isfinite(t).any(-1)
    if rows.any():
        r = t[rows]
        R = max(R, (r.max(-1) - np.where(np.isfinite(r), r, np.inf).min(-1)).max() / tau)
    one = U * (8 * R + 32 + 2 * np.log(z.shape[1]))
    return one, one


SIZES = [(1, 1, 1), (2, 2, 2), (3, 5, 3), (7, 33, 8), (5, 1021, 17), (33, 1024, 32),
         (4, 4096, 64), (3, 5000, 200), (2, 50304, 64), (9, 50303, 128), (1, 50304, 1024),
         (300, 257, 5), (2, 131072, 100), (1, 200001, 7)]


@pytest.mark.parametrize("N,V,K", SIZES)
@pytest.mark.parametrize("tau,ragged", [(1.0, False), (2.5, True)])
def test_loss_and_gradient(N, V, K, tau, ragged, rng):
    F = _F()
    z, top, ids = problem(rng, N, V, K, ragged)
    loss, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32), tau)
    rloss, rp, rq = recurrent.distill(z, top, ids, tau)
    bl, bg = bounds(z, top, tau)
    assert np.abs(loss.numpy() - rloss).max() <= tau * tau * bl
    grad = rng.standard_normal((N, 1)).astype(np.float32)
    d = F.distill_loss_backward(up(grad), up(z), up(top), up(ids, np.uint32), stats, tau).numpy()
    rd = recurrent.distill_backward(grad, z, top, ids, tau)
    # entry by entry: q and p are good to bg of themselves, before they cancel
    full = rq.copy()
    for n in range(N):
        np.add.at(full[n], ids[n].astype(np.int64), rp[n])
    assert (np.abs(d - rd) <= np.abs(grad) * tau * full * bg + 1e-37).all()


@pytest.mark.parametrize("N,V,K", [(1500, 7, 7), (1030, 31, 20), (1024, 256, 64), (1025, 257, 33),
                                   (1024, 500, 64), (1027, 513, 1), (1100, 1021, 40),
                                   (1024, 1024, 65), (1024, 1025, 64), (6, 2048, 128),
                                   (6, 2049, 128), (5, 2048, 129)])
@pytest.mark.parametrize("ragged", [False, True])
def test_many_short_rows(N, V, K, ragged, rng):
    """Both sides of the lengths, entries and rows where the kernels change, ids
    stored twice among them."""
    tau = 1.5
    F = _F()
    z, top, ids = problem(rng, N, V, K, ragged)
    ids[:, K // 2] = ids[:, 0]
    ids[::3, K - 1] = ids[::3, K // 3]
    loss, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32), tau)
    rloss, rp, rq = recurrent.distill(z, top, ids, tau)
    bl, bg = bounds(z, top, tau)
    assert np.abs(loss.numpy() - rloss).max() <= tau * tau * bl
    grad = rng.standard_normal((N, 1)).astype(np.float32)
    d = F.distill_loss_backward(up(grad), up(z), up(top), up(ids, np.uint32), stats, tau).numpy()
    rd = recurrent.distill_backward(grad, z, top, ids, tau)
    full = rq.copy()
    for n in range(N):
        np.add.at(full[n], ids[n].astype(np.int64), rp[n])
    assert (np.abs(d - rd) <= np.abs(grad) * tau * full * bg + 1e-37).all()


def test_gradient_against_differences(rng):
    """Central differences of the kernel's loss: the third derivative of the
    log-sum is below 1/4, so a step s is off by tau^2 s^2 / 24 / tau^3 and the
    loss's rounding over s."""
    F = _F()
    N, V, K, tau, s = 2, 12, 4, 1.5, 2.0 ** -5
    z, top, ids = problem(rng, N, V, K, False)
    _, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32), tau)
    ones = np.ones((N, 1), np.float32)
    d = F.distill_loss_backward(up(ones), up(z), up(top), up(ids, np.uint32), stats, tau).numpy()
    bl, _ = bounds(z, top, tau)
    for j in range(V):
        at = []
        for sign in (s, -s):
            v = z.copy()
            v[:, j] += sign
            at.append(F.distill_loss(up(v), up(top), up(ids, np.uint32), tau)[0].numpy())
        ref = (at[0].astype(np.float64) - at[1])[:, 0] / (2 * s)
        assert np.abs(d[:, j] - ref).max() <= tau * tau * bl / s + s * s / 24 / tau


def test_teacher_equal_to_student_has_no_loss(rng):
    F = _F()
    z = rng.standard_normal((4, 60)).astype(np.float32)
    ids = np.tile(np.arange(60, dtype=np.uint32), (4, 1))
    loss, stats = F.distill_loss(up(z), up(z + 2), up(ids, np.uint32), 2.0)
    bl, _ = bounds(z, z, 2.0)
    assert np.abs(loss.numpy()).max() <= 4 * bl + 4 * U * 16     # z + 2 rounds
    d = F.distill_loss_backward(up(np.ones((4, 1))), up(z), up(z + 2), up(ids, np.uint32), stats,
                                2.0).numpy()
    assert np.abs(d).max() <= 2 * 0.5 * (2 * bl + 16 * U)


def test_masks_and_extremes(rng):
    F = _F()
    z = (rng.standard_normal((6, 40)) * 2).astype(np.float32)
    ids = np.stack([rng.permutation(40)[:4] for _ in range(6)]).astype(np.uint32)
    top = rng.standard_normal((6, 4)).astype(np.float32)
    z[0, 5:] = -np.inf                       # all but five tokens forbidden
    ids[0] = [0, 1, 2, 3]
    z[1] = np.finfo(np.float32).min          # masked by the lowest value throughout
    z[2, 10:] = np.finfo(np.float32).min
    ids[2] = [1, 2, 3, 4]
    top[3] = -np.inf                         # no stored logit
    top[4, 1:] = -np.inf                     # one stored logit: minus its log-probability
    z[5] *= 40.0                             # far apart
    loss, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32), 1.0)
    ref, p, q = recurrent.distill(z, top, ids, 1.0)
    tol = U * (8 * 400 + 64)
    assert np.isfinite(loss.numpy()).all()
    assert np.abs(loss.numpy() - ref).max() <= tol * max(1, np.abs(ref).max())
    assert loss.numpy()[3, 0] == 0
    d = F.distill_loss_backward(up(np.ones((6, 1))), up(z), up(top), up(ids, np.uint32), stats)
    rd = recurrent.distill_backward(np.ones((6, 1)), z, top, ids, 1.0)
    assert np.abs(d.numpy() - rd).max() <= tol
    assert not d.numpy()[3].any() and not d.numpy()[0, 5:].any()
    # a forbidden token that the teacher wants costs everything
    ids[0, 0] = 20
    loss, _ = F.distill_loss(up(z), up(top), up(ids, np.uint32), 1.0)
    assert loss.numpy()[0, 0] == np.inf and np.isfinite(loss.numpy()[1:]).all()
    # a row without stored logits is nothing, whatever the student says; NaN stays in its row
    z[3, 7], z[4, 7] = np.nan, np.nan
    loss, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32), 1.0)
    d = F.distill_loss_backward(up(np.ones((6, 1))), up(z), up(top), up(ids, np.uint32), stats)
    assert loss.numpy()[3, 0] == 0 and not d.numpy()[3].any()
    assert np.isnan(loss.numpy()[4, 0]) and np.isnan(d.numpy()[4]).all()
    assert np.isfinite(d.numpy()[[0, 1, 2, 5]]).all()


def test_an_id_stored_twice(rng):
    F = _F()
    z, top, ids = problem(rng, 3, 50, 6, False)
    ids[:, 3] = ids[:, 1]
    ids[1, :] = ids[1, 0]
    loss, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32))
    bl, bg = bounds(z, top, 1.0)
    assert np.abs(loss.numpy() - recurrent.distill(z, top, ids, 1.0)[0]).max() <= bl
    one = np.ones((3, 1), np.float32)
    d = F.distill_loss_backward(up(one), up(z), up(top), up(ids, np.uint32), stats).numpy()
    assert np.abs(d - recurrent.distill_backward(one, z, top, ids, 1.0)).max() <= 2 * bg


def test_id_outside_the_vocabulary(rng):
    F = _F()
    import wxx_b200 as wxx

    z, top, ids = problem(rng, 4, 30, 5, False)
    ids[2, 1] = 30
    loss, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32))
    assert wxx.backend.device_status() == 2
    gone = top.copy()
    gone[2, 1] = -np.inf
    ok = ids.copy()
    ok[2, 1] = 0
    assert np.array_equal(loss.numpy(), F.distill_loss(up(z), up(gone), up(ok, np.uint32))[0].numpy())
    one = up(np.ones((4, 1)))
    d = F.distill_loss_backward(one, up(z), up(top), up(ids, np.uint32), stats).numpy()
    assert wxx.backend.device_status() == 2
    ref = F.distill_loss_backward(one, up(z), up(gone), up(ok, np.uint32), stats).numpy()
    assert np.array_equal(d, ref)
    # behind an absent entry any id will do
    gone[2, 1] = -np.inf
    F.distill_loss(up(z), up(gone), up(ids, np.uint32))
    assert wxx.backend.device_status() == 0


@pytest.mark.parametrize("N,V", [(6, 5000), (6, 900), (1030, 300)])
def test_absent_entries_beside_foreign_ones(N, V, rng):
    """A NaN or an infinity among a row's stored logits makes its loss NaN, and the
    gradient where it is stored; the entries that are not there stay without effect,
    whatever their ids."""
    F = _F()
    K = 40
    z, top, ids = problem(rng, N, V, K, False)
    top[:, 20:] = -np.inf
    ids[:, 20:] = np.uint32(0xFFFFFFFF)
    ids[3, 20:] = np.argsort(z[3])[:20]
    top[1, 0] = top[3, 7] = np.nan
    top[2, 3] = np.inf
    loss, stats = F.distill_loss(up(z), up(top), up(ids, np.uint32), 2.0)
    grad = np.ones((N, 1), np.float32)
    d = F.distill_loss_backward(up(grad), up(z), up(top), up(ids, np.uint32), stats, 2.0).numpy()
    loss = loss.numpy()
    safe = np.where(top == -np.inf, 0, ids)
    for n in range(N):
        if n not in (1, 2, 3):
            want = recurrent.distill(z[n:n + 1], top[n:n + 1], safe[n:n + 1], 2.0)[0]
            assert abs(loss[n, 0] - want[0, 0]) <= 4 * bounds(z[n:n + 1], top[n:n + 1], 2.0)[0]
            continue
        assert np.isnan(loss[n, 0])
        stored = np.zeros(V, bool)
        stored[ids[n, :20]] = True
        assert np.isnan(d[n, stored]).all() and np.isfinite(d[n, ~stored]).all()
    import wxx_b200 as wxx

    assert wxx.backend.device_status() == 0


def test_strided_logits_and_empty_batch(rng):
    F = _F()
    z, top, ids = problem(rng, 6, 101, 9, False)
    padded = np.full((6, 128), 99.0, np.float32)
    padded[:, 3:104] = z
    view = up(padded)[:, 3:104]
    a = F.distill_loss(view, up(top), up(ids, np.uint32), 2.0)
    b = F.distill_loss(up(z), up(top), up(ids, np.uint32), 2.0)
    assert np.abs(a[0].numpy() - b[0].numpy()).max() <= 4 * bounds(z, top, 2.0)[0]
    one = up(np.ones((6, 1)))
    da = F.distill_loss_backward(one, view, up(top), up(ids, np.uint32), a[1], 2.0).numpy()
    db = F.distill_loss_backward(one, up(z), up(top), up(ids, np.uint32), b[1], 2.0).numpy()
    assert np.abs(da - db).max() <= 4 * bounds(z, top, 2.0)[1]
    loss, stats = F.distill_loss(up(z[:0]), up(top[:0]), up(ids[:0], np.uint32))
    assert loss.shape == [0, 1]
    assert F.distill_loss_backward(up(np.ones((0, 1))), up(z[:0]), up(top[:0]),
                                   up(ids[:0], np.uint32), stats).shape == [0, 101]


def test_offsets_past_32_bits(rng):
    """43000 x 50304 logits (2^31 of them, 8.7 GB): the last rows against the same
    rows on their own."""
    F = _F()
    import wxx_b200 as wxx

    N, V, K, n = 43000, 50304, 4, 3
    z, top, ids = problem(rng, n, V, K, False)
    big = wxx.Tensor((N, V), value=0.25)
    F.assign(big.narrow(0, N - n, n), up(z))
    all_top, all_ids = np.zeros((N, K), np.float32), np.tile(np.arange(K, dtype=np.uint32), (N, 1))
    all_top[N - n:], all_ids[N - n:] = top, ids
    loss, stats = F.distill_loss(big, up(all_top), up(all_ids, np.uint32))
    ref, rstats = F.distill_loss(up(z), up(top), up(ids, np.uint32))
    # (a row on its own may be summed in more pieces)
    bl, bg = bounds(z, top, 1.0)
    assert np.abs(loss.numpy()[N - n:] - ref.numpy()).max() <= 2 * bl
    # uniform student over V against uniform teacher over K
    assert np.abs(loss.numpy()[0] - np.log(V / K)) <= bl
    grad = np.ones((N, 1), np.float32)
    d = F.distill_loss_backward(up(grad), big, up(all_top), up(all_ids, np.uint32), stats)
    tail = d.narrow(0, N - n, n).numpy()
    rd = F.distill_loss_backward(up(grad[:n]), up(z), up(top), up(ids, np.uint32), rstats).numpy()
    assert np.abs(tail - rd).max() <= 2 * bg
    assert wxx.backend.device_status() == 0


def test_module_with_mask_trains_the_logits(rng):
    import wxx_b200 as wxx

    F = _F()
    z, top, ids = problem(rng, 8, 30, 6, False)
    mask = np.array([1, 1, 0, 1, 1, 0, 1, 1], np.float32)
    tau = 2.0
    for m in (None, mask):
        leaf = wxx.Parameter(up(z))
        loss = wxx.nn.DistillLoss(tau)(leaf, up(top), up(ids, np.uint32),
                                       None if m is None else up(m))
        loss.backward()
        w = np.ones(8) if m is None else m
        rows = recurrent.distill(z, top, ids, tau)[0][:, 0]
        bl, bg = bounds(z, top, tau)
        assert abs(loss.item() - (rows * w).sum() / w.sum()) <= 2 * tau * tau * bl
        ref = recurrent.distill_backward((w / w.sum())[:, None], z, top, ids, tau)
        assert np.abs(leaf.grad.numpy() - ref).max() <= 2 * tau * bg


@pytest.mark.parametrize("N,V,sliced", [(1100, 300, False), (3, 1021, False), (4, 5001, False),
                                        (4, 6001, True), (2, 60001, False)])
@pytest.mark.parametrize("tau", [1.0, 1.5, 2.0])
def test_probabilities_of_far_logits(N, V, sliced, tau, rng):
    """Logits to 80 tau below the largest, which is 0, so that their distances are
    exact: the gradient off the one stored entry is grad tau q.  Relative, entry by
    entry: 4 u for the exponential, u each for its argument's correction and product,
    the same for the terms of the sum and 16 u for adding them in a tree, u each for its
    reciprocal and three products: 32 u."""
    F = _F()
    far = np.sort(rng.uniform(0, 80 * tau, (N, V)), -1)
    far[:, 0] = 0
    z = (-far).astype(np.float32)
    order = rng.permutation(V)
    z = np.ascontiguousarray(z[:, order])
    best = np.full((N, 1), int(np.flatnonzero(order == 0)[0]), np.uint32)
    tz = up(np.concatenate([z[:, :1], z, z[:, :2]], -1))[:, 1:1 + V] if sliced else up(z)
    top, ids = up(np.zeros((N, 1))), up(best, np.uint32)
    loss, stats = F.distill_loss(tz, top, ids, tau)
    grad = rng.uniform(0.5, 2, (N, 1)).astype(np.float32)
    d = F.distill_loss_backward(up(grad), tz, top, ids, stats, tau).numpy().astype(np.float64)
    _, _, q = recurrent.distill(z, np.zeros((N, 1)), best, tau)
    ref = q * grad.astype(np.float64) * tau
    others = np.arange(V) != best[0, 0]
    off = np.abs(d / ref - 1)[:, others].max() / U
    assert off <= 32, off


@pytest.mark.parametrize("N", [511, 512])
@pytest.mark.parametrize("V,K", [(1021, 17), (200, 64)])
def test_both_sides_of_many_rows(N, V, K, rng):
    """Short rows: a block a row below 512 of them, a warp a row from there."""
    test_loss_and_gradient(N, V, K, 1.5, True, rng)
