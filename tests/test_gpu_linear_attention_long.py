"""Linear attention over rows long enough to be worked on in many pieces, against its 64-bit
restatement: what reaches a piece from the ones before it."""

import numpy as np
import pytest

from oracle import retention

pytestmark = pytest.mark.gpu


def _F():
    import wxx_b200 as wxx

    return wxx.functional


def up(a, dtype=np.float32):
    return None if a is None else _F().from_numpy(np.asarray(a), dtype=dtype)


def normals(rng, *shapes):
    return [rng.standard_normal(s).astype(np.float32) for s in shapes]


@pytest.mark.parametrize("memory", [2, 8, 2000])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("d,T", [(32, 20000), (64, 9000)])
def test_only_a_reset_ends_a_value_that_is_not_finite(d, T, bad, memory, rng):
    """A NaN or an infinity near a row's start (backward: its end) reaches all that follows in
    its document, in all pieces, also where the decays over a piece are below 2^-149."""
    F = _F()
    H = 2
    q, k, v, do = normals(rng, *[(1, T, H * d)] * 4)
    h0, dlast = normals(rng, *[(1, H, d, d)] * 2)
    decay = np.log1p(-1 / np.full(H, memory, np.float64)).astype(np.float32)
    with_reset = np.zeros((1, T), np.uint32)
    with_reset[0, T // 2] = 1
    for reset in (None, with_reset):
        r = up(reset, np.uint32)
        for name in ("v", "h0"):
            given = {"v": v.copy(), "h0": h0.copy()}
            given[name][(0, 70, 3) if name == "v" else (0, 0, 2, 3)] = bad    # head 0, column 3
            o, last = F.linear_attention(up(q), up(k), up(given["v"]), up(decay), up(given["h0"]), r)
            hit = ~np.isfinite(o.numpy())
            want = np.zeros((1, T, H * d), bool)
            want[0, 70 if name == "v" else 0:T if reset is None else T // 2, 3] = True
            assert np.array_equal(hit, want)
            hit = ~np.isfinite(last.numpy())
            want = np.zeros((1, H, d, d), bool)
            if reset is None:
                want[0, 0, slice(None) if name == "v" else 2, 3] = True
            assert np.array_equal(hit, want)
        for name in ("do", "dlast"):
            given = {"do": do.copy(), "dlast": dlast.copy()}
            given[name][(0, T - 70, 3) if name == "do" else (0, 0, 2, 3)] = bad
            dv = F.linear_attention_backward(up(given["do"]), up(q), up(k), up(v), up(decay), up(h0),
                                             r, up(given["dlast"]))[2].numpy()
            want = np.zeros((1, T, H * d), bool)
            want[0, 0 if reset is None else T // 2:T - 69 if name == "do" else T, 3] = True
            assert np.array_equal(~np.isfinite(dv), want)


@pytest.mark.parametrize("memory", [2 ** 14, 2 ** 16, 2 ** 18])
@pytest.mark.parametrize("B,H,d", [(1, 2, 32), (1, 2, 64), (150, 1, 32)])
def test_long_memories(B, H, d, memory, rng):
    """Memories of 2^14 positions and more over 32768, in many pieces and (150 sequences) in few.
    A state is rounded once a chunk of 64 positions, 512 times, independently: sqrt(512) u / 2 = 12
    u of it; its products 8 u, its decays a few u for all chunks together: below 64 u = 4e-6 in the
    2-norm.  Decays that are rounded alike in every chunk, u / 2 of the state each, would be off by up
    to 256 u."""
    F = _F()
    T = 32768
    rows = min(B, 2)                             # these again and again
    q, k, v, do = normals(rng, *[(rows, T, H * d)] * 4)
    k, v, q, do = k + 0.5, v + 0.5, q + 0.5, do + 0.5
    h0, dlast = normals(rng, *[(rows, H, d, d)] * 2)
    h0, dlast = 100 * h0, 100 * dlast
    decay = np.full(H, np.log1p(-1 / memory), np.float32)

    def many(t):
        return up(np.ascontiguousarray(np.broadcast_to(t, (B // rows,) + t.shape)).reshape(
            (B,) + t.shape[1:]))

    def close(got, ref, what):
        got = got.numpy().astype(np.float64)
        for at in {0, B // rows - 1}:
            part = got[at * rows:(at + 1) * rows]
            e = np.linalg.norm(part - ref) / np.linalg.norm(ref)
            assert e < 4e-6, (what, e)

    refs = retention.linear_attention_long(do, q, k, v, decay, h0, dlast)
    args = [many(t) for t in (q, k, v)] + [up(decay), many(h0)]
    got = (*F.linear_attention(*args),
           *F.linear_attention_backward(many(do), *args, None, many(dlast)))
    for name, g, ref in zip(("o", "last", "dq", "dk", "dv", "dh0"), got, refs):
        close(g, ref, name)
    # what is left of h0 alone
    none = np.zeros_like(v)
    o, last = F.linear_attention(many(q), many(k), many(none), up(decay), many(h0))
    close(last, np.exp(T * decay.astype(np.float64))[None, :, None, None] * h0, "h0")


@pytest.mark.parametrize("d", [32, 64])
def test_sizes_of_a_chunk_do_not_meet(d, rng):
    """Positions of a chunk whose keys and values are more than 2^126 apart, the large ones
    later, or in another document: each output is as good as its own terms allow."""
    F = _F()
    T, H = 64, 1
    q, k, v = normals(rng, *[(1, T, d)] * 3)
    size = np.where(np.arange(T) < 20, 1e-10, np.where(np.arange(T) < 40, 1e12, 1e-12))
    k, v = ((t * size[None, :, None]).astype(np.float32) for t in (k, v))
    reset = np.zeros((1, T), np.uint32)
    reset[0, 40] = 1
    decay = np.float32([-0.01])
    for back in (False, True):
        if back:
            got = F.linear_attention_backward(up(v), up(k), up(q), up(q), up(decay), None,
                                              up(reset, np.uint32))[2].numpy()
            ref = retention.linear_attention_backward(v, k, q, q, decay, None, reset)[2]
            top = retention.linear_attention_backward(*map(np.abs, (v, k, q, q)), decay, None, reset)[2]
        else:
            got = F.linear_attention(up(q), up(k), up(v), up(decay), None, up(reset, np.uint32))[0].numpy()
            ref = retention.linear_attention(q, k, v, decay, None, reset)[0]
            top = retention.linear_attention(*map(np.abs, (q, k, v)), decay, None, reset)[0]
        # 3 * 2^-22 of the rows' lengths for halves, (64 + 8 sqrt(64) + d) u for the sums
        tol = (3 * 2.0 ** -22 + (128 + d) * 2.0 ** -24) * d
        worst = np.abs(got - ref).max(-1) / top.max(-1)
        assert worst.max() < tol, (back, worst)


@pytest.mark.parametrize("d,scale", [(64, 1e-36), (64, -1e-30), (32, 1e30), (32, 1e-33), (200, 1e-36)])
def test_scales_near_the_ends_of_the_range(d, scale, rng):
    """A scale multiplies: outputs and gradients are those of scale 1 times it, each term rounded
    as there (two roundings more), the states free of it."""
    F = _F()
    B, T, H = 2, 150, 2
    q, k, v, do = normals(rng, *[(B, T, H * d)] * 4)
    h0, dlast = normals(rng, *[(B, H, d, d)] * 2)
    dlast *= np.float32(scale)
    decay = np.log1p(-1 / np.float32([8, 100])).astype(np.float32)
    args = [up(t) for t in (q, k, v, decay, h0)]
    o, last = F.linear_attention(*args, scale=scale)
    scale = float(np.float32(scale))
    refs = (*retention.linear_attention(q, k, v, decay, h0, None, scale),
            *retention.linear_attention_backward(do, q, k, v, decay, h0, None, dlast, scale))
    got = (o, last, *F.linear_attention_backward(up(do), *args, None, up(dlast), scale=scale))
    for g, ref in zip(got, refs):
        e = np.linalg.norm(g.numpy().astype(np.float64) - ref) / np.linalg.norm(ref)
        assert e < 4e-6, e


def test_documents_after_their_last_token_take_as_long_as_others(rng):
    """Sequences that end early (keys and values of 0 from there on; backward: no gradient after
    the prompt): the state decays below 2^-60 there and goes on as any other, to the formula's
    values, and in about the time of a row of ordinary numbers."""
    import wxx_b200 as wxx

    F = _F()
    B, T, H, d, n = 40, 4096, 1, 64, 512
    q, k, v, do = normals(rng, *[(B, T, H * d)] * 4)
    kz, vz, doz = k.copy(), v.copy(), do.copy()
    kz[:, n:] = vz[:, n:] = 0
    doz[:, :T - n] = 0
    decay = np.log1p(-1 / np.float32([8])).astype(np.float32)
    ld, uq = up(decay), up(q)
    plain, ended = [up(t) for t in (k, v, do)], [up(t) for t in (kz, vz, doz)]
    o, last = F.linear_attention(uq, ended[0], ended[1], ld)
    grads = F.linear_attention_backward(ended[2], uq, plain[0], plain[1], ld)
    row = slice(3, 4)
    ro, rlast = retention.linear_attention(q[row], kz[row], vz[row], decay)
    refs = retention.linear_attention_backward(doz[row], q[row], k[row], v[row], decay)
    # Rows of an output against their own lengths: the decays over t positions, each good to t
    # log(memory) u, as far as a number and its state (times up to 2^4) are normal ones
    for got, ref in ((o, ro), (grads[1], refs[1]), (grads[2], refs[2])):
        got, ref = got.numpy()[row].astype(np.float64)[0], ref[0]
        size, off = np.linalg.norm(ref, axis=-1), np.linalg.norm(got - ref, axis=-1)
        normal = size > 2.0 ** -110
        assert normal.sum() > 1000 and (off[normal] < 1e-4 * size[normal]).all()
        assert (off[~normal] < 2.0 ** -109).all()
    assert np.abs(last.numpy()[row] - rlast).max() < 2.0 ** -120

    def ms(call):
        times = []
        for _ in range(6):
            a = wxx.backend.device.Event().record()
            keep = call()
            b = wxx.backend.device.Event().record()
            wxx.backend.device.synchronize()
            times.append(a.elapsed_ms(b))
            del keep
        return min(times)

    # (position by position the forward took 11 times as long)
    assert ms(lambda: F.linear_attention(uq, ended[0], ended[1], ld)) < \
        4 * ms(lambda: F.linear_attention(uq, plain[0], plain[1], ld))
    assert ms(lambda: F.linear_attention_backward(ended[2], uq, plain[0], plain[1], ld)) < \
        4 * ms(lambda: F.linear_attention_backward(plain[2], uq, plain[0], plain[1], ld))


@pytest.mark.parametrize("d,log_decay,T", [(32, -3.0, 200), (64, -1.5, 200), (64, -0.1, 12000),
                                           (32, -2.0, 12000)])
def test_large_numbers_behind_small_decays(d, log_decay, T, rng):
    """Keys and values of 1e12 to 1e15 at a row's first positions, little after them, queries of
    1e6: their part of later outputs counts where the decay itself is below 2^-126.  A position's
    decay, rounded each time, is off by up to t |log decay| u after t of them, t |log decay| below
    120 where the terms are above 1e-15: with the products and sums (128 + 2 d) u of the terms."""
    F = _F()
    H = 1
    q, k, v, do = normals(rng, *[(1, T, H * d)] * 4)
    q *= np.float32(1e6)
    k[:, :3] *= np.float32(1e12)
    v[:, :3] *= np.float32(1e15)
    k[:, 3:] *= np.float32(1e-15)
    v[:, 3:] *= np.float32(1e-10)
    decay = np.float32([log_decay])
    terms = [np.abs(t) for t in (q, k, v)]
    o, last = F.linear_attention(up(q), up(k), up(v), up(decay))
    ro, rlast = retention.linear_attention(q, k, v, decay)
    mo, mlast = retention.linear_attention(*terms, decay)
    for got, ref, size in ((o, ro, mo), (last, rlast, mlast)):
        off = np.abs(got.numpy() - ref)
        counts = size > 1e-15
        # halves: 3 * 2^-22 of the rows' lengths, up to d / 2 of their entries' products
        assert (off <= (3 * 2.0 ** -22 * d + (248 + 2 * d) * 2.0 ** -24) * size)[counts].all()
