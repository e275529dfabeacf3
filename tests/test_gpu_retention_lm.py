"""The recurrent language model with retentions on the GPU against its 64-bit restatement:
rotary positions, linear attention and the gated group norm as a model runs them together, in
training, prefill, decoding, beam search and in a recorded step.

Products run in 3xTF32 mode, good to 2^-21 of their terms' sizes, and the mixers' values to 2^-20
with their own roundings.  A head's norm divides by the head's size, so where its terms cancel it
passes errors on enlarged: the bound is twice what such errors do to the 64-bit model's logits
(``retention.lm_error``), and 1e-5 of the largest logit for the other layers."""

import numpy as np
import pytest

from oracle import init, recurrent, retention

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _faithful_products():
    import wxx_b200 as wxx

    wxx.set_matmul_mode("3xtf32")
    yield
    wxx.set_matmul_mode("tf32")


def _wxx():
    import wxx_b200 as wxx

    return wxx


def decays(H):
    return np.log1p(-1 / 2.0 ** np.linspace(3, 9, H)).astype(np.float32).astype(np.float64)


def build(V, D, H, L, seed=3):
    wxx = _wxx()
    wxx.manual_seed(seed)
    m = wxx.nn.RecurrentLM(V, D, H, L, mixer="retention")
    rng = np.random.default_rng(seed)
    sd = m.state_dict()
    for k, v in sd.items():            # weights large enough that the layers matter
        if v.ndim >= 2:
            sd[k] = (rng.standard_normal(v.shape) * (0.3 if "tok_emb" in k else 0.15)).astype(np.float32)
        elif "norm" in k:
            sd[k] = (v + rng.standard_normal(v.shape) * 0.1).astype(np.float32)
    m.load_state_dict(sd)
    wxx.manual_seed(None)
    return m, sd


def u32(a):
    return _wxx().functional.from_numpy(np.asarray(a), dtype=np.uint32)


def bound(ref, *args):
    return 2 * retention.lm_error(*args).max() + 1e-5 * np.abs(ref).max()


@pytest.mark.parametrize("V,D,H,L,B,T", [(50, 32, 4, 2, 2, 20), (97, 48, 3, 3, 3, 150),
                                         (64, 64, 1, 1, 1, 300), (33, 20, 2, 1, 2, 70)])
def test_forward_and_decode(V, D, H, L, B, T):
    wxx = _wxx()
    m, sd = build(V, D, H, L)
    ids = init.token_ids(1, B, T, V)
    reset = np.zeros((B, T), np.uint32)
    reset[:, 0] = 1
    reset[B - 1, T // 3] = 1
    ref = retention.lm_forward(sd, ids, L, H, decays(H), reset)
    tol = bound(ref, sd, ids, L, H, decays(H), reset)
    plain = retention.lm_forward(sd, ids, L, H, decays(H))
    ptol = bound(plain, sd, ids, L, H, decays(H))
    assert np.abs(m(u32(ids)).numpy() - plain).max() < ptol       # training mode, no reset
    with wxx.backend.inferenceMode():
        assert np.abs(m.forward(u32(ids), u32(reset)).numpy() - ref).max() < tol
        # the sequence in two calls, then token by token, the positions of either shape
        states = m.new_states(B)
        cut = T // 2
        a = m.forward(u32(ids[:, :cut]), None, states).numpy()
        b = m.forward(u32(ids[:, cut:T - 5]), None, states, cut).numpy()
        assert np.abs(np.concatenate([a, b], 1) - plain[:, :T - 5]).max() < ptol
        for t in range(T - 5, T):
            at = u32([t]) if t % 2 else u32(np.full((B, 1), t))
            z = m.decode(u32(ids[:, t:t + 1]), states, at).numpy()
            assert np.abs(z - plain[:, t]).max() < ptol
    assert wxx.backend.device_status() == 0


def test_sequences_at_different_lengths_decode_together():
    """A batch's rows at different positions: each row as it would be alone."""
    wxx = _wxx()
    V, D, H, L = 50, 32, 4, 2
    m, sd = build(V, D, H, L)
    lengths = [1, 9, 70]
    ids = init.token_ids(8, 3, 75, V)
    with wxx.backend.inferenceMode():
        states = m.new_states(3)
        for r, n in enumerate(lengths):
            alone = m.new_states(1)
            m.forward(u32(ids[r:r + 1, :n]), None, alone)
            for full, one in zip(states, alone):
                wxx.functional.assign(full.narrow(0, r, 1), one)
        for s in range(3):
            at = np.array(lengths) + s
            z = m.decode(u32([[ids[r, t]] for r, t in enumerate(at)]), states,
                         u32(at.reshape(3, 1))).numpy()
            for r, t in enumerate(at):
                one = ids[r:r + 1, :t + 1]
                ref = retention.lm_forward(sd, one, L, H, decays(H))
                assert np.abs(z[r] - ref[0, t]).max() < bound(ref, sd, one, L, H, decays(H))
    assert wxx.backend.device_status() == 0


def test_parameter_gradients_against_differences():
    """Along a random direction in every parameter, the gradient against central differences of
    the 64-bit model's loss.  A step of 1e-4 leaves 1e-8 of the third derivative; the products are
    good to 1e-4 of a gradient through two layers, and the mixers' own errors, of 2^-20 of their
    terms, move a derivative of this model by 2e-6 of the direction's length at most (counted in
    64 bits for each parameter), twice that is allowed."""
    wxx = _wxx()
    V, D, H, L, B, T, K = 40, 16, 2, 2, 2, 24, 8
    m, sd = build(V, D, H, L)
    ids = init.token_ids(2, B, T, V)
    reset = np.zeros((B, T), np.uint32)
    reset[1, 9] = 1
    rng = np.random.default_rng(0)
    teacher = rng.standard_normal((B * T, V)).astype(np.float32) * 2
    top, top_ids = wxx.functional.topk(wxx.functional.from_numpy(teacher), K)
    loss = wxx.nn.DistillLoss(1.5)(m.forward(u32(ids), u32(reset)).reshape((B * T, V)), top, top_ids)
    loss.backward()
    hids = top_ids.numpy().astype(np.int64)
    htop = top.numpy()

    def value(state):
        z = retention.lm_forward(state, ids, L, H, decays(H), reset).reshape(B * T, V)
        return recurrent.distill(z, htop, hids, 1.5)[0].mean()

    assert abs(loss.item() - value(sd)) < 1e-5 * max(1.0, value(sd))
    for name, p in m.named_parameters():
        if name.endswith(("ln1.weight", "ln1.bias", "ln2.weight", "ln2.bias", "ln_f.weight",
                          "ln_f.bias")):
            continue                    # aliases of weightg / weightb
        d = rng.standard_normal(p.shape)
        step = 1e-4 / np.sqrt(d.size)
        hi, lo = dict(sd), dict(sd)
        hi[name] = sd[name].astype(np.float64) + step * d
        lo[name] = sd[name].astype(np.float64) - step * d
        slope = (value(hi) - value(lo)) / (2 * step)
        got = (p.grad.numpy().astype(np.float64) * d).sum()
        scale = np.linalg.norm(p.grad.numpy()) * np.linalg.norm(d)
        assert abs(got - slope) < 1e-4 * scale + 4e-6 * np.linalg.norm(d), name


def test_training_step_replays_from_a_graph():
    """Recorded steps on new batches end where the eager ones do (the embedding gradient's
    atomic adds may reorder 32-bit sums, hence a tolerance), with an eager forward of
    the same parameters alive meanwhile."""
    wxx = _wxx()
    F = wxx.functional
    V, D, H, L, S, B = 64, 32, 2, 2, 70, 2
    rng = np.random.default_rng(11)
    batches = [rng.integers(0, V, size=(B, S)).astype(np.uint32) for _ in range(4)]

    def make():
        model, _ = build(V, D, H, L)
        opt = wxx.nn.AdamW(model.parameters(), lr=1e-3)
        ids, tgt = u32(batches[0]), u32(np.roll(batches[0], -1, axis=1).reshape(-1))

        def step():
            opt.zero_grad()
            loss = wxx.nn.CCELoss()(model(ids).reshape((B * S, V)), tgt)
            loss.backward()
            opt.step()
            return loss

        return model, ids, tgt, step

    def load(ids, tgt, k):
        F.assign(ids, u32(batches[k]))
        F.assign(tgt, u32(np.roll(batches[k], -1, axis=1).reshape(-1)))

    m_eager, ids, tgt, step = make()
    for k in range(4):
        load(ids, tgt, k)
        last_eager = float(step().numpy().reshape(-1)[0])
    m_graph, ids, tgt, step = make()
    alive = m_graph(ids)
    g = wxx.graph.capture(step)                 # its warm-up run is step 1 (batch 0)
    try:
        for k in range(1, 4):
            load(ids, tgt, k)
            out = g.replay()
        assert abs(float(out.numpy().reshape(-1)[0]) - last_eager) < 1e-4 * max(1.0, abs(last_eager))
        eager = dict(m_eager.named_parameters())
        for name, p in m_graph.named_parameters():
            a, b = p.numpy(), eager[name].numpy()
            assert np.linalg.norm(a - b) < 1e-3 * np.linalg.norm(b) + 1e-6, name
    finally:
        g.close()
    assert alive.shape[0] == B
    assert wxx.backend.device_status() == 0


def test_a_parameter_listed_twice_is_stepped_once():
    """LayerNorm's parameters have two names each; AdamW steps them like any other, to the bit,
    however its blocks are scheduled."""
    wxx = _wxx()
    F = wxx.functional
    rng = np.random.default_rng(5)
    sizes = [32, 4096, 70000]
    w0 = [rng.standard_normal(n).astype(np.float32) for n in sizes]
    grads = [[rng.standard_normal(n).astype(np.float32) for n in sizes] for _ in range(5)]

    def run(times):
        params = [wxx.Parameter(F.from_numpy(w)) for w in w0]
        opt = wxx.nn.AdamW([("", p) for p in params for _ in range(times)], lr=1e-2)
        for g in grads:
            for p, t in zip(params, g):
                p.grad = F.from_numpy(t)
            opt.step()
        return [p.numpy() for p in params]

    once = run(1)
    for _ in range(10):
        for a, b in zip(run(2), once):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("beams,n,stop", [(1, 12, None), (3, 12, None), (4, 16, 11), (8, 6, None)])
def test_beam_search_over_states(beams, n, stop):
    wxx = _wxx()
    V, D, H, L = 60, 32, 4, 2
    m, sd = build(V, D, H, L)
    prompt = init.token_ids(4, 2, 5, V)
    got, scores = m.beam_search(prompt, beams=beams, max_new_tokens=n, stop_token=stop)
    logits = lambda i: retention.lm_forward(sd, i, L, H, decays(H))  # noqa: E731
    ref, rscores, gap = recurrent.beam_search(logits, prompt, beams, n, stop)
    # A score is the sum of its new tokens' log-probabilities, and log p_i = z_i - log sum exp z
    # moves by at most twice the largest error e_t of its position's logits (the logarithm by a
    # mean of the errors): a score by 2 sum e_t over the positions that chose a token.  The
    # prompt's other positions, whose heads cancel most, do not enter.
    rows = ref.reshape(-1, ref.shape[-1])
    e = 2 * retention.lm_error(sd, rows, L, H, decays(H)) + 1e-5 * np.abs(logits(rows)).max(-1)
    tol = 2 * e[:, prompt.shape[1] - 1:-1].sum(1).max()
    assert gap > tol                       # proposals further apart than the scores' error
    assert got.shape[2] <= ref.shape[2]    # the search ends when every beam is finished
    assert np.array_equal(got, ref[:, :, :got.shape[2]])
    assert np.abs(scores - rscores).max() < tol
    from wxx_b200.nn.generation import beam_search

    again, s2 = beam_search(m, prompt, beams, n, stop, use_graph=False)
    assert np.array_equal(again, got) and np.array_equal(s2, scores)
    assert wxx.backend.device_status() == 0


def test_rotary_linear_attention_and_norm_in_a_row(rng):
    """The functional forms as a user runs them: queries and keys turned in one call from a
    projection's slice, the state carried from a prefill into single steps, the heads' norm with
    the gate; a whole sequence against the pieces and against 64 bits.  Each of o's values is off
    by up to 2^-20 of its terms; the norm enlarges it by the head's 1 / deviation."""
    F = _wxx().functional
    B, T, H, hd = 3, 100, 4, 24
    D = H * hd
    x = rng.standard_normal((B, T, 4 * D)).astype(np.float32)
    gamma = rng.standard_normal(D).astype(np.float32)
    f, ld = F.rotary_frequencies(hd), decays(H)
    decay = F.from_numpy(ld.astype(np.float32))
    up = F.from_numpy(x)
    ug = F.from_numpy(gamma)

    def part(lo, hi):
        return up.narrow(1, lo, hi - lo)

    def mix(p, lo, state):
        qk = F.rotary(p.narrow(2, 0, 2 * D), 2 * H, f, None, lo)
        return F.linear_attention(qk.narrow(2, 0, D), qk.narrow(2, D, D), p.narrow(2, 2 * D, D),
                                  decay, state, None, 0.2)

    def norm(o, p):
        return F.group_norm(o, H, ug, None, "silu", p.narrow(2, 3 * D, D))

    rows = (B * T, D)
    x64 = x.astype(np.float64)
    q, k = (retention.rotary(x64[:, :, s], H, np.array(f.frequencies))
            for s in (slice(0, D), slice(D, 2 * D)))
    ro, rlast = retention.linear_attention(q, k, x64[:, :, 2 * D:3 * D], ld, None, None, 0.2)
    terms = retention.linear_attention(np.abs(q), np.abs(k), np.abs(x64[:, :, 2 * D:3 * D]), ld,
                                       None, None, 0.2)[0]
    # a norm over one position's head: the samples are positions
    ry = retention.group_norm(ro.reshape(rows), H, gamma, None, "silu",
                              x64[:, :, 3 * D:].reshape(rows))[0].reshape(B, T, D)
    dev = np.sqrt(ro.reshape(B, T, H, hd).var(-1) + 1e-5)
    grown = (terms.reshape(B, T, H, hd).max(-1) * 2.0 ** -20 / dev)[..., None]
    tol = (4 * grown * (1 + np.abs(ry.reshape(B, T, H, hd))) * 4).reshape(B, T, D) + 1e-5

    def check(o, p, lo, hi):
        n = hi - lo
        y = norm(o.reshape((B * n, 1, D)), p.reshape((B * n, 1, 4 * D)))[0].numpy().reshape(B, n, D)
        e = np.abs(y - ry[:, lo:hi])
        assert (e < tol[:, lo:hi]).all()

    o, last = mix(up, 0, None)
    check(o, up, 0, T)
    assert np.abs(last.numpy() - rlast).max() < 1e-5 * np.abs(rlast).max()
    state = None
    for lo, hi in ((0, 33), (33, 97)):
        o, state = mix(part(lo, hi), lo, state)
        check(o, part(lo, hi), lo, hi)
    for t in range(97, T):
        p = part(t, t + 1)
        qk = F.rotary(p.narrow(2, 0, 2 * D), 2 * H, f, u32([t])).reshape((B, 2 * D))
        o = F.linear_attention_step(qk.narrow(1, 0, D), qk.narrow(1, D, D),
                                    p.reshape((B, 4 * D)).narrow(1, 2 * D, D), decay, state, 0.2)
        check(o, p, t, t + 1)
    assert np.abs(state.numpy() - rlast).max() < 1e-5 * np.abs(rlast).max()


def test_refusals():
    wxx = _wxx()
    F = wxx.functional
    for args in ((30, 16, None, 1), (30, 16, 3, 1), (30, 18, 2, 1), (30, 514, 1, 1)):
        with pytest.raises(ValueError):
            wxx.nn.RecurrentLM(*args, mixer="retention")
    with pytest.raises(ValueError):
        wxx.nn.RecurrentLM(30, 16, 2, 1, mixer="attention")
    with pytest.raises(ValueError):
        wxx.nn.GroupNorm(3, 16)
    m, _ = build(30, 16, 2, 1)
    with pytest.raises(RuntimeError):
        m.forward(u32([[1, 2]]), None, m.new_states(1))       # a state in training mode
    with wxx.backend.inferenceMode():
        with pytest.raises(ValueError):
            m.decode(u32([[1]]), m.new_states(1))             # no positions
        with pytest.raises(TypeError):
            m.decode(u32([[1]]), m.new_states(1), F.from_numpy(np.zeros(1, np.float32)))
        with pytest.raises(ValueError):
            m.decode(u32([[1]]), m.new_states(1), u32([1, 2]))
    q = F.from_numpy(np.zeros((1, 2, 4), np.float32))
    decay = wxx.Parameter(F.from_numpy(np.zeros(2, np.float32)))
    with pytest.raises(ValueError):
        wxx.autograd.linear_attention(q, q, q).forward(q, q, q, decay)
