"""The recurrent language model, distillation training and beam search on the
GPU against the 64-bit restatements.  Products run in 3xTF32 mode (2^-21 of a
product's terms), so logits of these small models are good to 1e-5 of their
largest entry, as for GPT2."""

import numpy as np
import pytest

from oracle import init, models, recurrent

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


def build(V, D, H, L, seed=3):
    wxx = _wxx()
    wxx.manual_seed(seed)
    m = wxx.nn.RecurrentLM(V, D, H, L)
    rng = np.random.default_rng(seed)
    sd = m.state_dict()
    for k, v in sd.items():            # weights large enough that the layers matter
        if v.ndim >= 2:
            sd[k] = (rng.standard_normal(v.shape) * (0.3 if "tok_emb" in k else 0.15)).astype(np.float32)
    m.load_state_dict(sd)
    wxx.manual_seed(None)
    return m, sd


def u32(a):
    return _wxx().functional.from_numpy(np.asarray(a), dtype=np.uint32)


@pytest.mark.parametrize("V,D,H,L,B,T", [(50, 32, None, 2, 2, 20), (97, 48, 12, 3, 3, 150),
                                         (64, 64, 2, 1, 1, 300)])
def test_forward_and_decode(V, D, H, L, B, T):
    wxx = _wxx()
    m, sd = build(V, D, H, L)
    ids = init.token_ids(1, B, T, V)
    reset = np.zeros((B, T), np.uint32)
    reset[:, 0] = 1
    reset[B - 1, T // 3] = 1
    ref = recurrent.lm_forward(sd, ids, L, reset)
    tol = 1e-5 * np.abs(ref).max()
    train = m(u32(ids)).numpy()                    # training mode, no reset
    plain = recurrent.lm_forward(sd, ids, L)
    assert np.abs(train - plain).max() < tol
    with wxx.backend.inferenceMode():
        got = m.forward(u32(ids), u32(reset)).numpy()
        assert np.abs(got - ref).max() < tol
        # the sequence in two calls, then token by token
        states = m.new_states(B)
        cut = T // 2
        a = m.forward(u32(ids[:, :cut]), None, states).numpy()
        b = m.forward(u32(ids[:, cut:T - 5]), None, states).numpy()
        assert np.abs(np.concatenate([a, b], 1) - plain[:, :T - 5]).max() < tol
        for t in range(T - 5, T):
            z = m.decode(u32(ids[:, t:t + 1]), states).numpy()
            assert np.abs(z - plain[:, t]).max() < tol
    assert wxx.backend.device_status() == 0


def test_parameter_gradients_against_differences():
    """Along a random direction in every parameter, the gradient against central
    differences of the 64-bit model's loss.  A step of 1e-4 leaves 1e-8 of the
    third derivative, so the bound is the gradient's own: products in 3xTF32 mode
    good to 1e-5 of their largest entry, through two layers' products."""
    wxx = _wxx()
    V, D, H, L, B, T, K = 40, 16, 4, 2, 2, 24, 8
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
        z = recurrent.lm_forward(state, ids, L, reset).reshape(B * T, V)
        return recurrent.distill(z, htop, hids, 1.5)[0].mean()

    assert abs(loss.item() - value(sd)) < 1e-5 * max(1.0, value(sd))
    names = dict(m.named_parameters())
    for name, p in names.items():
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
        assert abs(got - slope) < 1e-4 * scale + 1e-9, name


def test_distilling_a_teacher_lowers_the_loss():
    wxx = _wxx()
    F = wxx.functional
    V, B, T, K = 64, 4, 48, 16
    sd = init.gpt2_state_dict(0, V, 64, 2, 2, T)
    for k in sd:
        if sd[k].ndim >= 2:
            sd[k] = sd[k] * 6
    teacher = wxx.nn.GPT2(V, 64, 2, 2, max_len=T)
    teacher.load_state_dict(sd)
    ids = u32(init.token_ids(3, B, T, V))
    with wxx.backend.inferenceMode():
        top, top_ids = F.topk(teacher(ids).reshape((B * T, V)), K)
    wxx.manual_seed(1)
    student = wxx.nn.RecurrentLM(V, 64, 8, 2)
    wxx.manual_seed(None)
    opt = wxx.nn.AdamW(student.parameters(), lr=3e-3)
    loss_of = wxx.nn.DistillLoss(2.0)
    losses = []
    for _ in range(40):
        opt.zero_grad()
        loss = loss_of(student(ids).reshape((B * T, V)), top, top_ids)
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.5 * losses[0]
    assert wxx.backend.device_status() == 0


@pytest.mark.parametrize("beams,n,stop", [(1, 12, None), (3, 12, None), (4, 16, 11), (8, 6, None)])
def test_beam_search_over_states(beams, n, stop):
    wxx = _wxx()
    V, D, H, L = 60, 32, 8, 2
    m, sd = build(V, D, H, L)
    prompt = init.token_ids(4, 2, 5, V)
    got, scores = m.beam_search(prompt, beams=beams, max_new_tokens=n, stop_token=stop)
    ref, rscores, gap = recurrent.beam_search(lambda i: recurrent.lm_forward(sd, i, L), prompt,
                                              beams, n, stop)
    assert gap > 1e-4                      # proposals further apart than the logits' error
    assert got.shape[2] <= ref.shape[2]    # the search ends when every beam is finished
    assert np.array_equal(got, ref[:, :, :got.shape[2]])
    assert np.abs(scores - rscores).max() < 1e-4
    from wxx_b200.nn.generation import beam_search

    again, s2 = beam_search(m, prompt, beams, n, stop, use_graph=False)
    assert np.array_equal(again, got) and np.array_equal(s2, scores)
    assert wxx.backend.device_status() == 0


@pytest.mark.parametrize("beams,n,stop", [(2, 20, None), (4, 10, None), (5, 14, 7)])
def test_beam_search_over_caches(beams, n, stop):
    wxx = _wxx()
    V, D, H, L, S = 80, 64, 2, 2, 48
    sd = init.gpt2_state_dict(5, V, D, H, L, S)
    for k in sd:
        if sd[k].ndim >= 2:
            sd[k] = sd[k] * 8
    m = wxx.nn.GPT2(V, D, H, L, max_len=S)
    m.load_state_dict(sd)
    prompt = init.token_ids(6, 3, 6, V)
    got, scores = m.beam_search(prompt, beams=beams, max_new_tokens=n, stop_token=stop)
    ref, rscores, gap = recurrent.beam_search(lambda i: models.gpt2_forward(sd, i, H, L), prompt,
                                              beams, n, stop)
    assert gap > 1e-3                      # (the reference forward rounds to 32 bits)
    assert np.array_equal(got, ref[:, :, :got.shape[2]])
    assert np.abs(scores - rscores).max() < 1e-3
    assert wxx.backend.device_status() == 0


def test_beam_search_limits_and_refusals():
    wxx = _wxx()
    m, _ = build(30, 16, None, 1)
    ids, scores = m.beam_search(np.array([1, 2]), beams=2, max_new_tokens=0)
    assert ids.shape == (1, 2, 2) and not scores.any()
    for kw, err in [({"beams": 0}, ValueError), ({"beams": 17}, ValueError),
                    ({"stop_token": 30}, ValueError)]:
        with pytest.raises(err):
            m.beam_search(np.array([[1]]), **kw)
    with pytest.raises(ValueError):
        m.beam_search(np.zeros((1, 0), np.uint32))
    g = wxx.nn.GPT2(30, 32, 1, 1, max_len=8)
    ids, _ = g.beam_search(np.array([[1, 2, 3]]), beams=3, max_new_tokens=50)
    assert ids.shape == (1, 3, 8)
    # a length penalty only reorders and rescales
    a, s = m.beam_search(np.array([[1]]), beams=4, max_new_tokens=6)
    b, t = m.beam_search(np.array([[1]]), beams=4, max_new_tokens=6, length_penalty=1.0)
    assert np.array_equal(a, b) and np.allclose(s / 6, t, rtol=1e-6)
    with pytest.raises(RuntimeError):
        m.forward(u32([[1, 2]]), None, m.new_states(1))       # a state in training mode


def test_beam_append():
    wxx = _wxx()
    F = wxx.functional
    ids = u32(np.zeros((5, 4), np.uint32))
    n = u32([2])
    F.beam_append(ids, u32([9, 8, 7, 6, 5]), n)
    F.beam_append(ids, u32(np.arange(5)), n)
    ref = np.zeros((5, 4), np.uint32)
    ref[:, 2], ref[:, 3] = [9, 8, 7, 6, 5], np.arange(5)
    assert np.array_equal(ids.numpy(), ref) and n.numpy()[0] == 4
    F.beam_append(ids, u32(np.arange(5)), n)
    assert wxx.backend.device_status() == 2
    assert np.array_equal(ids.numpy(), ref) and n.numpy()[0] == 4
    with pytest.raises(ValueError):
        F.beam_append(ids, u32([1, 2]), n)
    with pytest.raises(TypeError):
        F.beam_append(ids, F.from_numpy(np.zeros(5, np.float32)), n)
