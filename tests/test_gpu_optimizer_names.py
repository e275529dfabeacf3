"""Parameters with two names in the optimisers."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _wxx():
    import wxx_b200 as wxx

    return wxx


def test_sgd_steps_a_parameter_with_two_names_once(rng):
    """w - lr grad, for LayerNorm's parameters (two names each) as for any other."""
    wxx = _wxx()
    F = wxx.functional
    ln = wxx.nn.LayerNorm(16)
    before = {n: p.numpy() for n, p in ln.named_parameters()}
    opt = wxx.nn.SGD(ln.parameters(), lr=0.25)
    grads = [rng.standard_normal(16).astype(np.float32) for _ in range(2)]
    ln.weightg.grad, ln.weightb.grad = (F.from_numpy(g) for g in grads)
    opt.step()
    for name, p in ln.named_parameters():
        g = grads[0] if name in ("weight", "weightg") else grads[1]
        assert np.array_equal(p.numpy(), before[name] + g * np.float32(-0.25)), name


def test_adamw_keeps_moments_once_for_each_parameter():
    wxx = _wxx()
    m = wxx.nn.Sequential(wxx.nn.Linear(4, 8), wxx.nn.LayerNorm(8))
    opt = wxx.nn.AdamW(m.parameters())
    assert len(opt.state) == len(opt.params) == len({id(p) for _, p in m.named_parameters()}) == 4
