"""Tensors that an autograd function is, and is not, constructed with."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _wxx():
    import wxx_b200 as wxx

    return wxx


def test_gradients_are_not_dropped(rng):
    """A tensor that needs a gradient is refused where the function is not constructed with it, in
    its place; without one it may be given to forward alone."""
    wxx = _wxx()
    F, autograd = wxx.functional, wxx.autograd

    def t(*shape, grad=True):
        x = F.from_numpy(rng.standard_normal(shape).astype(np.float32))
        return wxx.Parameter(x) if grad else x

    q, k, v, h0 = t(2, 5, 8), t(2, 5, 8), t(2, 5, 8), t(2, 2, 4, 4)
    decay = F.from_numpy(np.float32([-0.1, -0.2]))
    for given in ((q, k, v), (q, k), (q, k, h0, v)):
        with pytest.raises(ValueError):
            autograd.linear_attention(*given).forward(q, k, v, decay, h0)
    o = autograd.linear_attention(q, k, v, h0).forward(q, k, v, decay, h0)
    do = t(2, 5, 8, grad=False)
    o.backward(do)
    grads = F.linear_attention_backward(do, q, k, v, decay, h0)
    for p, g in zip((q, k, v, h0), grads):
        assert np.array_equal(p.grad.numpy(), g.numpy())
    state = t(2, 2, 4, 4, grad=False)
    autograd.linear_attention(q, k, v).forward(q, k, v, decay, state).backward(do)

    x, gamma, beta, gate = t(6, 8), t(8), t(8), t(6, 8)
    for given in ((x, gamma, beta), (x, gate), (x, gate, gamma, beta)):
        with pytest.raises(ValueError):
            autograd.group_norm(*given).forward(x, 2, gamma, beta, "silu", gate)
    dy = t(6, 8, grad=False)
    autograd.group_norm(x, gamma, beta, gate).forward(x, 2, gamma, beta, "silu", gate).backward(dy)
    _, mean, inv = F.group_norm(x, 2, gamma, beta, "silu", gate)
    for p, g in zip((x, gamma, beta, gate),
                    F.group_norm_backward(dy, x, mean, inv, 2, gamma, beta, "silu", gate)):
        assert np.array_equal(p.grad.numpy(), g.numpy())
    # no gamma and beta: nothing in their places; a gate without a gradient to forward alone
    x.grad = gate.grad = None
    autograd.group_norm(x, None, None, gate).forward(x, 2, None, None, "silu", gate).backward(dy)
    grads = F.group_norm_backward(dy, x, mean, inv, 2, None, None, "silu", gate)
    assert np.array_equal(x.grad.numpy(), grads[0].numpy())
    assert np.array_equal(gate.grad.numpy(), grads[3].numpy())
    plain = t(6, 8, grad=False)
    x.grad = None
    autograd.group_norm(x, gamma, beta).forward(x, 2, gamma, beta, "silu", plain).backward(dy)
    assert np.array_equal(x.grad.numpy(), F.group_norm_backward(dy, x, mean, inv, 2, gamma, beta, "silu",
                                                                plain)[0].numpy())
    with wxx.backend.inferenceMode():                # no gradients there
        autograd.linear_attention(q, k, v).forward(q, k, v, decay, h0)


def test_group_norm_module_without_a_gate_trains(rng):
    wxx = _wxx()
    F = wxx.functional
    m = wxx.nn.GroupNorm(2, 8, activation="gelu")
    x = wxx.Parameter(F.from_numpy(rng.standard_normal((3, 5, 8)).astype(np.float32)))
    dy = F.from_numpy(rng.standard_normal((3, 5, 8)).astype(np.float32))
    m(x).backward(dy)
    _, mean, inv = F.group_norm(x, 2, m.weight, m.bias, "gelu")
    grads = F.group_norm_backward(dy, x, mean, inv, 2, m.weight, m.bias, "gelu")
    for p, g in zip((x, m.weight, m.bias), grads):
        assert np.array_equal(p.grad.numpy(), g.numpy())
