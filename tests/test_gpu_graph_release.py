"""The last tensor of a closed graph freed while another graph is recorded."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_stale_arena_freed_inside_a_capture(rng):
    import wxx_b200 as wxx

    F = wxx.functional
    x = F.from_numpy(rng.standard_normal((64, 64)).astype(np.float32))
    first = wxx.graph.capture(lambda t: F.pointwise(t, t, 0), x)
    held = [first.replay()]
    first.close()                       # the tensor outlives its graph

    def step(t):
        if wxx.graph.capturing():
            held.clear()                # its arena goes now, inside the capture
        return F.pointwise(F.pointwise(t, t, 2), t, 0)

    second = wxx.graph.capture(step, x)
    expect = x.numpy() ** 2 + x.numpy()
    assert np.array_equal(second.replay().numpy(), expect)
    second.close()
    again = F.pointwise(x, x, 0)        # and the library goes on
    assert np.array_equal(again.numpy(), 2 * x.numpy())
    assert wxx.backend.device_status() == 0
