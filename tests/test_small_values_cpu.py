"""The bound that attention over small int8 values is held to refuses what is wrong there."""
import numpy as np
import pytest

from . import small_values
from . import verify_ref as ref
from .test_attention_gpu import Step


@pytest.mark.parametrize("value_scale", [1e-2, 1e-3, 1e-4, 1e-5])
def test_the_bound_sees_small_values(value_scale):
    s = small_values.step(Step, 1, 2, 1, 64, [(2, 4000)], value_scale)
    w = s.want()
    want, lse = w[:2]
    assert np.all(w[4] < 1.2), "one key leads"
    assert small_values.close(s, want, lse, w) == 0.0
    b, _ = small_values.bound(s, *w)
    assert np.all(b < 2.0 ** -7 * np.abs(want)), float(np.max(b / np.abs(want)))
    for wrong in (np.zeros_like(want), want * 1.02, want * 0.98):
        with pytest.raises(AssertionError):
            small_values.close(s, wrong, lse, w)
    small_values.close(s, want.astype(np.float16), lse, w)


def lost(s, w, lift):
    """What rounding lift * p * scale to f16 leaves of the result (the reference at the largest p), the sums in 64 bits."""
    rows, q = ref.rows_of(s.cache), s.q.astype(np.float64)
    out = np.zeros_like(w[0])
    for b, n in enumerate(s.lengths):
        pos = np.arange(n)
        page, slot = s.table[b, pos // s.page], pos % s.page
        for t in range(s.starts[b], s.starts[b + 1]):
            keep = n - (s.starts[b + 1] - s.starts[b]) + (t - s.starts[b]) + 1
            for h in range(s.heads):
                g = h * s.kv_heads // s.heads
                x = rows[page, slot, 0, g][:keep] @ q[t, h] * s.scale
                p = np.exp(x - x.max())
                sv = s.cache[1][page, g, slot, 1][:keep].astype(np.float64)
                out[t, h] = (lift * p * sv).astype(np.float16).astype(np.float64) @ s.cache[0][page, g, slot, 1][:keep] / (lift * p.sum())
    return out


@pytest.mark.parametrize("value_scale", [1e-3, 1e-4, 1e-5])
def test_a_lift_that_knows_nothing_of_the_values_is_seen(value_scale):
    """Probabilities times the scale, lifted by 16: f16's small numbers, refused. Lifted to where their products need it: taken."""
    s = small_values.step(Step, 2, 1, 1, 64, [(1, 4000)], value_scale)
    w = s.want()
    with pytest.raises(AssertionError):
        small_values.close(s, lost(s, w, 16.0), w[1], w)
    small_values.close(s, lost(s, w, 512.0 * 64 / value_scale), w[1], w)
