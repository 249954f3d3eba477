"""Packed attention where the scores of a row's first keys are beyond float32's range, minus infinity, and those behind them are numbers: the softmax over the
later keys, forward and backward.  Needs a B200: ``-m gpu``.  Bars: those of ``test_gpu_packed_attention``, of the later positions as a sequence of their own
(the weights of the others are exp(-1e38), 0 in float32 as in 64 bits)."""
import numpy as np
import pytest

from test_gpu_packed_attention import make, rounded, run, whole

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hidden", [63, 64, 65, 128, 150])
@pytest.mark.parametrize("level", [-1600.0, -200.0, 0.0, 900.0])
def test_first_keys_at_minus_infinity(dim, hidden, level):
    """Column 0 of the queries is 2^70; that of the first ``hidden`` keys is -2^70, so their scores overflow, that of the others such that a score is ``level`` and the rest's."""
    lengths, heads, kv_heads, at = [70, 333], 4, 2, 70
    arrays = make(np.random.default_rng(hidden + dim), sum(lengths), heads, kv_heads, dim)
    q, k = arrays[0].reshape(-1, heads, dim), arrays[1].reshape(-1, kv_heads, dim)
    q[at:, :, 0] = 2.0 ** 70
    k[at:at + hidden, :, 0] = -2.0 ** 70
    k[at + hidden:, :, 0] = rounded(np.full((333 - hidden, kv_heads), level * 2.0 ** -70))
    got = run(arrays, lengths, heads, kv_heads, dim)
    later = at + hidden
    want = whole([a[later:] for a in arrays], [333 - hidden], heads, kv_heads, dim, dim ** -0.5)
    for name, x, (y, bar) in zip(("out", "lse", "dq", "dk", "dv"), got, want):
        assert np.all(np.abs(x[later:] - y) <= bar + 1e-30), (name, np.max(np.abs(x[later:] - y) / (bar + 1e-30)))
    assert np.all(got[1][at:later] == -np.inf) and np.isnan(got[0][at:later]).all()      # nothing but minus infinity: 0 / 0, as in the formula
    alone = run([a[:at] for a in arrays], [at], heads, kv_heads, dim)
    for x, y, (_, bar) in zip(got, alone, whole([a[:at] for a in arrays], [at], heads, kv_heads, dim, dim ** -0.5)):
        assert np.all(np.abs(x[:at] - y) <= 2 * bar)
