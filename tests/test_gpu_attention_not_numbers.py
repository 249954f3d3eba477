"""Queries and keys that are no numbers, in attention over a shared prefix and own caches (``qutai_b200.kv_cache.prefix_attention``), by every
form it takes and however many parts a row is cut into: a row that meets a NaN is NaN in all its values and in its log-sum-exp, every
other row has the bits it has without.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# (batch, time, heads, kv_heads, prefix, lengths): one part and several, rows that share a tile and rows that fill it, joined by a warp and by
# eight, on the tensor cores with one launch and with two
SHAPES = [(2, 1, 4, 2, 0, [30, 5]), (2, 1, 4, 2, 300, [30, 5]), (1, 1, 2, 1, 9000, [40]), (40, 1, 4, 2, 130, [0] * 40), (40, 1, 4, 2, 700, [20] * 40),
          (3, 7, 6, 2, 200, [40, 9, 70]), (40, 1, 8, 2, 4096, [90] * 40), (300, 1, 4, 1, 2048, [150] * 300)]


def run(q, heads, cache, shared):
    from gpu_util import to_device, to_host
    from qutai_b200 import lib
    from qutai_b200.kv_cache import prefix_attention
    from qutai_b200.layers import Tensor

    out, lse = prefix_attention(Tensor(to_device(q, "bfloat16"), q.shape), heads, cache, shared)
    assert lib.device_status() == 0
    return to_host(out, (*q.shape[:2], heads, -1)), to_host(lse, (*q.shape[:2], heads))


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("batch,time,heads,kv_heads,prefix,lengths", SHAPES)
def test_queries_that_are_no_numbers(batch, time, heads, kv_heads, prefix, lengths, value, dim, dtype):
    """An infinite element of a query gives scores of both signs, whose softmax is none either."""
    from test_gpu_prefix_attention import make

    rng = np.random.default_rng(prefix)
    cache, _ = make(rng, batch, kv_heads, max(lengths) or 1, dim, dtype, lengths, 0.0)
    if not max(lengths):
        cache.rewind(cache.lengths, 0)
    shared = make(rng, 1, kv_heads, prefix, dim, dtype, [prefix], 0.0)[0] if prefix else None
    q = rng.standard_normal((batch, time, heads * dim))
    plain, plain_lse = run(q, heads, cache, shared)
    marked = np.zeros((batch, time, heads), dtype=bool)
    marked[-1, -1, heads - 1] = marked[0, -1, 0] = True
    if value == np.inf:
        marked[np.asarray(lengths) + prefix < 4] = False
    q.reshape(batch, time, heads, dim)[marked, 3] = value
    out, lse = run(q, heads, cache, shared)
    assert np.isnan(out[marked]).all() and np.isnan(lse[marked]).all()
    assert np.array_equal(out[~marked], plain[~marked]) and np.array_equal(lse[~marked], plain_lse[~marked])


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("batch,time,heads,kv_heads,prefix,lengths", SHAPES)
def test_keys_that_are_no_numbers(batch, time, heads, kv_heads, prefix, lengths, where, dtype):
    """A NaN key (of 8 bits: a NaN scale) of one head takes the rows of that head that see it, and no others."""
    from gpu_util import to_device, to_host
    from test_gpu_prefix_attention import make

    if not (prefix if where == "prefix" else lengths[0]):
        pytest.skip("holds nothing")
    rng = np.random.default_rng(prefix)
    cache, _ = make(rng, batch, kv_heads, max(lengths) or 1, 64, dtype, lengths, 0.0)
    if not max(lengths):
        cache.rewind(cache.lengths, 0)
    shared = make(rng, 1, kv_heads, prefix, 64, dtype, [prefix], 0.0)[0] if prefix else None
    q = rng.standard_normal((batch, time, heads * 64))
    plain, plain_lse = run(q, heads, cache, shared)
    holder = shared if where == "prefix" else cache
    storage = holder.k if dtype == "bfloat16" else holder.k_scale
    values = to_host(storage).reshape(holder.batch, kv_heads, holder.capacity, -1)
    values[0, kv_heads - 1, 2 if where == "prefix" else 0, 0] = np.nan
    storage.copy_from(to_device(values.reshape(-1), storage.dtype))
    out, lse = run(q, heads, cache, shared)
    marked = np.zeros((batch, time, heads), dtype=bool)
    group = heads // kv_heads
    marked[:, :, (kv_heads - 1) * group:] = True
    if where == "own":
        marked[1:] = False
        marked[0, :max(0, time - lengths[0])] = False
    assert np.isnan(out[marked]).all() and np.isnan(lse[marked]).all()
    assert np.array_equal(out[~marked], plain[~marked]) and np.array_equal(lse[~marked], plain_lse[~marked])
