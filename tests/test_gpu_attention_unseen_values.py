"""Values that a query does not see, in attention with several new positions a sequence (``qutai_b200.kv_cache.prefix_attention``): a NaN or an
infinity at a later position leaves the queries before it alone.  Needs a B200: ``-m gpu``.

Bar of the numbers: as in the test of the operator, 2^-9 * 1.05 of sum p |v| and of the output."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("time,heads,kv_heads,prefix,lengths", [(2, 2, 1, 0, [2, 64]), (5, 6, 2, 100, [5, 66, 131]), (4, 4, 1, 0, [70, 3]), (9, 16, 2, 640, [9, 300]),
                                                                (70, 2, 1, 30, [200, 70]), (150, 3, 1, 0, [150, 100])])
def test_later_values_are_not_seen(time, heads, kv_heads, prefix, lengths, value, dim, dtype):
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import prefix_attention
    from qutai_b200.layers import Tensor
    from test_gpu_prefix_attention import make

    if dtype == "int8" and value == -np.inf:
        pytest.skip("a scale is not negative")
    rng = np.random.default_rng(time + dim)
    batch, group = len(lengths), heads // kv_heads
    cache, own = make(rng, batch, kv_heads, max(lengths), dim, dtype, lengths, 0.0)
    shared, held = make(rng, 1, kv_heads, prefix, dim, dtype, [prefix], 0.0) if prefix else (None, None)
    # the last position of every sequence and one in the middle of the new ones; of bfloat16 three elements, of 8 bits the scale of them all
    storage = cache.v if dtype == "bfloat16" else cache.v_scale
    raw = to_host(storage).reshape(batch, kv_heads, cache.capacity, -1)
    for b, n in enumerate(lengths):
        for at in {n - 1, max(0, n - 1 - time // 2)}:
            columns = [0, dim // 2 + 1, dim - 1] if dtype == "bfloat16" else slice(None)
            own["v"][b, :, at, columns] = value
            raw[b, :, at, columns] = value
    storage.copy_from(to_device(raw.reshape(-1), storage.dtype))
    q = to_host(to_device(rng.standard_normal((batch, time, heads * dim)), "bfloat16"), (batch, time, heads, dim))
    out, lse = prefix_attention(Tensor(to_device(q, "bfloat16"), (batch, time, heads * dim)), heads, cache, shared)
    out, lse = to_host(out, q.shape), to_host(lse, (batch, time, heads))
    for b in range(batch):
        for t in range(time):
            n = max(0, min(lengths[b], lengths[b] - time + t + 1))
            for g in range(kv_heads):
                k, v = (own[name][b, g, :n] for name in "kv")
                if prefix:
                    k, v = (np.concatenate((held[name][0, g, :prefix], x)) for name, x in (("k", k), ("v", v)))
                rows = slice(g * group, (g + 1) * group)
                got = out[b, t, rows]
                if not len(k):
                    assert not got.any() and np.all(np.isneginf(lse[b, t, rows]))
                    continue
                s = q[b, t, rows] @ k.T / np.sqrt(dim)
                top = s.max(-1, keepdims=True)
                p = np.exp(s - top)
                total = p.sum(-1, keepdims=True)
                assert np.all(np.abs(lse[b, t, rows] - (top + np.log(total))[:, 0]) <= 1e-5 * (1 + np.abs(s).max()))
                seen = ~np.isfinite(v).all(0)                                    # columns with a value that is none
                assert not np.isfinite(got[:, seen]).any()
                clean = np.where(seen, 0.0, v)
                want, size = p @ clean / total, p @ np.abs(clean) / total
                error, bar = np.abs(got - want), 2.0 ** -9 * 1.05 * (size + np.abs(want)) + 1e-6
                assert np.all(error[:, ~seen] <= bar[:, ~seen]), (b, t, g)
