"""Attention over a shared prefix and each sequence's own cache (``qutai_b200.kv_cache.prefix_attention``) against the softmax in
64 bits.  Needs a B200: ``-m gpu``.

Bars: every probability is rounded to bfloat16 (2^-9) before it meets its value, so the output is off by at most 2^-9 sum p |v|, and by
2^-9 of itself for its own rounding; a twentieth more for float32 sums and exponentials.  A score is a float32 sum of dim products: the
log-sum-exp is held to 1e-5 of the largest score's size."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def make(rng, batch, kv_heads, capacity, dim, dtype, lengths, garbage):
    """A cache of ``lengths``, with rubbish behind them, as storages and as 64-bit values."""
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache
    from qutai_b200.storage import DeviceStorage

    values, storages = {}, {}
    behind = np.arange(capacity)[None, :] >= np.asarray(lengths)[:, None]
    for name, size in (("k", 1.0), ("v", 0.5)):
        x = rng.standard_normal((batch, kv_heads, capacity, dim)) * size
        if dtype == "bfloat16":
            x[np.broadcast_to(behind[:, None, :, None], x.shape)] = garbage
            storages[name] = to_device(x, "bfloat16")
            values[name] = to_host(storages[name], x.shape)
        else:
            scale = (np.abs(x).max(-1) / 127).astype(np.float32)
            q = np.rint(x / scale[..., None]).astype(np.int8)
            scale[np.broadcast_to(behind[:, None], scale.shape)] = garbage
            storages[name] = DeviceStorage.from_bytes(q.tobytes(), "int8")
            storages[name + "_scale"] = to_device(scale, "float32")
            values[name] = q * scale[..., None].astype(np.float64)
    cache = KVCache(batch, capacity, kv_heads, dim, dtype, lengths=to_device(np.asarray(lengths), "int32"), longest=capacity, **storages)
    return cache, values


def check(batch, time, heads, kv_heads, dim, *, prefix, lengths, dtype="bfloat16", prefix_room=0, room=0, sharp=1.0, garbage=np.nan, seed=0):
    from gpu_util import to_device, to_host
    from qutai_b200 import lib
    from qutai_b200.kv_cache import prefix_attention
    from qutai_b200.layers import Tensor

    rng = np.random.default_rng(seed + (prefix or 0) + heads)
    q = rng.standard_normal((batch, time, heads * dim)) * sharp
    q = to_host(to_device(q, "bfloat16"), q.shape)
    capacity = max(max(lengths), 1) + room
    cache, own = make(rng, batch, kv_heads, capacity, dim, dtype, lengths, garbage)
    shared, held = None, None
    if prefix is not None:
        shared, held = make(rng, 1, kv_heads, max(prefix + prefix_room, 1), dim, dtype, [prefix], garbage)
    out, lse = prefix_attention(Tensor(to_device(q, "bfloat16"), q.shape), heads, cache, shared)
    again = prefix_attention(Tensor(to_device(q, "bfloat16"), q.shape), heads, cache, shared)
    assert lib.device_status() == 0
    assert out.tobytes() == again[0].tobytes() and lse.tobytes() == again[1].tobytes()
    out, lse = to_host(out, (batch, time, heads, dim)), to_host(lse, (batch, time, heads))
    group = heads // kv_heads
    for b in range(batch):
        for t in range(time):
            n = max(0, min(lengths[b], lengths[b] - time + t + 1))
            for g in range(kv_heads):
                k, v = (own[name][b, g, :n] for name in "kv")
                if prefix:
                    k, v = (np.concatenate((held[name][0, g, :prefix], x)) for name, x in (("k", k), ("v", v)))
                rows = slice(g * group, (g + 1) * group)
                if not len(k):
                    assert not out[b, t, rows].any() and np.all(np.isneginf(lse[b, t, rows]))
                    continue
                s = q[b, t].reshape(heads, dim)[rows] @ k.T / np.sqrt(dim)
                top = s.max(-1, keepdims=True)
                p = np.exp(s - top)
                total = p.sum(-1, keepdims=True)
                want, size = p @ v / total, p @ np.abs(v) / total
                bar = 2.0 ** -9 * 1.05 * (size + np.abs(want)) + 1e-6
                assert np.all(np.abs(out[b, t, rows] - want) <= bar), (b, t, g, np.max(np.abs(out[b, t, rows] - want) / bar))
                assert np.all(np.abs(lse[b, t, rows] - (top + np.log(total))[:, 0]) <= 1e-5 * (1 + np.abs(s).max()))


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads,kv_heads,prefix,lengths", [
    (1, 1, 1, 1, [1]), (1, 4, 1, 0, [1]), (2, 4, 2, 64, [1, 64]), (3, 8, 2, 65, [63, 0, 129]), (5, 6, 2, 1003, [1, 2, 3, 300, 17]),
    (17, 16, 4, 200, list(range(17))), (40, 8, 8, 511, [7] * 40), (33, 10, 2, 4100, [70] * 33), (4, 64, 2, 300, [5, 600, 1, 0])])
def test_one_new_position_a_sequence(batch, heads, kv_heads, prefix, lengths, dim, dtype):
    check(batch, 1, heads, kv_heads, dim, prefix=prefix, lengths=lengths, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("time,lengths,dim", [(2, [2, 1], 64), (5, [5, 300, 3, 64, 0], 128), (5, [70, 64, 65, 2], 64), (17, [17, 40], 64), (130, [130, 200], 128),
                                              (200, [150], 64)])
def test_several_new_positions_see_no_later_ones(time, lengths, dim, dtype):
    """Also with fewer positions held than there are queries: the first ones see nothing of their own sequence."""
    check(len(lengths), time, 4, 2, dim, prefix=100, lengths=lengths, dtype=dtype)
    check(len(lengths), time, 3, 1, dim, prefix=None, lengths=lengths, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("garbage", [np.nan, np.inf, 3.0e38])
def test_what_lies_behind_the_lengths_is_not_seen(garbage, dtype):
    check(3, 1, 4, 2, 64, prefix=130, prefix_room=200, lengths=[0, 65, 10], room=300, garbage=garbage, dtype=dtype)
    check(40, 1, 8, 2, 128, prefix=700, prefix_room=900, lengths=[3] * 40, room=70, garbage=garbage, dtype=dtype)
    check(2, 9, 16, 2, 64, prefix=0, prefix_room=64, lengths=[4, 30], room=130, garbage=garbage, dtype=dtype)


@pytest.mark.parametrize("batch", [1, 40])
def test_rows_that_see_nothing(batch):
    check(batch, 1, 4, 2, 64, prefix=0, lengths=[0] * batch)
    check(batch, 1, 4, 2, 64, prefix=None, lengths=[0] * (batch - 1) + [3])


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_sharp_scores(dtype):
    """Scores of some hundreds: nearly one key has all the weight, in the prefix or in the sequence's own part."""
    check(6, 1, 8, 2, 64, prefix=900, lengths=[300, 1, 0, 50, 200, 64], sharp=60.0, dtype=dtype)
    check(70, 1, 8, 2, 128, prefix=300, lengths=[30] * 70, sharp=60.0, dtype=dtype)


def test_a_new_cache_that_holds_nothing_yet():
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache, prefix_attention
    from qutai_b200.layers import Tensor

    cache = KVCache(3, 50, 2, 64)
    out, lse = prefix_attention(Tensor(to_device(np.ones((3, 1, 256)), "bfloat16"), (3, 1, 256)), 4, cache)
    assert not to_host(out).any() and np.all(np.isneginf(to_host(lse)))


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_offsets_beyond_32_bits(dtype):
    """A head whose first key lies more than 2^31 elements into the cache; the rest of the buffer is never touched."""
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache, prefix_attention
    from qutai_b200.layers import Tensor

    batch, kv_heads, capacity, dim = 3, 1, 11_200_000, 128
    cache = KVCache(batch, capacity, kv_heads, dim, dtype)
    start = capacity - 70
    cache.rewind(to_device(np.array([0, 0, start]), "int32"), start)
    rng = np.random.default_rng(0)
    x = rng.standard_normal((batch, 70, dim))
    new = Tensor(to_device(x, "bfloat16"), x.shape)
    cache.append(new, new, counts=to_device(np.array([0, 0, 70]), "int32"))
    back = to_host(cache.read(start, 70, dtype="float32")[0].storage, (batch, 70, dim))
    assert not back[:2].any() and np.abs(back[2] - x[2]).max() <= (0.02 if dtype == "bfloat16" else 0.02)
    # the last sequence alone, its first `start` positions left out: the same rows at the front of a small cache
    small = KVCache(1, 70, kv_heads, dim, dtype)
    row = Tensor(to_device(x[2:], "bfloat16"), (1, 70, dim))
    small.append(row, row)
    q = to_device(rng.standard_normal((1, 1, dim)), "bfloat16")
    want = to_host(prefix_attention(Tensor(q, (1, 1, dim)), 1, small)[0])
    places = (batch - 1) * kv_heads * capacity + start
    view = {name: getattr(cache, name).view(places * dim, 70 * dim) for name in "kv"}
    if dtype == "int8":
        view.update({name: getattr(cache, name).view(places, 70) for name in ("k_scale", "v_scale")})
    tail = KVCache(1, 70, kv_heads, dim, dtype, lengths=to_device(np.array([70]), "int32"), longest=70, **view)
    assert np.array_equal(to_host(prefix_attention(Tensor(q, (1, 1, dim)), 1, tail)[0]), want)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,time,heads,kv_heads,prefix", [(50, 1, 6, 2, 129), (33, 3, 5, 1, 640), (70, 1, 7, 7, 2000), (2, 40, 9, 3, 333), (1, 300, 2, 1, 128), (9, 1, 64, 1, 191),
                                                              (3, 1, 200, 1, 500), (300, 1, 4, 2, 1024)])
def test_rows_that_fill_tiles_over_a_prefix(batch, time, heads, kv_heads, prefix, dim, dtype):
    """Groups of heads that do not divide a tile of rows, new positions in several tiles, prefixes that end in and at blocks of keys."""
    rng = np.random.default_rng(prefix)
    check(batch, time, heads, kv_heads, dim, prefix=prefix, lengths=[int(n) for n in rng.integers(0, time + 70, batch)], dtype=dtype, prefix_room=40)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,time,heads,kv_heads,prefix,room", [
    (17, 1, 1, 1, 61700, 0), (4, 1, 32, 4, 8193, 0), (50, 1, 6, 2, 129, 3500), (33, 3, 5, 1, 2200, 0), (70, 1, 7, 7, 2171, 0), (2, 40, 9, 3, 333, 1300), (1, 300, 2, 1, 1800, 0),
    (9, 1, 64, 1, 128, 1800), (9, 1, 64, 1, 1951, 1), (3, 1, 128, 1, 2816, 0), (3, 1, 200, 1, 500, 2000), (600, 1, 4, 2, 511, 1), (40, 1, 8, 2, 0, 4000), (40, 1, 8, 2, 1, 4000)])
def test_long_prefixes(batch, time, heads, kv_heads, prefix, room, dim, dtype):
    """The same where the prefix is long for the number of rows, or could be, by what the host knows of it."""
    rng = np.random.default_rng(prefix)
    check(batch, time, heads, kv_heads, dim, prefix=prefix, lengths=[int(n) for n in rng.integers(0, time + 70, batch)], dtype=dtype, prefix_room=room)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("garbage", [np.nan, np.inf, 3.0e38])
def test_what_lies_behind_a_long_prefix_is_not_seen(garbage, dtype):
    check(40, 1, 8, 2, 128, prefix=700, prefix_room=3300, lengths=[3, 70, 0, 64] * 10, room=70, garbage=garbage, dtype=dtype)
    check(70, 1, 8, 1, 64, prefix=2300, prefix_room=50, lengths=[30] * 70, room=1, garbage=garbage, dtype=dtype, sharp=60.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("prefix,room", [(200, 0), (150, 800), (0, 700), (150, 7000), (0, 7000)])
def test_a_prefix_and_nothing_of_their_own(prefix, room, dtype):
    """A new cache: the prefix alone, in one part or several, and a prefix that holds nothing where there could be much."""
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache, prefix_attention
    from qutai_b200.layers import Tensor

    rng = np.random.default_rng(prefix)
    batch, heads, kv_heads, dim = 40, 4, 2, 64
    shared, held = make(rng, 1, kv_heads, prefix + room, dim, dtype, [prefix], np.nan)
    q = to_host(to_device(rng.standard_normal((batch, heads, dim)), "bfloat16"), (batch, heads, dim))
    out, lse = prefix_attention(Tensor(to_device(q, "bfloat16"), (batch, 1, heads * dim)), heads, KVCache(batch, 5, kv_heads, dim, dtype), shared)
    out, lse = to_host(out, q.shape), to_host(lse, (batch, heads))
    if not prefix:
        assert not out.any() and np.all(np.isneginf(lse))
        return
    for h in range(heads):
        k, v = (held[name][0, h // 2, :prefix] for name in "kv")
        s = q[:, h] @ k.T / 8
        p = np.exp(s - s.max(-1, keepdims=True))
        want, size = p @ v / p.sum(-1, keepdims=True), p @ np.abs(v) / p.sum(-1, keepdims=True)
        assert np.all(np.abs(out[:, h] - want) <= 2.0 ** -9 * 1.05 * (size + np.abs(want)) + 1e-6)
        assert np.all(np.abs(lse[:, h] - s.max(-1) - np.log(p.sum(-1))) <= 1e-5 * (1 + np.abs(s).max()))


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("batch", [24, 400])
def test_scores_that_grow_along_the_prefix(batch, dtype):
    """The maximum of a row rises by more than 2^8 from block to block: everything summed so far is rescaled each time."""
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache, prefix_attention
    from qutai_b200.layers import Tensor

    rng = np.random.default_rng(3)
    heads, dim, prefix = 4, 64, 700
    k = rng.standard_normal((1, prefix, dim)) * 0.3
    k[..., 0] = np.arange(prefix) * 2.0                 # scores up to 175 apart over the prefix, 16 from block to block
    v = rng.standard_normal((1, prefix, dim))
    shared, cache = KVCache(1, prefix, 1, dim, dtype), KVCache(batch, 4, 1, dim, dtype)
    shared.append(Tensor(to_device(k, "bfloat16"), k.shape), Tensor(to_device(v, "bfloat16"), v.shape))
    k, v = (to_host(x.storage, (prefix, dim)) for x in shared.read(0, prefix, dtype="float32"))
    q = rng.standard_normal((batch, heads, dim))
    q[..., 0] = 1.0
    q = to_host(to_device(q, "bfloat16"), q.shape)
    out, lse = prefix_attention(Tensor(to_device(q, "bfloat16"), (batch, 1, heads * dim)), heads, cache, shared)
    s = q @ k.T / 8
    p = np.exp(s - s.max(-1, keepdims=True))
    want, size = p @ v / p.sum(-1, keepdims=True), p @ np.abs(v) / p.sum(-1, keepdims=True)
    assert np.all(np.abs(to_host(out, q.shape) - want) <= 2.0 ** -9 * 1.05 * (size + np.abs(want)) + 1e-6)
    assert np.all(np.abs(to_host(lse, (batch, heads)) - s.max(-1) - np.log(p.sum(-1))) <= 1e-5 * (1 + np.abs(s).max()))


def test_another_stream_than_the_default_one():
    import ctypes

    from gpu_util import to_device
    from qutai_b200 import lib
    from qutai_b200.kv_cache import prefix_attention
    from qutai_b200.layers import Tensor

    rng = np.random.default_rng(8)
    cache, _ = make(rng, 80, 2, 30, 64, "bfloat16", [int(n) for n in rng.integers(0, 31, 80)], np.nan)
    shared, _ = make(rng, 1, 2, 300, 64, "bfloat16", [300], np.nan)
    q = Tensor(to_device(rng.standard_normal((80, 1, 256)), "bfloat16"), (80, 1, 256))
    want = [s.tobytes() for s in prefix_attention(q, 4, cache, shared)]
    stream = ctypes.c_uint64()
    lib.call("qmoe_stream_create", ctypes.byref(stream))
    got = prefix_attention(q, 4, cache, shared, stream=stream.value)
    lib.call("qmoe_stream_sync", stream.value)
    assert [s.tobytes() for s in got] == want
    lib.call("qmoe_stream_destroy", stream.value)
