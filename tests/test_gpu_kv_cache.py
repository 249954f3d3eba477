"""The key/value cache (``qutai_b200.kv_cache.KVCache``): what is appended comes back, quantised or not, where it belongs.  Needs a
B200: ``-m gpu``.

An 8-bit value is the nearest multiple of max |x| / 127, so half a scale bounds its error; the numbers themselves are whole and
are compared exactly with the same division in float32."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def rounded(a, dtype):
    from gpu_util import to_device, to_host

    return to_host(to_device(a, dtype), np.shape(a))


def given(a, dtype):
    from gpu_util import to_device
    from qutai_b200.layers import Tensor

    return Tensor(to_device(a, dtype), a.shape)


def int8_of(storage, shape):
    return np.frombuffer(storage.tobytes(), dtype=np.int8).reshape(shape)


def quantised(x):
    """x [..., dim] in float32 steps: numbers and scales"""
    x = x.astype(np.float32)
    scale = np.abs(x).max(-1) / np.float32(127)
    q = np.divide(x, scale[..., None], out=np.zeros_like(x), where=scale[..., None] > 0)
    return np.clip(np.rint(q), -127, 127), scale


@pytest.mark.parametrize("source", ["bfloat16", "float32"])
@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("batch,kv_heads,dim,times", [(1, 1, 64, [1]), (3, 2, 64, [5, 1, 130]), (64, 4, 64, [1, 1]), (2, 3, 128, [70, 33]),
                                                      (5, 1, 8, [2, 3]), (2, 2, 40, [9]), (1, 2, 256, [17])])
def test_what_is_appended_is_read_back(batch, kv_heads, dim, times, dtype, source):
    from gpu_util import to_host
    from qutai_b200.kv_cache import KVCache

    rng = np.random.default_rng(batch * dim)
    capacity = sum(times) + 3
    cache = KVCache(batch, capacity, kv_heads, dim, dtype)
    held = {name: [] for name in "kv"}
    for time in times:
        new = {name: rounded(rng.standard_normal((batch, time, kv_heads, dim)) * np.exp(rng.standard_normal((batch, time, kv_heads, 1))), source) for name in "kv"}
        cache.append(*(given(new[name].reshape(batch, time, -1), source) for name in "kv"))
        for name in "kv":
            held[name].append(new[name])
    total = sum(times)
    assert cache.longest == total and to_host(cache.lengths).tolist() == [total] * batch
    for name, read in zip("kv", cache.read(0, capacity, dtype="float32")):
        x, got = np.concatenate(held[name], 1), to_host(read.storage, (batch, capacity, kv_heads, dim))
        assert not got[:, total:].any()                 # whatever lies behind the length
        if dtype == "bfloat16":
            assert np.array_equal(got[:, :total], rounded(x, "bfloat16"))
            continue
        q, scale = quantised(x)
        stored = int8_of(getattr(cache, name), (batch, kv_heads, capacity, dim))[:, :, :total].transpose(0, 2, 1, 3)
        assert np.array_equal(stored, q)
        assert np.array_equal(to_host(getattr(cache, name + "_scale"), (batch, kv_heads, capacity))[:, :, :total].transpose(0, 2, 1), scale)
        assert np.array_equal(got[:, :total], (q.astype(np.float32) * scale[..., None]).astype(np.float64))
        assert np.all(np.abs(got[:, :total] - x) <= 0.5001 * scale[..., None])
    part = cache.read(1, total, dtype="bfloat16")[0]
    whole = to_host(cache.read(0, capacity, dtype="bfloat16")[0].storage, (batch, capacity, -1))
    assert np.array_equal(to_host(part.storage, (batch, total, -1)), whole[:, 1:total + 1])


@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
def test_sequences_of_different_lengths_and_a_rewind(dtype):
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache

    rng = np.random.default_rng(1)
    batch, time, width = 4, 6, 128
    cache = KVCache(batch, 20, 2, 64, dtype)
    counts = np.array([0, 6, 3, 99])                    # more than there are rows: all of them
    first, second = (rounded(rng.standard_normal((batch, time, width)), "bfloat16") for _ in range(2))
    cache.append(given(first, "bfloat16"), given(first, "bfloat16"), counts=to_device(counts, "int32"))
    kept, longest = cache.lengths, cache.longest
    assert to_host(cache.lengths).tolist() == [0, 6, 3, 6] and longest == 6
    cache.append(given(second, "bfloat16"), given(second, "bfloat16"))
    assert to_host(cache.lengths).tolist() == [6, 12, 9, 12] and cache.longest == 12
    reference = KVCache(1, 40, 2, 64, dtype)
    for b, n in enumerate([0, 6, 3, 6]):
        reference.rewind(to_device([0], "int32"), 0)
        whole = np.concatenate((first[b, :n], second[b]))[None]
        reference.append(given(whole, "bfloat16"), given(whole, "bfloat16"))
        for mine, other in zip(cache.read(0, n + 6), reference.read(0, n + 6)):
            assert np.array_equal(to_host(mine.storage, (batch, -1))[b], to_host(other.storage))
    cache.rewind(kept, longest)
    assert not to_host(cache.read(0, 12)[0].storage, (batch, 12, width))[0].any()
    assert np.array_equal(to_host(cache.lengths), [0, 6, 3, 6])


def test_nothing_appended_and_values_that_need_care():
    from gpu_util import to_host
    from qutai_b200.kv_cache import KVCache
    from qutai_b200.layers import Tensor
    from qutai_b200.storage import DeviceStorage

    cache = KVCache(2, 8, 1, 64, "int8")
    none = Tensor(DeviceStorage(0, "bfloat16"), (2, 0, 64))
    cache.append(none, none)
    assert cache.longest == 0 and not to_host(cache.lengths).any()
    x = np.zeros((2, 4, 64), dtype=np.float32)
    x[0, 1] = 1e-44                                     # below what a scale can express: zeros
    x[0, 2, 5] = np.inf
    x[0, 3, 7] = np.nan
    x[1, 1] = 3.0e38
    x[1, 2] = np.linspace(-127, 127, 64)
    cache.append(given(x, "float32"), given(x, "float32"))
    got = to_host(cache.read(0, 4, dtype="float32")[0].storage, (2, 4, 64))
    assert not got[0, 0].any() and not got[1, 0].any() and np.abs(got[0, 1]).max() <= 1.1e-44
    assert np.isnan(got[0, 2]).all() and np.isnan(got[0, 3]).all()      # not silently numbers
    assert np.allclose(got[1, 1], 3.0e38, rtol=1e-6) and np.abs(got[1, 2] - x[1, 2]).max() <= 0.5001


def test_columns_of_one_projection():
    from gpu_util import to_host
    from qutai_b200.kv_cache import KVCache
    from qutai_b200.rotary import Columns

    rng = np.random.default_rng(2)
    fused = rounded(rng.standard_normal((3, 5, 256 + 128)), "bfloat16")
    tensor = given(fused, "bfloat16")
    cache = KVCache(3, 5, 2, 64)
    cache.append(Columns(tensor, 128, 128), Columns(tensor, 256, 128))
    for read, start in zip(cache.read(0, 5), (128, 256)):
        assert np.array_equal(to_host(read.storage, (3, 5, 128)), fused[..., start:start + 128])
