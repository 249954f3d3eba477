"""How exact attention over a shared prefix and own caches is (``qutai_b200.kv_cache.prefix_attention``), and that its offsets hold 64 bits.  Needs
a B200: ``-m gpu``.

Bars.  A row's weight lies on a few keys only, the others' scores being 60 below: what is off is then
  the output's own rounding to bfloat16, half of a unit in its eighth bit: 2^-8 of it;
  a probability, cut into two bfloat16 numbers: the first, cut off, leaves less than 2^-7 of the power of two below it, the second holds that in units of
    2^-15 or finer, half of which is lost: 2^-16 of it;
  a score, a float32 sum of dim products and its rounded exponent: e = (dim + 8) 2^-24 sum |q k| / sqrt(dim), which moves output and weights by 2 e;
  the exponential, 2^-22, and float32 sums of at most n / 16 steps on two chains, 2^-22 n / 16, n the number of keys;
  a hundredth more for the rounding of what these are off by.
With every probability in ONE bfloat16 number, off by up to 2^-8 of it, the bar is not met: shown on the host."""
import numpy as np
import pytest

SHAPES = [(2, 1, 4, 2, 40, [9, 30]), (40, 1, 4, 2, 200, [20] * 40), (3, 7, 6, 2, 130, [40, 9, 70]), (64, 1, 8, 2, 2000, [30] * 64), (40, 1, 16, 4, 700, [0] * 40)]


def make_case(rng, batch, time, heads, kv_heads, prefix, lengths, dim, rounded):
    """Queries and keys in which one key of ten, and one at the very front, counts."""
    q = rounded(rng.standard_normal((batch, time, heads, dim)))
    q[..., 0] = 8.0
    data = {}
    for name, count, held in (("prefix", 1, prefix), ("own", batch, max(max(lengths), 1))):
        k, v = rng.standard_normal((count, kv_heads, held, dim)), rng.standard_normal((count, kv_heads, held, dim))
        far = rng.random((count, kv_heads, held)) > 4.0 / max(held, 8)
        far[:, :, 0] = False
        k[..., 0] = np.where(far, -7.5 * np.sqrt(dim), 0.0)
        data[name] = rounded(k), rounded(v)
    return q, data


def rows_of(q, data, lengths, prefix, b, t, g, group, time):
    n = max(0, min(lengths[b], lengths[b] - time + t + 1))
    k, v = (np.concatenate((shared[0, g, :prefix], own[b, g, :n])) for shared, own in zip(data["prefix"], data["own"]))
    return q[b, t, g * group:(g + 1) * group], k, v


def bf16(x):
    bits = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return (((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16 << 16).astype(np.uint32)).view(np.float32).astype(np.float64)


def formula(q, k, v, one_number=False):
    """The output in 64 bits and its bar; ``one_number``: with every probability rounded to bfloat16, a mistake."""
    dim, n = q.shape[-1], len(k)
    s = q @ k.T / np.sqrt(dim)
    p = np.exp(s - s.max(-1, keepdims=True))
    total = p.sum(-1, keepdims=True)
    weight = p / total
    e = ((dim + 8) * 2.0 ** -24 * (np.abs(q) @ np.abs(k).T / np.sqrt(dim)) * (weight > 1e-12)).max(-1, keepdims=True)
    want, size = weight @ v, weight @ np.abs(v)
    bar = 2.0 ** -8 * np.abs(want) + 1.01 * (2.0 ** -16 + 2 * e + 2.0 ** -22 * (1 + n / 16)) * size
    return (bf16((bf16(p) if one_number else p) @ v / total) if one_number else want), want, bar


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,time,heads,kv_heads,prefix,lengths", SHAPES)
def test_the_bar_tells_one_number_from_two(batch, time, heads, kv_heads, prefix, lengths, dim):
    q, data = make_case(np.random.default_rng(prefix), batch, time, heads, kv_heads, prefix, lengths, dim, bf16)
    worst = 0.0
    for b in range(batch):
        for g in range(kv_heads):
            got, want, bar = formula(*rows_of(q, data, lengths, prefix, b, time - 1, g, heads // kv_heads, time), one_number=True)
            worst = max(worst, (np.abs(got - want) / bar).max())
    assert worst > 1.5


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("batch,time,heads,kv_heads,prefix,lengths", SHAPES)
def test_probabilities_keep_sixteen_bits(batch, time, heads, kv_heads, prefix, lengths, dim, dtype):
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache, prefix_attention
    from qutai_b200.layers import Tensor

    q, data = make_case(np.random.default_rng(prefix), batch, time, heads, kv_heads, prefix, lengths, dim, bf16)
    caches, held = {}, {}
    for name, count, long in (("prefix", 1, [prefix]), ("own", batch, lengths)):
        k, v = data[name]
        capacity = k.shape[2]
        caches[name] = KVCache(count, capacity, kv_heads, dim, dtype)
        flat = lambda x: x.transpose(0, 2, 1, 3).reshape(count, capacity, -1)  # noqa: E731
        given = [Tensor(to_device(flat(x), "bfloat16"), (count, capacity, kv_heads * dim)) for x in (k, v)]
        caches[name].append(*given, counts=to_device(np.asarray(long), "int32"))
        back = [to_host(x.storage, (count, capacity, kv_heads, dim)).transpose(0, 2, 1, 3) for x in caches[name].read(0, capacity, dtype="float32")]
        held[name] = back
    caches["own"].rewind(caches["own"].lengths, max(lengths))
    out, _ = prefix_attention(Tensor(to_device(q, "bfloat16"), (batch, time, heads * dim)), heads, caches["own"], caches["prefix"])
    out = to_host(out, q.shape)
    group = heads // kv_heads
    for b in range(batch):
        for t in range(time):
            for g in range(kv_heads):
                want, _, bar = formula(*rows_of(q, held, lengths, prefix, b, t, g, group, time))
                error = np.abs(out[b, t, g * group:(g + 1) * group] - want)
                assert np.all(error <= bar), (b, t, g, (error / bar).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "int8"])
@pytest.mark.parametrize("where", ["own", "prefix", "prefix by tensor memory"])
def test_attention_reads_beyond_32_bits(where, dtype):
    """The last head's (the last sequence's) keys lie more than 2^31 elements into the cache that the kernel is given: the same bits as from a
    small cache with the same keys."""
    from gpu_util import to_device, to_host
    from qutai_b200.kv_cache import KVCache, prefix_attention
    from qutai_b200.layers import Tensor

    rng = np.random.default_rng(0)
    dim, rows = 128, 70
    batch, kv_heads, capacity = (3, 1, 11_200_000) if where == "own" else (1, 2, 17_000_000)
    count = {"own": rows, "prefix": 300, "prefix by tensor memory": 1500}[where]
    x = rng.standard_normal((batch, count, kv_heads * dim))
    new = Tensor(to_device(x, "bfloat16"), x.shape)
    results = []
    for room in (capacity, count + 5):
        held = KVCache(batch, room, kv_heads, dim, dtype)
        held.append(new, new)
        if where == "own":
            q = Tensor(to_device(np.random.default_rng(1).standard_normal((batch, 1, 2 * dim)), "bfloat16"), (batch, 1, 2 * dim))
            results.append([s.tobytes() for s in prefix_attention(q, 2, held)])
        else:
            queries = 40 if where == "prefix" else 128
            own = KVCache(queries, 5, kv_heads, dim, dtype)
            q = Tensor(to_device(np.random.default_rng(1).standard_normal((queries, 1, 4 * dim)), "bfloat16"), (queries, 1, 4 * dim))
            results.append([s.tobytes() for s in prefix_attention(q, 4, own, held)])
        del held
    assert results[0] == results[1]
    last = np.frombuffer(results[0][1], dtype=np.float32)
    assert np.isfinite(last).all()
