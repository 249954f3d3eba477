"""Sampling (``qutai_b200.sampling.sample``) against a plain implementation on the host.  Needs a B200: ``-m gpu``.

Tokens are compared exactly.  The host forms weights from float64 exponentials of the same float32 arguments and rounds them to whole numbers of
2^-31; a weight that rounds the other way moves a running sum by 2^-31 of the largest weight, so a different token would take a
uniform number within about 1e-7 of a boundary.  Log-probabilities: float32 rounding of the argument and of the result, 1e-6 of their size + 1."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ONE = 2.0 ** 31


def plain(logits, uniform, temperature, top_k, top_p, min_p):
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float32) + np.float32(0)
    largest = x.max()
    if largest == -np.inf:
        return -1, -np.inf
    greedy = not temperature > 0
    with np.errstate(all="ignore"):
        inverse = np.float32(1) if greedy else np.float32(1) / np.float32(temperature)
        z = np.where(x == largest, np.float32(0), (x - largest) * inverse)
        z = np.where(np.isneginf(x - largest), -np.inf, z)
        weight = np.exp(z.astype(np.float64))
    mass = np.rint(weight * ONE)
    order = np.argsort(-x, kind="stable")
    if greedy:
        order = order[:1]
    elif 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        before = np.cumsum(mass[order]) - mass[order]
        order = order[(before == 0) | (before < float(np.float32(top_p)) * mass[order].sum())]
    order = np.sort(order[weight[order].astype(np.float32) >= np.float32(min(min_p, 1))])
    running = np.cumsum(mass[order])
    target = min(np.floor(float(np.float32(uniform)) * running[-1]), running[-1] - 1)
    token = order[np.searchsorted(running, target, side="right")]
    return int(token), z[token] - np.log(mass.sum() / ONE)


def check(logits, uniforms, dtype="float32", **settings):
    from gpu_util import to_device, to_host
    from qutai_b200.layers import Tensor
    from qutai_b200.sampling import sample

    rows = len(logits)
    storage = to_device(logits, dtype)
    logits = to_host(storage, logits.shape)
    arguments, each = {}, {}
    for name, default in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
        value = settings.get(name, default)
        each[name] = np.broadcast_to(value, rows)
        arguments[name] = to_device(np.asarray(value), "int32" if name == "top_k" else "float32") if np.ndim(value) else value
    tokens, log_probs = sample(Tensor(storage, logits.shape), to_device(uniforms, "float32"), **arguments)
    tokens, log_probs = to_host(tokens), to_host(log_probs)
    for n in range(rows):
        token, log_prob = plain(logits[n], uniforms[n], *(each[name][n] for name in ("temperature", "top_k", "top_p", "min_p")))
        assert tokens[n] == token, (n, {name: each[name][n] for name in each})
        assert log_probs[n] == log_prob or abs(log_probs[n] - log_prob) <= 1e-6 * (1 + abs(log_prob)), n
    return tokens


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 31), (5, 1000), (64, 4099), (2, 32000), (3, 131071), (300, 260)])
@pytest.mark.parametrize("settings", [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
                                      dict(temperature=1.3, top_k=50, top_p=0.95, min_p=0.02), dict(temperature=0.8, top_k=700, top_p=0.5)])
def test_tokens_and_log_probabilities(rows, vocab, settings, dtype):
    rng = np.random.default_rng(rows * vocab)
    check(rng.standard_normal((rows, vocab)) * 2.5, rng.random(rows), dtype, **settings)


def test_every_row_with_settings_of_its_own():
    rng = np.random.default_rng(9)
    rows = 96
    check(rng.standard_normal((rows, 3001)) * 3, rng.random(rows), "bfloat16", temperature=rng.choice([0.0, 0.2, 0.9, 1.5], rows),
          top_k=rng.choice([0, 1, 7, 300, 3000, 3001, 5000], rows), top_p=rng.choice([1.0, 0.3, 0.9, 1e-9], rows), min_p=rng.choice([0.0, 0.01, 0.6, 1.0, 3.0], rows))


@pytest.mark.parametrize("vocab", [1, 7, 1024, 40000, 140001])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=3), dict(top_p=0.5), dict(top_k=30000, top_p=0.7), dict(top_p=1e-6), dict(temperature=0.0)])
def test_equal_logits_go_by_their_index(vocab, settings):
    uniforms = np.array([0.0, 0.2, 0.5, 0.999999])
    tokens = check(np.full((4, vocab), -3.25), uniforms, **settings)
    kept = vocab
    if settings.get("top_k"):
        kept = min(kept, settings["top_k"])
    if settings.get("top_p"):
        kept = max(1, int(np.ceil(kept * float(np.float32(settings["top_p"])))))
    if "temperature" in settings:
        kept = 1
    assert tokens.max() < kept and tokens[0] == 0
    # two levels, the boundary among many equal ones of either
    levels = np.where(np.arange(vocab) % 3 == 1, 1.0, 0.0)[None].repeat(4, 0)
    check(levels, uniforms, **settings)


def test_infinities_and_numbers_that_are_none():
    inf, nan, low = np.inf, np.nan, -3.4028235e38
    rows = np.array([[-inf, -inf, -inf, -inf], [nan, nan, nan, nan], [-inf, nan, 2.0, -inf], [1.0, inf, 0.0, inf], [low, low, low, low], [low, 3.0e38, -inf, 2.9e38],
                     [0.0, -0.0, 0.0, -0.0], [-inf, -inf, -inf, 5.0]])
    for uniform in (0.0, 0.6, 0.99):
        for settings in (dict(), dict(top_k=2), dict(top_p=0.5), dict(temperature=0.0), dict(min_p=0.5), dict(temperature=1e-30), dict(temperature=np.inf),
                         dict(temperature=1e-42, top_k=2, top_p=0.9)):
            check(rows, np.full(len(rows), uniform), **settings)


def test_masked_tokens_are_never_drawn():
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((200, 5003))
    logits[:, rng.random(5003) < 0.9] = -np.inf
    tokens = check(logits, rng.random(200), top_k=600, top_p=0.99)
    assert np.isfinite(logits[np.arange(200), tokens]).all()


def test_uniform_numbers_draw_by_the_weights():
    """Equally spaced numbers take every token as often as its weight says, to one draw."""
    logits = np.log(np.array([1.0, 2.0, 3.0, 4.0]))[None].repeat(1000, 0)
    tokens = check(logits, (np.arange(1000) + 0.5) / 1000)
    assert np.abs(np.bincount(tokens, minlength=4) - [100, 200, 300, 400]).max() <= 1


def test_a_wide_spread_and_a_narrow_one():
    rng = np.random.default_rng(6)
    check(rng.standard_normal((8, 50021)) * 40, rng.random(8), top_p=0.999)
    check(rng.standard_normal((8, 50021)) * 1e-3, rng.random(8), top_p=0.6, top_k=40000)
    check(1000 + rng.standard_normal((8, 50021)) * 1e-4, rng.random(8), "float32", top_p=0.3)
    spikes = rng.standard_normal((8, 50021)) * 0.01
    spikes[:, 777] = 30.0
    check(spikes, rng.random(8), "bfloat16", top_p=0.9)


def test_no_rows():
    from qutai_b200.layers import Tensor
    from qutai_b200.sampling import sample
    from qutai_b200.storage import DeviceStorage

    tokens, log_probs = sample(Tensor(DeviceStorage(0, "float32"), (0, 50)), DeviceStorage(0, "float32"))
    assert tokens.size == 0 and log_probs.size == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [700001, 1999999])
def test_vocabularies_that_no_shared_memory_holds(vocab, dtype):
    rng = np.random.default_rng(8)
    check(rng.standard_normal((2, vocab)), rng.random(2), dtype, top_p=0.8, top_k=vocab - 5)
    check(rng.standard_normal((2, vocab)) * 4, rng.random(2), dtype, top_k=100)
    check(np.zeros((1, vocab)), rng.random(1), dtype, top_p=0.5)


def test_more_tokens_than_there_are_with_any_weight():
    """Half of the row masked, or too small to weigh anything: top-k beyond the rest takes all of it."""
    rng = np.random.default_rng(10)
    logits = rng.standard_normal((4, 3000))
    logits[:, ::2] = -np.inf
    logits[2:, 1::4] = -200.0
    check(logits, rng.random(4), top_k=2000, top_p=0.9)
    check(logits, rng.random(4), top_k=2000)


@pytest.mark.parametrize("top_k", [300, 600, 1500, 2040, 2060, 6000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_lists_of_every_length(top_k, dtype):
    """The candidates in one comparison, in a histogram of their own, in the row's: the same tokens by the same rule."""
    rng = np.random.default_rng(top_k)
    logits = rng.standard_normal((6, 20011)) * 2.0
    logits[3:] = np.round(logits[3:] * 2) / 2           # few levels, every one many times
    check(logits, rng.random(6), dtype, top_k=top_k)
    check(logits, rng.random(6), dtype, top_k=top_k, top_p=0.7, temperature=0.9, min_p=0.01)


@pytest.mark.parametrize("settings", [{"top_k": 600}, {"top_k": 2040, "top_p": 0.7}, {"top_p": 0.9}, {"top_k": 6000, "top_p": 0.8, "min_p": 0.01}, {"min_p": 0.01}])
@pytest.mark.parametrize("rows", [5, 300])
def test_every_call_gives_the_same(rows, settings):
    """The same bits from the same arguments, twenty calls in a row, on rows of few and of many different logits."""
    from gpu_util import to_device
    from qutai_b200.layers import Tensor
    from qutai_b200.sampling import sample

    rng = np.random.default_rng(rows)
    logits = rng.standard_normal((rows, 20011)) * 2.0
    logits[::2] = np.round(logits[::2] * 2) / 2
    logits = Tensor(to_device(logits, "bfloat16"), logits.shape)
    uniforms = to_device(rng.random(rows), "float32")
    first = [x.tobytes() for x in sample(logits, uniforms, **settings)]
    for _ in range(20):
        assert [x.tobytes() for x in sample(logits, uniforms, **settings)] == first
