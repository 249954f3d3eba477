"""Calls of one shape on two streams with neither waited for: each gives what it gives alone.  Needs a B200: ``-m gpu``."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture
def streams():
    from qutai_b200 import lib

    made = [ctypes.c_uint64() for _ in range(2)]
    for stream in made:
        lib.call("qmoe_stream_create", ctypes.byref(stream))
    yield [stream.value for stream in made]
    for stream in made:
        lib.call("qmoe_stream_sync", stream.value)
        lib.call("qmoe_stream_destroy", stream.value)


def overlapped(calls, streams, rounds=12):
    """``calls``: two functions of a stream that return storages.  Their results alone, and side by side round after round."""
    from qutai_b200 import lib

    alone = []
    for call, stream in zip(calls, streams):
        results = call(stream)
        lib.call("qmoe_stream_sync", stream)
        alone.append([s.tobytes(stream) for s in results])
    kept = [[call(stream) for call, stream in zip(calls, streams)] for _ in range(rounds)]
    for results in kept:
        for want, got, stream in zip(alone, results, streams):
            assert [s.tobytes(stream) for s in got] == want


def test_attention_over_a_prefix(streams):
    from gpu_util import to_device
    from qutai_b200.kv_cache import prefix_attention
    from qutai_b200.layers import Tensor
    from test_gpu_prefix_attention import make

    calls = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        cache, _ = make(rng, 80, 2, 300, 64, "bfloat16", [int(n) for n in rng.integers(0, 301, 80)], 0.0)
        shared, _ = make(rng, 1, 2, 5000, 64, "bfloat16", [5000], 0.0)
        q = Tensor(to_device(rng.standard_normal((80, 1, 256)), "bfloat16"), (80, 1, 256))
        calls.append(lambda stream, q=q, cache=cache, shared=shared: prefix_attention(q, 4, cache, shared, stream=stream))
    overlapped(calls, streams)


def test_norm_and_rotation_backward(streams):
    from gpu_util import to_device
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import norm_rope_backward

    calls = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        given = lambda *shape: Tensor(to_device(rng.standard_normal(shape), "bfloat16"), shape)  # noqa: E731
        q, k, gq, gk = given(2, 700, 512), given(2, 700, 128), given(2, 700, 512), given(2, 700, 128)
        w = Tensor(to_device(rng.standard_normal(64), "float32"), (64,))
        calls.append(lambda stream, a=(gq, gk, q, k, w, w): norm_rope_backward(*a, 8, 2, stream=stream))
    overlapped(calls, streams)


def test_two_generators(streams):
    from qutai_b200 import lib
    from qutai_b200.generate import Generator
    from qutai_b200.decoder import Config, Decoder
    from gpu_util import to_device

    config = Config(vocab_size=96, d_model=256, n_heads=4, n_kv_heads=2, n_layers=2, n_experts=2, top_k=2, d_expert=64, qk_norm=True)
    generators = [Generator(Decoder(config, seed=seed, stream=stream)) for seed, stream in zip((1, 2), streams)]
    lib.call("qmoe_stream_sync", 0)
    ids = to_device(np.arange(30) % 96, "int64")
    alone = []
    for generator, stream in zip(generators, streams):
        generator.prefill(list(range(40)))
        generator.start(30, 6)
        alone.append([generator.step(ids).storage.tobytes(stream) for _ in range(6)])
    for generator in generators:
        generator.prefill(list(range(40)))
        generator.start(30, 6)
    kept = [[generator.step(ids).storage for generator in generators] for _ in range(6)]
    for i, pair in enumerate(kept):
        for which, (logits, stream) in enumerate(zip(pair, streams)):
            assert logits.tobytes(stream) == alone[which][i], (i, which)
