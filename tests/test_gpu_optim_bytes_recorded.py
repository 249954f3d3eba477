"""Steps of ``AdamW(state_bits=8)`` between ``qmoe_graph_begin`` and ``qmoe_graph_end``: a replay is the next ordinary step, bit for bit, from whatever the gradients
hold then.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

from test_gpu_packed_recorded import Recording

pytestmark = pytest.mark.gpu

SIZES = (300, 4096, 9001)


def made(seed, stream, shadows=True, rate=1e-2):
    from gpu_util import to_device
    from qutai_b200 import lib
    from qutai_b200.layers import Tensor
    from qutai_b200.optim import AdamW
    from qutai_b200.storage import DeviceStorage

    rng = np.random.default_rng(seed)
    parameters = [Tensor(to_device(rng.standard_normal(n), "float32"), (n,), requires_grad=True) for n in SIZES]
    for p in parameters:
        p.grad = Tensor(DeviceStorage.zeros(p.storage.size, "float32", stream), p.shape)
    copies = {}
    for p in parameters if shadows else ():
        copies[p] = DeviceStorage(p.storage.size, "bfloat16", stream=stream)
        lib.call("qmoe_cast_bf16", p.storage.ptr, copies[p].ptr, p.storage.size, stream)
        copies[p].mark_derived_from(p.storage)
    return AdamW(parameters, learning_rate=rate, state_bits=8, shadows=copies, stream=stream)


def gradients(optimizer, seed):
    rng = np.random.default_rng(seed)
    for p in optimizer.parameters:
        p.grad.storage.upload_bytes(rng.standard_normal(p.storage.size).astype(np.float32).tobytes(), optimizer.stream)


def everything(optimizer):
    values = []
    for p in optimizer.parameters:
        a, b = optimizer.averages[p], optimizer.square_averages[p]
        storages = (p.storage, a.codes, a.scales, b.codes, b.scales, *((optimizer.shadows[p],) if p in optimizer.shadows else ()))
        values.append([s.tobytes(optimizer.stream) for s in storages])
    return values


@pytest.mark.parametrize("shadows", [False, True])
def test_replays_are_the_next_steps(shadows):
    with Recording() as r:
        plain, recorded = made(1, r.stream, shadows), made(1, r.stream, shadows)
        for optimizer in (plain, recorded):
            gradients(optimizer, 0)
            optimizer.step()
        r.lib.call("qmoe_graph_begin", r.stream)
        before = [p.storage.generation for p in recorded.parameters]
        recorded.step()
        import ctypes

        graph = ctypes.c_uint64()
        r.lib.call("qmoe_graph_end", r.stream, ctypes.byref(graph))
        r.graphs.append(graph.value)
        # the recording is no step
        assert set(recorded.steps.values()) == {1} and [p.storage.generation for p in recorded.parameters] == before
        assert everything(recorded) == everything(plain)
        # replays, ordinary steps among them, and the host told or not told of the replays
        for i, kind in enumerate(("replay", "replay", "step", "replay", "told", "step", "step", "replay", "told", "replay", "told"), 1):
            if kind == "told":
                recorded.replayed()
                assert recorded.steps == dict(zip(recorded.parameters, plain.steps.values()))
                continue
            for optimizer in (plain, recorded):
                gradients(optimizer, i)
            plain.step()
            if kind == "step":
                recorded.step()
            else:
                r.replay(graph.value)
            assert everything(recorded) == everything(plain), (i, kind)
        assert len(set(plain.steps.values())) == 1 and plain.steps[plain.parameters[0]] == 9
        assert all(new > old for new, old in zip([p.storage.generation for p in recorded.parameters], before))
        if shadows:
            assert all(recorded.shadows[p].is_derived_from(p.storage) for p in recorded.parameters)
        # a number of steps of one's own counts, in an ordinary step
        for optimizer in (plain, recorded):
            for p in optimizer.parameters:
                optimizer.steps[p] = 40
            gradients(optimizer, 99)
            optimizer.step()
        assert everything(recorded) == everything(plain)
        for optimizer in (plain, recorded):
            gradients(optimizer, 100)
        plain.step()
        r.replay(graph.value)
        recorded.replayed()
        assert everything(recorded) == everything(plain) and set(recorded.steps.values()) == {42}


def test_more_parameters_than_travel_with_a_launch():
    """Forty parameters of which three have gradients when the step is recorded; then all take ordinary steps, the three by the device's count."""
    from gpu_util import to_device
    from qutai_b200.layers import Tensor
    from qutai_b200.optim import AdamW

    def forty(stream):
        rng = np.random.default_rng(5)
        return AdamW([Tensor(to_device(rng.standard_normal(100 + n), "float32"), (100 + n,), requires_grad=True) for n in range(40)], learning_rate=1e-2, state_bits=8,
                     stream=stream)

    def give(optimizer, seed, count):
        rng = np.random.default_rng(seed)
        for i, p in enumerate(optimizer.parameters):
            values = rng.standard_normal(p.storage.size).astype(np.float32)
            if i >= count:
                p.grad = None
            elif p.grad is None:
                p.grad = Tensor(to_device(values, "float32"), p.shape)
            else:
                p.grad.storage.upload_bytes(values.tobytes(), optimizer.stream)

    def state(optimizer):
        return [[s.tobytes(optimizer.stream) for s in (p.storage, optimizer.averages[p].codes, optimizer.square_averages[p].codes)] for p in optimizer.averages]

    import ctypes

    with Recording() as r:
        plain, recorded = forty(r.stream), forty(r.stream)
        for optimizer in (plain, recorded):
            give(optimizer, 0, 3)
            optimizer.step()
        r.lib.call("qmoe_graph_begin", r.stream)
        recorded.step()
        graph = ctypes.c_uint64()
        r.lib.call("qmoe_graph_end", r.stream, ctypes.byref(graph))
        r.graphs.append(graph.value)
        held = [p.grad for p in recorded.parameters]           # a replay reads them
        for seed, count in ((1, 3), (2, 3), (3, 40), (4, 40), (5, 3)):
            for optimizer in (plain, recorded):
                give(optimizer, seed, count)
            plain.step()
            if count == 3 and seed < 5:
                r.replay(graph.value)
            else:
                recorded.step()
            assert state(recorded) == state(plain), seed
        recorded.replayed()
        assert list(recorded.steps.values()) == list(plain.steps.values()) and sorted(set(plain.steps.values())) == [2, 6]
        assert held


def test_a_first_step_or_another_number_of_steps_is_not_recorded():
    with Recording() as r:
        optimizer = made(2, r.stream)
        gradients(optimizer, 1)
        for prepare in (lambda: None, lambda: optimizer.steps.update({p: 7 for p in optimizer.parameters})):
            prepare()
            r.lib.call("qmoe_graph_begin", r.stream)
            with pytest.raises(RuntimeError, match="recorded after"):
                optimizer.step()
            r.lib.load().qmoe_graph_abandon(r.stream)
            if not optimizer.steps:
                optimizer.step()
        assert set(optimizer.steps.values()) == {7}
        optimizer.step()
        assert set(optimizer.steps.values()) == {8}


def test_states_of_a_recording_outlive_their_optimizer():
    """Another call does not get the blocks that a replay writes to."""
    from qutai_b200.storage import DeviceStorage

    with Recording() as r:
        optimizer = made(3, r.stream)
        gradients(optimizer, 1)
        parameters = optimizer.parameters
        kept = [(p, p.grad) for p in parameters]
        graph, _ = r.record(optimizer.step)
        sizes = [(s.size, s.dtype) for p in parameters for state in (optimizer.averages[p], optimizer.square_averages[p]) for s in (state.codes, state.scales)]
        shadows = optimizer.shadows
        del optimizer, parameters
        others = [DeviceStorage.zeros(size, dtype, r.stream) for size, dtype in sizes]
        for _ in range(2):
            r.replay(graph)
        assert not any(any(s.tobytes(r.stream)) for s in others)
        assert kept and shadows
