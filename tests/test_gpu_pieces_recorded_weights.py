"""A recorded loss in pieces and what its head is used for afterwards: the copy of a float32 weight, the rows kept for the backward.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

from test_gpu_packed_recorded import Recording

pytestmark = pytest.mark.gpu


def problem(seed, stream, rows=300):
    from gpu_util import to_device
    from qutai_b200.layers import Tensor

    rng = np.random.default_rng(seed)
    x = Tensor(to_device(rng.standard_normal((rows, 64)), "bfloat16"), (rows, 64))
    w = Tensor(to_device(rng.standard_normal((1500, 64)), "float32"), (1500, 64))
    return x, w, to_device(rng.integers(-1, 1500, rows), "int64")


def fill(stream):
    """Storages of many sizes, so that a block that was let go of is in use again."""
    from qutai_b200.storage import DeviceStorage

    return [DeviceStorage(size // 4, "float32", stream=stream) for size in [512 * n for n in range(1, 130)] + [65536 * n for n in range(1, 20)] for _ in range(3)]


def test_a_recorded_loss_keeps_the_copy_of_its_weight():
    from qutai_b200.head import PiecewiseHead

    with Recording() as r:
        head = PiecewiseHead(r.stream)
        first, second = problem(1, r.stream), problem(2, r.stream)

        def work(given):
            loss = head.forward(*given)
            return (loss.storage, *(t.storage for t in head.backward()))

        want = [s.tobytes(r.stream) for s in work(first)]
        graph, results = r.record(lambda: work(first))
        other = work(second)                                   # another weight: another copy
        held = fill(r.stream)
        for s in held:
            s.fill_zero(r.stream)
        r.replay(graph)
        assert [s.tobytes(r.stream) for s in results] == want
        assert not any(any(s.tobytes(r.stream)) for s in held)
        assert other


def test_a_recorded_backward_keeps_the_rows_of_its_forward():
    from qutai_b200.head import PiecewiseHead

    with Recording() as r:
        head = PiecewiseHead(r.stream)
        first, second = problem(3, r.stream), problem(4, r.stream)
        head.forward(*first)
        graph, results = r.record(lambda: [t.storage for t in head.backward()])
        r.replay(graph)
        want = [s.tobytes(r.stream) for s in results]
        head.forward(*second)
        head.backward()
        held = fill(r.stream)
        for s in held:
            s.fill_zero(r.stream)
        r.replay(graph)
        assert [s.tobytes(r.stream) for s in results] == want


def test_a_recorded_cast_is_none_before_its_replay():
    """The weight changes between the last plain call and the recording: the copy is stale until something has written it."""
    from qutai_b200.head import PiecewiseHead

    with Recording() as r:
        head = PiecewiseHead(r.stream)
        x, w, targets = problem(5, r.stream)
        head.forward(x, w, targets)
        changed = problem(6, r.stream)[1]
        w.storage.copy_from(changed.storage, r.stream)
        import ctypes

        r.lib.call("qmoe_graph_begin", r.stream)
        loss = head.forward(x, w, targets)
        graph = ctypes.c_uint64()
        r.lib.call("qmoe_graph_end", r.stream, ctypes.byref(graph))
        r.graphs.append(graph.value)
        want = PiecewiseHead(r.stream).forward(x, changed, targets).storage.tobytes(r.stream)
        assert head.forward(x, w, targets).storage.tobytes(r.stream) == want
        r.replay(graph.value)
        assert loss.storage.tobytes(r.stream) == want
