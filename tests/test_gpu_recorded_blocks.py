"""Memory of recorded calls between ``qmoe_graph_begin`` and the graph's end.  Needs a B200: ``-m gpu``."""
import ctypes

import numpy as np
import pytest

from test_gpu_packed_recorded import Recording, operands

pytestmark = pytest.mark.gpu


def held():
    from qutai_b200 import storage

    storage.release_recorded()
    return sum(s.nbytes for kept in storage._recorded.values() for s in kept)


def test_graphs_that_are_destroyed_give_their_blocks_back(monkeypatch):
    from gpu_util import to_device
    from qutai_b200 import lib
    from qutai_b200.attention import packed_attention_backward, packed_attention_forward
    from qutai_b200.head import PiecewiseHead
    from qutai_b200.layers import Tensor

    rng = np.random.default_rng(1)
    x, w = (Tensor(to_device(rng.standard_normal(shape), "bfloat16"), shape) for shape in ((300, 64), (1500, 64)))
    targets = to_device(rng.integers(-1, 1500, 300), "int64")
    made = []
    call = lib.call
    monkeypatch.setattr(lib, "call", lambda name, *args: (made.append(name) if name == "qmoe_malloc" else None, call(name, *args))[1])
    with Recording() as r:
        head = PiecewiseHead(r.stream, piece_bytes=1 << 19)
        tensors, gradient, sequences = operands(1, [300, 129], 4, 2, 64, r.stream)

        def work():
            out, lse = packed_attention_forward(*tensors, 4, 2, sequences, stream=r.stream)
            grads = packed_attention_backward(gradient, *tensors, out, lse, 4, 2, sequences, stream=r.stream)
            loss = head.forward(x, w, targets)
            return (out, lse, *grads, loss.storage, *(t.storage for t in head.backward()))

        want = [s.tobytes(r.stream) for s in work()]
        before, counts = held(), []
        for _ in range(12):
            graph, results = r.record(work)
            assert held() > before
            r.replay(graph)
            assert [s.tobytes(r.stream) for s in results] == want
            del results
            r.lib.call("qmoe_graph_destroy", r.graphs.pop())
            assert held() == before
            counts.append(len(made))
        assert counts[-1] == counts[2]                        # nothing more from the device

        # one that ends without a graph
        r.lib.call("qmoe_graph_begin", r.stream)
        work()
        assert held() > before
        r.lib.call("qmoe_graph_abandon", r.stream)
        assert held() == before

        # two graphs, destroyed one by one
        first, second = r.record(work)[0], r.record(work)[0]
        both = held()
        r.lib.call("qmoe_graph_destroy", first)
        r.graphs.remove(first)
        one = held()
        assert before < one < both
        r.replay(second)
        r.lib.call("qmoe_graph_destroy", second)
        r.graphs.remove(second)
        assert held() == before


def test_numbers_of_recordings():
    from qutai_b200 import lib
    from qutai_b200.storage import DeviceStorage

    handle = lib.load()
    with Recording() as r:
        target = DeviceStorage(64, "int32", stream=r.stream)
        assert handle.qmoe_capture_number(r.stream) == 0
        numbers = []
        for _ in range(2):
            r.lib.call("qmoe_graph_begin", r.stream)
            numbers.append(handle.qmoe_capture_number(r.stream))
            assert numbers[-1] and not handle.qmoe_capture_over(numbers[-1])
            r.lib.call("qmoe_memset", target.ptr, 0, 64, r.stream)
            graph = ctypes.c_uint64()
            r.lib.call("qmoe_graph_end", r.stream, ctypes.byref(graph))
            r.graphs.append(graph.value)
        assert numbers[0] != numbers[1] and handle.qmoe_capture_number(r.stream) == 0
        for number in numbers:
            assert not handle.qmoe_capture_over(number)
            r.lib.call("qmoe_graph_destroy", r.graphs.pop(0))
            assert handle.qmoe_capture_over(number)
