"""The storages that the packed attention's backward writes to are named as those of its forward, of the rotations and of the loss in pieces: ``out``.
No GPU: a device call is noted instead of made."""
import pytest

from qutai_b200 import attention, lib
from qutai_b200.attention import packed_attention_backward
from test_packed_training_arguments import Sequences, storage, tensor


def backward(monkeypatch, **names):
    noted, plan = [], Sequences([60, 40], monkeypatch)
    with monkeypatch.context() as m:
        m.setattr(lib, "call", lambda name, *args: noted.append((name, args)))
        m.setattr(attention, "DeviceStorage", lambda size, dtype, stream=0: storage(size, dtype, 10 << 20))
        results = packed_attention_backward(storage(12800, ptr=4 << 20), tensor(100, 128), tensor(100, 64, ptr=2 << 20), tensor(100, 64, ptr=3 << 20),
                                            storage(12800, ptr=5 << 20), storage(200, "float32", 6 << 20), 2, 1, plan, **names)
    return results, noted


def given():
    return storage(12800, ptr=7 << 20), storage(6400, ptr=8 << 20), storage(6400, ptr=9 << 20)


@pytest.mark.parametrize("name", ["out", "results"])
def test_results_go_to_the_given_storages(monkeypatch, name):
    results, noted = backward(monkeypatch, **{name: given()})
    assert [s.ptr for s in results] == [7 << 20, 8 << 20, 9 << 20]
    (function, (reference, stream)), = noted
    a = reference._obj
    assert function == "qmoe_packed_attention_backward" and stream == 0
    assert (a.grad_out, a.out, a.lse, a.delta, a.dq, a.dk, a.dv) == tuple(n << 20 for n in (4, 5, 6, 10, 7, 8, 9))


def test_both_names_at_once_and_storages_of_other_sizes_are_refused(monkeypatch):
    for names in (dict(out=given(), results=given()), dict(out=given()[:2]), dict(out=(*given()[:2], storage(6399, ptr=9 << 20)))):
        with pytest.raises(ValueError):
            backward(monkeypatch, **names)
