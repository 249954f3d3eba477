"""What a recorded step of ``AdamW(state_bits=8)`` hands to the device: no number of its own, a count there.  No GPU: device calls are noted."""
import ctypes

import pytest

from qutai_b200 import lib, optim, storage
from qutai_b200.layers import Tensor
from qutai_b200.optim import AdamW
from test_packed_training_arguments import storage as wrapped


class Device:
    """Addresses, and the items of each step."""

    def __init__(self):
        self.next, self.steps, self.capturing, self.counts = 1 << 20, [], 0, []

    def qmoe_stream_capturing(self, stream):
        return int(bool(self.capturing and stream))

    def qmoe_capture_number(self, stream):
        return self.capturing if stream else 0

    def qmoe_capture_over(self, number):
        return 0

    def call(self, name, *args):
        if name == "qmoe_malloc":
            self.next += 1 << 20
            ctypes.cast(args[0], ctypes.POINTER(ctypes.c_uint64))[0] = self.next
        if name == "qmoe_adamw_bytes":
            items, count = args[:2]
            self.steps.append([(items[i].count, items[i].number, items[i].step) for i in range(count)])
        if name == "qmoe_memcpy_d2h":
            (ctypes.c_int64 * len(self.counts)).from_address(args[0].value)[:] = self.counts


@pytest.fixture
def device(monkeypatch):
    made = Device()
    monkeypatch.setattr(lib, "load", lambda: made)
    monkeypatch.setattr(lib, "call", made.call)
    monkeypatch.setattr(storage, "_cache", {})
    monkeypatch.setattr(storage, "_recorded", {})
    monkeypatch.setattr(storage, "_release", lambda *_: None)
    return made


def optimizer(stream):
    parameters = [Tensor(wrapped(300, "float32", n << 30), (300,), requires_grad=True) for n in (1, 2)]
    for p in parameters:
        p.grad = Tensor(wrapped(300, "float32", 5 << 30), (300,))
    return AdamW(parameters, state_bits=8, stream=stream)


def test_on_the_default_stream_nothing_is_counted(device):
    o = optimizer(0)
    o.step()
    o.step()
    o.replayed()
    assert [[item[:2] for item in step] for step in device.steps] == [[(0, 0)] * 2] * 2 and set(o.steps.values()) == {2}


def test_a_recorded_step_has_the_number_that_the_device_counts(device):
    o = optimizer(3)
    device.capturing = 11
    with pytest.raises(RuntimeError):
        o.step()
    device.capturing = 0
    o.step()
    (first, second), = device.steps
    assert first[1] == second[1] == 1 and first[0] and second[0] == first[0] + 16
    device.capturing = 11
    generations = [p.storage.generation for p in o.parameters]
    o.step()
    assert [item[:2] for item in device.steps[-1]] == [(first[0], 0), (second[0], 0)]
    assert set(o.steps.values()) == {1} and [p.storage.generation for p in o.parameters] == generations
    assert len(storage._recorded[11]) == 9                       # two states of codes and scales each, and the counts
    device.capturing = 0
    o.step()                                                     # ordinary again: replays may have come between
    assert [item[1] for item in device.steps[-1]] == [0, 0] and set(o.steps.values()) == {2}
    device.counts = [6, 0, 2, 0]
    generations = [p.storage.generation for p in o.parameters]
    o.replayed()
    assert list(o.steps.values()) == [6, 2] and [p.storage.generation - g for p, g in zip(o.parameters, generations)] == [1, 0]
    o.steps[o.parameters[1]] = 9
    o.step()
    assert [item[1] for item in device.steps[-1]] == [0, 10] and list(o.steps.values()) == [7, 10]


def test_a_count_is_checked(library_path):
    item = lib.ByteItem(*[1 << 20] * 7, 0, 0, 300, 0, 1e-3, 1.0, 1 << 20, 1)
    for field, value in (("count", (1 << 20) + 4), ("number", -1)):
        bad = lib.ByteItem.from_buffer_copy(item)
        setattr(bad, field, value)
        with pytest.raises(ValueError, match="count"):
            lib.call("qmoe_adamw_bytes", ctypes.byref(bad), 1, 0, 1e-3, 0.9, 0.999, 1e-8, 0.01, 0)
