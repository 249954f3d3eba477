"""What a recorded loss in pieces holds for its replays, on the fake device (no GPU)."""
import pytest

from qutai_b200 import lib, storage
from qutai_b200.head import PiecewiseHead
from test_optim_bytes_recorded import device  # noqa: F401
from test_packed_training_arguments import storage as wrapped, tensor


@pytest.mark.parametrize("weight", ["float32", "bfloat16"])
def test_every_block_of_its_own(device, monkeypatch, weight):  # noqa: F811
    device.qmoe_pieces_table_words = lambda rows: 8 + rows
    device.qmoe_pieces_scratch_bytes = lambda a, backward: 4096
    calls, call = [], lib.call
    monkeypatch.setattr(lib, "call", lambda name, *args: (calls.append((name, args)), call(name, *args))[1])
    head = PiecewiseHead(3)
    given = tensor(10, 64), tensor(500, 64, dtype=weight, ptr=2 << 20), wrapped(10, "int64", 3 << 20)
    head.forward(*given)
    head.backward()
    assert not storage._recorded
    device.capturing = 9
    head.forward(*given)
    forward = lib.Pieces.from_buffer_copy(calls[-1][1][0]._obj)
    device.capturing = 0
    addresses = {s.ptr for s in storage._recorded[9]}
    wanted = {getattr(forward, name) for name in ("tables", "inputs", "lse", "row_loss", "scratch")} | ({forward.weight} if weight == "float32" else set())
    assert addresses == wanted
    device.capturing = 10                       # the backward alone, in another recording
    head.backward()
    backward = calls[-1][1][0]._obj
    addresses = {s.ptr for s in storage._recorded[10]}
    assert addresses == (wanted - {forward.scratch}) | {backward.scratch}


def test_a_recorded_cast_marks_nothing(device, monkeypatch):  # noqa: F811
    device.qmoe_pieces_table_words = lambda rows: 8 + rows
    device.qmoe_pieces_scratch_bytes = lambda a, backward: 4096
    names, call = [], lib.call
    monkeypatch.setattr(lib, "call", lambda name, *args: (names.append(name), call(name, *args))[1])
    head = PiecewiseHead(3)
    given = tensor(10, 64), tensor(500, 64, dtype="float32", ptr=2 << 20), wrapped(10, "int64", 3 << 20)
    for capturing, casts in ((5, 1), (0, 2), (0, 2), (6, 2)):
        device.capturing = capturing
        head.forward(*given)
        assert names.count("qmoe_cast_bf16") == casts
