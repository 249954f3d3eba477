"""The table of a plan that a recorded call of packed attention reads lives as long as the recording: a replay that found another call's numbers there would read
and write anywhere.  On the fake device (no GPU)."""
import pytest

from qutai_b200 import lib, storage
from qutai_b200.attention import PackedSequences, packed_attention_backward, packed_attention_forward
from test_optim_bytes_recorded import device  # noqa: F401
from test_packed_training_arguments import storage as wrapped, tensor


@pytest.mark.parametrize("backward", [False, True])
def test_the_table_outlives_its_plan(device, monkeypatch, backward):  # noqa: F811
    released, tables = [], []
    monkeypatch.setattr(storage, "_release", lambda address, size, stream: released.append(address))
    call = lib.call

    def noted(name, *args):
        if name.startswith("qmoe_packed"):
            tables.append(args[0]._obj.table)
        return call(name, *args)

    monkeypatch.setattr(lib, "call", noted)
    plan = PackedSequences([60, 40], 3)
    q, k, v = tensor(100, 128), tensor(100, 64, ptr=2 << 20), tensor(100, 64, ptr=3 << 20)
    device.capturing = 21
    if backward:
        packed_attention_backward(wrapped(12800, ptr=4 << 20), q, k, v, wrapped(12800, ptr=5 << 20), wrapped(200, "float32", 6 << 20), 2, 1, plan, stream=3)
    else:
        packed_attention_forward(q, k, v, 2, 1, plan, stream=3)
    device.capturing = 0
    del plan
    assert tables and tables[0] not in released
    storage._recorded.clear()
    assert tables[0] in released


def test_an_ordinary_call_keeps_nothing(device):  # noqa: F811
    plan = PackedSequences([60, 40], 3)
    packed_attention_forward(tensor(100, 128), tensor(100, 64, ptr=2 << 20), tensor(100, 64, ptr=3 << 20), 2, 1, plan, stream=3)
    assert not storage._recorded
