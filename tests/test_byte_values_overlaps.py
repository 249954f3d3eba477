"""The numbers that 8-bit states stand for go to storages apart from one another and from the states.  No GPU: a refusal comes before a launch."""
import ctypes

import pytest

from qutai_b200 import lib
from qutai_b200.layers import Tensor
from qutai_b200.optim import AdamW, ByteState
from test_packed_training_arguments import storage

FIELDS = ("average", "average_scale", "root", "root_scale", "average_out", "square_out")
SIZES = {"average": 1000, "average_scale": 16, "root": 1000, "root_scale": 16, "average_out": 4000, "square_out": 4000}


def items():
    made = (lib.ByteItem * 3)()
    for i, item in enumerate(made):
        item.size = 1000
        for j, field in enumerate(FIELDS):
            setattr(item, field, (i * 6 + j + 1) << 20)
    return made


@pytest.mark.parametrize("output", ["average_out", "square_out"])
def test_outputs_over_anything_are_refused(library_path, output):
    for i in range(3):
        for field in FIELDS:
            if (i, field) == (1, output):
                continue
            for by in (0, SIZES[field] - 4, -3996):              # the same place, its last word, and one that reaches into it
                bad = items()
                setattr(bad[1], output, getattr(bad[i], field) + by)
                with pytest.raises(ValueError, match="overlaps"):
                    lib.call("qmoe_byte_values", bad, 3, 0, 0)


def test_one_storage_for_both_is_refused(library_path):
    parameter = Tensor(storage(300, "float32"), (300,), requires_grad=True)
    optimizer = AdamW([parameter], state_bits=8)
    optimizer.averages[parameter], optimizer.square_averages[parameter] = (
        ByteState(storage(300, "int8", n << 20), storage(2, "float32", (n + 1) << 20)) for n in (2, 4))
    optimizer._values_table.fill = lambda rows: (lambda table: (table, 1, 0))((lib.ByteItem * 1)(lib.ByteItem(*rows[0])))
    with pytest.raises(ValueError, match="overlaps"):
        optimizer.values_of_states(out={parameter: (storage(300, "float32", 6 << 20),) * 2})
