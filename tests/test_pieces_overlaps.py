"""Every buffer that the loss in pieces writes lies apart from all that the call reads and from the others that it writes.  No GPU: a refusal comes before a launch."""
import ctypes
from itertools import combinations

import pytest

from qutai_b200 import lib

FIELDS = ("hidden", "weight", "targets", "loss", "tables", "inputs", "lse", "row_loss", "gradient", "d_hidden", "d_weight", "scratch")
WRITES = {"forward": ("loss", "tables", "inputs", "lse", "row_loss", "scratch"), "backward": ("d_hidden", "d_weight", "scratch")}
READS = {"forward": ("hidden", "weight", "targets"), "backward": ("weight", "targets", "tables", "inputs", "lse", "gradient")}


def structure():
    a = lib.Pieces(10, 64, 500, 256, lib.QMOE_BF16, lib.QMOE_BF16, *[0] * 12)
    for i, field in enumerate(FIELDS):
        setattr(a, field, (i + 1) << 20)
    return a


@pytest.mark.parametrize("function", ["forward", "backward"])
def test_one_buffer_over_another_is_refused(library_path, function):
    writes = WRITES[function]
    pairs = [*combinations(writes, 2), *((w, r) for w in writes for r in READS[function])]
    for first, second in pairs:
        for moved, other in ((first, second), (second, first)):
            bad = structure()
            setattr(bad, moved, getattr(bad, other))
            with pytest.raises(ValueError, match="overlap"):
                lib.call("qmoe_pieces_" + function, ctypes.byref(bad), 0)


def test_the_last_byte_of_one_in_the_first_of_another_is_refused(library_path):
    """10 rows count as 128 in the buffers that are kept."""
    sizes = {"hidden": 10 * 64 * 2, "weight": 500 * 64 * 2, "targets": 80, "inputs": 128 * 64 * 2, "lse": 512, "row_loss": 512,
             "tables": 4 * int(lib.load().qmoe_pieces_table_words(10))}
    for moved, other in (("lse", "hidden"), ("lse", "inputs"), ("row_loss", "lse"), ("row_loss", "targets"), ("row_loss", "tables"), ("row_loss", "weight")):
        bad = structure()
        setattr(bad, moved, getattr(bad, other) + sizes[other] - 4)
        with pytest.raises(ValueError, match="overlap"):
            lib.call("qmoe_pieces_forward", ctypes.byref(bad), 0)
