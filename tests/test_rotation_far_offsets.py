"""Offsets at which the frequencies' 64 bits no longer give every angle are refused.  No GPU: the refusal comes before a launch."""
import ctypes

import pytest

from qutai_b200 import lib
from qutai_b200.rotary import Rotation, rotate_backward, rotate_forward
from test_packed_training_arguments import storage, tensor


@pytest.mark.parametrize("offset", [2 ** 37, -2 ** 37, 2 ** 61])
def test_far_offsets_are_refused(library_path, offset):
    rotation = Rotation(64)
    for function in (rotate_forward, rotate_backward):
        with pytest.raises(ValueError, match="2\\^37"):
            function(tensor(2, 3, 128), tensor(2, 3, 64, ptr=1 << 21), 2, 1, rotation, offset=offset, out=(storage(768), storage(384, ptr=1 << 21)))
    a = lib.Rotate(2, 3, 2, 1, 64, 64, lib.QMOE_BF16, rotation._code, 0, 0, offset, 128, 64, 1 << 20, 1 << 21, 0, 1 << 20, 1 << 21, rotation._address)
    with pytest.raises(ValueError, match="2\\^37"):
        lib.call("qmoe_rotate", ctypes.byref(a), 0)
