"""Rotation at the farthest offsets that are taken, against angles in 60 decimal digits.  Needs a B200: ``-m gpu``."""
from decimal import Decimal, localcontext

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")


@pytest.mark.parametrize("offset", [2 ** 37 - 1, 1 - 2 ** 37, 2 ** 36 + 12345])
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_far_offsets(offset, layout):
    """A head of ones and zeros shows cosines and sines.  The table is off by 2^-27 of a turn there, the kernel's angle by 2^-26 and 2^-32 more (together 1.5e-7),
    its sine and cosine by 2^-22: 6e-7 with room."""
    from gpu_util import to_device, to_host
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import Rotation, rotate_forward

    dim, places = 64, [0, 1, -1, 77, 2 ** 31 - 1, -2 ** 31]
    x = np.zeros((1, len(places), dim))
    first = np.arange(0, dim, 2) if layout == "interleaved" else np.arange(dim // 2)
    second = first + 1 if layout == "interleaved" else first + dim // 2
    x[..., first] = 1
    q = Tensor(to_device(x, "float32"), x.shape)
    out = rotate_forward(q, Tensor(to_device(x, "float32"), x.shape), 1, 1, Rotation(dim, layout=layout), positions=to_device(np.array(places), "int32"), offset=offset)[0]
    got = to_host(out, (len(places), dim))
    with localcontext() as context:
        context.prec = 60
        for row, place in zip(got, places):
            for i in range(dim // 2):
                angle = float((Decimal(place + offset) * Decimal(10000) ** (Decimal(-2 * i) / dim)) % (2 * PI))
                assert abs(row[first[i]] - np.cos(angle)) < 6e-7 and abs(row[second[i]] - np.sin(angle)) < 6e-7
