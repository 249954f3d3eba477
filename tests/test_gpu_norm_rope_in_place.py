"""Norm and rotation written over their own operands: the bits they have elsewhere.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("batch,time,heads,kv_heads,dim", [(1, 1, 16, 4, 64), (2, 301, 7, 3, 64), (3, 40, 5, 2, 24), (2, 700, 40, 8, 128)])
def test_outputs_on_their_own_operands(batch, time, heads, kv_heads, dim, dtype):
    from gpu_util import to_device
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import norm_rope_backward, norm_rope_forward
    from qutai_b200.storage import DeviceStorage

    rng = np.random.default_rng(dim)
    given = lambda h: Tensor(to_device(rng.standard_normal((batch, time, h * dim)), dtype), (batch, time, h * dim))  # noqa: E731
    copied = lambda x: Tensor(x.storage.copy(), x.shape)  # noqa: E731
    q, k, gq, gk = given(heads), given(kv_heads), given(heads), given(kv_heads)
    w = Tensor(to_device(rng.standard_normal(dim), "float32"), (dim,))
    want = [s.tobytes() for s in norm_rope_forward(q, k, w, w, heads, kv_heads)]
    own = copied(q), copied(k)
    norm_rope_forward(*own, w, w, heads, kv_heads, out=[x.storage for x in own])
    assert [x.storage.tobytes() for x in own] == want
    want = [s.tobytes() for s in norm_rope_backward(gq, gk, q, k, w, w, heads, kv_heads)]
    for over in ("gradients", "operands"):
        a, b, c, d = copied(gq), copied(gk), copied(q), copied(k)
        on = (a, b) if over == "gradients" else (c, d)
        out = [x.storage for x in on] + [DeviceStorage(dim, "float32") for _ in range(2)]
        norm_rope_backward(a, b, c, d, w, w, heads, kv_heads, out=out)
        assert [s.tobytes() for s in out] == want
