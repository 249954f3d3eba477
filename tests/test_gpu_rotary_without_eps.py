"""Norm and rotation with an epsilon of zero (or one that 32 bits hold as zero), on heads that leave places of a warp's pass empty.  The bars
are those of ``test_gpu_rotary``.  Needs a B200: ``-m gpu``."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 64), (3, 3, 64), (5, 2, 64), (1, 1, 128), (3, 2, 24), (1, 3, 8)])
def test_places_without_a_head_add_nothing(heads, kv_heads, dim, dtype, eps, monkeypatch):
    import test_gpu_rotary

    monkeypatch.setattr(test_gpu_rotary, "EPS", eps)
    test_gpu_rotary.check(3, 11, heads, kv_heads, dim, dtype, seed=dim)
