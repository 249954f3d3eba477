"""A row's own ``min_p`` that is NaN is no limit, as in the formula (no weight is below a NaN).  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=40), dict(top_k=700, top_p=0.9), dict(top_p=0.95), dict(temperature=0.0), dict(temperature=np.inf)])
@pytest.mark.parametrize("rows", [5, 400])
def test_a_limit_that_is_no_number(rows, settings, dtype):
    from gpu_util import to_device
    from qutai_b200.layers import Tensor
    from qutai_b200.sampling import sample

    rng = np.random.default_rng(rows)
    logits = Tensor(to_device(rng.standard_normal((rows, 5003)) * 2, dtype), (rows, 5003))
    uniforms = to_device(rng.random(rows), "float32")
    limits = np.where(np.arange(rows) % 2, 0.1, np.nan)
    got = sample(logits, uniforms, min_p=to_device(limits, "float32"), **settings)
    want = sample(logits, uniforms, min_p=to_device(np.nan_to_num(limits), "float32"), **settings)
    assert [x.tobytes() for x in got] == [x.tobytes() for x in want]
