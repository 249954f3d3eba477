"""A ``Generator`` that is given another prompt forgets the continuations of the one before.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("between", ["prefill", "generate"])
def test_a_step_after_another_prompt_needs_a_start(between):
    from gpu_util import to_device, to_host
    from qutai_b200.generate import Generator
    from test_gpu_generate import decoder

    model = decoder(True)
    generator = Generator(model)
    ids = to_device(np.array([1, 2]), "int64")
    generator.prefill([3, 4, 5])
    generator.start(2, 4)
    generator.step(ids)
    if between == "prefill":
        generator.prefill([6, 7])
    else:
        generator.generate([6, 7], 2, 1)
    with pytest.raises(RuntimeError):
        generator.step(ids)
    generator.start(2, 4)
    got = to_host(generator.step(ids).storage)
    fresh = Generator(model)
    fresh.prefill([6, 7])
    fresh.start(2, 4)
    assert np.array_equal(got, to_host(fresh.step(ids).storage))


def test_a_prompt_that_is_refused_leaves_the_one_before():
    from gpu_util import to_device
    from qutai_b200.generate import Generator
    from test_gpu_generate import decoder

    generator = Generator(decoder(False))
    generator.prefill([3, 4, 5])
    generator.start(2, 4)
    with pytest.raises(ValueError):
        generator.prefill([96])
    generator.step(to_device(np.array([1, 2]), "int64"))
