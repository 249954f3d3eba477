"""An 8-bit AdamW that was saved and resumed takes the steps of one that was not, bit for bit.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_a_resumed_optimizer_takes_the_same_steps(tmp_path):
    from gpu_util import to_device
    from qutai_b200 import checkpoint
    from qutai_b200.layers import Tensor
    from qutai_b200.optim import AdamW, ByteState

    sizes = (300, 4096, 70001)

    def states(optimizer):
        return [(f"{i}.{kind}.{part}", getattr(state[p], part)) for i, p in enumerate(optimizer.parameters)
                for kind, state in (("average", optimizer.averages), ("root", optimizer.square_averages)) for part in ("codes", "scales")]

    def made(values):
        return AdamW([Tensor(to_device(v, "float32"), v.shape, requires_grad=True) for v in values], learning_rate=1e-2, state_bits=8)

    def step(optimizer, seed):
        rng = np.random.default_rng(seed)
        for p in optimizer.parameters:
            p.grad = Tensor(to_device(rng.standard_normal(p.storage.size), "float32"), p.shape)
        optimizer.step()

    rng = np.random.default_rng(0)
    first = made([rng.standard_normal(n).astype(np.float32) for n in sizes])
    for t in range(3):
        step(first, t)
    checkpoint.save_sharded(tmp_path, states(first), metadata={"steps": [first.steps[p] for p in first.parameters]}, chunk_bytes=5000)
    second = made([np.frombuffer(p.storage.tobytes(), np.float32) for p in first.parameters])
    for p in second.parameters:
        second.averages[p], second.square_averages[p] = ByteState.zeros(p.storage.size), ByteState.zeros(p.storage.size)
    steps = checkpoint.load_sharded(tmp_path, states(second), verify=True, chunk_bytes=5000)["steps"]
    second.steps = dict(zip(second.parameters, steps))
    for t in range(3, 6):
        step(first, t)
        step(second, t)
        assert [p.storage.tobytes() for p in first.parameters] == [p.storage.tobytes() for p in second.parameters]
        assert [s.tobytes() for _, s in states(first)] == [s.tobytes() for _, s in states(second)]
