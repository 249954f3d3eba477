"""Packed attention right behind the kernel that writes its table of blocks, on one stream.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_the_table_may_come_from_the_kernel_before(dim):
    """The table at the end of a buffer of 256 MB that one kernel fills (a sum with zeros: small whole numbers are float32 values that it keeps).  What lay there is
    the table of another packing of the same rows."""
    from gpu_util import to_device
    from qutai_b200 import lib
    from qutai_b200.attention import PackedSequences, packed_attention_backward, packed_attention_forward
    from qutai_b200.layers import Tensor
    from qutai_b200.storage import DeviceStorage

    lengths, other, heads, kv_heads = [300, 84, 129], [129, 84, 300], 4, 2
    rng, rows, size = np.random.default_rng(dim), sum(lengths), 1 << 26
    tensors = [Tensor(to_device(rng.standard_normal((rows, h * dim)), "bfloat16"), (rows, h * dim)) for h in (heads, kv_heads, kv_heads)]
    gradient = to_device(rng.standard_normal((rows, heads * dim)), "bfloat16")

    def work(forward, backward):
        out, lse = packed_attention_forward(*tensors, heads, kv_heads, forward)
        return out, lse, *packed_attention_backward(gradient, *tensors, out, lse, heads, kv_heads, backward)

    plan, stale = PackedSequences(lengths), PackedSequences(other)
    assert (plan.blocks, plan.longest, plan.pairs) == (stale.blocks, stale.longest, stale.pairs)
    want = [s.tobytes() for s in work(plan, plan)]
    words = plan.table.size
    source, zeros, target = DeviceStorage.zeros(size, "float32"), DeviceStorage.zeros(size, "float32"), DeviceStorage.zeros(size, "float32")
    end = DeviceStorage.wrap(target.ptr + 4 * (size - words), words, "int32", owner=target)
    DeviceStorage.wrap(source.ptr + 4 * (size - words), words, "int32", owner=source).copy_from(plan.table)
    fresh = PackedSequences(lengths)
    fresh.table = end

    def write():
        end.copy_from(stale.table)
        lib.call("qmoe_stream_sync", 0)
        lib.call("qmoe_add", source.ptr, zeros.ptr, target.ptr, lib.QMOE_F32, size, 0)

    for _ in range(5):
        write()
        results = work(fresh, fresh)
        assert end.tolist() == plan.table.tolist()
        assert [s.tobytes() for s in results] == want
        out, lse = results[:2]
        write()              # and right before the backward
        grads = packed_attention_backward(gradient, *tensors, out, lse, heads, kv_heads, fresh)
        assert [s.tobytes() for s in grads] == want[2:]
