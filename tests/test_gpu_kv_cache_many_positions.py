"""More heads of positions in one call than 2^31 threads could hold one each, which a cache takes all the same (``qutai_b200.kv_cache``): what
is appended comes back bit for bit.  Needs a B200: ``-m gpu``."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_nine_million_heads_of_positions_in_one_call():
    from qutai_b200.kv_cache import KVCache
    from qutai_b200.layers import Tensor
    from qutai_b200.storage import DeviceStorage

    batch, time, kv_heads, dim = 16, 65600, 8, 8
    bits = np.random.default_rng(0).integers(0, 1 << 14, batch * time * kv_heads * dim, dtype=np.uint16)         # small positive numbers
    shape = (batch, time, kv_heads * dim)
    new = Tensor(DeviceStorage.from_bytes(bits.tobytes(), "bfloat16"), shape)
    cache = KVCache(batch, time, kv_heads, dim)
    cache.append(new, new)
    for read in cache.read(0, time):
        assert np.array_equal(np.frombuffer(read.storage.tobytes(), dtype=np.uint16), bits)
