"""Eight-bit tensors in rank-sharded checkpoint files (``qutai_b200.checkpoint``), on host-memory stand-ins for the device storages."""
import pytest

from qutai_b200 import checkpoint
from test_checkpoint_sharded import HostStorage


class Bytes(HostStorage):
    WIDTH = {**HostStorage.WIDTH, "int8": 1}

    def view(self, start, size):
        assert 0 <= start and start + size <= self.size
        return Bytes(size, self.dtype, self._data, self, self._start + start * self.WIDTH[self.dtype])


@pytest.mark.parametrize("chunk", [1, 7, 256, 1 << 20])
def test_codes_and_scales_come_back_as_they_were(tmp_path, chunk):
    codes, scales = bytes((i * 37 + 11) % 256 for i in range(1001)), bytes(range(16))

    def named():
        return [("w.average.codes", Bytes(1001, "int8")), ("w.average.scales", Bytes(4))]

    written = named()
    for (_, storage), data in zip(written, (codes, scales)):
        storage.upload_bytes(data)
    checkpoint.save_sharded(tmp_path, written, metadata={"step": 3}, chunk_bytes=chunk)
    read = [(name, type(s)(s.size, s.dtype)) for name, s in named()]
    assert checkpoint.load_sharded(tmp_path, read, verify=True, chunk_bytes=max(chunk, 4)) == {"step": 3}
    assert [s.tobytes() for _, s in read] == [codes, scales]
    with pytest.raises(ValueError):
        checkpoint.load_sharded(tmp_path, [("w.average.codes", Bytes(1001, "float32"))])
