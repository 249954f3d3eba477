"""Blocks that recorded calls took for themselves, on a fake device (no GPU): out of the cache while their recording's graph is there, in it again afterwards."""
import pytest

from qutai_b200 import lib, storage
from test_storage_cache import FakeDevice, fake  # noqa: F401


@pytest.fixture
def device(fake):  # noqa: F811
    """The fake allocator, with recordings: ``capturing`` {stream: number}, ``over`` the numbers of those that are no more."""
    fake.capturing, fake.over, fake.made = {}, set(), 0
    fake.qmoe_capture_number = lambda stream: fake.capturing.get(stream, 0)
    fake.qmoe_stream_capturing = lambda stream: int(stream in fake.capturing)
    fake.qmoe_capture_over = lambda number: number in fake.over
    plain = fake.malloc

    def malloc(out, size):
        fake.made += 1
        plain(out, size)

    fake.malloc = malloc
    return fake


def test_a_block_belongs_to_its_recording_until_that_is_over(device, monkeypatch):
    monkeypatch.setattr(storage, "_recorded", type(storage._recorded)())
    device.capturing[5] = 77
    a = storage.DeviceStorage(1 << 18, stream=5)
    address = a.ptr
    storage.done_with(a, 5)
    del a
    b = storage.DeviceStorage(1 << 18, stream=5)              # recorded too: not the other call's block
    assert b.ptr != address
    del device.capturing[5]
    c = storage.DeviceStorage(1 << 18, stream=5)
    assert c.ptr != address
    device.over.add(77)                                       # the graph is destroyed
    d = storage.DeviceStorage(1 << 18, stream=5)
    assert d.ptr == address and device.made == 3


def test_only_recorded_calls_keep_their_blocks(device, monkeypatch):
    monkeypatch.setattr(storage, "_recorded", type(storage._recorded)())
    for stream in (0, 5):
        a = storage.DeviceStorage(1 << 18, stream=stream)
        storage.done_with(a, stream)
        del a
    assert storage._cached_bytes == 2 << 20 and not storage._recorded


def test_recording_again_and_again_takes_no_more_memory(device, monkeypatch):
    monkeypatch.setattr(storage, "_recorded", type(storage._recorded)())
    for number in range(1, 50):
        device.capturing[5] = number
        for _ in range(2):
            a = storage.DeviceStorage(1 << 17, stream=5)
            storage.done_with(a, 5)
            del a
        del device.capturing[5]
        device.over.add(number)
    assert device.made <= 4
    storage.empty_cache()                                     # what is left of recordings that are over goes back to the device as well
    assert not device.live and not storage._recorded


def test_threads_record_and_let_go_at_once(device, monkeypatch):
    """A recording that another thread makes, or lets go of, while the list is looked through."""
    monkeypatch.setattr(storage, "_recorded", {1: [], 2: [], 3: []})

    def over(number):
        storage._recorded.setdefault(number + 10, [])
        storage._recorded.pop(2, None)
        return number < 3

    device.qmoe_capture_over = over
    storage.release_recorded()
    assert set(storage._recorded) == {3, 11, 13} or set(storage._recorded) == {3, 11, 12, 13}
