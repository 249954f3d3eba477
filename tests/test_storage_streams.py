"""Blocks of the storage cache and streams, on a fake allocator (no GPU): a block goes back to work on the stream it was taken for and on no
other, whose kernels may still be using what another stream's call let go of."""
import ctypes

import pytest

from qutai_b200 import lib, storage
from qutai_b200.attention import attention_backward
from qutai_b200.kv_cache import KVCache, prefix_attention
from qutai_b200.layers import Tensor
from qutai_b200.rotary import norm_rope_backward
from qutai_b200.sampling import sample


class FakeDevice:
    """Hands out addresses, notes the structures of the calls."""

    def __init__(self):
        self.next, self.calls, self.freed = 0x10000, [], []

    def qmoe_free(self, address):
        self.freed.append(address)
        return 0

    def qmoe_prefix_attention_scratch(self, *_):
        return 4096

    def qmoe_norm_rope_partials(self, *_):
        return 1024

    def call(self, name, *args):
        if name == "qmoe_malloc":
            ctypes.cast(args[0], ctypes.POINTER(ctypes.c_uint64))[0] = self.next
            self.next += 1 << 32
        else:
            self.calls.append((name, args))


@pytest.fixture
def fake(monkeypatch):
    device = FakeDevice()
    monkeypatch.setattr(lib, "load", lambda: device)
    monkeypatch.setattr(lib, "call", device.call)
    monkeypatch.setattr(storage, "_cache", {})
    monkeypatch.setattr(storage, "_cached_bytes", 0)
    return device


def tensor(*shape, dtype="bfloat16"):
    size = 1
    for n in shape:
        size *= n
    return Tensor(storage.DeviceStorage(size, dtype), shape)


def test_a_block_is_reused_on_its_own_stream(fake):
    first = storage.DeviceStorage(1 << 18, "float32", stream=7)
    address = first.ptr
    del first
    other = storage.DeviceStorage(1 << 18, "float32", stream=8)
    plain = storage.DeviceStorage(1 << 18, "float32")
    assert address not in (other.ptr, plain.ptr)
    assert storage.DeviceStorage(1 << 18, "float32", stream=7).ptr == address


def test_what_is_made_for_a_stream_belongs_to_it(fake):
    for make in (lambda: storage.DeviceStorage.zeros(1 << 18, "float32", 7), lambda: storage.DeviceStorage.from_values([0.0] * 10, "float32", 7),
                 lambda: storage.DeviceStorage(10, "float32").copy(7)):
        made = make()
        address, size = made.ptr, made.size
        del made
        assert storage.DeviceStorage(size, "float32", stream=8).ptr != address
        assert storage.DeviceStorage(size, "float32", stream=7).ptr == address


def test_the_longest_waiting_block_leaves_whatever_its_stream(fake, monkeypatch):
    monkeypatch.setattr(storage, "CACHE_LIMIT_BYTES", 3 << 20)
    blocks = [storage.DeviceStorage(1 << 18, "float32", stream=s) for s in (7, 8, 0)]
    addresses = [b.ptr for b in blocks]
    small = storage.DeviceStorage(1 << 16, "float32", stream=9)
    del blocks[0], blocks[0], blocks[0]
    del small
    assert fake.freed == [addresses[0]] and storage._cached_bytes == (2 << 20) + (1 << 18)
    storage.empty_cache()
    assert len(fake.freed) == 4 and storage._cached_bytes == 0 and not storage._cache


def last_struct(fake, name):
    args = [args for called, args in fake.calls if called == name][-1]
    return args[0]._obj, args[-1]


def addresses(fake, name, fields):
    struct, stream = last_struct(fake, name)
    return {getattr(struct, field) for field in fields}, stream


@pytest.mark.parametrize("case", ["prefix_attention", "norm_rope_backward", "attention_backward", "sample"])
def test_two_streams_share_no_scratch_and_no_dropped_output(fake, case):
    q, k, w = tensor(2, 3, 128), tensor(2, 3, 64), tensor(64, dtype="float32")
    g, gk = tensor(2, 3, 128), tensor(2, 3, 64)
    cache, lse = KVCache(2, 10, 1, 64), tensor(12, dtype="float32")
    logits, uniforms = tensor(2, 64), storage.DeviceStorage(2, "float32")
    if case == "prefix_attention":
        name, fields, run = "qmoe_prefix_attention", ("scratch", "out", "lse"), lambda s: prefix_attention(q, 2, cache, stream=s)
    elif case == "norm_rope_backward":
        name, fields = "qmoe_norm_rope_backward", ("partials", "dq", "dk", "d_q_weight", "d_k_weight")
        run = lambda s: norm_rope_backward(g.storage, gk.storage, q, k, w, w, 2, 1, stream=s)  # noqa: E731
    elif case == "attention_backward":
        name, fields = "qmoe_attention_backward", ("delta", "dq", "dk", "dv")
        run = lambda s: attention_backward(g.storage, q, k, k, g.storage, lse.storage, 2, 1, s)  # noqa: E731
    else:
        name, fields, run = "qmoe_sample", ("tokens", "log_probs"), lambda s: sample(logits, uniforms, stream=s)
    run(7)
    on_seven, stream = addresses(fake, name, fields)
    assert stream == 7 and 0 not in on_seven
    run(8)
    on_eight, stream = addresses(fake, name, fields)
    assert stream == 8 and not on_seven & on_eight
    run(7)
    assert addresses(fake, name, fields)[0] == on_seven
