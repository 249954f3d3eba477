"""The stream that ``prefix_attention`` runs on: the cache's, whose appends it has to come behind, unless another is given.  No GPU."""
import pytest

from qutai_b200 import lib
from qutai_b200.kv_cache import prefix_attention
from test_decoding_arguments import cache, storage, tensor


@pytest.mark.parametrize("given,wanted", [(dict(), 7), (dict(stream=9), 9), (dict(stream=0), 0)])
def test_attention_follows_its_cache(library_path, monkeypatch, given, wanted):
    calls = []
    monkeypatch.setattr(lib, "call", lambda name, *args: calls.append((name, args[-1])))
    out = (storage(256), storage(4, "float32"))
    monkeypatch.setattr("qutai_b200.kv_cache.DeviceStorage", lambda size, dtype, **_: storage(size, dtype))
    prefix_attention(tensor(2, 1, 128), 2, cache(kv_heads=1, stream=7), out=out, **given)
    assert calls == [("qmoe_prefix_attention", wanted)]
