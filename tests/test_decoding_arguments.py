"""What the operators of decoding refuse, and that their structures match the C layout.  No GPU: every refusal comes before a launch."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT
from qutai_b200 import lib
from qutai_b200.kv_cache import KVCache, prefix_attention
from qutai_b200.layers import Tensor
from qutai_b200.rotary import Columns, norm_rope_backward, norm_rope_forward
from qutai_b200.sampling import sample
from qutai_b200.storage import DeviceStorage


def storage(size, dtype="bfloat16", ptr=1 << 20):
    return DeviceStorage.wrap(ptr, size, dtype)


def tensor(*shape, dtype="bfloat16", ptr=1 << 20):
    size = 1
    for n in shape:
        size *= n
    return Tensor(storage(size, dtype, ptr), shape)


def test_structures_match_the_c_layout(tmp_path):
    header = os.path.join(ROOT, "include", "qutai_moe.h")
    structures = {"qmoe_norm_rope_t": lib.NormRope, "qmoe_cache_t": lib.Cache, "qmoe_prefix_attention_t": lib.PrefixAttention, "qmoe_sample_t": lib.Sample}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for name, structure in structures.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));' for field, _ in structure._fields_]
    source, binary = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", str(binary), str(source)], check=True)
    reported = dict(line.rsplit(" ", 1) for line in subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, structure in structures.items():
        assert int(reported[name]) == ctypes.sizeof(structure)
        for field, _ in structure._fields_:
            assert int(reported[f"{name}.{field}"]) == getattr(structure, field).offset, (name, field)


@pytest.mark.parametrize("change", [
    dict(q=tensor(2, 3, 256)), dict(k=tensor(2, 4, 64)), dict(q=tensor(6, 128)), dict(heads=3), dict(kv_heads=0), dict(k=tensor(2, 3, 64, dtype="float32")),
    dict(q=tensor(2, 3, 128, dtype="int32"), k=tensor(2, 3, 64, dtype="int32")), dict(w=tensor(32, dtype="float32")), dict(w=tensor(64)),
    dict(starts=storage(3, "int32")), dict(starts=storage(2, "float32")), dict(eps=-1.0), dict(theta=0.0), dict(q=tensor(2, 3, 128, ptr=(1 << 20) + 2)),
    dict(out=(storage(768), storage(383))), dict(out=(storage(768),)), dict(q=tensor(2, 3, 24), k=tensor(2, 3, 12), w=tensor(12, dtype="float32")),
    dict(q=tensor(2, 3, 1024), k=tensor(2, 3, 512), w=tensor(512, dtype="float32"))])
def test_norm_rope_refuses(library_path, change):
    a = dict(q=tensor(2, 3, 128), k=tensor(2, 3, 64), w=tensor(64, dtype="float32"), heads=2, kv_heads=1, out=(storage(768), storage(384)))
    a.update(change)
    options = {name: a[name] for name in ("starts", "eps", "theta", "out") if name in a}
    with pytest.raises(ValueError):
        norm_rope_forward(a["q"], a["k"], a["w"], a["w"], a["heads"], a["kv_heads"], **options)


def test_norm_rope_backward_refuses_gradients_of_another_size(library_path):
    q, k, w = tensor(2, 3, 128), tensor(2, 3, 64), tensor(64, dtype="float32")
    for gq, gk in ((storage(767), storage(384)), (storage(768), storage(384, "float32"))):
        with pytest.raises(ValueError):
            norm_rope_backward(gq, gk, q, k, w, w, 2, 1)


def test_columns_stay_inside_their_tensor():
    for start, width in ((-1, 8), (0, 0), (64, 65)):
        with pytest.raises(ValueError):
            Columns(tensor(2, 3, 128), start, width)
    part = Columns(tensor(2, 3, 128), 64, 64)
    assert (part.shape, part.pitch, part.ptr) == ((2, 3, 64), 128, (1 << 20) + 128)


def cache(batch=2, capacity=10, kv_heads=2, dim=64, dtype="bfloat16", longest=4, **changes):
    places = batch * kv_heads * capacity
    buffers = dict(k=storage(places * dim, dtype), v=storage(places * dim, dtype), lengths=storage(batch, "int32"))
    if dtype == "int8":
        buffers.update(k_scale=storage(places, "float32"), v_scale=storage(places, "float32"))
    buffers.update(changes)
    return KVCache(batch, capacity, kv_heads, dim, dtype, longest=longest, **buffers)


def test_a_cache_refuses_buffers_that_do_not_fit(library_path):
    for bad in (dict(dtype="float32"), dict(batch=0), dict(capacity=-1), dict(longest=11), dict(longest=-1), dict(k=storage(5)), dict(v=None), dict(lengths=storage(3, "int32")),
                dict(lengths=storage(2, "float32")), dict(k_scale=storage(40, "float32")), dict(dtype="int8", k_scale=storage(39, "float32"))):
        with pytest.raises(ValueError):
            cache(**bad)
    c = cache()
    for lengths, longest in ((storage(1, "int32"), 0), (storage(2, "int32"), 11), (storage(2, "int64"), 1)):
        with pytest.raises(ValueError):
            c.rewind(lengths, longest)


def test_append_and_read_refuse(library_path):
    c, after = cache(), storage(2, "int32", 1 << 21)
    good = tensor(2, 3, 128)
    for k, v, options in ((tensor(2, 7, 128), tensor(2, 7, 128), {}), (good, tensor(2, 3, 64), {}), (tensor(1, 3, 128), tensor(1, 3, 128), {}),
                          (good, tensor(2, 3, 128, dtype="float32"), {}), (tensor(2, 3, 128, dtype="int8"), tensor(2, 3, 128, dtype="int8"), {}),
                          (good, good, dict(counts=storage(3, "int32"))), (good, good, dict(counts=storage(2, "int64"))),
                          (good, good, dict(lengths_out=c.lengths)), (good, good, dict(lengths_out=storage(1, "int32"))),
                          (tensor(2, 3, 128, ptr=(1 << 20) + 8), good, {})):
        with pytest.raises(ValueError):
            c.append(k, v, **{"lengths_out": after, **options})
        assert c.longest == 4                        # a refused call changes nothing
    for start, count, options in ((-1, 2, {}), (0, 11, {}), (10, 1, {}), (0, 2, dict(dtype="int8")), (0, 2, dict(out=(storage(512), storage(511)))),
                                  (0, 2, dict(out=(storage(512, ptr=(1 << 20) + 2), storage(512))))):
        with pytest.raises(ValueError):
            c.read(start, count, **{"out": (storage(512), storage(512)), **options})


def test_prefix_attention_refuses(library_path):
    good = dict(q=tensor(2, 1, 256), heads=4, cache=cache(), prefix=cache(batch=1))
    for change in (dict(q=tensor(3, 1, 256)), dict(heads=3), dict(heads=0), dict(q=tensor(2, 1, 256, dtype="float32")), dict(q=tensor(2, 256)), dict(prefix=cache(batch=2)),
                   dict(prefix=cache(batch=1, kv_heads=1)), dict(prefix=cache(batch=1, dtype="int8")), dict(prefix=cache(batch=1, dim=128)),
                   dict(q=tensor(2, 1, 256, ptr=(1 << 20) + 4)), dict(q=tensor(2, 1, 128), cache=cache(dim=32), prefix=None),
                   dict(q=tensor(2, 0, 256)), dict(q=tensor(2, 1, 192), heads=3, prefix=None)):
        a = {**good, **change}
        out = (storage(a["q"].size), storage(a["q"].size // a["cache"].dim, "float32"))
        with pytest.raises(ValueError):
            prefix_attention(a["q"], a["heads"], a["cache"], a["prefix"], out=out)


def test_sample_refuses(library_path):
    good = dict(logits=tensor(3, 50), uniforms=storage(3, "float32"))
    out = (storage(3, "int64"), storage(3, "float32"))
    for change in (dict(logits=tensor(150)), dict(logits=tensor(3, 50, dtype="int32")), dict(uniforms=storage(2, "float32")), dict(uniforms=storage(3)),
                   dict(temperature=-0.5), dict(temperature=float("nan")), dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=-0.1), dict(top_k=-1),
                   dict(top_k=storage(3, "float32")), dict(top_p=storage(2, "float32")), dict(logits=tensor(3, 50, ptr=(1 << 20) + 1)),
                   dict(out=(storage(3, "int32"), storage(3, "float32"))), dict(out=(storage(3, "int64", (1 << 20) + 4), storage(3, "float32")))):
        a = {**good, "out": out, **change}
        with pytest.raises(ValueError):
            sample(a.pop("logits"), a.pop("uniforms"), **a)
