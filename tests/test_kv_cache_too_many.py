"""A cache refuses more heads of positions in a call than its kernels can number, also where their number passes 64 bits.  No GPU: every
refusal comes before a launch."""
import pytest

from test_decoding_arguments import cache, storage, tensor


@pytest.mark.parametrize("batch,kv_heads,time", [(1 << 20, 1 << 20, 1 << 24), (1 << 20, 1 << 14, 1 << 30), (1, 1 << 20, 1 << 11), (3, 1, 1 << 30)])
def test_more_heads_of_positions_than_there_are_numbers(library_path, batch, kv_heads, time):
    c = cache(batch=batch, kv_heads=kv_heads, capacity=time, dim=8, longest=0)
    new = tensor(batch, time, kv_heads * 8)
    with pytest.raises(ValueError, match="2147483647"):
        c.append(new, new, lengths_out=storage(batch, "int32", 1 << 40))
    with pytest.raises(ValueError, match="2147483647"):
        c.read(0, time, out=(storage(new.size), storage(new.size)))
