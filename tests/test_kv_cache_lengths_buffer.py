"""The new lengths of an append lie in a buffer of their own: parts of the append still read the old lengths and the counts when others write them.
No GPU: every refusal comes before a launch."""
import pytest

from test_decoding_arguments import cache, storage, tensor

NEW = 1 << 21


@pytest.mark.parametrize("lengths,counts", [(1 << 22, NEW), (1 << 22, NEW + 4), (1 << 22, NEW - 4), (NEW + 4, 1 << 22), (NEW - 4, 1 << 22), (NEW, None)])
@pytest.mark.parametrize("time", [0, 3])
def test_new_lengths_that_overlap_what_is_read(library_path, lengths, counts, time):
    c = cache(batch=2, lengths=storage(2, "int32", lengths))
    new = tensor(2, time, 128)
    with pytest.raises(ValueError, match="of their own"):
        c.append(new, new, counts=None if counts is None else storage(2, "int32", counts), lengths_out=storage(2, "int32", NEW))
