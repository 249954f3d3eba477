"""A ``top_k`` that 32 bits do not hold: all tokens, and refused where it is negative.  No GPU."""
import pytest

from qutai_b200 import lib
from qutai_b200.sampling import sample
from test_decoding_arguments import storage, tensor

OUT = (storage(3, "int64"), storage(3, "float32"))


@pytest.mark.parametrize("top_k,wanted", [(0, 0), (7, 7), (50, 50), (51, 50), (2 ** 31, 50), (2 ** 32 + 5, 50), (2 ** 70, 50)])
def test_counts_beyond_the_vocabulary(monkeypatch, top_k, wanted):
    given = []
    monkeypatch.setattr(lib, "call", lambda name, args, stream: given.append(args._obj.top_k))
    sample(tensor(3, 50), storage(3, "float32"), top_k=top_k, out=OUT)
    assert given == [wanted]


@pytest.mark.parametrize("top_k", [-1, -2 ** 31 - 1, -2 ** 32, -2 ** 32 + 5])
def test_negative_counts(library_path, top_k):
    with pytest.raises(ValueError):
        sample(tensor(3, 50), storage(3, "float32"), top_k=top_k, out=OUT)


def test_a_count_is_a_whole_number():
    with pytest.raises(TypeError):
        sample(tensor(3, 50), storage(3, "float32"), top_k=5.0, out=OUT)
