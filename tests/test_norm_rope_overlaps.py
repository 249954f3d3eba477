"""Where the outputs of norm and rotation may not lie: on an operand, unless it is their own, row on row.  Elsewhere rows would be written before they
are read.  No GPU: every refusal comes before a launch."""
import pytest

from qutai_b200 import rotary
from qutai_b200.layers import Tensor
from qutai_b200.rotary import Columns, norm_rope_backward, norm_rope_forward
from test_decoding_arguments import storage, tensor

MB = 1 << 20
Q, K, FUSED, W = 16 * MB, 32 * MB, 64 * MB, 128 * MB
Q_SIZE, K_SIZE = 6 * 128, 6 * 64
w = tensor(64, dtype="float32", ptr=W)
q, k = tensor(2, 3, 128, ptr=Q), tensor(2, 3, 64, ptr=K)
fused = Tensor(storage(6 * 256, ptr=FUSED), (2, 3, 256))
columns = Columns(fused, 0, 128), Columns(fused, 128, 64)


@pytest.mark.parametrize("operands,out", [
    ((q, k), (Q + 16, K)), ((q, k), (Q, K + 16)), ((q, k), (K, 49 * MB)), ((q, k), (48 * MB, Q)), ((q, k), (48 * MB, 48 * MB + 16)), ((q, k), (Q + 2 * Q_SIZE - 16, K)),
    ((q, k), (Q - 2 * Q_SIZE + 16, K)), (columns, (FUSED, 49 * MB)), (columns, (48 * MB, FUSED + 2 * 128)), (columns, (48 * MB, FUSED + 2 * 192))])
def test_forward(library_path, operands, out):
    with pytest.raises(ValueError, match="its own operand"):
        norm_rope_forward(*operands, w, w, 2, 1, out=(storage(Q_SIZE, ptr=out[0]), storage(K_SIZE, ptr=out[1])))


@pytest.mark.parametrize("dq,dk", [(Q + 16, 49 * MB), (52 * MB + 16, 49 * MB), (53 * MB, 49 * MB), (48 * MB, 52 * MB), (K, 49 * MB), (48 * MB, 48 * MB)])
def test_backward(library_path, dq, dk, monkeypatch):
    monkeypatch.setattr(rotary, "DeviceStorage", lambda size, dtype, **_: storage(size, dtype, 80 * MB))
    gradients = storage(Q_SIZE, ptr=52 * MB), storage(K_SIZE, ptr=53 * MB)
    out = storage(Q_SIZE, ptr=dq), storage(K_SIZE, ptr=dk), storage(64, "float32", 84 * MB), storage(64, "float32", 85 * MB)
    with pytest.raises(ValueError, match="its own operand"):
        norm_rope_backward(*gradients, q, k, w, w, 2, 1, out=out)
