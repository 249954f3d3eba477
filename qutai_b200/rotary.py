"""Norm and rotation of query and key heads in one pass, over ``qmoe_norm_rope_forward`` / ``qmoe_norm_rope_backward``.

Every head of every row is divided by its root mean square, multiplied by a weight (one for the query heads, one for the key
heads) and turned by the angles of its position as ``qmoe_rope`` turns it; queries and keys go through in one launch.
Upstream rotates unnormalised heads (src/qutai/lm/layers.py:316-349), so these functions have no counterpart there.
float32 or bfloat16, any head width that is a multiple of 8 up to 256.  Dependency-free: ctypes and the standard library only.
"""
from __future__ import annotations

import ctypes

from . import lib
from .storage import DeviceStorage


class Columns:
    """Columns ``[start, start + width)`` of a tensor [batch, time, total] as an operand [batch, time, width] whose rows lie ``total``
    elements apart: the queries, keys or values in the output of one projection for all three."""

    def __init__(self, tensor, start, width):
        if len(tensor.shape) != 3 or start < 0 or width <= 0 or start + width > tensor.shape[2]:
            raise ValueError("columns outside the tensor [batch, time, width]")
        self.tensor, self.start = tensor, start
        self.shape = (*tensor.shape[:2], width)
        self.pitch = tensor.shape[2]

    @property
    def dtype(self):
        return self.tensor.storage.dtype

    @property
    def ptr(self):
        return self.tensor.storage.ptr + self.start * lib.ITEM_BYTES[self.dtype]


def operand(x):
    """``(address, dtype, row pitch)`` of a tensor [batch, time, width] or of ``Columns``."""
    if isinstance(x, Columns):
        return x.ptr, x.dtype, x.pitch
    return x.storage.ptr, x.storage.dtype, x.shape[-1]


def _describe(q, k, q_weight, k_weight, heads, kv_heads, eps, theta, starts, offset):
    if len(q.shape) != 3 or len(k.shape) != 3 or q.shape[:2] != k.shape[:2]:
        raise ValueError("q must be [batch, time, heads * dim] and k [batch, time, kv_heads * dim]")
    batch, time, width = q.shape
    if heads <= 0 or kv_heads <= 0 or width % heads or k.shape[2] * heads != kv_heads * width:
        raise ValueError("the widths of q and k must be heads and kv_heads times the same head width")
    dim = width // heads
    (q_ptr, dtype, q_pitch), (k_ptr, k_dtype, k_pitch) = operand(q), operand(k)
    if dtype not in lib.DTYPE_CODES or k_dtype != dtype:
        raise ValueError("q and k must be float32 or bfloat16, both the same")
    for weight in (q_weight, k_weight):
        if weight.storage.dtype != "float32" or weight.storage.size != dim:
            raise ValueError("the weights must hold one float32 value for each element of a head")
    if starts is not None and (starts.dtype != "int32" or starts.size != batch):
        raise ValueError("starts must hold one int32 position for each sequence")
    # (fields in their order: one call instead of one for each)
    a = lib.NormRope(batch, time, heads, kv_heads, dim, lib.DTYPE_CODES[dtype], int(offset), q_pitch, k_pitch, eps, theta, q_ptr, k_ptr,
                     q_weight.storage.ptr, k_weight.storage.ptr, 0 if starts is None else starts.ptr)
    return a, dtype, dim


def outputs(given, wanted, stream):
    """``given`` storages, checked against ``wanted`` [(size, dtype), ...], or new ones for ``stream``."""
    if given is None:
        return tuple(DeviceStorage(size, dtype, stream=stream) for size, dtype in wanted)
    given = tuple(given)
    if len(given) != len(wanted) or any(s.size != size or s.dtype != dtype for s, (size, dtype) in zip(given, wanted)):
        raise ValueError("out must be storages of " + ", ".join(f"{size} x {dtype}" for size, dtype in wanted))
    return given


def norm_rope_forward(q, k, q_weight, k_weight, heads, kv_heads, *, eps=1e-6, theta=10000.0, starts=None, offset=0, out=None, stream=0):
    """``q`` [batch, time, heads * dim], ``k`` [batch, time, kv_heads * dim] (tensors or ``Columns``), weights of ``dim`` float32 values.  Row
    ``t`` of sequence ``b`` is position ``offset + starts[b] + t`` (``starts``: int32 storage on the device, none: 0).  Returns the
    storages of the normalised, rotated queries and keys (dense); ``out``: two storages to write to instead of new ones."""
    a, dtype, dim = _describe(q, k, q_weight, k_weight, heads, kv_heads, eps, theta, starts, offset)
    rows = a.batch * a.time
    q_out, k_out = outputs(out, ((rows * heads * dim, dtype), (rows * kv_heads * dim, dtype)), stream)
    a.q_out, a.k_out = q_out.ptr, k_out.ptr
    lib.call("qmoe_norm_rope_forward", ctypes.byref(a), stream)
    return q_out, k_out


def norm_rope_backward(grad_q, grad_k, q, k, q_weight, k_weight, heads, kv_heads, *, eps=1e-6, theta=10000.0, starts=None, offset=0, out=None,
                       stream=0):
    """``grad_q``, ``grad_k``: storages (or tensors) like the forward's outputs; the other arguments are the forward's.  Returns ``(dq, dk,
    d_q_weight, d_k_weight)`` as storages, the weights' gradients float32."""
    a, dtype, dim = _describe(q, k, q_weight, k_weight, heads, kv_heads, eps, theta, starts, offset)
    rows = a.batch * a.time
    wanted = ((rows * heads * dim, dtype), (rows * kv_heads * dim, dtype))
    gradients = [getattr(g, "storage", g) for g in (grad_q, grad_k)]
    if any(g.size != size or g.dtype != dtype for g, (size, dtype) in zip(gradients, wanted)):
        raise ValueError("the gradients must have the sizes and the dtype of the forward's outputs")
    results = outputs(out, (*wanted, (dim, "float32"), (dim, "float32")), stream)
    partials = DeviceStorage(int(lib.load().qmoe_norm_rope_partials(a.batch, a.time, heads, kv_heads, dim)), "float32", stream=stream)
    a.grad_q, a.grad_k = (g.ptr for g in gradients)
    a.dq, a.dk, a.d_q_weight, a.d_k_weight = (s.ptr for s in results)
    a.partials = partials.ptr
    lib.call("qmoe_norm_rope_backward", ctypes.byref(a), stream)
    return results
