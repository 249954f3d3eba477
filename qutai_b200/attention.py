"""Causal self-attention with grouped key/value heads over ``qmoe_attention_forward`` / ``qmoe_attention_backward``.

Upstream's ``attention(q, k, v, heads, kv_heads)`` (src/qutai/lm/layers.py:119-130) takes ``q`` [batch, time,
heads * dim] and ``k``, ``v`` [batch, time, kv_heads * dim], calls the backend's ``attention`` (output and the
log-sum-exp of every row) and records a backward that calls ``attention_backward`` with the saved storages.
``attention`` here has that signature and returns a tensor whose ``parents`` / ``backward_rule`` are what upstream's
``record`` would have filled in.  bfloat16 and head width 64 only — the case of upstream's tensor-core kernels
(src/qutai/backends/cuda/lm.cu:91-285).

``packed_attention`` is the same within each of many sequences of different lengths that lie behind one another in one tensor of rows
(``PackedSequences``), for head widths 64 and 128, over ``qmoe_packed_attention_forward`` / ``qmoe_packed_attention_backward``; upstream
has rectangular batches only.  Dependency-free: ctypes and the standard library only.
"""
from __future__ import annotations

import ctypes
from array import array
from math import isfinite

from . import lib
from .layers import Tensor
from .rotary import operand, outputs
from .storage import DeviceStorage, done_with


def _describe(q, k, v, heads, kv_heads):
    if len(q.shape) != 3 or tuple(k.shape) != tuple(v.shape) or len(k.shape) != 3 or k.shape[:2] != q.shape[:2]:
        raise ValueError("q must be [batch, time, heads * dim] and k, v [batch, time, kv_heads * dim]")
    batch, time, features = q.shape
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads or features % heads:
        raise ValueError("heads must be a positive multiple of kv_heads and divide the width of q")
    dim = features // heads
    if k.shape[2] != kv_heads * dim:
        raise ValueError("the width of k and v must be kv_heads * dim")
    for tensor in (q, k, v):
        if tensor.storage.dtype != "bfloat16":
            raise ValueError("attention takes bfloat16 tensors")
    a = lib.Attention()
    a.batch, a.time, a.heads, a.kv_heads, a.dim, a.dtype = batch, time, heads, kv_heads, dim, lib.QMOE_BF16
    a.q, a.k, a.v = q.storage.ptr, k.storage.ptr, v.storage.ptr
    return a


def attention_forward(q, k, v, heads, kv_heads, stream=0):
    """Returns ``(out, lse)`` as device storages (bfloat16 [batch * time * heads * dim], float32 [batch * time * heads])."""
    a = _describe(q, k, v, heads, kv_heads)
    out = DeviceStorage(q.storage.size, "bfloat16", stream=stream)
    lse = DeviceStorage(a.batch * a.time * a.heads, "float32", stream=stream)
    a.out, a.lse = out.ptr, lse.ptr
    lib.call("qmoe_attention_forward", ctypes.byref(a), stream)
    return out, lse


def attention_backward(gradient, q, k, v, out, lse, heads, kv_heads, stream=0):
    """``gradient``: storage (or tensor) like ``out``.  Returns ``(dq, dk, dv)`` as device storages."""
    a = _describe(q, k, v, heads, kv_heads)
    gradient = getattr(gradient, "storage", gradient)
    if gradient.dtype != "bfloat16" or gradient.size != q.storage.size:
        raise ValueError("the gradient must be bfloat16 and shaped like the output")
    dq = DeviceStorage(q.storage.size, "bfloat16", stream=stream)
    dk = DeviceStorage(k.storage.size, "bfloat16", stream=stream)
    dv = DeviceStorage(v.storage.size, "bfloat16", stream=stream)
    delta = DeviceStorage(lse.size, "float32", stream=stream)
    a.out, a.lse, a.grad_out, a.delta = out.ptr, lse.ptr, gradient.ptr, delta.ptr
    a.dq, a.dk, a.dv = dq.ptr, dk.ptr, dv.ptr
    lib.call("qmoe_attention_backward", ctypes.byref(a), stream)
    return dq, dk, dv


def attention(q, k, v, heads, kv_heads, stream=0):
    """Upstream's ``attention`` (src/qutai/lm/layers.py:119-130)."""
    out, lse = attention_forward(q, k, v, heads, kv_heads, stream)
    result = Tensor(out, q.shape)
    result.parents = (q, k, v)
    result.backward_rule = lambda gradient: attention_backward(gradient, q, k, v, out, lse, heads, kv_heads, stream)
    return result


class PackedSequences:
    """Sequences of ``lengths`` positions (none among them is no error), one behind the other in one tensor of rows: where each starts and which blocks
    of 128 positions it has, on the device.  ``rows``: up to the last one's end.  A program keeps one for each packing it runs."""

    BLOCK = 128

    def __init__(self, lengths, stream=0):
        self.lengths = tuple(int(n) for n in lengths)
        if any(n < 0 for n in self.lengths):
            raise ValueError("a length must not be negative")
        self.rows, self.stream, starts = 0, stream, []
        for n in self.lengths:
            starts.append(self.rows)
            self.rows += n
        if self.rows >= 2 ** 31 - 512:
            raise ValueError("too many rows")
        self.starts = tuple(starts)
        # the blocks with the most key blocks before them first: the grid then ends in its shortest pieces
        items = [(block, start, n) for start, n in zip(starts, self.lengths) for block in range(-(-n // self.BLOCK))]
        items.sort(key=lambda item: -item[0])
        self.blocks, self.longest, self.pairs = len(items), items[0][0] + 1 if items else 0, sum(item[0] + 1 for item in items)
        # how many have more than a half, a quarter and an eighth of the longest one's
        self.above = tuple(sum((item[0] + 1) * part > self.longest for item in items) for part in (2, 4, 8))
        table = array("i", (value for block, start, n in items for value in (start, n, block, 0)))
        self.table = DeviceStorage.from_bytes(table.tobytes(), "int32", stream) if items else None
        self._positions = None

    @property
    def positions(self):
        """int32 storage [rows] of every row's place in its sequence, made when first asked for."""
        if self._positions is None:
            values = array("i")
            for n in self.lengths:
                values.extend(range(n))
            self._positions = DeviceStorage.from_bytes(values.tobytes(), "int32", self.stream)
        return self._positions


def _describe_packed(q, k, v, heads, kv_heads, sequences, scale):
    rows = q.shape[-2] if len(q.shape) > 1 else 0
    for tensor in (q, k, v):
        if len(tensor.shape) not in (2, 3) or (len(tensor.shape) == 3 and tensor.shape[0] != 1) or tensor.shape[-2] != rows:
            raise ValueError("q must be [rows, heads * dim] and k, v [rows, kv_heads * dim]")
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads or q.shape[-1] % heads:
        raise ValueError("heads must be a positive multiple of kv_heads and divide the width of q")
    dim = q.shape[-1] // heads
    if k.shape[-1] != kv_heads * dim or v.shape[-1] != kv_heads * dim:
        raise ValueError("the width of k and v must be kv_heads * dim")
    if dim not in (64, 128):
        raise ValueError("the head width must be 64 or 128")
    if sequences.rows > rows:
        raise ValueError("the sequences hold more rows than the tensors")
    scale = dim ** -0.5 if scale is None else scale
    if not scale > 0 or not isfinite(scale):
        raise ValueError("the scale must be a positive number")
    operands = [operand(tensor) for tensor in (q, k, v)]
    if any(dtype != "bfloat16" for _, dtype, _ in operands):
        raise ValueError("packed attention takes bfloat16 tensors")
    a = lib.PackedAttention(sequences.rows, sequences.blocks, sequences.longest, sequences.pairs, heads, kv_heads, dim, lib.QMOE_BF16,
                            *(pitch for _, _, pitch in operands), scale, 0, 0 if sequences.table is None else sequences.table.ptr,
                            *(address for address, _, _ in operands))
    a.above_half, a.above_quarter, a.above_eighth = sequences.above
    return a, rows, dim


def _made(given, wanted, rows, used, stream):
    """``given`` storages, or new ones whose rows behind the last sequence hold zeros (those of given ones stay as they are)."""
    results = outputs(given, wanted, stream)
    if given is None and used < rows:
        for storage in results:
            width = storage.size // rows * lib.ITEM_BYTES[storage.dtype]
            lib.call("qmoe_memset", storage.ptr + used * width, 0, (rows - used) * width, stream)
    return results


def packed_attention_forward(q, k, v, heads, kv_heads, sequences, *, scale=None, out=None, stream=0):
    """``q`` [rows, heads * dim], ``k``, ``v`` [rows, kv_heads * dim], bfloat16 (tensors, or ``rotary.Columns`` of a tensor [1, rows, width]), the rows of
    ``sequences`` one behind the other and any number of rows behind them.  ``scale`` of the scores: by default dim^-0.5.  Returns ``(out, lse)``, storages
    of bfloat16 [rows * heads * dim] and float32 [rows * heads]; ``out``: two storages to write to, whose rows behind the last
    sequence stay as they are."""
    a, rows, dim = _describe_packed(q, k, v, heads, kv_heads, sequences, scale)
    result = _made(out, ((rows * heads * dim, "bfloat16"), (rows * heads, "float32")), rows, sequences.rows, stream)
    if sequences.blocks:
        a.out, a.lse = (storage.ptr for storage in result)
        lib.call("qmoe_packed_attention_forward", ctypes.byref(a), stream)
        done_with(sequences.table, stream)       # a replay reads it, whether or not the plan is still there
    return result


def packed_attention_backward(gradient, q, k, v, attended, lse, heads, kv_heads, sequences, *, scale=None, out=None, results=None, stream=0):
    """``gradient``: storage (or tensor) like the forward's output; ``attended`` and ``lse`` are what the forward returned, the other arguments the
    forward's.  Returns ``(dq, dk, dv)`` as dense storages; ``out``: three storages to write to, whose rows behind the last sequence stay as they are
    (``results``: another name of it)."""
    if results is not None:
        if out is not None:
            raise ValueError("out and results are two names of the storages to write to")
        out = results
    a, rows, dim = _describe_packed(q, k, v, heads, kv_heads, sequences, scale)
    gradient = getattr(gradient, "storage", gradient)
    wide, narrow = rows * heads * dim, rows * kv_heads * dim
    for storage, size, dtype in ((gradient, wide, "bfloat16"), (attended, wide, "bfloat16"), (lse, rows * heads, "float32")):
        if storage.size != size or storage.dtype != dtype:
            raise ValueError("the gradient, attended and lse must have the sizes and dtypes of the forward's results")
    result = _made(out, ((wide, "bfloat16"), (narrow, "bfloat16"), (narrow, "bfloat16")), rows, sequences.rows, stream)
    if sequences.blocks:
        delta = DeviceStorage(sequences.rows * heads, "float32", stream=stream)
        a.out, a.lse, a.grad_out, a.delta = attended.ptr, lse.ptr, gradient.ptr, delta.ptr
        a.dq, a.dk, a.dv = (storage.ptr for storage in result)
        lib.call("qmoe_packed_attention_backward", ctypes.byref(a), stream)
        done_with(delta, stream)
        done_with(sequences.table, stream)
    return result


def packed_attention(q, k, v, heads, kv_heads, sequences, *, scale=None, stream=0):
    """``packed_attention_forward`` as a tensor recorded with parents ``(q, k, v)``, like ``attention``."""
    out, lse = packed_attention_forward(q, k, v, heads, kv_heads, sequences, scale=scale, stream=stream)
    result = Tensor(out, q.shape)
    result.parents = (q, k, v)
    result.backward_rule = lambda gradient: packed_attention_backward(gradient, q, k, v, out, lse, heads, kv_heads, sequences, scale=scale, stream=stream)
    return result
