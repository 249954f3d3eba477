"""Rotation of query and key heads: with their norm in one pass, over ``qmoe_norm_rope_forward`` / ``qmoe_norm_rope_backward``, or alone with
other layouts and frequencies and a position for every row, over ``qmoe_rotate``.

Every head of every row is divided by its root mean square, multiplied by a weight (one for the query heads, one for the key
heads) and turned by the angles of its position as ``qmoe_rope`` turns it; queries and keys go through in one launch.
Upstream rotates unnormalised heads (src/qutai/lm/layers.py:316-349), so these functions have no counterpart there.
float32 or bfloat16, any head width that is a multiple of 8 up to 256.

``Rotation`` says how heads are turned alone: neighbouring elements or halves of a head as pairs, all of a head or its first
elements, frequencies as they are or scaled for contexts longer than the ones that a model was trained on (``Scaling``).
``rotate_forward`` and ``rotate_backward`` take every row's position from the device, so rows of packed sequences or of sequences that are
decoded side by side go through in one launch.  Any head width from 2 to 256.  Dependency-free: ctypes and the standard library only.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from decimal import Decimal, localcontext
from math import isfinite

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


_PI = Decimal("3.14159265358979323846264338327950288419716939937510")


@dataclass(frozen=True)
class Scaling:
    """Frequencies for contexts ``factor`` times as long as the ``original`` one.  ``kind`` "linear": every frequency divided by the factor;
    "base": theta multiplied by factor^(w / (w - 2)) for ``w`` turned elements, which keeps the fastest pair and divides the slowest by the factor;
    "bands": a pair that turns at least ``high`` times over the original context keeps its frequency, one that turns less than
    ``low`` times has it divided by the factor, between them a share of both, linear in the number of turns."""
    kind: str
    factor: float
    original: float | None = None
    low: float = 1.0
    high: float = 4.0

    def __post_init__(self):
        if self.kind not in ("linear", "base", "bands"):
            raise ValueError("a scaling is linear, base or bands")
        if not self.factor >= 1 or not isfinite(self.factor):
            raise ValueError("a scaling's factor must be a finite number from 1 on")
        if self.kind == "bands" and (self.original is None or not self.original > 0 or not 0 < self.low < self.high):
            raise ValueError("bands need an original context above 0 and 0 < low < high")


# The table's frequencies are off by up to 2^-64 of a turn for each position: here 2^-27, half of what the kernel's rounding of an angle takes
FARTHEST = 2 ** 37


class Rotation:
    """How heads of ``dim`` elements are turned: the first ``width`` of them (all by default) in pairs, neighbours with ``layout``
    "interleaved" (``qmoe_rope``'s), elements ``width / 2`` apart with "halves"; pair ``i`` by theta^(-2 i / width) radians
    for each position, or what ``scaling`` makes of that."""

    def __init__(self, dim, *, theta=10000.0, layout="interleaved", width=None, scaling=None):
        width = dim if width is None else width
        if not 2 <= dim <= 256:
            raise ValueError("the head width must lie between 2 and 256")
        if width % 2 or not 2 <= width <= dim:
            raise ValueError("the turned width must be an even number of a head's elements")
        if layout not in ("interleaved", "halves"):
            raise ValueError("the layout is interleaved or halves")
        if not 1e-15 <= theta <= 1e30:      # (40 digits hold the turns of a position, up to 1e15, and their fraction's 64 bits)
            raise ValueError("theta must lie between 1e-15 and 1e30")
        self.dim, self.theta, self.layout, self.width, self.scaling = dim, theta, layout, width, scaling
        # what counts of an angle is its fraction of a turn, held in 64 bits: an integer product with the position keeps all of them
        with localcontext() as context:
            context.prec = 40
            base, turn = Decimal(theta), 2 * _PI
            if scaling is not None and scaling.kind == "base" and width > 2:
                base *= Decimal(scaling.factor) ** (Decimal(width) / (width - 2))
            ratio, rates = base ** (Decimal(-2) / width), [Decimal(1)]
            for _ in range(width // 2 - 1):
                rates.append(rates[-1] * ratio)
            if scaling is not None and scaling.kind == "linear":
                rates = [rate / Decimal(scaling.factor) for rate in rates]
            elif scaling is not None and scaling.kind == "bands":
                low, high = Decimal(scaling.low), Decimal(scaling.high)
                kept = [min(Decimal(1), max(Decimal(0), (rate * Decimal(scaling.original) / turn - low) / (high - low))) for rate in rates]
                rates = [rate * share + rate / Decimal(scaling.factor) * (1 - share) for rate, share in zip(rates, kept)]
            parts = [int(rate / turn % 1 * 2 ** 64) for rate in rates]
        self.frequencies = tuple(float(rate) for rate in rates)          # radians a position
        self._turns = (ctypes.c_uint64 * len(parts))(*parts)
        self._address = ctypes.addressof(self._turns)
        self._code = lib.ROTATE_HALVES if layout == "halves" else lib.ROTATE_NEIGHBOURS


def _rotate(q, k, heads, kv_heads, rotation, positions, offset, out, stream, backward):
    if len(q.shape) != 3 or len(k.shape) != 3 or q.shape[:2] != k.shape[:2]:
        raise ValueError("q must be [batch, time, heads * dim] and k [batch, time, kv_heads * dim]")
    batch, time, width = q.shape
    dim = rotation.dim
    if heads <= 0 or kv_heads <= 0 or width != heads * dim or k.shape[2] != kv_heads * dim:
        raise ValueError("the widths of q and k must be heads and kv_heads times the rotation's head width")
    (q_ptr, dtype, q_pitch), (k_ptr, k_dtype, k_pitch) = operand(q), operand(k)
    if dtype not in lib.DTYPE_CODES or k_dtype != dtype:
        raise ValueError("q and k must be float32 or bfloat16, both the same")
    rows = batch * time
    if positions is not None and (positions.dtype != "int32" or positions.size != rows):
        raise ValueError("positions must hold one int32 position for each row")
    if not -FARTHEST < offset < FARTHEST:
        raise ValueError("the offset must lie within 2^37 of 0, where the angles are as exact as anywhere")
    q_out, k_out = outputs(out, ((rows * heads * dim, dtype), (rows * kv_heads * dim, dtype)), stream)
    if rows:
        a = lib.Rotate(batch, time, heads, kv_heads, dim, rotation.width, lib.DTYPE_CODES[dtype], rotation._code, backward, 0, int(offset), q_pitch, k_pitch,
                       q_ptr, k_ptr, 0 if positions is None else positions.ptr, q_out.ptr, k_out.ptr, rotation._address)
        lib.call("qmoe_rotate", ctypes.byref(a), stream)
    return q_out, k_out


def rotate_forward(q, k, heads, kv_heads, rotation, *, positions=None, offset=0, out=None, stream=0):
    """``q`` [batch, time, heads * dim], ``k`` [batch, time, kv_heads * dim] (tensors or ``Columns``, float32 or bfloat16), turned as ``rotation`` says.  Row
    ``r`` of all rows is at ``offset + positions[r]`` (int32 storage [batch * time] on the device; none: row ``t`` of every sequence
    at ``offset + t``).  Returns the storages of the turned queries and keys (dense); ``out``: two storages to write to instead of new ones,
    which may be the operands' own where those are dense."""
    return _rotate(q, k, heads, kv_heads, rotation, positions, offset, out, stream, 0)


def rotate_backward(grad_q, grad_k, heads, kv_heads, rotation, *, positions=None, offset=0, out=None, stream=0):
    """``grad_q``, ``grad_k``: gradients of the forward's outputs, tensors or ``Columns`` shaped like its operands; the other arguments are the
    forward's.  Returns the storages of the gradients of the operands."""
    return _rotate(grad_q, grad_k, heads, kv_heads, rotation, positions, offset, out, stream, 1)
