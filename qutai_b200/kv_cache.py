"""A key/value cache for decoding and attention over it, over ``qmoe_cache_append`` / ``qmoe_cache_read`` / ``qmoe_prefix_attention``.

``KVCache`` holds the keys and values of a batch of sequences, in bfloat16 or quantised to 8 bits with a scale for each head and
position, and each sequence's length on the device.  ``prefix_attention`` lets new queries see a prefix that all
sequences share (a cache of batch 1, read once for all of them) and what their own sequence holds.  No upstream counterpart.
Dependency-free: ctypes and the standard library only.
"""
from __future__ import annotations

import ctypes

from . import lib
from .layers import Tensor
from .rotary import operand, outputs
from .storage import DeviceStorage


class KVCache:
    """Keys and values [batch, kv_heads, capacity, dim].  ``dtype`` "bfloat16" or "int8".  ``lengths`` (int32 [batch], on the device)
    says what each sequence holds; ``longest`` is the host's bound on it, by which the work is cut up: after ``append``
    with ``counts`` it may lie above every sequence's length, never below.  ``append`` and ``read`` run on ``stream``; work on another stream that
    reads the cache has to be over before the next ``append``, which lets go of the lengths before it.  The buffers are made here unless they are given
    (``k``, ``v``, ``lengths`` and, for int8, ``k_scale``, ``v_scale`` as storages; ``longest`` then says how long they are)."""

    def __init__(self, batch, capacity, kv_heads, dim, dtype="bfloat16", *, k=None, v=None, k_scale=None, v_scale=None, lengths=None,
                 longest=0, stream=0):
        if dtype not in lib.CACHE_CODES:
            raise ValueError("a cache is bfloat16 or int8")
        if min(batch, capacity, kv_heads, dim) <= 0:
            raise ValueError("batch, capacity, kv_heads and dim must be positive")
        if not 0 <= longest <= capacity:
            raise ValueError("longest must lie between 0 and the capacity")
        places = batch * kv_heads * capacity
        wanted = [("k", k, places * dim, dtype), ("v", v, places * dim, dtype)]
        if dtype == "int8":
            wanted += [("k_scale", k_scale, places, "float32"), ("v_scale", v_scale, places, "float32")]
        elif k_scale is not None or v_scale is not None:
            raise ValueError("a bfloat16 cache has no scales")
        given = [storage is not None for _, storage, _, _ in wanted] + [lengths is not None]
        if any(given) and not all(given):
            raise ValueError("give all of a cache's buffers or none")
        self.batch, self.capacity, self.kv_heads, self.dim, self.dtype, self.stream = batch, capacity, kv_heads, dim, dtype, stream
        self.k_scale = self.v_scale = None
        for name, storage, size, kind in wanted:
            if storage is None:
                storage = DeviceStorage(size, kind, stream=stream)
            elif storage.size != size or storage.dtype != kind:
                raise ValueError(f"{name} must hold {size} values of {kind}")
            setattr(self, name, storage)
        if lengths is None:
            if longest:
                raise ValueError("a new cache holds nothing")
            lengths = DeviceStorage.zeros(batch, "int32", stream)
        self._struct = lib.Cache()
        c = self._struct
        c.batch, c.capacity, c.kv_heads, c.dim, c.dtype = batch, capacity, kv_heads, dim, lib.CACHE_CODES[dtype]
        c.k, c.v = self.k.ptr, self.v.ptr
        if self.k_scale is not None:
            c.k_scale, c.v_scale = self.k_scale.ptr, self.v_scale.ptr
        self.rewind(lengths, longest)

    def rewind(self, lengths, longest):
        """From here on the sequences hold ``lengths`` (an int32 storage, kept, not copied) positions, at most ``longest`` of them:
        back to a point that was held earlier, or, with zeros, to nothing."""
        if lengths.dtype != "int32" or lengths.size != self.batch:
            raise ValueError("lengths must hold one int32 value for each sequence")
        if not 0 <= longest <= self.capacity:
            raise ValueError("longest must lie between 0 and the capacity")
        self.lengths, self.longest = lengths, longest
        self._struct.lengths = lengths.ptr

    def append(self, k, v, *, counts=None, lengths_out=None):
        """``k``, ``v`` [batch, time, kv_heads * dim], float32 or bfloat16 (tensors or ``rotary.Columns``), behind what the sequences hold; with
        ``counts`` (int32 storage) only the first ``counts[b]`` rows of sequence ``b``.  ``lengths`` becomes a new storage
        (``lengths_out``, if given)."""
        if len(k.shape) != 3 or tuple(k.shape) != tuple(v.shape) or k.shape[0] != self.batch or k.shape[2] != self.kv_heads * self.dim:
            raise ValueError("k and v must be [batch, time, kv_heads * dim]")
        time = k.shape[1]
        if self.longest + time > self.capacity:
            raise ValueError(f"{time} more positions exceed the cache's capacity of {self.capacity} ({self.longest} held)")
        (k_ptr, dtype, k_pitch), (v_ptr, v_dtype, v_pitch) = operand(k), operand(v)
        if dtype not in lib.DTYPE_CODES or v_dtype != dtype:
            raise ValueError("k and v must be float32 or bfloat16, both the same")
        if counts is not None and (counts.dtype != "int32" or counts.size != self.batch):
            raise ValueError("counts must hold one int32 value for each sequence")
        after, = outputs(None if lengths_out is None else (lengths_out,), ((self.batch, "int32"),), self.stream)
        lib.call("qmoe_cache_append", ctypes.byref(self._struct), k_ptr, v_ptr, lib.DTYPE_CODES[dtype], k_pitch, v_pitch, time,
                 0 if counts is None else counts.ptr, after.ptr, self.stream)
        self.rewind(after, self.longest + time)

    def read(self, start, count, *, dtype="bfloat16", out=None):
        """Positions ``[start, start + count)`` of every sequence as tensors ``(k, v)`` [batch, count, kv_heads * dim] of ``dtype``; zeros behind a
        sequence's length.  ``out``: two storages to write to instead of new ones."""
        if dtype not in lib.DTYPE_CODES:
            raise ValueError("positions are read as float32 or bfloat16")
        if start < 0 or count < 0 or start + count > self.capacity:
            raise ValueError("positions outside the cache")
        size = self.batch * count * self.kv_heads * self.dim
        k, v = outputs(out, ((size, dtype), (size, dtype)), self.stream)
        lib.call("qmoe_cache_read", ctypes.byref(self._struct), start, count, k.ptr, v.ptr, lib.DTYPE_CODES[dtype], self.stream)
        shape = (self.batch, count, self.kv_heads * self.dim)
        return Tensor(k, shape), Tensor(v, shape)


def prefix_attention(q, heads, cache, prefix=None, *, out=None, stream=None):
    """``q`` [batch, time, heads * dim] (bfloat16), the queries of the last ``time`` positions of every sequence of ``cache``, whose keys
    and values are in it already: query ``t`` sees all of ``prefix`` (a ``KVCache`` of batch 1, or none) and the first
    ``length - time + t + 1`` positions of its own sequence.  Returns ``(out, lse)``, storages of bfloat16 [batch * time * heads * dim] and float32
    [batch * time * heads]; a query that sees nothing gives zeros and -infinity, one with a score that is NaN or +infinity NaN.  Head
    width 64 or 128.  ``stream``: by default the cache's, behind what was appended to it."""
    stream = cache.stream if stream is None else stream
    if len(q.shape) != 3 or q.shape[0] != cache.batch or heads <= 0 or q.shape[2] != heads * cache.dim:
        raise ValueError("q must be [batch, time, heads * dim] with the batch and head width of the cache")
    if q.storage.dtype != "bfloat16":
        raise ValueError("prefix_attention takes bfloat16 queries")
    rows = cache.batch * q.shape[1] * heads
    result = outputs(out, ((rows * cache.dim, "bfloat16"), (rows, "float32")), stream)
    q_ptr, out_ptr = q.storage.ptr, result[0].ptr
    if (q_ptr | out_ptr) & 15:
        raise ValueError("q and the output must be 16-byte aligned")
    a = lib.PrefixAttention(q.shape[1], heads, 0, 0 if prefix is None else prefix.longest, cache.longest, q_ptr, out_ptr, result[1].ptr)
    own, shared = ctypes.byref(cache._struct), None if prefix is None else ctypes.byref(prefix._struct)
    nbytes = lib.load().qmoe_prefix_attention_scratch(ctypes.byref(a), own, shared)
    scratch = DeviceStorage(nbytes // 4, "float32", stream=stream) if nbytes else None
    a.scratch = scratch.ptr if nbytes else 0
    lib.call("qmoe_prefix_attention", ctypes.byref(a), own, shared, stream)
    return result
