"""Drawing one token a row by temperature, top-k, top-p and min-p from given uniform numbers, over ``qmoe_sample``.

The random numbers are an input, so a run can be repeated, and sums of weights are formed in whole numbers, so the same logits,
settings and numbers give the same tokens whatever the batch around them.  No upstream counterpart.  Dependency-free: ctypes and
the standard library only.
"""
from __future__ import annotations

import ctypes

from . import lib
from .rotary import outputs


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, stream=0):
    """``logits`` [rows, vocab], float32 or bfloat16; ``uniforms`` a float32 storage of ``rows`` numbers in [0, 1).  Every setting is a number, or a storage
    with one for each row (float32, ``top_k`` int32).  Kept are the ``top_k`` largest logits (0: all), of these the shortest run from
    the largest that holds ``top_p`` of the weight, of these the ones of at least ``min_p`` times the largest weight; temperature 0
    takes the largest logit.  Returns ``(tokens, log_probs)``: storages of int64 and float32; ``log_probs`` are those of the tokens among all
    of their row at its temperature (at 1 for temperature 0).  A row of nothing but -infinity and NaN gives -1 and -infinity."""
    if len(logits.shape) != 2:
        raise ValueError("logits must be [rows, vocab]")
    rows, vocab = logits.shape
    if logits.storage.dtype not in lib.DTYPE_CODES:
        raise ValueError("logits must be float32 or bfloat16")
    if uniforms.dtype != "float32" or uniforms.size != rows:
        raise ValueError("uniforms must hold one float32 number for each row")
    a = lib.Sample(rows, vocab, lib.DTYPE_CODES[logits.storage.dtype], 0, 1.0, 1.0, 0.0, 0.0, logits.storage.ptr, uniforms.ptr)
    for name, value, dtype in (("temperature", temperature, "float32"), ("top_k", top_k, "int32"), ("top_p", top_p, "float32"), ("min_p", min_p, "float32")):
        if not hasattr(value, "ptr"):
            # (the field holds 32 bits: a count beyond the vocabulary is all of it, a negative one is refused whatever its size)
            setattr(a, name, max(-1, min(value, vocab)) if name == "top_k" else value)
        elif value.dtype != dtype or value.size != rows:
            raise ValueError(f"{name} must be a number or hold one {dtype} value for each row")
        else:
            setattr(a, name + "s", value.ptr)
    tokens, log_probs = outputs(out, ((rows, "int64"), (rows, "float32")), stream)
    a.tokens, a.log_probs = tokens.ptr, log_probs.ptr
    lib.call("qmoe_sample", ctypes.byref(a), stream)
    return tokens, log_probs
