"""The language-model head with its cross-entropy loss, over ``qmoe_head_forward`` / ``qmoe_head_backward``.

Upstream's ``projection_loss(hidden, weight, labels, chunk_size, *, prepared_labels=None)``
(src/qutai/lm/layers.py:187-257, called from ``Decoder.loss`` src/qutai/lm/decoder.py:143-175) drops the last
position of every sequence, multiplies by the (tied embedding) weight chunk by chunk, takes each row's
``log sum exp - picked logit`` for labels other than -100 and divides by the number of counted rows; its backward
forms every chunk's logits again.  ``projection_loss`` here keeps that signature and meaning — ``chunk_size`` is
accepted and ignored: the logits of all rows are formed once and kept (see ``csrc/head.cu``) — and returns a tensor
whose ``parents`` / ``backward_rule`` are what upstream's ``record`` would have filled in, so either autograd can
walk it.

``PiecewiseHead`` is the loss for steps whose logits are too many to keep: rows with a target each (packed sequences, a part
of the rows without one), the vocabulary a piece at a time, over ``qmoe_pieces_forward`` / ``qmoe_pieces_backward``.  It costs a fourth product
(``csrc/pieces.cu``) and keeps a number a row.  Dependency-free: ctypes and the standard library only.
"""
from __future__ import annotations

import ctypes
from array import array

from . import lib
from .layers import Tensor
from .storage import DeviceStorage, done_with

ROW_PAD = 128


def prepare_labels(labels, stream=0):
    """Token ids ``[batch][time]`` (nested sequences, -100 = no target) as an int64 device storage, the form
    ``projection_loss`` takes as ``prepared_labels``.  Upstream's ``prepare_labels`` uploads the targets
    ``row[1:]`` of every sequence (src/qutai/lm/layers.py:193-196, src/qutai/backends/cuda_lm.py); here the whole
    ``[batch, time]`` table goes up and the kernels read position ``t + 1`` for row ``t``."""
    flat = array("q", (int(label) for row in labels for label in row))
    return DeviceStorage.from_bytes(flat.tobytes(), "int64", stream)


class LMHead:
    """Buffers and the two calls of one head.  ``forward`` leaves the loss (fp32 scalar on the device) and keeps
    the gradient of the logits; ``backward`` returns ``(d_hidden, d_weight)``."""

    def __init__(self, stream=0):
        self.stream = stream
        self._buffers, self._key = {}, None
        self._operand = None      # bf16 copy of an fp32 weight, and whose it is
        self._operand_of_weight = None
        self._call = None

    def _buffer(self, name, size, dtype):
        current = self._buffers.get(name)
        if current is None or current.size < size or current.dtype != dtype:
            current = self._buffers[name] = DeviceStorage(size, dtype, stream=self.stream)
        return current

    def _weight_operand(self, weight, dtype):
        if weight.storage.dtype == dtype:
            return weight.storage
        if weight.storage.dtype != "float32" or dtype != "bfloat16":
            raise ValueError("the head's weight must have the activations' dtype, or be float32 with bfloat16 activations")
        shadow = self._operand
        of = weight.storage.ptr, weight.storage.size
        if shadow is None or self._operand_of_weight not in (None, of) or shadow.size != weight.storage.size:
            shadow = self._operand = DeviceStorage(weight.storage.size, "bfloat16", stream=self.stream)
        self._operand_of_weight = of
        if not shadow.is_derived_from(weight.storage):
            lib.call("qmoe_cast_bf16", weight.storage.ptr, shadow.ptr, weight.storage.size, self.stream)
            if not (self.stream and lib.load().qmoe_stream_capturing(self.stream)):      # (a recorded cast has not run)
                shadow.mark_derived_from(weight.storage)
        return shadow

    def forward(self, hidden, weight, labels):
        """``hidden`` [batch, time, width] (bfloat16 or float32), ``weight`` [vocab, width], ``labels`` an int64
        device storage of batch * time token ids (``prepare_labels``) or nested sequences."""
        if len(hidden.shape) != 3 or len(weight.shape) != 2 or weight.shape[1] != hidden.shape[2]:
            raise ValueError("hidden must be [batch, time, width] and weight [vocab, width]")
        batch, time, width = hidden.shape
        vocab = weight.shape[0]
        if time < 2:
            raise ValueError("a sequence needs at least two positions to have a target")
        dtype = hidden.storage.dtype
        if dtype not in lib.DTYPE_CODES:
            raise ValueError("hidden must be float32 or bfloat16")
        if not isinstance(labels, DeviceStorage):
            labels = prepare_labels(labels, self.stream)
        if labels.dtype != "int64" or labels.size != batch * time:
            raise ValueError("labels must hold batch * time int64 token ids")
        rows = batch * (time - 1)
        bound = (rows + ROW_PAD - 1) // ROW_PAD * ROW_PAD
        operand = self._weight_operand(weight, dtype)
        h = lib.Head()
        h.batch, h.time, h.dtype, h.width, h.vocab, h.rows_bound = batch, time, lib.DTYPE_CODES[dtype], width, vocab, bound
        h.hidden, h.weight, h.labels = hidden.storage.ptr, operand.ptr, labels.ptr
        h.inputs = self._buffer("inputs", bound * width, dtype).ptr
        h.logits = self._buffer("logits", bound * vocab, dtype).ptr
        h.row_loss = self._buffer("row_loss", rows, "float32").ptr
        h.meta = self._buffer("meta", 8, "float32").ptr
        loss = DeviceStorage(1, "float32", stream=self.stream)
        h.loss = loss.ptr
        lib.call("qmoe_head_forward", ctypes.byref(h), self.stream)
        self._call = (h, hidden, weight, labels, loss)
        return Tensor(loss, ())

    def backward(self, gradient=None, *, need_hidden=True, need_weight=True):
        """``gradient``: fp32 device storage (or tensor) of one element, ``None`` = 1.  Returns ``(d_hidden,
        d_weight)`` — the first in the dtype of ``hidden`` with zero rows at the last positions, the second fp32 —
        ``None`` for the one not asked for."""
        if self._call is None:
            raise RuntimeError("backward needs a forward first")
        h, hidden, weight, labels, loss = self._call
        dtype = hidden.storage.dtype
        d_hidden = d_weight = None
        h.d_inputs = h.d_hidden = h.d_weight = 0
        if need_hidden:
            d_hidden = DeviceStorage(hidden.storage.size, dtype, stream=self.stream)
            h.d_inputs = self._buffer("d_inputs", h.rows_bound * h.width, dtype).ptr
            h.d_hidden = d_hidden.ptr
        if need_weight:
            d_weight = DeviceStorage(weight.storage.size, "float32", stream=self.stream)
            h.d_weight = d_weight.ptr
        if not (need_hidden or need_weight):
            return None, None
        storage = getattr(gradient, "storage", gradient)
        if storage is not None and (storage.dtype != "float32" or storage.size != 1):
            raise ValueError("the incoming gradient must be one float32 value on the device")
        lib.call("qmoe_head_backward", ctypes.byref(h), 0 if storage is None else storage.ptr, self.stream)
        return (None if d_hidden is None else Tensor(d_hidden, hidden.shape),
                None if d_weight is None else Tensor(d_weight, weight.shape))


def projection_loss(hidden, weight, labels, chunk_size=None, *, prepared_labels=None, head=None):
    """Upstream's ``projection_loss`` (src/qutai/lm/layers.py:187-257): the mean cross-entropy of predicting token
    ``t + 1`` from position ``t``.  Returns the loss as a tensor recorded with parents ``(hidden, weight)``."""
    head = head or LMHead()
    loss = head.forward(hidden, weight, labels if prepared_labels is None else prepared_labels)

    def backward(gradient):
        d_hidden, d_weight = head.backward(gradient, need_hidden=getattr(hidden, "requires_grad", True),
                                           need_weight=getattr(weight, "requires_grad", True))
        return (None if d_hidden is None else d_hidden.storage, None if d_weight is None else d_weight.storage)

    loss.parents, loss.backward_rule = (hidden, weight), backward
    return loss


class PiecewiseHead(LMHead):
    """The mean cross-entropy of rows that have a target each, with the logits formed a piece of the vocabulary at a time, in the
    backward again, and never kept.  ``piece_bytes``: how much of them (of their gradient) there may be at a time.  ``operand_of``: an ``LMHead`` of the
    same weight, whose bfloat16 copy of it serves both.  A recorded call (``qmoe_graph_begin``) multiplies with the copy of a float32 weight as it is at each replay:
    after an update of the weight one plain ``forward`` renews it."""

    def __init__(self, stream=0, *, piece_bytes=256 << 20, operand_of=None):
        if piece_bytes <= 0:
            raise ValueError("piece_bytes must be positive")
        if operand_of is not None and operand_of.stream != stream:
            raise ValueError("heads that share a copy of their weight have one stream")
        super().__init__(stream)
        self.piece_bytes, self._operand_of = piece_bytes, operand_of

    def _weight_operand(self, weight, dtype):
        return super()._weight_operand(weight, dtype) if self._operand_of is None else self._operand_of._weight_operand(weight, dtype)

    def _piece(self, rows, vocab, item):
        """Classes of a piece: whole tiles, as many as fit ``piece_bytes``, the pieces as even as tiles allow."""
        most = max(256, self.piece_bytes // (rows * item) // 256 * 256)
        count = -(-vocab // most)
        return -(-(-(-vocab // count)) // 256) * 256

    def forward(self, hidden, weight, targets, *, out=None):
        """``hidden`` [..., width] (bfloat16 or float32), ``weight`` [vocab, width] of the same dtype, or float32 beside bfloat16 rows,
        ``targets`` an int64 device storage with the class that each row has to predict; any number that is no class (-100): none.  Returns the loss
        (float32, of one element; ``out``: the storage to write to): 0 where no row has a target."""
        if len(hidden.shape) < 2 or len(weight.shape) != 2 or weight.shape[1] != hidden.shape[-1]:
            raise ValueError("hidden must be [..., width] and weight [vocab, width]")
        (vocab, width), dtype = weight.shape, hidden.storage.dtype
        rows = hidden.storage.size // width if width else 0
        if dtype not in lib.DTYPE_CODES:
            raise ValueError("hidden must be float32 or bfloat16")
        if rows == 0 or vocab == 0:
            raise ValueError("the loss needs rows and classes")
        if targets.dtype != "int64" or targets.size != rows:
            raise ValueError("targets must hold one int64 class for each row")
        if out is not None and (out.dtype != "float32" or out.size != 1):
            raise ValueError("out must be a storage of one float32 value")
        operand = self._weight_operand(weight, dtype)
        item, bound = lib.ITEM_BYTES[dtype], -(-rows // ROW_PAD) * ROW_PAD
        # the rows kept for the backward are this call's own: another forward, recorded or not, leaves them alone
        self._call = None
        new = lambda size, kind: DeviceStorage(size, kind, stream=self.stream)  # noqa: E731
        kept = new(int(lib.load().qmoe_pieces_table_words(rows)), "int32"), new(bound * width, dtype), new(bound, "float32"), new(bound, "float32")
        loss = new(1, "float32") if out is None else out
        a = lib.Pieces(rows, width, vocab, self._piece(rows, vocab, item), lib.DTYPE_CODES[dtype], lib.DTYPE_CODES[weight.storage.dtype],
                       hidden.storage.ptr, operand.ptr, targets.ptr, loss.ptr, *(storage.ptr for storage in kept))
        scratch = self._scratch(a, 0)
        lib.call("qmoe_pieces_forward", ctypes.byref(a), self.stream)
        self._hold(scratch, operand, weight, kept)
        self._call = (a, hidden, weight, operand, targets, loss, kept)
        return Tensor(loss, ())

    def _hold(self, scratch, operand, weight, kept):
        """What a recorded call reads and writes beside its caller's storages: also after another loss has taken its place here."""
        for storage in (scratch, *kept, *(() if operand is weight.storage else (operand,))):
            done_with(storage, self.stream)

    def _scratch(self, a, backward):
        scratch = DeviceStorage(-(-int(lib.load().qmoe_pieces_scratch_bytes(ctypes.byref(a), backward)) // 4), "float32", stream=self.stream)
        a.scratch = scratch.ptr
        return scratch

    def backward(self, gradient=None, *, need_hidden=True, need_weight=True, out=None):
        """``gradient``: float32 device storage (or tensor) of one element, ``None`` = 1.  Returns ``(d_hidden, d_weight)`` of the
        last forward, in the dtypes of ``hidden`` and ``weight``, ``None`` for the one not asked for; rows without a target get zeros.  ``out``:
        two storages to write to instead of new ones.  ``hidden``, ``weight`` and ``targets`` may not have changed since the forward."""
        if self._call is None:
            raise RuntimeError("backward needs a forward first")
        a, hidden, weight, operand, targets, loss, kept = self._call
        if not (need_hidden or need_weight):
            return None, None
        storage = getattr(gradient, "storage", gradient)
        if storage is not None and (storage.dtype != "float32" or storage.size != 1):
            raise ValueError("the incoming gradient must be one float32 value on the device")
        results = []
        for i, (tensor, needed) in enumerate(((hidden, need_hidden), (weight, need_weight))):
            given = None if out is None else out[i]
            if needed and given is not None and (given.size != tensor.storage.size or given.dtype != tensor.storage.dtype):
                raise ValueError("out must be storages like hidden and weight")
            if needed and given is None:
                given = DeviceStorage(tensor.storage.size, tensor.storage.dtype, stream=self.stream)
            results.append(given if needed else None)
        a.gradient = 0 if storage is None else storage.ptr
        a.d_hidden, a.d_weight = (0 if result is None else result.ptr for result in results)
        scratch = self._scratch(a, 1)
        lib.call("qmoe_pieces_backward", ctypes.byref(a), self.stream)
        self._hold(scratch, operand, weight, kept)
        return tuple(None if result is None else Tensor(result, tensor.shape) for result, tensor in zip(results, (hidden, weight)))


def piecewise_projection_loss(hidden, weight, targets, *, head=None):
    """``PiecewiseHead``'s loss as a tensor recorded with parents ``(hidden, weight)``, like ``projection_loss``; ``targets``: int64 device
    storage, one class for each row of ``hidden``."""
    head = head or PiecewiseHead()
    loss = head.forward(hidden, weight, targets)
    call = head._call

    def backward(gradient):
        head._call = call           # of this loss, whatever the head has been used for since
        d_hidden, d_weight = head.backward(gradient, need_hidden=getattr(hidden, "requires_grad", True),
                                           need_weight=getattr(weight, "requires_grad", True))
        return (None if d_hidden is None else d_hidden.storage, None if d_weight is None else d_weight.storage)

    loss.parents, loss.backward_rule = (hidden, weight), backward
    return loss
