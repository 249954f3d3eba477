"""``AdamW`` and ``clip_grad_norm`` for parameters that live on the device, mirroring the upstream
optimizer interface (src/qutai/nn/optimizers.py:19-31, :121-153): per-parameter step counters and moments,
parameters whose ``grad`` is ``None`` are skipped, ``clip_grad_norm`` returns the norm before clipping.

Upstream launches one kernel per parameter tensor; here every tensor that has a gradient goes into one
table and one launch (``qmoe_adamw_multi`` / ``qmoe_clip_grad_norm``).  When ``shadows`` maps a parameter
to a bf16 storage, the step also writes the rounded parameter there, so a layer whose tensor-core operands
are those storages need not convert its weights again (``SparseMoE.operand_shadows``).

``AdamW(..., state_bits=8)`` holds both moments in 8 bits with a scale for every 256 elements (``qmoe_adamw_bytes``): 2 bytes and a
thirty-second of state an element instead of 8.
"""
from __future__ import annotations

import ctypes
import struct
from itertools import chain
from math import isfinite

from . import lib
from .storage import DeviceStorage, done_with


def _parameters(source):
    """A model, a layer or an iterable of tensors; a shared parameter is kept once (upstream ``_parameters``)."""
    if hasattr(source, "parameters"):
        source = source.parameters()
    return tuple(dict.fromkeys(source))


_ITEM = "5Q2q2f"       # lib.OptimItem: values, grad, exp_avg, exp_avg_sq, shadow, size, first_chunk, c1, c2
_BYTE_ITEM = "9Q2q2fQq"    # lib.ByteItem: values, grad, average, its scale, root, its scale, shadow, two outputs, size, first_chunk, step, root_factor, count, number
STATE_BLOCK = 256      # elements of an 8-bit moment that share a scale


class _Table:
    """Host item array plus the device buffer it is copied into, grown on demand."""

    def __init__(self, stream, kind=lib.OptimItem, layout=_ITEM):
        self.capacity, self.items, self.device, self.stream = 0, None, None, stream
        self.kind, self.layout = kind, layout

    def fill(self, rows):
        if len(rows) > self.capacity:
            self.capacity = max(64, 2 * len(rows))
            self.items = (self.kind * self.capacity)()
            self.device = DeviceStorage(self.capacity * ctypes.sizeof(self.kind) // 4, "int32", stream=self.stream)
        struct.pack_into(self.layout * len(rows), self.items, 0, *chain.from_iterable(rows))
        return self.items, len(rows), self.device.ptr


class ByteState:
    """One moment of a parameter in 8 bits: ``codes`` (int8 storage, one for each element) and ``scales`` (float32, one for every
    ``STATE_BLOCK`` elements).  The first moment's codes are e4m3 numbers; the second moment is held by its root, whose codes are numbers of 4 exponent and
    4 mantissa bits without a sign (``qmoe_adamw_bytes`` in the header says which).  ``AdamW.values_of_states`` gives what they stand for; a checkpoint holds the
    codes and scales themselves (``checkpoint.save_sharded`` takes both), since values do not lead back to their codes."""

    def __init__(self, codes, scales):
        if codes.dtype != "int8" or scales.dtype != "float32" or scales.size != -(-codes.size // STATE_BLOCK):
            raise ValueError(f"a state is int8 codes and one float32 scale for every {STATE_BLOCK} of them")
        self.codes, self.scales = codes, scales

    @classmethod
    def zeros(cls, size, stream=0):
        return cls(DeviceStorage.zeros(size, "int8", stream), DeviceStorage.zeros(-(-size // STATE_BLOCK), "float32", stream))


def clip_grad_norm(parameters, max_norm=1.0, *, stream=0, scratch=None):
    """Scale all gradients so that their joint L2 norm is at most ``max_norm``; returns the norm before
    clipping (reading it waits for the device, as upstream's download does)."""
    if not isfinite(max_norm) or max_norm < 0:
        raise ValueError("max_norm must be a non-negative finite number")
    gradients = [p.grad for p in _parameters(parameters) if p.grad is not None]
    if not gradients:
        return 0.0
    if any(g.dtype != "float32" for g in gradients):
        raise ValueError("gradients must be float32")
    table = _Table(stream)
    items, count, device = table.fill([(0, g.storage.ptr, 0, 0, 0, g.storage.size, 0, 1.0, 1.0) for g in gradients])
    scratch = scratch or DeviceStorage(int(lib.load().qmoe_clip_scratch_bytes()) // 4, "int32", stream=stream)
    lib.call("qmoe_clip_grad_norm", items, count, device, float(max_norm), scratch.ptr, stream)
    host = (ctypes.c_double * 2)()
    lib.call("qmoe_memcpy_d2h", ctypes.cast(host, ctypes.c_void_p), scratch.ptr, 16, stream)
    lib.call("qmoe_stream_sync", stream)
    norm = float(host[0])
    if not isfinite(norm):
        raise ValueError("the gradients contain non-finite values")
    return norm


def clip_grad_norm_sharded(replicated, sharded, max_norm=1.0, *, stream=0):
    """``clip_grad_norm`` for one rank of an expert-parallel job (no counterpart upstream, which is single-device):
    the gradients of ``replicated`` parameters are the same on every rank and count once, those of ``sharded``
    parameters (this rank's experts) exist only here and count together with the other ranks'.  Every rank calls it
    at the same point; all return the same norm and scale by the same factor.  Built from the single-rank kernels:
    two passes that only measure (replicated, sharded), one all-reduce of the sharded square, and one pass over all
    local gradients whose limit is chosen so that the kernel's own ``max_norm / norm`` comes out as
    ``max_norm / joint norm``."""
    if not isfinite(max_norm) or max_norm < 0:
        raise ValueError("max_norm must be a non-negative finite number")
    replicated, sharded = _parameters(replicated), _parameters(sharded)
    measure_only = 1.7e308      # the largest limit the kernel takes: nothing is scaled, the norm is reported
    norm_replicated = clip_grad_norm(replicated, measure_only, stream=stream)
    norm_sharded = clip_grad_norm(sharded, measure_only, stream=stream)
    square = DeviceStorage.from_values([norm_sharded * norm_sharded], "float32", stream)
    lib.call("qmoe_ep_all_reduce_f32", square.ptr, 1, stream)
    joint = (norm_replicated * norm_replicated + float(square.tolist(stream)[0])) ** 0.5
    if not isfinite(joint):
        raise ValueError("the gradients contain non-finite values")
    local = (norm_replicated * norm_replicated + norm_sharded * norm_sharded) ** 0.5
    if joint > max_norm and local > 0:
        # the kernel scales by limit / local when local > limit: limit = max_norm * local / joint gives max_norm / joint
        clip_grad_norm(tuple(replicated) + tuple(sharded), max_norm * local / joint, stream=stream)
    return joint


class AdamW:
    """Adam with decoupled weight decay; state per parameter object (``steps``, ``averages``,
    ``square_averages``), created when the parameter first has a gradient.  ``state_bits``: 32, averages in float32
    storages, or 8, averages as ``ByteState`` (learning rate and epsilon are then read as they are at each step, like the others).

    A step with 8-bit states on a stream of its own can be recorded (``qmoe_graph_begin``), once one has been taken by itself, for up to 32 parameters with
    gradients.  Each replay is the next step, counted on the device, from what the same gradient storages hold then, with the recorded learning rate and
    settings.  ``replayed()`` tells the host about replays."""

    def __init__(self, parameters, *, learning_rate=0.001, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 shadows=None, stream=0, state_bits=32):
        if state_bits not in (8, 32):
            raise ValueError("the moments are held in 8 or in 32 bits")
        if learning_rate < 0 or weight_decay < 0 or eps < 0:
            raise ValueError("learning rate, weight decay and eps must not be negative")
        if len(betas) != 2 or any(beta < 0 or beta >= 1 for beta in betas):
            raise ValueError("betas must be two numbers in [0, 1)")
        self.parameters = _parameters(parameters)
        if any(p.dtype != "float32" for p in self.parameters):
            raise ValueError("parameters must be float32")
        self.learning_rate, self.betas, self.eps, self.weight_decay = learning_rate, tuple(betas), eps, weight_decay
        self.shadows = dict(shadows or {})
        self.stream = stream
        self.steps, self.averages, self.square_averages = {}, {}, {}
        self.state_bits = state_bits
        self._table = _Table(self.stream) if state_bits == 32 else _Table(self.stream, lib.ByteItem, _BYTE_ITEM)
        self._values_table = _Table(self.stream, lib.ByteItem, _BYTE_ITEM)
        # 8 bits on a stream that can be recorded: two words on the device for each parameter, of which the first is its steps; what ``steps`` was when they were
        # written; and whether a recording counts there, so that the host's number may be behind
        self._counts, self._counted, self._recorded = None, {}, False

    def _state(self, states, parameter):
        """The parameter's moment in ``states``, zeros before its first step."""
        size, state = parameter.storage.size, states.get(parameter)
        if state is None:
            make = DeviceStorage.zeros if self.state_bits == 32 else ByteState.zeros
            state = states[parameter] = make(size, stream=self.stream)
        elif self.state_bits == 8 and (not isinstance(state, ByteState) or state.codes.size != size):
            raise ValueError("an 8-bit state must be a ByteState of its parameter's size")
        return state

    def _row(self, parameter, gradient, shadow, step, count=0, number=0):
        beta1, beta2 = self.betas
        average, square = self._state(self.averages, parameter), self._state(self.square_averages, parameter)
        shadow = 0 if shadow is None else shadow.ptr
        if self.state_bits == 32:
            return (parameter.storage.ptr, gradient.storage.ptr, average.ptr, square.ptr, shadow, parameter.storage.size, 0,
                    1 - beta1 ** step, 1 - beta2 ** step)
        return (parameter.storage.ptr, gradient.storage.ptr, average.codes.ptr, average.scales.ptr, square.codes.ptr, square.scales.ptr, shadow, 0, 0,
                parameter.storage.size, 0, self.learning_rate / (1 - beta1 ** step), (1 - beta2 ** step) ** -0.5, count, number)

    def values_of_states(self, out=None):
        """``{parameter: (average, square average)}`` as float32 storages, what 8-bit states stand for, in one launch, to be looked at or compared.  ``out``:
        such a dict, of the storages to write to (all parameters that have a state, or some of them)."""
        if self.state_bits != 8:
            if out is not None:
                raise ValueError("states of 32 bits are the values themselves")
            return {parameter: (average, self.square_averages[parameter]) for parameter, average in self.averages.items()}
        if out is None:
            out = {parameter: tuple(DeviceStorage(parameter.storage.size, "float32", stream=self.stream) for _ in range(2)) for parameter in self.averages}
        rows = []
        for parameter, (average_out, square_out) in out.items():
            if parameter not in self.averages:
                raise ValueError("a parameter without a state has no values")
            average, square, size = self._state(self.averages, parameter), self._state(self.square_averages, parameter), parameter.storage.size
            if any(s.dtype != "float32" or s.size != size for s in (average_out, square_out)):
                raise ValueError("a state's values are float32 and as many as its parameter's")
            rows.append((0, 0, average.codes.ptr, average.scales.ptr, square.codes.ptr, square.scales.ptr, 0, average_out.ptr, square_out.ptr, size, 0, 0.0, 0.0, 0, 0))
        if rows:
            items, count, device = self._values_table.fill(rows)
            lib.call("qmoe_byte_values", items, count, device, self.stream)
            for pair in out.values():
                for storage in pair:
                    storage.touch()
        return out

    def zero_grad(self):
        for parameter in self.parameters:
            parameter.zero_grad()

    def step(self):
        beta1, beta2 = self.betas
        rows, updated, steps = [], [], {}
        counting = self.state_bits == 8 and self.stream != 0
        recording = counting and bool(lib.load().qmoe_stream_capturing(self.stream))
        for i, parameter in enumerate(self.parameters):
            gradient = parameter.grad
            if gradient is None:
                continue
            if gradient.storage.size != parameter.storage.size or gradient.dtype != "float32":
                raise ValueError("a gradient must be float32 and have its parameter's size")
            step = self.steps.get(parameter, 0) + 1
            shadow = self.shadows.get(parameter)
            if shadow is not None and (shadow.dtype != "bfloat16" or shadow.size != parameter.storage.size):
                raise ValueError("a shadow must be a bfloat16 storage of its parameter's size")
            kept = number = 0
            if counting:
                in_step = parameter in self._counted and self._counted[parameter] == step - 1
                if recording and not (in_step and parameter in self.averages and parameter in self.square_averages):
                    raise RuntimeError("a step is recorded after one by itself, from the states and the number of steps that it left")
                if self._counts is None:
                    self._counts = DeviceStorage.zeros(2 * len(self.parameters), "int64", self.stream)
                kept, number = self._counts.ptr + 16 * i, 0 if recording or (self._recorded and in_step) else step
            rows.append(self._row(parameter, gradient, shadow, step, kept, number))
            steps[parameter] = step
            updated.append((parameter.storage, shadow))
        if not rows:
            return
        items, count, device = self._table.fill(rows)
        written = self._written(updated)
        lib.call("qmoe_adamw_multi" if self.state_bits == 32 else "qmoe_adamw_bytes", items, count, device, self.learning_rate, beta1, beta2, self.eps,
                 self.weight_decay, self.stream)
        if recording:       # nothing has run; the states and the counts live as long as the recording
            self._recorded = True
            for parameter in steps:
                for state in (self.averages[parameter], self.square_averages[parameter]):
                    done_with(state.codes, self.stream)
                    done_with(state.scales, self.stream)
            done_with(self._counts, self.stream)
            return
        self.steps.update(steps)
        if counting:
            self._counted.update(steps)
        self._mark(written)

    @staticmethod
    def _written(updated):
        """Change tracking (storage.py), before a step is launched: the parameters' generation grows.  A bf16 copy that was current before the
        step and whose every updated part was rewritten by this launch is current afterwards as well; a copy of
        an allocation in which some updated parameter had no shadow is left stale for its owner to rebuild."""
        groups = {}
        for master, shadow in updated:
            group = groups.setdefault(id(master._root), dict(master=master, shadows={}, complete=True))
            if shadow is None:
                group["complete"] = False
            else:
                group["shadows"][id(shadow._root)] = shadow
        for group in groups.values():
            group["current"] = [s for s in group["shadows"].values() if group["complete"] and len(group["shadows"]) == 1
                                and s.is_derived_from(group["master"])]
        return list(groups.values())

    @staticmethod
    def _mark(written):
        for group in written:
            group["master"].touch()
            for shadow in group["current"]:
                shadow.mark_derived_from(group["master"])

    def replayed(self):
        """Behind replays of recorded steps: waits for them, brings ``steps`` up to date with the device, and marks as changed the parameters that they wrote (bf16 copies
        in ``shadows`` were written with them)."""
        if self._counts is None:
            return
        counts, updated = self._counts.tolist(self.stream), []
        for i, parameter in enumerate(self.parameters):
            taken = counts[2 * i]
            if parameter in self._counted and taken != self._counted[parameter]:
                self.steps[parameter] = self._counted[parameter] = taken
                updated.append((parameter.storage, self.shadows.get(parameter)))
        self._mark(self._written(updated))
