"""The operators of decoding many continuations of one prompt, as a list of measurable cases.

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, ``run`` is one pass through an
operator, ``work`` the bytes and operations that pass cannot do without, ``exact`` the operator's definition in 64 bits.
With ``own`` false ``run`` computes the operators from elementary torch operations in 32 bits; with ``own`` true it calls
``qutai_b200``.

Kinds of case:
  rotary     norm of every query and key head and the rotation of its position in one pass
             (``qutai_b200.rotary.norm_rope_forward``), with ``train`` its backward as well (``norm_rope_backward``)
  cache      new keys and values written behind the positions that each sequence of a key/value cache holds, quantised to
             8 bits as they are written, and everything the sequences then hold read back (``qutai_b200.kv_cache.KVCache``)
  attention  new queries of a batch over a prefix of keys and values that all sequences share and over each sequence's own
             cache (``qutai_b200.kv_cache.prefix_attention``)
  sample     one token a row by temperature, top-k, top-p and min-p from given uniform numbers (``qutai_b200.sampling.sample``)
"""
import math

import numpy as np
import torch

own = False

TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int8": torch.int8}
BYTES = {"float32": 4, "bfloat16": 2, "int8": 1}
EPS, THETA = 1e-6, 10000.0
ONE = 2.0 ** 31          # the weight of a row's largest logit, as a whole number (see _plain_sample)


# -- the cases ----------------------------------------------------------------------------------------------------
def _named(name, case):
    return case if name is None else dict(case, name=name)


def _rotary(name, batch, time, heads, kv_heads, dim, *, dtype="bfloat16", train=False, held=0):
    return _named(name, dict(kind="rotary", batch=batch, time=time, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, train=train, held=held))


def _cache(name, batch, time, kv_heads, dim, *, held, dtype="int8", source="bfloat16"):
    return _named(name, dict(kind="cache", batch=batch, time=time, kv_heads=kv_heads, dim=dim, held=held, dtype=dtype, source=source))


def _attention(name, batch, time, heads, kv_heads, dim, *, prefix, held, dtype="bfloat16"):
    return _named(name, dict(kind="attention", batch=batch, time=time, heads=heads, kv_heads=kv_heads, dim=dim, prefix=prefix, held=held, dtype=dtype))


def _sample(name, rows, vocab, *, dtype="bfloat16", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False):
    return _named(name, dict(kind="sample", rows=rows, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                             mixed=mixed))


def listed():
    return [
        # A step of decoding: one new position in each of 64 sequences, every sequence at a position of its own.
        _rotary("rotary_decode_64", 64, 1, 16, 4, 64, held=4096),
        # A training step of the 12-block model (4 x 2048 positions, 16 heads in 4 groups), forward and backward.
        _rotary("rotary_train", 4, 2048, 16, 4, 64, train=True),
        # float32 activations, wider heads, an odd number of positions: forward and backward.
        _rotary("rotary_train_float32", 3, 1003, 8, 2, 128, dtype="float32", train=True),
        # A step of decoding for 64 sequences of up to 300 positions: one position appended to each, all read back.
        _cache("cache_decode_64", 64, 1, 4, 64, held=300),
        # Prompts of up to 2048 positions written in one go and read back.
        _cache("cache_prefill", 4, 2048, 4, 64, held=0),
        # The smallest call: four continuations of a short prompt, a few positions each.
        _attention("attention_small", 4, 1, 16, 4, 64, prefix=512, held=16),
        # Decoding 64 continuations of a prompt of 4096 positions over an 8-bit cache.
        _attention("attention_decode_int8", 64, 1, 16, 4, 64, prefix=4096, held=512, dtype="int8"),
        # Five drafted positions a sequence checked in one pass, odd batch and prompt, wider heads, some sequences with less behind them.
        _attention("attention_verify", 13, 5, 8, 2, 128, prefix=1003, held=300),
        # Many continuations of a long document at width 2048: the largest pass.
        _attention("attention_large", 128, 1, 32, 8, 64, prefix=32768, held=1024),
        # One sequence, a 32000-token vocabulary, the usual settings of a chat.
        _sample("sample_one", 1, 32000, temperature=0.8, top_k=50, top_p=0.95),
        # A batch whose requests bring their own settings, greedy ones and masked tokens among them, float32 logits.
        _sample("sample_64_mixed", 64, 32000, dtype="float32", mixed=True),
        # A large batch over a wide vocabulary of odd size, truncated by mass alone.
        _sample("sample_256_wide", 256, 131071, top_p=0.9, min_p=0.02),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case from the ranges above: sizes log-uniform, most of them no multiple of a tile."""
    largest = work(_attention(None, 128, 1, 32, 8, 64, prefix=32768, held=1024))
    while True:
        case = _drawn(rng)
        if all(mine <= most for mine, most in zip(work(case).values(), largest.values())):
            return case


def _drawn(rng):
    kind = rng.choice(["rotary", "cache", "attention", "attention", "sample", "sample"])
    if kind == "rotary":
        kv_heads, train = rng.choice([1, 2, 3, 4, 8]), rng.random() < 0.5
        batch, time = _log(rng, 1, 64), 1 if not train and rng.random() < 0.4 else _log(rng, 1, 2048)
        time = min(time, max(1, 16384 // batch))
        return _rotary(None, batch, time, kv_heads * rng.choice([1, 2, 4]), kv_heads, rng.choice([32, 64, 64, 128]),
                       dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), train=train, held=0 if train else _log(rng, 1, 100000))
    if kind == "cache":
        batch, time = _log(rng, 1, 64), 1 if rng.random() < 0.4 else _log(rng, 1, 2048)
        held = rng.choice([0, _log(rng, 1, 2048)])
        time, held = min(time, max(1, 16384 // batch)), min(held, 32768 // batch)
        return _cache(None, batch, time, rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), held=held, dtype=rng.choice(["int8", "int8", "bfloat16"]),
                      source=rng.choice(["bfloat16", "float32"]))
    if kind == "attention":
        kv_heads, dtype = rng.choice([1, 2, 4, 8]), rng.choice(["bfloat16", "int8"])
        dim, time = rng.choice([64, 64, 128]), rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 256)])
        batch, prefix = _log(rng, 1, 128), 0 if rng.random() < 0.15 else _log(rng, 1, 32768)
        batch = min(batch, max(1, 1024 // time))
        held = min(_log(rng, 1, 1024), 131072 // batch)
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        return _attention(None, batch, time, heads, kv_heads, dim, prefix=prefix, held=held, dtype=dtype)
    vocab = _log(rng, 1000, 131072)
    rows = _log(rng, 1, 256)
    return _sample(None, rows, vocab, dtype=rng.choice(["bfloat16", "float32"]), temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                   top_k=rng.choice([0, 0, 1, 20, 200, vocab // 2]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.05, 0.5]),
                   mixed=rng.random() < 0.3)


# -- inputs -------------------------------------------------------------------------------------------------------
def _lengths(generator, case, low):
    """What each sequence holds: anything from ``low`` to ``held`` positions, the first as many as there may be."""
    held = case["held"]
    lengths = torch.randint(min(low, held), held + 1, (case["batch"],), generator=generator, device="cuda", dtype=torch.int32)
    lengths[0] = held
    return lengths


def _quantised(values):
    """8-bit values and the scale of every last axis."""
    scale = values.abs().amax(-1) / 127.0
    return torch.where(scale[..., None] > 0, values / scale[..., None], 0.0).round().clamp(-127, 127).to(torch.int8), scale


def _filled(generator, case, batch, capacity, lengths):
    """A cache as torch tensors, [batch, kv_heads, capacity, dim]: keys as a norm leaves them (with a channel that stands out),
    values around one half; zeros behind each sequence's length."""
    shape = (batch, case["kv_heads"], capacity, case["dim"])
    k = torch.randn(shape, generator=generator, device="cuda")
    k[..., 3] *= 4.0
    v = torch.randn(shape, generator=generator, device="cuda") * 0.5
    free = torch.arange(capacity, device="cuda")[None, :] >= lengths[:, None]
    for values in (k, v):
        values.masked_fill_(free[:, None, :, None], 0.0)
    if case["dtype"] == "bfloat16":
        return dict(k=k.to(torch.bfloat16), v=v.to(torch.bfloat16), lengths=lengths)
    (k, k_scale), (v, v_scale) = _quantised(k), _quantised(v)
    return dict(k=k, v=v, k_scale=k_scale, v_scale=v_scale, lengths=lengths)


def _inputs(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda shape, dtype="float32": torch.randn(shape, generator=generator, device="cuda").to(TORCH[dtype])  # noqa: E731
    kind, data = case["kind"], {}
    if kind == "rotary":
        shape, dim = (case["batch"], case["time"]), case["dim"]
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            data[name] = normal((*shape, heads * dim), case["dtype"])
            data[name + "_weight"] = 1.0 + 0.1 * normal((dim,))
            if case["train"]:
                data["d" + name] = normal((*shape, heads * dim), case["dtype"])
        if case["held"]:
            data["starts"] = _lengths(generator, case, 0)
    elif kind == "cache":
        shape, lengths = (case["batch"], case["time"], case["kv_heads"] * case["dim"]), _lengths(generator, case, 0)
        data.update(_filled(generator, case, case["batch"], case["held"] + case["time"], lengths))
        data["new_k"], data["new_v"] = normal(shape, case["source"]), normal(shape, case["source"])
        # prompts of different lengths lie side by side; a step of decoding has one position for everybody
        data["counts"] = torch.randint(1, case["time"] + 1, (case["batch"],), generator=generator, device="cuda", dtype=torch.int32)
        data["counts"][0] = case["time"]
    elif kind == "attention":
        data["q"] = normal((case["batch"], case["time"], case["heads"] * case["dim"]), "bfloat16")
        # the new positions' own keys are in the cache already: most sequences hold at least those
        lengths = _lengths(generator, dict(case, held=case["held"] + case["time"]), 1)
        if case["prefix"]:
            prefix = torch.full((1,), case["prefix"], device="cuda", dtype=torch.int32)
            data["prefix"] = _filled(generator, case, 1, case["prefix"], prefix)
        data["cache"] = _filled(generator, case, case["batch"], case["held"] + case["time"], lengths)
    else:
        rows, vocab = case["rows"], case["vocab"]
        data["logits"] = (2.5 * normal((rows, vocab))).to(TORCH[case["dtype"]])
        data["uniforms"] = torch.rand(rows, generator=generator, device="cuda")
        for name in ("temperature", "top_k", "top_p", "min_p"):
            data[name] = case[name]
        if case["mixed"]:      # every request with its own settings; some tokens are forbidden
            choose = lambda values: torch.tensor(values, device="cuda")[torch.randint(len(values), (rows,), generator=generator, device="cuda")]  # noqa: E731
            data["temperature"] = choose([0.0, 0.5, 0.8, 1.0, 1.3])
            data["top_k"] = choose([0, 1, 40, 500]).to(torch.int32)
            data["top_p"], data["min_p"] = choose([1.0, 0.95, 0.7]), choose([0.0, 0.0, 0.1])
            data["logits"].masked_fill_(torch.rand((rows, vocab), generator=generator, device="cuda") < 0.05, -math.inf)
    return data


def _storage(tensor):
    """A torch tensor as a storage of the package, over the same memory."""
    from qutai_b200.storage import DeviceStorage

    names = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.int8: "int8", torch.int32: "int32", torch.int64: "int64"}
    return DeviceStorage.wrap(tensor.data_ptr(), tensor.numel(), names[tensor.dtype], owner=tensor)


def _given(tensor):
    from qutai_b200.layers import Tensor

    return Tensor(_storage(tensor), tuple(tensor.shape))


def _handle(case, held, longest):
    """The package's cache over the tensors of ``held``."""
    from qutai_b200.kv_cache import KVCache

    batch, kv_heads, capacity, dim = held["k"].shape
    scales = {name: _storage(held[name]) for name in ("k_scale", "v_scale") if name in held}
    return KVCache(batch, capacity, kv_heads, dim, case["dtype"], k=_storage(held["k"]), v=_storage(held["v"]), lengths=_storage(held["lengths"]),
                   longest=longest, **scales)


def prepare(case, seed):
    """The inputs, the same for both forms; for the package's calls also the handles and output buffers that a program makes once."""
    data = _inputs(case, seed)
    state = dict(case=case, data=data)
    if not own:
        return state
    kind = case["kind"]
    empty = lambda shape, dtype: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
    if kind == "rotary":
        state["handles"] = {name: (_storage if name == "starts" else _given)(value) for name, value in data.items()}
        state["out"] = [torch.empty_like(data[name]) for name in ("q", "k")]
        if case["train"]:
            state["out"] += [torch.empty_like(data[name]) for name in ("q", "k", "q_weight", "k_weight")]
    elif kind == "cache":
        longest = case["held"] + case["time"]
        state["cache"] = _handle(case, data, case["held"])
        state["held"] = _storage(data["lengths"])
        state["new"] = _given(data["new_k"]), _given(data["new_v"])
        state["counts"] = _storage(data["counts"])
        shape = (case["batch"], longest, case["kv_heads"] * case["dim"])
        state["out"] = [empty(shape, torch.bfloat16), empty(shape, torch.bfloat16), empty((case["batch"],), torch.int32)]
    elif kind == "attention":
        state["q"] = _given(data["q"])
        state["prefix"] = _handle(case, data["prefix"], case["prefix"]) if "prefix" in data else None
        state["cache"] = _handle(case, data["cache"], case["held"] + case["time"])
        state["out"] = [torch.empty_like(data["q"]), empty((case["batch"], case["time"], case["heads"]), torch.float32)]
    else:
        state["logits"], state["uniforms"] = _given(data["logits"]), _storage(data["uniforms"])
        state["settings"] = {name: _storage(data[name]) if case["mixed"] else data[name] for name in ("temperature", "top_k", "top_p", "min_p")}
        state["out"] = [empty((case["rows"],), torch.int64), empty((case["rows"],), torch.float32)]
    state["buffers"] = [_storage(tensor) for tensor in state["out"]]
    return state


# -- the plain forms ----------------------------------------------------------------------------------------------
def _turn(case, data):
    """cos and sin of every position's angles, [batch, time, 1, dim / 2].  The angle is a place on the circle: it is formed in 64
    bits (at position 100000 32 bits leave it four digits), its cosine and sine are held in 32."""
    position = torch.arange(case["time"], device="cuda", dtype=torch.float64)[None, :]
    if "starts" in data:
        position = position + data["starts"].double()[:, None]
    angle = position[..., None, None] * THETA ** (-torch.arange(0, case["dim"], 2, device="cuda", dtype=torch.float64) / case["dim"])
    return angle.cos().float(), angle.sin().float()


def _rotated(x, cos, sin):
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * cos - odd * sin, even * sin + odd * cos), -1).flatten(-2)


def _plain_rotary(case, data):
    shape, dim = (case["batch"], case["time"], -1, case["dim"]), case["dim"]
    cos, sin = _turn(case, data)
    outputs, gradients, weights = [], [], []
    for name in ("q", "k"):
        x, weight = data[name].float().view(shape), data[name + "_weight"]
        inverse = torch.rsqrt((x * x).sum(-1, keepdim=True) / dim + EPS)
        normed = x * inverse
        outputs.append(_rotated(normed * weight, cos, sin).to(data[name].dtype).view(data[name].shape))
        if case["train"]:
            g = _rotated(data["d" + name].float().view(shape), cos, -sin)
            weights.append((g * normed).sum((0, 1, 2)))
            g = g * weight
            gradients.append((inverse * (g - normed * ((g * normed).sum(-1, keepdim=True) / dim))).to(data[name].dtype).view(data[name].shape))
    return outputs + gradients + weights


def _values(held, name):
    values = held[name].float()
    return values * held[name + "_scale"][..., None] if name + "_scale" in held else values


def _plain_cache(case, data):
    batch, time, kv_heads, dim = case["batch"], case["time"], case["kv_heads"], case["dim"]
    new = torch.arange(time, device="cuda")[None, :] < data["counts"][:, None]
    sequence, step = new.nonzero(as_tuple=True)
    position = data["lengths"][sequence] + step
    lengths = data["lengths"] + data["counts"]
    outputs = []
    for name in ("k", "v"):
        source = data["new_" + name].view(batch, time, kv_heads, dim)[sequence, step]
        if case["dtype"] == "int8":
            values, scale = _quantised(source.float())
            data[name][sequence, :, position] = values
            data[name + "_scale"][sequence, :, position] = scale
        else:
            data[name][sequence, :, position] = source.to(torch.bfloat16)
        held = torch.arange(case["held"] + time, device="cuda")[None, :] < lengths[:, None]
        values = torch.where(held[:, None, :, None], _values(data, name), 0.0)
        outputs.append(values.to(torch.bfloat16).transpose(1, 2).reshape(batch, case["held"] + time, kv_heads * dim))
    outputs.append(lengths)
    if case["dtype"] == "int8":
        outputs += [data["k_scale"], data["v_scale"]]
    return outputs


def _plain_attention(case, data):
    batch, time, kv_heads, dim = case["batch"], case["time"], case["kv_heads"], case["dim"]
    q = data["q"].float().view(batch, time, kv_heads, -1, dim) * dim ** -0.5
    cache, positions = data["cache"], case["held"] + time
    # query t of a sequence is its position length - time + t
    last = cache["lengths"][:, None] - time + torch.arange(time, device="cuda")
    seen = torch.arange(positions, device="cuda") <= last[..., None]
    scores = torch.einsum("btgrd,bgsd->btgrs", q, _values(cache, "k"))
    scores.masked_fill_(~seen[:, :, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if "prefix" in data:
        shared = torch.einsum("btgrd,gsd->btgrs", q, _values(data["prefix"], "k")[0])
        top = torch.maximum(top, shared.amax(-1, keepdim=True))
    base = torch.where(top > -math.inf, top, 0.0)
    weights = torch.exp(scores - base)
    total = weights.sum(-1, keepdim=True)
    out = torch.einsum("btgrs,bgsd->btgrd", weights, _values(cache, "v"))
    if "prefix" in data:
        weights = torch.exp(shared - base)
        total = total + weights.sum(-1, keepdim=True)
        out = out + torch.einsum("btgrs,gsd->btgrd", weights, _values(data["prefix"], "v")[0])
    out = torch.where(total > 0, out / total, 0.0)
    return [out.to(torch.bfloat16).view(data["q"].shape), (base + total.log()).view(batch, time, -1)]


def _per_row(value, rows, dtype):
    return value.to(dtype) if torch.is_tensor(value) else torch.full((rows,), value, device="cuda", dtype=dtype)


def _plain_sample(case, data):
    """A token's weight is exp((logit - largest) / temperature), held as a whole number of 2^-31: sums of whole numbers do not
    depend on their order, so the kept set and the token are the same in every implementation.  Logits that are not numbers
    are never drawn.  Kept are the ``top_k`` largest logits (of equal ones those of lower index), of these the shortest run
    from the largest that holds ``top_p`` of their weight, of these the ones that weigh ``min_p`` of the largest; drawn is the
    token at which the running sum of the kept weights, by index, passes uniform times their sum.  Temperature 0 takes
    the first of the largest, with the log-probability of temperature 1.  A row without a finite logit gives -1."""
    rows, vocab = data["logits"].shape
    temperature, uniform = _per_row(data["temperature"], rows, torch.float32), data["uniforms"]
    top_k, top_p, min_p = _per_row(data["top_k"], rows, torch.int64), _per_row(data["top_p"], rows, torch.float32), _per_row(data["min_p"], rows, torch.float32)
    logits = data["logits"].float()
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    largest = logits.amax(-1, keepdim=True)
    greedy = ~(temperature > 0)
    inverse = torch.where(greedy, 1.0, 1.0 / torch.where(greedy, 1.0, temperature))[:, None]
    apart = logits - largest
    weight = torch.exp(apart * inverse)
    weight = torch.where(logits == largest, 1.0, torch.where(apart == -math.inf, 0.0, weight))
    whole = (weight * ONE).round().to(torch.int64)
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(vocab, device="cuda")
    limit = torch.where((top_k <= 0) | (top_k > vocab), vocab, top_k)
    limit = torch.where(greedy, 1, limit)
    sorted_whole = torch.where(rank < limit[:, None], whole.gather(-1, order), 0)
    before = sorted_whole.cumsum(-1) - sorted_whole
    mass = sorted_whole.sum(-1)
    keep = (rank < limit[:, None]) & ((before == 0) | (top_p >= 1)[:, None] | (before.double() < top_p.double()[:, None] * mass.double()[:, None]))
    keep = keep & ~(weight.gather(-1, order) < min_p.clamp(max=1.0)[:, None])
    kept = torch.zeros_like(whole).scatter_(-1, order, torch.where(keep, sorted_whole, 0))
    running = kept.cumsum(-1)
    target = torch.minimum((uniform.double() * running[:, -1].double()).to(torch.int64), running[:, -1] - 1)
    token = (running <= target[:, None]).sum(-1)
    log_probability = ((apart.gather(-1, token.clamp(max=vocab - 1)[:, None]) * inverse)[:, 0].double() - (whole.sum(-1).double() / ONE).log()).float()
    none = largest[:, 0] == -math.inf
    return [torch.where(none, -1, token), torch.where(none, -math.inf, log_probability)]


PLAIN = {"rotary": _plain_rotary, "cache": _plain_cache, "attention": _plain_attention, "sample": _plain_sample}


# -- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return PLAIN[kind](case, state["data"])
    out, buffers = state["out"], state["buffers"]
    if kind == "rotary":
        from qutai_b200.rotary import norm_rope_backward, norm_rope_forward

        h = state["handles"]
        settings = dict(eps=EPS, theta=THETA, starts=h.get("starts"))
        norm_rope_forward(h["q"], h["k"], h["q_weight"], h["k_weight"], case["heads"], case["kv_heads"], out=buffers[:2], **settings)
        if case["train"]:
            norm_rope_backward(h["dq"], h["dk"], h["q"], h["k"], h["q_weight"], h["k_weight"], case["heads"], case["kv_heads"], out=buffers[2:], **settings)
        return out
    if kind == "cache":
        cache, data = state["cache"], state["data"]
        cache.rewind(state["held"], case["held"])
        cache.append(*state["new"], counts=state["counts"], lengths_out=buffers[2])
        cache.read(0, case["held"] + case["time"], out=buffers[:2])
        return out + ([data["k_scale"], data["v_scale"]] if case["dtype"] == "int8" else [])
    if kind == "attention":
        from qutai_b200.kv_cache import prefix_attention

        prefix_attention(state["q"], case["heads"], state["cache"], state["prefix"], out=buffers)
        return out
    from qutai_b200.sampling import sample

    sample(state["logits"], state["uniforms"], out=buffers, **state["settings"])
    return out


# -- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "rotary":
        values, size = case["batch"] * case["time"] * (case["heads"] + case["kv_heads"]) * case["dim"], BYTES[case["dtype"]]
        # forward: read and written; backward: input and gradient read, gradient written
        return {"bytes": float(values * size * (5 if case["train"] else 2)), "flops": values * (30.0 if case["train"] else 9.0)}
    if kind == "cache":
        row = 2 * case["kv_heads"] * case["dim"]                      # values of a position, keys and values together
        # stored: a scale of 4 bytes for each head's `dim` values of one byte, or two bytes a value
        stored = row + 8 * case["kv_heads"] if case["dtype"] == "int8" else 2 * row
        new, held = case["batch"] * (case["time"] + 1) / 2, case["batch"] * case["held"] / 2
        whole = case["batch"] * (case["held"] + case["time"])
        return {"bytes": new * (row * BYTES[case["source"]] + stored) + (new + held) * stored + whole * row * 2.0, "flops": 4.0 * row * (new + whole)}
    if kind == "attention":
        stored = 2 * case["kv_heads"] * (case["dim"] + 4 if case["dtype"] == "int8" else 2 * case["dim"])
        rows, own_positions = case["batch"] * case["time"] * case["heads"], case["time"] / 2 + (case["held"] + 1) / 2
        return {"bytes": stored * (case["prefix"] + case["batch"] * own_positions) + rows * (4.0 * case["dim"] + 4),
                "flops": 4.0 * case["dim"] * rows * (case["prefix"] + own_positions)}
    values = case["rows"] * case["vocab"]
    return {"bytes": float(values * BYTES[case["dtype"]] + 16 * case["rows"]), "flops": 4.0 * values}


# -- the definitions in 64 bits --------------------------------------------------------------------------------------
def _exact_rotary(case, data):
    """By complex numbers: a pair is a number, a rotation a factor of modulus one."""
    b, t, dim = case["batch"], case["time"], case["dim"]
    place = torch.arange(t, device="cuda", dtype=torch.float64).expand(b, t)
    if "starts" in data:
        place = place + data["starts"].to(torch.float64).reshape(b, 1)
    rate = torch.exp(torch.arange(dim // 2, device="cuda", dtype=torch.float64) * (-2.0 * math.log(THETA) / dim))
    factor = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), place.reshape(b, t, 1, 1) * rate)
    pairs = lambda x: torch.view_as_complex(x.reshape(b, t, -1, dim // 2, 2).contiguous())  # noqa: E731
    flat = lambda z: torch.view_as_real(z).reshape(b, t, -1)  # noqa: E731
    first, second, third = [], [], []
    for name in ("q", "k"):
        x, w = data[name].double().reshape(b, t, -1, dim), data[name + "_weight"].double()
        length = torch.sqrt(torch.mean(x ** 2, dim=-1, keepdim=True) + EPS)
        first.append(flat(pairs(x / length * w) * factor))
        if case["train"]:
            g = flat(pairs(data["d" + name].double()) * factor.conj()).reshape(b, t, -1, dim)
            third.append(torch.sum(g * x / length, dim=(0, 1, 2)))
            second.append((g * w / length - x * torch.mean(g * w * x, dim=-1, keepdim=True) / length ** 3).reshape(b, t, -1))
    return first + second + third


def _exact_cache(case, data):
    b, t, h, dim, total = case["batch"], case["time"], case["kv_heads"], case["dim"], case["held"] + case["time"]
    held, counts = data["lengths"].long(), data["counts"].long()
    at = torch.arange(total, device="cuda").reshape(1, total)
    fresh = (at >= held[:, None]) & (at < (held + counts)[:, None])
    outputs, scales = [], []
    for name in ("k", "v"):
        source = data["new_" + name].double().reshape(b, t, h, dim)
        picked = torch.gather(source, 1, (at - held[:, None]).clamp(0, t - 1)[:, :, None, None].expand(b, total, h, dim)).permute(0, 2, 1, 3)
        old = data[name].double()
        if case["dtype"] == "int8":
            old_scale = data[name + "_scale"].double()
            step = torch.amax(torch.abs(picked), dim=-1) / 127
            stored = torch.round(picked / torch.where(step == 0, 1.0, step)[..., None]) * step[..., None]
            scales.append(torch.where(fresh[:, None, :], step, old_scale))
            old = old * old_scale[..., None]
        else:
            stored = picked
        values = torch.where(fresh[:, None, :, None], stored, torch.where((at < held[:, None])[:, None, :, None], old, 0.0))
        outputs.append(values.permute(0, 2, 1, 3).reshape(b, total, h * dim))
    return outputs + [None] + scales


def _exact_attention(case, data):
    b, t, heads, g, dim = case["batch"], case["time"], case["heads"], case["kv_heads"], case["dim"]
    q = data["q"].double().reshape(b, t, g, heads // g, dim).permute(0, 2, 1, 3, 4)          # [b, g, t, r, dim]
    out = torch.empty((b, t, heads, dim), device="cuda", dtype=torch.float64)
    lse = torch.empty((b, t, heads), device="cuda", dtype=torch.float64)
    value = lambda held, name, n: held[name][n].double() * (held[name + "_scale"][n].double()[..., None] if name + "_scale" in held else 1.0)  # noqa: E731
    shared = [value(data["prefix"], name, 0) for name in ("k", "v")] if "prefix" in data else None
    for n in range(b):
        k, v = value(data["cache"], "k", n), value(data["cache"], "v", n)
        length = int(data["cache"]["lengths"][n])
        behind = 0
        if shared is not None:
            behind = shared[0].shape[1]
            k, v = torch.cat((shared[0], k), 1), torch.cat((shared[1], v), 1)
        rows = q[n].reshape(g, t * (heads // g), dim)
        s = torch.bmm(rows, k.transpose(1, 2)).reshape(g, t, heads // g, -1) / math.sqrt(dim)
        limit = (torch.arange(t, device="cuda") + (length - t + 1)).clamp(min=0) + behind
        s = torch.where(torch.arange(k.shape[1], device="cuda") < limit[None, :, None, None], s, -math.inf)
        log_sum = torch.logsumexp(s, -1)
        p = torch.where(limit[None, :, None, None] > 0, torch.exp(s - log_sum[..., None]), 0.0)
        o = torch.bmm(p.reshape(g, t * (heads // g), -1), v).reshape(g, t, heads // g, dim)
        out[n] = o.permute(1, 0, 2, 3).reshape(t, heads, dim)
        lse[n] = log_sum.permute(1, 0, 2).reshape(t, heads)
    return [out.reshape(b, t, heads * dim), lse]


def _exact_sample(case, data):
    """Row by row on the host; the token itself is no computed number, its log-probability is."""
    logits = data["logits"].double().cpu().numpy()
    rows, vocab = logits.shape
    setting = lambda name: data[name].double().cpu().numpy() if torch.is_tensor(data[name]) else np.full(rows, float(data[name]))  # noqa: E731
    temperature, top_k, top_p, min_p, uniform = (setting(name) for name in ("temperature", "top_k", "top_p", "min_p", "uniforms"))
    if not torch.is_tensor(data["top_p"]):                   # the operators hold a setting in 32 bits
        temperature, top_p, min_p = (np.float32(values).astype(np.float64) for values in (temperature, top_p, min_p))
    result = np.empty(rows)
    for n in range(rows):
        x = logits[n]
        if not np.isfinite(x).any():
            result[n] = -math.inf
            continue
        greedy = temperature[n] <= 0
        z = (x - x.max()) / (1.0 if greedy else temperature[n])
        p = np.exp(z)
        order = np.argsort(-x, kind="stable")
        if greedy:
            order = order[:1]
        elif 0 < top_k[n] < vocab:
            order = order[:int(top_k[n])]
        mass = p[order]
        if top_p[n] < 1:
            order = order[np.cumsum(mass) - mass < top_p[n] * mass.sum()]
        order = np.sort(order[p[order] >= min_p[n]])
        running = np.cumsum(p[order])
        token = order[min(np.searchsorted(running, uniform[n] * running[-1], side="right"), len(order) - 1)]
        result[n] = z[token] - math.log(p.sum())
    return [None, result]


def exact(case, seed):
    data = _inputs(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_rotary(case, data)
    if kind == "cache":
        return _exact_cache(case, data)
    if kind == "attention":
        return _exact_attention(case, data)
    return _exact_sample(case, data)
