"""The operators of training on packed documents in little memory, as a list of measurable cases.

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, ``run`` is one pass through an
operator, ``work`` the bytes and operations that pass cannot do without, ``exact`` the operator's definition in 64 bits.
With ``own`` false ``run`` computes the operators from elementary torch operations in 32 bits; with ``own`` true it calls
``qutai_b200``.

Kinds of case:
  rotary     query and key heads turned by the angles of each row's own position: pairs side by side or in halves, part of a
             head, frequencies scaled for long contexts (``qutai_b200.rotary.rotate_forward``), with ``train`` its backward too
             (``rotate_backward``)
  attention  causal attention within each of many sequences that lie behind one another in one batch of rows
             (``qutai_b200.attention.packed_attention_forward``), with ``train`` its backward too (``packed_attention_backward``)
  loss       softmax cross entropy over a vocabulary, its logits formed a piece of the vocabulary at a time and never kept, and
             the gradients of the hidden rows and of the table (``qutai_b200.head.PiecewiseHead``)
  adamw      one step over many tensors with both moments held in 8 bits (``qutai_b200.optim.AdamW(state_bits=8)``), and what the
             moments then stand for, as a checkpoint holds them
"""
import math

import torch

own = False

TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "bfloat16": 2}
THETA = 10000.0
BANDS = dict(factor=8.0, original=4096, low=1.0, high=4.0)         # the scaling of the cases that have one
RATE, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
BLOCK = 256                                                        # elements of a moment that share a scale
LARGEST = 448.0, 491520.0                                          # largest values of the first and second moment's codes


# -- the cases ----------------------------------------------------------------------------------------------------
def _named(name, case):
    return case if name is None else dict(case, name=name)


def _rotary(name, rows, heads, kv_heads, dim, *, turned, layout, scaled=False, far=0, dtype="bfloat16", train=False):
    return _named(name, dict(kind="rotary", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, turned=turned, layout=layout, scaled=scaled, far=far,
                             dtype=dtype, train=train))


def _attention(name, lengths, heads, kv_heads, dim, *, train=True, spare=0):
    return _named(name, dict(kind="attention", lengths=",".join(map(str, lengths)), heads=heads, kv_heads=kv_heads, dim=dim, train=train, spare=spare))


def _loss(name, rows, width, vocab, *, dtype="bfloat16", none=0.0):
    return _named(name, dict(kind="loss", rows=rows, width=width, vocab=vocab, dtype=dtype, none=none))


def _adamw(name, sizes, *, shadow=True, steps=10, tight=False):
    return _named(name, dict(kind="adamw", sizes=",".join(map(str, sizes)), shadow=shadow, steps=steps, tight=tight))


def listed():
    return [
        # A step of decoding: one position in each of 64 sequences, far apart, frequencies scaled for a long context.
        _rotary("rotary_decode_64", 64, 16, 4, 64, turned=64, layout="halves", scaled=True, far=100000),
        # A training step of the 12-block model (8192 positions, 16 heads in 4 groups), documents packed: forward and backward.
        _rotary("rotary_train", 8192, 16, 4, 64, turned=64, layout="interleaved", train=True),
        # float32 activations, wide heads of which a part is turned, an odd number of rows: forward and backward.
        _rotary("rotary_train_part", 3001, 8, 2, 128, turned=48, layout="halves", dtype="float32", train=True),
        # The smallest call: a handful of short documents, one of them empty, one a single token, rows behind the last one.
        _attention("attention_small", [1, 7, 0, 33, 130], 8, 2, 64, spare=21),
        # A training step of the 12-block model on documents as they come: a few long ones, many short ones.
        _attention("attention_train", [2048, 1501, 1024, 777, 640, 512, 400, 333, 257, 200, 150, 129, 100, 64, 31, 17, 9], 16, 4, 64),
        # Wide heads, every query head with a key head of its own, odd lengths.
        _attention("attention_train_wide", [1999, 1003, 600, 301, 130, 66], 8, 8, 128),
        # Prompts of very different lengths run in one go before decoding: the longest sequences, forward alone.
        _attention("attention_prompts", [8192, 4096, 2048, 1200, 801, 47], 32, 8, 128, train=False),
        # float32 activations, a small odd vocabulary, a quarter of the rows without a target.
        _loss("loss_float32", 301, 256, 5003, dtype="float32", none=0.25),
        # A training step of the 12-block model: 32000 classes, document ends without a target.
        _loss("loss_train", 8192, 1024, 32000, none=0.002),
        # A wide model over a large vocabulary of odd size, most of an instruction's rows without a target.
        _loss("loss_wide", 8191, 2048, 131071, none=0.5),
        # A few small tensors, sizes that end inside a block: what a call costs at least.
        _adamw("adamw_small", [64, 1000, 4096, 513, 1], shadow=False, tight=True),
        # A model's table, its projections, its experts and their norms.
        _adamw("adamw_model", [32768000] + [1048576, 262144, 262144, 1048576, 16384, 1024, 1024] * 12 + [33554432] * 6 + [1024]),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case from the ranges above: sizes log-uniform, most of them no multiple of a tile."""
    most = {}
    for case in listed():
        for name, amount in work(case).items():
            most[case["kind"], name] = max(most.get((case["kind"], name), 0), amount)
    while True:
        case = _drawn(rng)
        if all(amount <= most[case["kind"], name] for name, amount in work(case).items()):
            return case


def _drawn(rng):
    kind = rng.choice(["rotary", "attention", "attention", "loss", "loss", "adamw"])
    if kind == "rotary":
        kv_heads, train, dim = rng.choice([1, 2, 3, 4, 8]), rng.random() < 0.6, rng.choice([32, 64, 64, 96, 128, 256])
        turned = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        return _rotary(None, _log(rng, 1, 8192), kv_heads * rng.choice([1, 2, 4]), kv_heads, dim, turned=turned, layout=rng.choice(["interleaved", "halves"]),
                       scaled=rng.random() < 0.5, far=rng.choice([0, _log(rng, 1, 100000)]), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), train=train)
    if kind == "attention":
        kv_heads, train, dim = rng.choice([1, 2, 4, 8]), rng.random() < 0.7, rng.choice([64, 64, 128])
        heads = kv_heads * rng.choice([1, 2, 3, 4])
        lengths = [_log(rng, 64, 4096 if train else 8192)] + [rng.choice([0, 1, _log(rng, 1, 2048), _log(rng, 1, 2048)]) for _ in range(rng.randint(0, 12))]
        rng.shuffle(lengths)
        return _attention(None, lengths, heads, kv_heads, dim, train=train, spare=rng.choice([0, 0, rng.randint(1, 200)]))
    if kind == "loss":
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        rows, width, vocab = _log(rng, 1, 8192), 8 * _log(rng, 8, 256), _log(rng, 500, 131072)
        if dtype == "float32":
            rows, width, vocab = min(rows, 700), min(width, 512), min(vocab, 12000)
        return _loss(None, rows, width, vocab, dtype=dtype, none=rng.choice([0.0, 0.01, 0.3, 0.8]))
    sizes = [_log(rng, 1, 1 << 24) for _ in range(rng.randint(1, 40))]
    return _adamw(None, sizes, shadow=rng.random() < 0.7, steps=_log(rng, 1, 10000), tight=rng.random() < 0.2)


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _places(case):
    """Where each tensor of an adamw case lies in the flat buffers that hold all of them, and how long those are."""
    places, end = [], 0
    for size in map(int, case["sizes"].split(",")):
        places.append(slice(end, end + size))
        end += size if case["tight"] else -(-size // 64) * 64
    return places, end


# -- the second moment's codes ----------------------------------------------------------------------------------------
# The root of the second moment is held as a number of 4 exponent and 4 mantissa bits without a sign: code c stands for
# c below 16 and for (16 + c % 16) 2^(c / 16 - 1) from there on, whole numbers up to 491520 (code 254); 255 is no number.
def _root_values(codes):
    c = codes.to(torch.int32) & 255
    power, part = (c >> 4).clamp(min=1), c & 15
    value = torch.where(c < 16, part, (16 + part) << (power - 1)).float()
    return torch.where(c == 255, math.nan, value)


def _root_codes(q):
    """Nearest code, ties to the even one; a positive value never becomes 0 (it divides)."""
    bits = q.view(torch.int32)
    high = ((bits + 0x3FFFF + ((bits >> 19) & 1)) >> 19) - 2080
    code = torch.where(q < 16, torch.where(q > 0, q.round().clamp(min=1), 0.0).to(torch.int32), high)
    return torch.where(torch.isfinite(q), code, 255).to(torch.uint8).view(torch.int8)


def _blocks(values):
    return torch.nn.functional.pad(values, (0, -values.numel() % BLOCK)).view(-1, BLOCK)


def _encoded(values, largest, floor, code):
    """Codes of a vector and the scale of every block of it; values that are no finite numbers have no part in the scale."""
    blocks = _blocks(values)
    top = torch.where(torch.isfinite(blocks), blocks.abs(), 0.0).amax(-1)
    held = top > floor
    inverse = torch.where(held, torch.full_like(top, largest) / top, 0.0)
    scaled = torch.where(torch.isfinite(blocks), blocks * inverse[:, None], math.nan)
    return code(scaled).view(-1)[:values.numel()], torch.where(held, top * (1.0 / largest), 0.0)


def _signed_codes(q):
    return q.to(torch.float8_e4m3fn).view(torch.int8)


def _signed_values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _decoded(values, scales):
    return (_blocks(values) * scales[:, None]).view(-1)[:values.numel()]


# -- inputs -------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda shape, dtype="float32": torch.randn(shape, generator=generator, device="cuda").to(TORCH[dtype])  # noqa: E731
    uniform = lambda shape: torch.rand(shape, generator=generator, device="cuda")  # noqa: E731
    kind, data = case["kind"], {}
    if kind == "rotary":
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            shape = (case["rows"], heads * case["dim"])
            data[name] = normal(shape, case["dtype"])
            if case["train"]:
                data["d" + name] = normal(shape, case["dtype"])
        # sequences at places of their own, or documents one behind the other, each from position 0 on
        places = (uniform((case["rows"],)) * case["far"]).to(torch.int32)
        row = torch.arange(case["rows"], device="cuda", dtype=torch.int32)
        starts = torch.where(uniform((case["rows"],)) < 0.005, row, 0)
        data["positions"] = places if case["far"] else (row - starts.cummax(0).values).to(torch.int32)
    elif kind == "attention":
        rows = sum(_lengths(case)) + case["spare"]
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"]), ("v", case["kv_heads"]), ("dout", case["heads"])):
            data[name] = normal((rows, heads * case["dim"]), "bfloat16")
    elif kind == "loss":
        data["hidden"] = normal((case["rows"], case["width"]), case["dtype"])
        data["weight"] = (normal((case["vocab"], case["width"])) * (2.0 * case["width"] ** -0.5)).to(TORCH[case["dtype"]])
        targets = torch.randint(case["vocab"], (case["rows"],), generator=generator, device="cuda")
        data["targets"] = torch.where(uniform((case["rows"],)) < case["none"], -100, targets)
    else:
        places, total = _places(case)
        flat = lambda dtype=torch.float32: torch.zeros(total, device="cuda", dtype=dtype)  # noqa: E731
        data.update(values=flat(), tensors=[])
        if case["shadow"]:
            data["shadow"] = flat(torch.bfloat16)
        for place in places:
            size, values = place.stop - place.start, data["values"][place]
            level = torch.exp(1.5 * normal((size,)))            # gradients of very different sizes beside one another
            gradient = 1e-3 * level * normal((size,))
            average, average_scale = _encoded(3e-4 * level * normal((size,)), LARGEST[0], 2.0 ** -100, _signed_codes)
            root, root_scale = _encoded(1e-3 * level, LARGEST[1], 0.0, _root_codes)
            values.copy_(0.02 * normal((size,)))
            held = dict(place=place, values=values, gradient=gradient, average=average, average_scale=average_scale, root=root, root_scale=root_scale)
            if case["shadow"]:
                held["shadow"] = data["shadow"][place].copy_(values)
            data["tensors"].append(held)
    return data


def _storage(tensor):
    """A torch tensor as a storage of the package, over the same memory."""
    from qutai_b200.storage import DeviceStorage

    names = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.int8: "int8", torch.int32: "int32", torch.int64: "int64"}
    return DeviceStorage.wrap(tensor.data_ptr(), tensor.numel(), names[tensor.dtype], owner=tensor)


def _given(tensor, shape=None):
    from qutai_b200.layers import Tensor

    return Tensor(_storage(tensor), tuple(shape or tensor.shape))


def prepare(case, seed):
    """The inputs, the same for both forms, with the buffers that outputs go to; for the package's calls also the handles that a
    program makes once."""
    data = _inputs(case, seed)
    state = dict(case=case, data=data)
    kind = case["kind"]
    empty = lambda shape, dtype=torch.float32: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
    if kind == "rotary":
        state["out"] = [torch.empty_like(data[name]) for name in ("q", "k")] * (2 if case["train"] else 1)
        state["out"] = [torch.empty_like(tensor) for tensor in state["out"]]
    elif kind == "attention":
        rows = data["q"].shape[0]
        state["out"] = [torch.zeros_like(data["q"]), torch.zeros((rows, case["heads"]), device="cuda")]      # rows behind the last sequence stay as they are
        if case["train"]:
            state["out"] += [torch.zeros_like(data[name]) for name in ("q", "k", "v")]
    elif kind == "loss":
        state["out"] = [empty((1,)), torch.empty_like(data["hidden"]), torch.empty_like(data["weight"])]
    else:
        state["step"] = case["steps"]
        state["out"] = [data["values"], torch.zeros_like(data["values"]), torch.zeros_like(data["values"])] + ([data["shadow"]] if case["shadow"] else [])
    if own:
        _handles(case, data, state)
    return state


def _handles(case, data, state):
    kind = case["kind"]
    if kind == "rotary":
        from qutai_b200.rotary import Rotation, Scaling

        state["rotation"] = Rotation(case["dim"], theta=THETA, layout=case["layout"], width=case["turned"],
                                     scaling=Scaling("bands", **BANDS) if case["scaled"] else None)
        state["given"] = {name: _given(data[name], (1, *data[name].shape)) for name in ("q", "k", "dq", "dk") if name in data}
        state["positions"] = _storage(data["positions"])
    elif kind == "attention":
        from qutai_b200.attention import PackedSequences

        state["sequences"] = PackedSequences(_lengths(case))
        state["given"] = {name: _given(data[name]) for name in ("q", "k", "v", "dout")}
    elif kind == "loss":
        from qutai_b200.head import PiecewiseHead

        state["head"] = PiecewiseHead()
        state["given"] = _given(data["hidden"]), _given(data["weight"]), _storage(data["targets"])
    else:
        from qutai_b200.optim import AdamW, ByteState

        parameters, shadows = [_given(held["values"]) for held in data["tensors"]], {}
        for parameter, held in zip(parameters, data["tensors"]):
            parameter.grad = _given(held["gradient"])
            if case["shadow"]:
                shadows[parameter] = _storage(held["shadow"])
        optimizer = AdamW(parameters, learning_rate=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY, shadows=shadows, state_bits=8)
        for parameter, held in zip(parameters, data["tensors"]):
            optimizer.steps[parameter] = case["steps"]
            optimizer.averages[parameter] = ByteState(_storage(held["average"]), _storage(held["average_scale"]))
            optimizer.square_averages[parameter] = ByteState(_storage(held["root"]), _storage(held["root_scale"]))
        state["optimizer"] = optimizer
        state["buffers"] = {parameter: (_storage(state["out"][1][held["place"]]), _storage(state["out"][2][held["place"]]))
                            for parameter, held in zip(parameters, data["tensors"])}
        return
    state["buffers"] = [_storage(tensor) for tensor in state["out"]]


# -- the plain forms ----------------------------------------------------------------------------------------------
def _rates(case):
    """Radians per position of every turned pair, 64 bits.  Scaled by bands: a wavelength that fits ``high`` times into the original context
    is kept, one that fits less than ``low`` times is stretched by the factor, between them by a share of both."""
    rate = THETA ** (-torch.arange(0, case["turned"], 2, device="cuda", dtype=torch.float64) / case["turned"])
    if not case["scaled"]:
        return rate
    kept = ((rate * BANDS["original"] / (2 * math.pi) - BANDS["low"]) / (BANDS["high"] - BANDS["low"])).clamp(0, 1)
    return rate * kept + rate / BANDS["factor"] * (1 - kept)


def _turned(case, x, cos, sin):
    heads, half = x.float().view(case["rows"], -1, case["dim"]), case["turned"] // 2
    part, rest = heads[..., :case["turned"]], heads[..., case["turned"]:]
    if case["layout"] == "halves":
        a, b = part[..., :half], part[..., half:]
        part = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((part, rest), -1).view(x.shape).to(x.dtype)


def _plain_rotary(case, data):
    # an angle is a place on the circle: formed in 64 bits (at position 100000 32 bits leave it four digits), its cosine and sine held in 32
    angle = data["positions"].double()[:, None, None] * _rates(case)
    cos, sin = angle.cos().float(), angle.sin().float()
    result = [_turned(case, data["q"], cos, sin), _turned(case, data["k"], cos, sin)]
    if case["train"]:
        result += [_turned(case, data["dq"], cos, -sin), _turned(case, data["dk"], cos, -sin)]
    return result


def _plain_attention(case, data, out):
    dim, group, start = case["dim"], case["heads"] // case["kv_heads"], 0
    for length in _lengths(case):
        if not length:
            continue
        rows = slice(start, start + length)
        start += length
        heads = lambda name, n: data[name][rows].float().view(length, n, -1, dim).permute(1, 2, 0, 3)  # noqa: E731
        q, k, v = heads("q", case["kv_heads"]), heads("k", case["kv_heads"]), heads("v", case["kv_heads"])
        later = torch.ones((length, length), dtype=torch.bool, device="cuda").triu(1)
        scores = (q @ k.transpose(-1, -2) * dim ** -0.5).masked_fill_(later, -math.inf)         # [kv_heads, group, length, length]
        lse = scores.logsumexp(-1, keepdim=True)
        p = scores.sub_(lse).exp_()
        o = p @ v
        flat = lambda x: x.permute(2, 0, 1, 3).reshape(length, -1)  # noqa: E731
        out[0][rows], out[1][rows] = flat(o).to(torch.bfloat16), flat(lse)
        if case["train"]:
            g = heads("dout", case["kv_heads"])
            ds = p * (g @ v.transpose(-1, -2) - (g * o).sum(-1, keepdim=True)) * dim ** -0.5
            out[2][rows] = flat(ds @ k).to(torch.bfloat16)
            out[3][rows] = flat((ds.transpose(-1, -2) @ q).sum(1, keepdim=True)).to(torch.bfloat16)
            out[4][rows] = flat((p.transpose(-1, -2) @ g).sum(1, keepdim=True)).to(torch.bfloat16)
    return out


def _plain_loss(case, data):
    counted = (data["targets"] != -100).nonzero().squeeze(1)
    x, w, target = data["hidden"][counted].float(), data["weight"].float(), data["targets"][counted]
    logits = x @ w.T
    lse = logits.logsumexp(-1)
    share = 1.0 / max(counted.numel(), 1)
    loss = (lse - logits.gather(1, target[:, None])[:, 0]).sum(dtype=torch.float64) * share
    gradient = logits.sub_(lse[:, None]).exp_()
    gradient[torch.arange(counted.numel(), device="cuda"), target] -= 1.0
    gradient *= share
    d_hidden = torch.zeros_like(data["hidden"])
    d_hidden[counted] = (gradient @ w).to(d_hidden.dtype)
    return [loss.float().view(1), d_hidden, (gradient.T @ x).to(data["weight"].dtype)]


def _plain_adamw(case, data, out, step):
    first, second = 1 - BETAS[0] ** step, 1 - BETAS[1] ** step
    for held in data["tensors"]:
        g = held["gradient"]
        m = _decoded(_signed_values(held["average"]), held["average_scale"]) * BETAS[0] + g * (1 - BETAS[0])
        root = _decoded(_root_values(held["root"]), held["root_scale"])
        v = root * root * BETAS[1] + g * g * (1 - BETAS[1])
        root = v.sqrt()
        held["values"].copy_(held["values"] * (1 - RATE * DECAY) - RATE / first * m / (root / math.sqrt(second) + EPS))
        held["average"], held["average_scale"] = _encoded(m, LARGEST[0], 2.0 ** -100, _signed_codes)
        held["root"], held["root_scale"] = _encoded(root, LARGEST[1], 0.0, _root_codes)
        if case["shadow"]:
            held["shadow"].copy_(held["values"])
        root = _decoded(_root_values(held["root"]), held["root_scale"])
        out[1][held["place"]] = _decoded(_signed_values(held["average"]), held["average_scale"])
        out[2][held["place"]] = root * root
    return out


def run(state):
    """One pass, and its outputs."""
    case, data, kind = state["case"], state["data"], state["case"]["kind"]
    if kind == "adamw":
        state["step"] += 1
    if not own:
        if kind == "rotary":
            return _plain_rotary(case, data)
        if kind == "attention":
            return _plain_attention(case, data, state["out"])
        return _plain_loss(case, data) if kind == "loss" else _plain_adamw(case, data, state["out"], state["step"])
    if kind == "adamw":
        optimizer = state["optimizer"]
        optimizer.step()
        optimizer.values_of_states(out=state["buffers"])
        return state["out"]
    buffers = state["buffers"]
    if kind == "rotary":
        from qutai_b200.rotary import rotate_backward, rotate_forward

        given = state["given"]
        rotate_forward(given["q"], given["k"], case["heads"], case["kv_heads"], state["rotation"], positions=state["positions"], out=buffers[:2])
        if case["train"]:
            rotate_backward(given["dq"], given["dk"], case["heads"], case["kv_heads"], state["rotation"], positions=state["positions"], out=buffers[2:])
    elif kind == "attention":
        from qutai_b200.attention import packed_attention_backward, packed_attention_forward

        given = state["given"]
        out, lse = packed_attention_forward(given["q"], given["k"], given["v"], case["heads"], case["kv_heads"], state["sequences"], out=buffers[:2])
        if case["train"]:
            packed_attention_backward(given["dout"], given["q"], given["k"], given["v"], out, lse, case["heads"], case["kv_heads"], state["sequences"],
                                      out=buffers[2:])
    else:
        head = state["head"]
        head.forward(*state["given"], out=buffers[0])
        head.backward(out=buffers[1:])
    return state["out"]


# -- the definitions in 64 bits --------------------------------------------------------------------------------------
def _exact_rotary(case, data):
    """By complex numbers: a pair is a number, a rotation a factor of modulus one."""
    n, half, dim = case["rows"], case["turned"] // 2, case["dim"]
    rate = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-math.log(THETA) / half))
    if case["scaled"]:
        fits = BANDS["original"] / (2 * math.pi / rate)
        smooth = (fits - BANDS["low"]) / (BANDS["high"] - BANDS["low"])
        between = (1 - smooth) * rate / BANDS["factor"] + smooth * rate
        rate = torch.where(fits < BANDS["low"], rate / BANDS["factor"], torch.where(fits > BANDS["high"], rate, between))
    factor = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), data["positions"].to(torch.float64).reshape(n, 1, 1) * rate)
    outputs = []
    for name in ("q", "k", "dq", "dk") if case["train"] else ("q", "k"):
        x = data[name].double().reshape(n, -1, dim)
        part = x[..., :2 * half]
        pairs = part.reshape(n, -1, 2, half).transpose(-1, -2) if case["layout"] == "halves" else part.reshape(n, -1, half, 2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * (factor.conj() if name[0] == "d" else factor))
        part = (z.transpose(-1, -2) if case["layout"] == "halves" else z).reshape(n, -1, 2 * half)
        outputs.append(torch.cat((part, x[..., 2 * half:]), -1).reshape(n, -1))
    return outputs


def _exact_attention(case, data):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    rows = data["q"].shape[0]
    new = lambda n: torch.zeros((rows, n, dim), device="cuda", dtype=torch.float64)  # noqa: E731
    out, lse = new(heads), torch.zeros((rows, heads), device="cuda", dtype=torch.float64)
    dq, dk, dv = new(heads), new(kv_heads), new(kv_heads)
    at = 0
    for length in _lengths(case):
        if length:
            of = lambda name, h: data[name][at:at + length].view(length, -1, dim)[:, h].double()  # noqa: E731
            seen = torch.ones((length, length), device="cuda", dtype=torch.bool).tril()
            for h in range(heads):
                g = h * kv_heads // heads
                q, k, v = of("q", h), of("k", g), of("v", g)
                s = torch.where(seen, torch.mm(q, k.T) / math.sqrt(dim), -math.inf)
                top = torch.amax(s, 1, keepdim=True)
                e = torch.exp(s - top)
                total = torch.sum(e, 1, keepdim=True)
                p = e / total
                out[at:at + length, h] = torch.mm(p, v)
                lse[at:at + length, h] = (top + torch.log(total))[:, 0]
                if case["train"]:
                    do = of("dout", h)
                    dp = torch.mm(do, v.T)
                    ds = p * (dp - torch.sum(p * dp, 1, keepdim=True)) / math.sqrt(dim)
                    dq[at:at + length, h] = torch.mm(ds, k)
                    dk[at:at + length, g] += torch.mm(ds.T, q)
                    dv[at:at + length, g] += torch.mm(p.T, do)
        at += length
    results = [out.reshape(rows, -1), lse]
    return results + ([x.reshape(rows, -1) for x in (dq, dk, dv)] if case["train"] else [])


def _exact_loss(case, data):
    rows, width, vocab = case["rows"], case["width"], case["vocab"]
    w = data["weight"].double()
    count = max(1, int((data["targets"] >= 0).sum()))
    loss = torch.zeros((), device="cuda", dtype=torch.float64)
    d_hidden = torch.zeros((rows, width), device="cuda", dtype=torch.float64)
    d_weight = torch.zeros((vocab, width), device="cuda", dtype=torch.float64)
    for begin in range(0, rows, 1024):
        part = slice(begin, min(begin + 1024, rows))
        x, target = data["hidden"][part].double(), data["targets"][part]
        valid = (target >= 0).double()[:, None]
        one = torch.nn.functional.one_hot(target.clamp(min=0), vocab).double()
        z = torch.mm(x, w.T)
        log_p = z - torch.logsumexp(z, 1, keepdim=True)
        loss -= torch.sum(valid * one * log_p) / count
        g = (torch.exp(log_p) - one) * valid / count
        d_hidden[part] = torch.mm(g, w)
        d_weight += torch.mm(g.T, x)
    return [loss.reshape(1), d_hidden, d_weight]


def _exact_adamw(case, data):
    """A moment in 8 bits is no computed number; the parameters are."""
    t = case["steps"] + 1
    result = torch.zeros_like(data["values"], dtype=torch.float64)
    for held in data["tensors"]:
        n = held["values"].numel()
        per_element = lambda scale: scale.double().repeat_interleave(BLOCK)[:n]  # noqa: E731
        g = held["gradient"].double()
        m = held["average"].view(torch.float8_e4m3fn).to(torch.float64) * per_element(held["average_scale"])
        c = held["root"].view(torch.uint8).to(torch.float64)
        power = torch.clamp(torch.floor(c / 16), min=1.0)
        root = (c - 16 * (power - 1)) * 2.0 ** (power - 1) * per_element(held["root_scale"])
        m = (BETAS[0] * m + (1 - BETAS[0]) * g) / (1 - BETAS[0] ** t)
        v = (BETAS[1] * root ** 2 + (1 - BETAS[1]) * g ** 2) / (1 - BETAS[1] ** t)
        p = held["values"].double()
        result[held["place"]] = p - RATE * DECAY * p - RATE * m / (torch.sqrt(v) + EPS)
    return [result, None, None] + ([result] if case["shadow"] else [])


def exact(case, seed):
    if case["kind"] == "loss" and case["rows"] * case["vocab"] * case["width"] > 2.5e12:
        return None
    data = _inputs(case, seed)
    return dict(rotary=_exact_rotary, attention=_exact_attention, loss=_exact_loss, adamw=_exact_adamw)[case["kind"]](case, data)


# -- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    """``bytes``: inputs read and outputs written once; ``flops``: products and sums as two operations."""
    kind = case["kind"]
    if kind == "rotary":
        elements = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"] * (2 if case["train"] else 1)
        return dict(bytes=elements * 2 * BYTES[case["dtype"]] + 4 * case["rows"], flops=elements * 3)
    if kind == "attention":
        lengths, heads, kv_heads, dim = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
        rows, pairs = sum(lengths), sum(n * (n + 1) // 2 for n in lengths)
        q, kv, lse = rows * heads * dim * 2, rows * kv_heads * dim * 2, rows * heads * 4
        if not case["train"]:
            return dict(bytes=2 * q + 2 * kv + lse, flops=4 * pairs * heads * dim)
        return dict(bytes=4 * q + 4 * kv + lse, flops=14 * pairs * heads * dim)
    if kind == "loss":
        rows, width, vocab, item = case["rows"], case["width"], case["vocab"], BYTES[case["dtype"]]
        counted = rows * (1 - case["none"])
        return dict(bytes=int(2 * item * width * (rows + vocab) + 8 * rows), flops=int(6 * counted * width * vocab))
    sizes = [int(size) for size in case["sizes"].split(",")]
    scales = sum(-(-size // BLOCK) for size in sizes)
    return dict(bytes=sum(sizes) * (4 + 4 + 4 + 2 + 2 + 8 + (2 if case["shadow"] else 0)) + 16 * scales, flops=sum(sizes) * 20)
