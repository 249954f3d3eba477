"""Continuations of a prompt (``qutai_b200.generate.Generator``) against running the whole sequence again, and a decoder with
normalised query and key heads against the formula and against itself.  Needs a B200: ``-m gpu``.

Both ways of a decoder's step run in bfloat16 but round at different places (a row among other rows, attention in parts): the logits
of one position agree to the bars of the decoder's own test, 6e-2 of the largest.  Every expert takes part, so that no rounding sends a row elsewhere."""
import numpy as np
import pytest

from oracle import moe_oracle as oracle

pytestmark = pytest.mark.gpu

TOL = 6e-2


def decoder(qk_norm, seed=11, heads=4, kv_heads=2):
    from gpu_util import to_device
    from qutai_b200.decoder import Config, Decoder

    model = Decoder(Config(vocab_size=96, d_model=64 * heads, n_heads=heads, n_kv_heads=kv_heads, n_layers=2, n_experts=2, top_k=2, d_expert=64, qk_norm=qk_norm), seed=seed)
    rng = np.random.default_rng(seed)
    for name, parameter in model.named_parameters():        # weights that make something of their input
        scale = 0.3 if "norm" in name else 0.5 if name == "embedding.weight" else 1.5 * parameter.shape[-1] ** -0.5
        values = rng.standard_normal(parameter.shape) * scale + (1 if "norm" in name else 0)
        parameter.storage.copy_from(to_device(values, "float32"))
    return model


def logits_of(generator, tokens):
    from gpu_util import to_host

    result = generator.prefill(tokens)
    return to_host(result.storage)


@pytest.mark.parametrize("cache_dtype,tol", [("bfloat16", TOL), ("int8", 2 * TOL)])       # 8 bits: half a part in 127 of every key and value on top
@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("prompt,samples", [(1, 1), (7, 3), (150, 40), (64, 70)])
def test_steps_agree_with_running_the_whole_sequence_again(prompt, samples, qk_norm, cache_dtype, tol):
    from gpu_util import to_device, to_host
    from qutai_b200.generate import Generator

    model = decoder(qk_norm)
    rng = np.random.default_rng(prompt)
    head = rng.integers(0, 96, prompt).tolist()
    tails = rng.integers(0, 96, (samples, 5))
    generator, whole = Generator(model, cache_dtype=cache_dtype), Generator(model)
    generator.prefill(head)
    generator.start(samples, 5)
    for i in range(5):
        got = to_host(generator.step(to_device(tails[:, i], "int64")).storage, (samples, 96))
        for b in {0, samples // 2, samples - 1}:
            want = logits_of(whole, head + tails[b, :i + 1].tolist())
            assert oracle.max_rel_err(got[b], want) <= tol, (i, b)


@pytest.mark.parametrize("cache_dtype", ["bfloat16", "int8"])
def test_greedy_tokens_and_repeated_draws(cache_dtype):
    from qutai_b200.generate import Generator

    generator = Generator(decoder(True), cache_dtype=cache_dtype)
    prompt = list(range(3, 40))
    tokens, scores = generator.generate(prompt, 4, 6, temperature=0.0)
    assert all(row == tokens[0] for row in tokens) and len(tokens[0]) == 6           # the same prompt, the same choice
    assert all(np.isfinite(row).all() and max(row) <= 0 for row in scores)
    once, again = (generator.generate(prompt, 9, 8, temperature=1.2, top_p=0.95, seed=5) for _ in range(2))
    assert once == again
    assert once[0] != generator.generate(prompt, 9, 8, temperature=1.2, top_p=0.95, seed=6)[0]
    assert len({tuple(row) for row in once[0]}) > 1
    stop = once[0][2][3]
    stopped, _ = generator.generate(prompt, 9, 8, temperature=1.2, top_p=0.95, seed=5, stop_token=stop)
    assert all(row == full[:full.index(stop) + 1] if stop in full else row == full for row, full in zip(stopped, once[0]))


def test_a_larger_batch_draws_the_same_tokens():
    """The numbers of a continuation are its own: two of them alone draw what they draw among others."""
    from gpu_util import to_device
    from qutai_b200.generate import Generator

    generator = Generator(decoder(True))
    numbers = np.random.default_rng(1).random((4, 6))
    uniforms = lambda n: to_device(numbers[:, :n].reshape(-1), "float32")  # noqa: E731
    few = generator.generate([5, 6, 7], 2, 4, uniforms=uniforms(2), temperature=0.9)[0]
    many = generator.generate([5, 6, 7], 6, 4, uniforms=uniforms(6), temperature=0.9)[0]
    assert few[0][0] == many[0][0] and few[1][0] == many[1][0]                       # the first token has the very same logits


def test_refusals():
    from gpu_util import to_device
    from qutai_b200.generate import Generator

    model = decoder(False)
    with pytest.raises(ValueError):
        Generator(model, cache_dtype="float32")
    generator = Generator(model)
    with pytest.raises(RuntimeError):
        generator.start(2, 3)
    for prompt in ([], [96], [-1]):
        with pytest.raises(ValueError):
            generator.prefill(prompt)
    generator.prefill([1, 2])
    with pytest.raises(RuntimeError):
        generator.step(to_device(np.zeros(2), "int64"))
    generator.start(2, 1)
    for ids in (to_device(np.zeros(3), "int64"), to_device(np.zeros(2), "int32")):
        with pytest.raises(ValueError):
            generator.step(ids)
    generator.step(to_device(np.zeros(2), "int64"))
    with pytest.raises(ValueError, match="capacity"):
        generator.step(to_device(np.zeros(2), "int64"))
    with pytest.raises(ValueError):
        generator.generate([1], 0, 4)
    with pytest.raises(ValueError):
        generator.generate([1], 2, 4, uniforms=to_device(np.zeros(7), "float32"))


@pytest.mark.parametrize("heads,kv_heads,time", [(4, 2, 37), (3, 1, 130)])
def test_attention_with_normalised_heads_matches_the_formula(heads, kv_heads, time):
    """``GQA`` with ``qk_norm``, forward and backward, against its pieces in 64 bits: projections, norm and rotation, causal attention."""
    from test_gpu_rotary import formula, formula_backward

    from gpu_util import to_device, to_host
    from qutai_b200.decoder import GQA, Config

    batch, width, dim = 2, 64 * heads, 64
    config = Config(vocab_size=8, d_model=width, n_heads=heads, n_kv_heads=kv_heads, n_layers=1, n_experts=1, top_k=1, d_expert=8, norm_eps=1e-5, qk_norm=True)
    layer = GQA(config, seed=1)
    rng, weights = np.random.default_rng(heads), {}
    for name, weight in layer.named_weights():
        values = rng.standard_normal(weight.shape) * (0.2 if "norm" in name else 1.5 * width ** -0.5) + (1 if "norm" in name else 0)
        weight.storage.copy_from(to_device(values, "float32"))
        weights[name] = oracle.round_bf16(values) if "norm" not in name else np.float32(values).astype(np.float64)
    x, dy = (oracle.round_bf16(rng.standard_normal((batch * time, width))) for _ in range(2))
    y, saved = layer.forward(to_device(x, "bfloat16"), batch, time)
    dx = layer.backward(to_device(dy, "bfloat16"), saved, batch, time)
    positions = np.broadcast_to(np.arange(float(time)), (batch, time))
    split = lambda a: a.reshape(batch, time, -1, dim)  # noqa: E731
    flat = lambda a: a.reshape(batch, time, -1)  # noqa: E731
    raw = {name: x @ weights[name].T for name in "qkv"}
    q = formula(split(raw["q"]), weights["q_norm"], positions, 10000.0)
    k = formula(split(raw["k"]), weights["k_norm"], positions, 10000.0)
    out, lse = oracle.attention_forward(flat(q), flat(k), flat(raw["v"]), heads, kv_heads)
    rows = out.reshape(batch * time, width)
    d_rows = dy @ weights["out"]
    dq, dk, dv = oracle.attention_backward(flat(d_rows), flat(q), flat(k), flat(raw["v"]), out, lse, heads, kv_heads)
    dq, dwq, _ = formula_backward(split(dq), split(raw["q"]), weights["q_norm"], positions, 10000.0)
    dk, dwk, _ = formula_backward(split(dk), split(raw["k"]), weights["k_norm"], positions, 10000.0)
    flatten = lambda a: a.reshape(batch * time, -1)  # noqa: E731
    wanted = dict(y=rows @ weights["out"].T, dx=flatten(dq) @ weights["q"] + flatten(dk) @ weights["k"] + flatten(dv) @ weights["v"], q_norm=dwq, k_norm=dwk,
                  q=flatten(dq).T @ x, k=flatten(dk).T @ x, v=flatten(dv).T @ x, out=dy.T @ rows)
    got = dict(y=to_host(y, (batch * time, width)), dx=to_host(dx, (batch * time, width)))
    got.update({name: to_host(weight.grad.storage, weight.shape) for name, weight in layer.named_weights()})
    errors = {name: oracle.max_rel_err(got[name], want) for name, want in wanted.items()}
    assert max(errors.values()) <= TOL, errors


def test_a_decoder_with_normalised_heads_trains():
    from gpu_util import to_host
    from qutai_b200.decoder import Config, Decoder
    from qutai_b200.optim import AdamW

    model = Decoder(Config(vocab_size=64, d_model=128, n_heads=2, n_kv_heads=1, n_layers=2, n_experts=4, top_k=2, d_expert=64, qk_norm=True), seed=3)
    names = [name for name, _ in model.named_parameters()]
    assert [n for n in names if n.startswith("blocks.1.attn.")] == [f"blocks.1.attn.{n}.weight" for n in ("q", "k", "v", "out", "q_norm", "k_norm")]
    tokens = np.random.default_rng(0).integers(0, 64, (2, 40)).tolist()
    optimizer = AdamW(model.parameters(), learning_rate=3e-3)
    losses = []
    for _ in range(12):
        model.zero_grad()
        losses.append(to_host(model.loss(tokens).storage)[0])
        model.backward()
        optimizer.step()
    assert losses[-1] < 0.7 * losses[0] and np.isfinite(losses).all()
    assert np.abs(to_host(model.blocks[0].attn.q_norm.weight.storage) - 1).max() > 1e-3
