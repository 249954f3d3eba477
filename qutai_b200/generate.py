"""Many continuations of one prompt from a ``Decoder``: the prompt runs once, its keys and values become a prefix that all
continuations share (``kv_cache.prefix_attention``), every continuation keeps its own positions in a ``KVCache``, and one token a
continuation and step is drawn on the device (``sampling.sample``); nothing waits for the host between steps.  No upstream counterpart.
Dependency-free.

``python -m qutai_b200.generate`` draws from a small decoder with random weights and prints what a step takes.
"""
from __future__ import annotations

import random
from array import array

from . import lib
from .decoder import _add, _rms_norm
from .kv_cache import KVCache, prefix_attention
from .layers import Tensor
from .sampling import sample
from .storage import DeviceStorage


class Generator:
    """``decoder``: a ``Decoder`` on one GPU.  ``cache_dtype``: "bfloat16", or "int8" for keys and values of 8 bits."""

    def __init__(self, decoder, *, cache_dtype="bfloat16"):
        if decoder.world != 1:
            raise ValueError("generation runs on one GPU")
        if cache_dtype not in lib.CACHE_CODES:
            raise ValueError("a cache is bfloat16 or int8")
        self.decoder, self.cache_dtype, self.stream = decoder, cache_dtype, decoder.stream
        self.prefix = self.caches = None
        self._operand = DeviceStorage(decoder.embedding.weight.size, "bfloat16", stream=self.stream)

    def _cache(self, batch, capacity):
        attention = self.decoder.blocks[0].attn
        return [KVCache(batch, capacity, attention.kv_heads, attention.dim, self.cache_dtype, stream=self.stream) for _ in self.decoder.blocks]

    def _embedded(self, ids, rows):
        c = self.decoder.config
        x = DeviceStorage(rows * c.d_model, "bfloat16", stream=self.stream)
        lib.call("qmoe_embedding", self.decoder.embedding.weight.storage.ptr, ids.ptr, x.ptr, lib.QMOE_BF16, rows, c.d_model, c.vocab_size, self.stream)
        return x

    def _logits(self, x, rows):
        """float32 logits [rows, vocab] of the residual rows ``x`` through the final norm and the tied table."""
        c, table = self.decoder.config, self.decoder.embedding.weight.storage
        if not self._operand.is_derived_from(table):
            lib.call("qmoe_cast_bf16", table.ptr, self._operand.ptr, table.size, self.stream)
            self._operand.mark_derived_from(table)
        hidden, _ = _rms_norm(x, self.decoder.norm, rows, c.d_model, self.stream)
        logits = DeviceStorage(rows * c.vocab_size, "float32", stream=self.stream)
        lib.call("qmoe_gemm", hidden.ptr, lib.QMOE_BF16, self._operand.ptr, lib.QMOE_BF16, logits.ptr, lib.QMOE_F32, rows, c.d_model, c.vocab_size,
                 0, 1, 0, self.stream)
        return Tensor(logits, (rows, c.vocab_size))

    def _feed_forward(self, block, x, y, rows):
        middle = _add(x, y, self.stream)
        return block.feed_forward(Tensor(middle, (rows, block.width)))[0].storage

    def prefill(self, prompt):
        """Run ``prompt`` (token ids) and keep its keys and values as the prefix; the continuations of a prompt before it are gone, and ``start`` makes
        room for new ones.  Returns the logits [1, vocab] behind its last token."""
        tokens, c = [int(t) for t in prompt], self.decoder.config
        if not tokens or any(not 0 <= t < c.vocab_size for t in tokens):
            raise ValueError("the prompt must be a non-empty list of token ids")
        time, width = len(tokens), c.d_model
        self.prefix = self.caches = None        # until all blocks have run there is nothing to go on from
        held = self._cache(1, time)
        x = self._embedded(DeviceStorage.from_bytes(array("q", tokens).tobytes(), "int64", self.stream), time)
        for block, prefix in zip(self.decoder.blocks, held):
            normed, _ = _rms_norm(x, block.attn_norm, time, width, self.stream)
            y, (_, _, k, v, *_) = block.attn.forward(normed, 1, time)
            prefix.append(k, v)
            x = self._feed_forward(block, x, y, time)
        logits = self._logits(x.view((time - 1) * width, width), 1)
        self.prefix = held
        return logits

    def start(self, batch, new_tokens):
        """Empty caches for ``batch`` continuations of up to ``new_tokens`` positions each."""
        if self.prefix is None:
            raise RuntimeError("start needs a prefill first")
        self.caches = self._cache(batch, new_tokens)

    def step(self, ids):
        """One position of every continuation: ``ids`` an int64 storage with their newest tokens.  Returns the logits [batch, vocab]."""
        if self.caches is None:
            raise RuntimeError("step needs a start first")
        batch, width = self.caches[0].batch, self.decoder.config.d_model
        if ids.dtype != "int64" or ids.size != batch:
            raise ValueError("ids must hold one int64 token id for each continuation")
        position = self.prefix[0].longest + self.caches[0].longest
        x = self._embedded(ids, batch)
        for block, prefix, cache in zip(self.decoder.blocks, self.prefix, self.caches):
            normed, _ = _rms_norm(x, block.attn_norm, batch, width, self.stream)
            (q, k, v), _ = block.attn.project(normed, batch, 1, position)
            cache.append(k, v)
            attended, _ = prefix_attention(q, block.attn.heads, cache, prefix, stream=self.stream)
            x = self._feed_forward(block, x, block.attn.out.forward(attended, batch), batch)
        return self._logits(x, batch)

    def generate(self, prompt, samples, new_tokens, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed=None, uniforms=None, stop_token=None):
        """``samples`` continuations of ``prompt``, ``new_tokens`` tokens each.  The settings are ``sampling.sample``'s (numbers, or storages with one
        for each continuation).  ``uniforms``: float32 storage [new_tokens * samples] of the numbers to draw with, step by step; by
        default ``random.Random(seed)`` makes them.  Returns ``(tokens, log_probs)`` as lists; with ``stop_token`` a continuation ends with it."""
        if samples <= 0 or new_tokens <= 0:
            raise ValueError("samples and new_tokens must be positive")
        if uniforms is None:
            rng = random.Random(seed)
            uniforms = DeviceStorage.from_values([min(rng.random(), 1 - 2 ** -24) for _ in range(samples * new_tokens)], "float32", self.stream)
        elif uniforms.dtype != "float32" or uniforms.size != samples * new_tokens:
            raise ValueError("uniforms must hold new_tokens * samples float32 numbers")
        first = self.prefill(prompt)
        vocab = first.shape[1]
        # the first draw of every continuation is from the prompt's last row
        zeros = DeviceStorage.zeros(samples, "int32", self.stream)
        logits = Tensor(DeviceStorage(samples * vocab, "float32", stream=self.stream), (samples, vocab))
        lib.call("qmoe_gather_rows", first.storage.ptr, logits.storage.ptr, zeros.ptr, samples, 1, 4 * vocab, self.stream)
        if new_tokens > 1:
            self.start(samples, new_tokens - 1)
        tokens, log_probs = DeviceStorage(samples * new_tokens, "int64", stream=self.stream), DeviceStorage(samples * new_tokens, "float32", stream=self.stream)
        for i in range(new_tokens):
            out = tokens.view(i * samples, samples), log_probs.view(i * samples, samples)
            sample(logits, uniforms.view(i * samples, samples), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, out=out, stream=self.stream)
            if i + 1 < new_tokens:
                logits = self.step(out[0])
        drawn, scores = tokens.tolist(self.stream), log_probs.tolist(self.stream)
        result = [drawn[b::samples] for b in range(samples)], [scores[b::samples] for b in range(samples)]
        if stop_token is not None:
            for row, score in zip(*result):
                if stop_token in row:
                    end = row.index(stop_token) + 1
                    del row[end:], score[end:]
        return result


def main(arguments=None):
    import argparse
    import time

    from .decoder import Config, Decoder

    parser = argparse.ArgumentParser(description="draw continuations of a random prompt from a decoder with random weights")
    parser.add_argument("--samples", type=int, default=64)
    parser.add_argument("--prompt", type=int, default=2048)
    parser.add_argument("--new-tokens", type=int, default=64)
    parser.add_argument("--cache", default="bfloat16", choices=sorted(lib.CACHE_CODES))
    parser.add_argument("--blocks", type=int, default=4)
    options = parser.parse_args(arguments)
    config = Config(vocab_size=32000, d_model=1024, n_heads=16, n_kv_heads=4, n_layers=options.blocks, n_experts=16, top_k=2, d_expert=2048, qk_norm=True)
    generator = Generator(Decoder(config, seed=0), cache_dtype=options.cache)
    prompt = [random.Random(1).randrange(config.vocab_size) for _ in range(options.prompt)]
    settings = dict(temperature=0.8, top_k=50, top_p=0.95, seed=2)
    generator.generate(prompt, options.samples, 4, **settings)                       # workspaces, operand copies
    took = []
    for count in (1, options.new_tokens):
        began = time.perf_counter()
        tokens, _ = generator.generate(prompt, options.samples, count, **settings)
        took.append(time.perf_counter() - began)
    steps = max(1, options.new_tokens - 1)
    print(f"{options.samples} continuations of {options.prompt} tokens, {options.cache} cache: prompt and first token {took[0] * 1e3:.2f} ms, "
          f"{(took[1] - took[0]) / steps * 1e3:.3f} ms a step, {options.samples * steps / max(took[1] - took[0], 1e-9):.0f} tokens/s; first: {tokens[0][:8]}")


if __name__ == "__main__":
    main()
