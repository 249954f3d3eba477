"""A row's largest probability is an exact 1 before the division by the sum, so it brings no rounding of its own: packed attention is as near to the exact result as
attention over a rectangular batch.  Needs a B200: ``-m gpu``.

Bar of an output: every other probability is held in bfloat16, half a step off (2^-8), the largest is not: (2^-8 (p without the largest) + e) |v| summed, and one
rounding of the result, 2^-8 |out|; ``e`` is the float32 arithmetic's share as in ``test_gpu_packed_attention``."""
import numpy as np
import pytest

from test_gpu_packed_attention import H, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1.0, 2.0, 3.0])
def test_the_largest_probability_is_not_rounded(dim, size):
    lengths, heads, kv_heads, scale = [900, 257, 64], 4, 2, dim ** -0.5
    arrays = make(np.random.default_rng(dim), sum(lengths), heads, kv_heads, dim, size)
    out = run(arrays, lengths, heads, kv_heads, dim)[0]
    q, k, v = (a.reshape(len(a), -1, dim) for a in arrays[:3])
    at = 0
    for n in lengths:
        part, seen = slice(at, at + n), np.tril(np.ones((n, n), bool))
        for h in range(heads):
            qh, kh, vh = q[part, h], k[part, h // 2], v[part, h // 2]
            s = np.where(seen, qh @ kh.T * scale, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            others = np.where(s == s.max(1, keepdims=True), 0.0, p)
            d = (dim / 16 + 4) * 2.0 ** -22 * np.where(seen, np.abs(qh) @ np.abs(kh).T * scale, 0)
            e = 2 * d.max(1, keepdims=True) + 2.0 ** -20 * (1 + np.abs(np.where(seen, s, 0)).max(1, keepdims=True)) + (n / 16 + 16) * 2.0 ** -22
            want = p @ vh
            bar = (H * others + e * p) @ np.abs(vh) + H * np.abs(want)
            error = np.abs(out[part, h] - want)
            assert np.all(error <= bar), (h, np.max(error / bar))
        at += n
