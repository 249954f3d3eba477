"""Norm and rotation of query and key heads (``qutai_b200.rotary``) against the formula in 64 bits, its gradients against the
formula's and against differences of the formula.  Needs a B200: ``-m gpu``.

Bars: a bfloat16 output is one rounding (2^-9 of the value) of a float32 result, so 2^-8 of the value bounds it with room for a
tie that falls the other way; float32 outputs pass through about ten roundings of 2^-24, 1e-6 of the head's size.  A weight's gradient is a sum of
``n`` float32 products in chains of at most a few dozen additions: 4e-6 of the sum of their sizes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = 1e-5


def turned(x, positions, theta, sign=1):
    """x [batch, time, heads, dim], positions [batch, time]"""
    dim = x.shape[-1]
    angle = sign * positions[..., None, None] * theta ** (-np.arange(0, dim, 2) / dim)
    y = np.empty_like(x)
    y[..., 0::2] = x[..., 0::2] * np.cos(angle) - x[..., 1::2] * np.sin(angle)
    y[..., 1::2] = x[..., 0::2] * np.sin(angle) + x[..., 1::2] * np.cos(angle)
    return y


def formula(x, weight, positions, theta):
    return turned(x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * weight, positions, theta)


def formula_backward(g, x, weight, positions, theta):
    r = np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    g = turned(g, positions, theta, -1)
    terms = g * x / r
    dx = (g * weight - x / r * (g * weight * x / r).mean(-1, keepdims=True)) / r
    return dx, terms.sum((0, 1, 2)), np.abs(terms).sum((0, 1, 2))


def rounded(a, dtype):
    from gpu_util import to_device, to_host

    return to_host(to_device(a, dtype), np.shape(a))


def make(rng, batch, time, heads, kv_heads, dim, dtype):
    shape = lambda h: (batch, time, h, dim)  # noqa: E731
    data = {name: rounded(rng.standard_normal(shape(h)) * scale, dtype)
            for name, h, scale in (("q", heads, 2.0), ("k", kv_heads, 0.1), ("gq", heads, 1.0), ("gk", kv_heads, 1.0))}
    for name in ("wq", "wk"):
        data[name] = rounded(1 + 0.2 * rng.standard_normal(dim), "float32")
    return data


def near(got, want, dtype):
    size = np.sqrt((want * want).mean(-1, keepdims=True))
    bar = 2.0 ** -8 * np.abs(want) + 1e-6 * size if dtype == "bfloat16" else 1e-6 * (np.abs(want) + 4 * size)
    assert np.all(np.abs(got - want) <= bar + 1e-30), np.max(np.abs(got - want) / (bar + 1e-30))


def check(batch, time, heads, kv_heads, dim, dtype, *, theta=10000.0, starts=None, offset=0, columns=False, seed=0):
    from gpu_util import to_device, to_host
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import Columns, norm_rope_backward, norm_rope_forward

    d = make(np.random.default_rng(seed), batch, time, heads, kv_heads, dim, dtype)
    flat = lambda a: a.reshape(batch, time, -1)  # noqa: E731
    given = lambda a: Tensor(to_device(a, dtype if a.ndim > 1 else "float32"), a.shape)  # noqa: E731
    if columns:      # queries, keys and something else beside one another, as one projection leaves them
        fused = given(np.concatenate((flat(d["q"]), flat(d["k"]), np.full((batch, time, 8), 7.0)), -1))
        q, k = Columns(fused, 0, heads * dim), Columns(fused, heads * dim, kv_heads * dim)
    else:
        q, k = given(flat(d["q"])), given(flat(d["k"]))
    wq, wk = given(d["wq"]), given(d["wk"])
    settings = dict(eps=EPS, theta=theta, offset=offset, starts=None if starts is None else to_device(np.array(starts), "int32"))
    positions = offset + (np.zeros(batch) if starts is None else np.array(starts, dtype=np.float64))[:, None] + np.arange(time)
    outs = norm_rope_forward(q, k, wq, wk, heads, kv_heads, **settings)
    grads = norm_rope_backward(to_device(d["gq"], dtype), to_device(d["gk"], dtype), q, k, wq, wk, heads, kv_heads, **settings)
    for i, (x, w, g) in enumerate((("q", "wq", "gq"), ("k", "wk", "gk"))):
        near(to_host(outs[i], d[x].shape), formula(d[x], d[w], positions, theta), dtype)
        dx, dw, size = formula_backward(d[g], d[x], d[w], positions, theta)
        near(to_host(grads[i], d[x].shape), dx, dtype)
        assert np.all(np.abs(to_host(grads[2 + i]) - dw) <= 4e-6 * size + 1e-30)
    again = norm_rope_backward(to_device(d["gq"], dtype), to_device(d["gk"], dtype), q, k, wq, wk, heads, kv_heads, **settings)
    for a, b in zip(grads, again):
        assert a.tobytes() == b.tobytes()          # fixed order of the sums: the same bits on every run


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("batch,time,heads,kv_heads,dim", [(1, 1, 1, 1, 8), (64, 1, 16, 4, 64), (3, 37, 8, 2, 128), (1, 1003, 16, 4, 64), (2, 5, 3, 3, 256),
                                                           (5, 7, 7, 1, 24), (2, 9, 6, 2, 40), (1, 300, 40, 8, 80), (4, 700, 4, 1, 32)])
def test_norm_and_rotation_match_the_formula(batch, time, heads, kv_heads, dim, dtype):
    check(batch, time, heads, kv_heads, dim, dtype, seed=time + dim)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_positions_far_out_keep_their_angles(dtype):
    """At position two million 32 bits leave an angle of 2e6 an error of 0.1; negative positions turn the other way."""
    check(4, 3, 4, 2, 64, dtype, starts=[0, 131071, 2000003, 2147483000], offset=5, theta=10000.0)
    check(2, 2, 2, 2, 64, dtype, starts=[-7, 12], offset=-100, theta=500000.0)
    check(1, 3, 2, 1, 64, "float32", offset=2 ** 40, theta=1.0)


def test_heads_out_of_one_projections_rows():
    check(3, 50, 8, 2, 64, "bfloat16", columns=True)
    check(2, 5, 3, 1, 40, "float32", columns=True)


def test_gradients_against_differences():
    """d/dx of sum(g * y) by central differences of the formula in 64 bits, for a few elements of each operand."""
    from gpu_util import to_device, to_host
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import norm_rope_backward

    rng = np.random.default_rng(5)
    shape, theta = (2, 3, 2, 16), 100.0
    d = make(rng, 2, 3, 2, 2, 16, "float32")
    positions = np.broadcast_to(np.arange(3.0), (2, 3))
    given = lambda a: Tensor(to_device(a, "float32"), a.shape)  # noqa: E731
    flat = lambda a: a.reshape(2, 3, 32)  # noqa: E731
    got = norm_rope_backward(to_device(d["gq"], "float32"), to_device(d["gk"], "float32"), given(flat(d["q"])), given(flat(d["k"])), given(d["wq"]),
                             given(d["wk"]), 2, 2, eps=EPS, theta=theta)
    value = lambda x, w, g: (formula(x, w, positions, theta) * g).sum()  # noqa: E731
    for i, (x, w, g) in enumerate((("q", "wq", "gq"), ("k", "wk", "gk"))):
        dx, dw = to_host(got[i], shape), to_host(got[2 + i])
        for _ in range(12):
            at, h = tuple(rng.integers(0, n) for n in shape), 1e-4 * np.abs(d[x]).mean()
            up, down = d[x].copy(), d[x].copy()
            up[at] += h
            down[at] -= h
            want = (value(up, d[w], d[g]) - value(down, d[w], d[g])) / (2 * h)
            assert abs(dx[at] - want) <= 1e-4 * np.abs(dx).mean() + 1e-4 * abs(want)       # h^2 of the third derivative, and float32
            j = at[3]
            up, down = d[w].copy(), d[w].copy()
            up[j] += 1e-4
            down[j] -= 1e-4
            want = (value(d[x], up, d[g]) - value(d[x], down, d[g])) / 2e-4
            assert abs(dw[j] - want) <= 1e-4 * np.abs(dw).mean() + 1e-4 * abs(want)


def test_no_rows_give_no_outputs_and_zero_gradients():
    from gpu_util import to_device, to_host
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import norm_rope_backward, norm_rope_forward
    from qutai_b200.storage import DeviceStorage

    w = Tensor(to_device(np.ones(64), "float32"), (64,))
    q, k = Tensor(DeviceStorage(0, "bfloat16"), (2, 0, 128)), Tensor(DeviceStorage(0, "bfloat16"), (2, 0, 64))
    assert [s.size for s in norm_rope_forward(q, k, w, w, 2, 1)] == [0, 0]
    dq, dk, dwq, dwk = norm_rope_backward(q, k, q, k, w, w, 2, 1)
    assert dq.size == dk.size == 0 and not to_host(dwq).any() and not to_host(dwk).any()


def test_a_head_of_zeros_stays_finite():
    from gpu_util import to_device, to_host
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import norm_rope_backward, norm_rope_forward

    w = Tensor(to_device(np.ones(64), "float32"), (64,))
    x = Tensor(to_device(np.zeros((1, 2, 64)), "bfloat16"), (1, 2, 64))
    g = to_device(np.ones((1, 2, 64)), "bfloat16")
    assert not to_host(norm_rope_forward(x, x, w, w, 1, 1)[0]).any()
    assert all(np.isfinite(to_host(s)).all() for s in norm_rope_backward(g, g, x, x, w, w, 1, 1))


def test_another_stream_than_the_default_one():
    import ctypes

    from gpu_util import to_device, to_host
    from qutai_b200 import lib
    from qutai_b200.layers import Tensor
    from qutai_b200.rotary import norm_rope_forward

    stream = ctypes.c_uint64()
    lib.call("qmoe_stream_create", ctypes.byref(stream))
    d = make(np.random.default_rng(3), 2, 11, 4, 2, 64, "bfloat16")
    given = lambda a: Tensor(to_device(a, "bfloat16" if a.ndim > 1 else "float32"), a.shape)  # noqa: E731
    q, k = given(d["q"].reshape(2, 11, -1)), given(d["k"].reshape(2, 11, -1))
    outs = norm_rope_forward(q, k, given(d["wq"]), given(d["wk"]), 4, 2, eps=EPS, stream=stream.value)
    lib.call("qmoe_stream_sync", stream.value)
    near(to_host(outs[0], d["q"].shape), formula(d["q"], d["wq"], np.broadcast_to(np.arange(11.0), (2, 11)), 10000.0), "bfloat16")
    lib.call("qmoe_stream_destroy", stream.value)
