"""The 64-bit layers against differences, and the codes of 8-bit states."""

import numpy as np
import pytest

from oracle import layers as L


def _difference(f, x, i, h=1e-6):
    a, b = x.copy(), x.copy()
    a.flat[i] += h
    b.flat[i] -= h
    return (f(a) - f(b)) / (2 * h)


@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_gradients_are_those_of_differences(residual):
    rng = np.random.default_rng(0)
    x, dy = rng.normal(size=(3, 7)), rng.normal(size=(3, 7))
    r = rng.normal(size=(3, 7)) if residual else None
    gamma, beta = 1 + 0.1 * rng.normal(size=7), rng.normal(size=7)

    def loss(x=x, r=r, gamma=gamma, beta=beta):
        return (L.layer_norm(x, r, 0.6, gamma, beta, 1e-3)["y"] * dy).sum()

    f = L.layer_norm(x, r, 0.6, gamma, beta, 1e-3)
    g = L.layer_norm_backward(x, dy, f["mean"], f["rstd"], r, 0.6, gamma)
    # The differences' own error: h^2 times a third derivative, and 2^-53 / h.
    for i in range(x.size):
        assert abs(_difference(lambda v: loss(x=v), x, i) - g["dx"].flat[i]) < 1e-7
        if residual:
            assert abs(_difference(lambda v: loss(r=v), r, i) - g["dresidual"].flat[i]) < 1e-7
    for i in range(7):
        assert abs(_difference(lambda v: loss(gamma=v), gamma, i) - g["dgamma"][i]) < 1e-7
        assert abs(_difference(lambda v: loss(beta=v), beta, i) - g["dbeta"][i]) < 1e-7


@pytest.mark.parametrize("causal,shared,lengths", [(False, False, False), (True, True, False),
                                                   (True, False, True), (False, True, True)])
def test_attention_gradients_are_those_of_differences(causal, shared, lengths):
    rng = np.random.default_rng(1)
    b, tq, tk, hq, hk, d = 2, 4, 5, 4, 2, 3
    q, k, v = rng.normal(size=(b, tq, hq, d)), rng.normal(size=(b, tk, hk, d)), \
        rng.normal(size=(b, tk, hk, d))
    bias = rng.normal(size=(1, hq, tq, tk) if shared else (b, hq, tq, tk))
    dout = rng.normal(size=q.shape)
    kw = dict(causal=causal)
    if lengths:
        kw.update(q_lengths=[3, 0], k_lengths=[5, 2])

    def loss(q=q, k=k, v=v, bias=bias):
        return (L.attention(q, k, v, 0.7, bias, **kw)["out"] * dout).sum()

    g = L.attention_backward(q, k, v, dout, 0.7, bias, **kw)
    db = g["dbias"].sum(0, keepdims=True) if shared else g["dbias"]
    for name, x, want in (("q", q, g["dq"]), ("k", k, g["dk"]), ("v", v, g["dv"]),
                          ("bias", bias, db)):
        for i in range(0, x.size, 3):
            got = _difference(lambda t: loss(**{name: t}), x, i)
            assert abs(got - want.flat[i]) < 1e-7, (name, i)


def test_rows_that_see_nothing_are_zero():
    rng = np.random.default_rng(2)
    q, k, v, dout = (rng.normal(size=(1, 3, 1, 2)) for _ in range(4))
    bias = np.zeros((1, 1, 3, 3))
    bias[0, 0, 1] = -np.inf
    k[0, 2] = np.nan
    g = L.attention_backward(q, k, v, dout, 1.0, bias, k_lengths=[2], q_lengths=[2])
    assert np.all(g["out"][0, 1:] == 0) and np.all(g["lse"][0, 0, 1:] == -np.inf)
    assert np.all(g["dq"][0, 1:] == 0) and np.all(g["dk"][0, 2] == 0)
    assert all(np.all(np.isfinite(g[n])) for n in ("dq", "dk", "dv", "dbias"))


def test_adamw_is_the_formula():
    p, m, v = L.adamw(np.array([1.0]), np.array([0.5]), np.array([0.0]), np.array([0.0]), 1, 0.1,
                      0.9, 0.99, 1e-8, weight_decay=0.5, factor=2.0)
    # After one step m / bc1 = g and v / bc2 = g^2: the update is the sign.
    assert abs(p[0] - (1.0 * (1 - 0.05) - 0.1)) < 1e-7 and abs(m[0] - 0.1) < 1e-15
    assert abs(v[0] - 0.01) < 1e-15
    assert L.clip_factor(4.0, 1.0) == 0.5 and L.clip_factor(4.0, 3.0, 2.0) == 2.0 * 3 / 4


def test_code_values():
    # OCP e4m3: 448 the largest, 2^-9 the smallest; eight bits without a sign.
    assert L.M_VALUES[0x7E] == 448 and L.M_VALUES[1] == 2.0 ** -9 and L.M_VALUES[0x88] == -2.0 ** -6
    assert L.V_VALUES[0xFF] == 122880 and L.V_VALUES[1] == 2.0 ** -17 and L.V_VALUES[0] == 0
    assert np.all(np.diff(L.V_VALUES) > 0) and np.all(np.diff(L.M_VALUES[:127]) > 0)


@pytest.mark.parametrize("n", [1, 255, 256, 1000])
def test_nearest_codes_are_off_by_half_a_step(n):
    rng = np.random.default_rng(n)
    m = (rng.normal(size=n) * 10.0 ** rng.uniform(-6, 0, n)).astype(np.float32)
    code, scale = L.encode_m(m)
    got, s = L.decode_m(code, scale), scale[L._blocks(n)].astype(np.float64)
    # 2^-4 relative for normal codes, half of 2^-9 scales below, and fp32's roundings.
    assert np.all(np.abs(got - m) <= np.maximum(2.0 ** -4 * np.abs(m), 2.0 ** -10 * s) * (1 + 1e-6))
    v = m * m
    code, scale = L.encode_v(v)
    got, s = L.decode_v(code, scale), scale[L._blocks(n)].astype(np.float64)
    assert np.all(np.abs(got - v) <= np.maximum(2.0 ** -4 * v, 2.0 ** -17 * s) * (1 + 1e-6))
    assert np.all((code > 0) == (v > 0))


def test_zeros_have_codes_of_zero():
    code, scale = L.encode_m(np.zeros(300, np.float32))
    assert not code.any() and np.all(scale == np.float32(2.0 ** -100))
    code, scale = L.encode_v(np.zeros(300, np.float32))
    assert not code.any() and np.all(scale == np.float32(2.0 ** -120))


def test_stochastic_codes_are_right_on_average():
    n, rounds = 256, 4000
    rng = np.random.default_rng(3)
    v = (rng.random(n) + 0.01).astype(np.float32)
    m = rng.normal(size=n).astype(np.float32)
    total_m, total_v = np.zeros(n), np.zeros(n)
    for step in range(rounds):
        bits = L.random_bits(7, step, np.arange(n))
        total_m += L.decode_m(*L.encode_m(m, bits))
        total_v += L.decode_v(*L.encode_v(v, bits))
    # A step is 1/8 of the value at most: a deviation of 1/16 / sqrt(4000) of it
    # (a thousandth); six of those.
    assert np.all(np.abs(total_v / rounds - v) < 6 * v / 16 / np.sqrt(rounds))
    assert np.all(np.abs(total_m / rounds - m) < 6 * np.abs(m) / 16 / np.sqrt(rounds) + 1e-4)


def test_random_bits_depend_on_seed_step_and_place():
    a = L.random_bits(1, 1, np.arange(4096))
    for other in (L.random_bits(2, 1, np.arange(4096)), L.random_bits(1, 2, np.arange(4096)),
                  L.random_bits(1, 1, np.arange(4096, 8192))):
        same = np.mean((a[:, None] >> np.arange(32, dtype=np.uint32) & 1)
                       == (other[:, None] >> np.arange(32, dtype=np.uint32) & 1))
        # 131072 fair bits: a deviation of 0.0014; six of those.
        assert abs(same - 0.5) < 0.0084
    assert np.unique(a).size > 4090
    # Bits are fair one by one: 4096 of them, six deviations of 1/128.
    share = (a[:, None] >> np.arange(32, dtype=np.uint32) & 1).mean(0)
    assert np.all(np.abs(share - 0.5) < 6 / 128)
