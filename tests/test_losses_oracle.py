"""Pins oracle.losses: gradients against central differences in 64 bits,
values against closed forms."""

import numpy as np
import pytest

from oracle import losses


def _rows(seed, rows=5, vocab=9):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(rows, vocab)) * 2
    moves = [sorted(rng.choice(vocab, size=rng.integers(2, vocab), replace=False))
             for _ in range(rows)]
    moves[1] = [3, 3, 5, vocab + 4, -2]  # twice the same, and two outside
    actions = np.array([m[0] for m in moves])
    return rng, x, moves, actions


def _differences(f, x, step=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        hi, lo = x.copy(), x.copy()
        hi[i] += step
        lo[i] -= step
        g[i] = (f(hi) - f(lo)) / (2 * step)
    return g


@pytest.mark.parametrize("listed", [True, False])
@pytest.mark.parametrize("temp", [1.0, 0.7])
def test_policy_gradient_is_the_derivative(listed, temp):
    rng, x, moves, actions = _rows(1)
    kw = dict(temp=temp, old_logp=rng.normal(size=5) * 0.1 - 1.5, advantage=rng.normal(size=5),
              weight=np.array([1.0, 0.5, 2.0, 0.0, 1.0]), ref=x + 0.3 * rng.normal(size=x.shape),
              clip_low=0.2, clip_high=0.3, kl_coef=0.4, entropy_coef=0.2)
    m = moves if listed else None
    got = losses.policy_loss(x, m, actions, **kw)["grad"]
    want = _differences(lambda v: losses.policy_loss(v, m, actions, **kw)["loss"].sum(), x)
    # Central differences: third derivatives are below 10, so 10 h^2 / 6, and
    # the rounding of sums near 10 over 2 h: 10 * 2^-52 / 1e-6 = 2e-9.
    np.testing.assert_allclose(got, want, rtol=0, atol=2e-8)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
@pytest.mark.parametrize("average", [False, True])
def test_preference_gradient_is_the_derivative(kind, average):
    rng, x, moves, actions = _rows(2, rows=7)
    actions[2] = -1
    off = [0, 2, 4, 5, 6]
    kw = dict(kind=kind, beta=0.5, average=average, ref_logp=rng.normal(size=7) - 1.5,
              weight=np.array([0.7, 1.3]),
              label_smoothing=0.1 if kind == "sigmoid" else 0.0)
    got = losses.preference_loss(x, moves, actions, off, **kw)["grad"][:6]
    want = _differences(
        lambda v: losses.preference_loss(v, moves, actions, off, **kw)["loss"].sum(), x)
    assert np.all(want[6] == 0)
    np.testing.assert_allclose(got, want[:6], rtol=0, atol=5e-8)


def test_closed_forms():
    # Equal logits: p = 1/n, entropy ln n; a reference with one logit higher
    # by ln 2: q = 2/(n+1) there and 1/(n+1) elsewhere.
    x = np.zeros((1, 4))
    ref = x.copy()
    ref[0, 1] = np.log(2.0)
    out = losses.policy_loss(x, None, [2], old_logp=[np.log(0.25)], advantage=[3.0], ref=ref,
                             kl_coef=1.0)
    assert np.isclose(out["entropy"][0], np.log(4))
    kl = 0.25 * np.log(0.25 / 0.4) + 0.75 * np.log(0.25 / 0.2)
    assert np.isclose(out["kl"][0], kl) and np.isclose(out["loss"][0], kl - 3.0)
    # Ratio 2 and 1/2: clipped where that lowers the objective, and only there.
    for old, adv, want, moving in ((0.125, 1.0, -1.2, False), (0.125, -1.0, 2.0, True),
                                   (0.5, 1.0, -0.5, True), (0.5, -1.0, 0.8, False)):
        o = losses.policy_loss(x, None, [2], old_logp=[np.log(old)], advantage=[adv])
        assert np.isclose(o["loss"][0], want)
        assert np.any(o["grad"] != 0) == moving
    # A pair of the same sequence: h = 0, ln 2.
    o = losses.preference_loss(np.zeros((2, 4)), None, [1, 1], [0, 1, 2])
    assert np.isclose(o["loss"][0], np.log(2)) and o["margin"][0] == 0


def test_empty_rows_are_zero():
    x = np.full((2, 3), -np.inf)
    out = losses.policy_loss(x, [[0, 1], []], [0, 0], advantage=[1.0, 1.0], ref=x, kl_coef=1.0,
                             entropy_coef=1.0)
    assert all(np.all(v == 0) for v in out.values())


def test_clip_scales_to_the_norm():
    rng = np.random.default_rng(0)
    t = [rng.normal(size=n) for n in (1, 7, 100)]
    norm, got = losses.clip(t, 2.0)
    assert np.isclose(norm, np.linalg.norm(np.concatenate(t)))
    assert np.isclose(np.linalg.norm(np.concatenate(got)), 2.0)
    norm, got = losses.clip(t, 1e9)
    assert all(np.array_equal(a, b) for a, b in zip(t, got))
