"""An action that a mask has taken out of its row counts as none."""

import numpy as np
import pytest

from oracle import losses


@pytest.mark.parametrize("moves", [None, [[4, 1, 2], [4, 1, 2], [4, 1, 2]]])
def test_a_masked_action_is_none(moves):
    rng = np.random.default_rng(1)
    x = rng.normal(size=(3, 6))
    x[0, 1] = x[2, 1] = -np.inf
    kw = dict(old_logp=[-np.inf, -2.0, -1.0], advantage=[1.0, 1.0, -1.0], entropy_coef=0.1)
    got = losses.policy_loss(x, moves, [1, 1, 1], **kw)
    want = losses.policy_loss(x, moves, [-1, 1, -1], **kw)
    for k in got:
        assert np.array_equal(got[k], want[k]) and np.isfinite(got[k]).all()
    assert got["logp"][0] == got["logp"][2] == 0.0 and got["logp"][1] < 0


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
def test_in_either_line_of_a_pair(kind):
    rng = np.random.default_rng(2)
    x = rng.normal(size=(4, 6))
    x[1, 3] = x[2, 0] = -np.inf
    got = losses.preference_loss(x, None, [1, 3, 0, 2], [0, 2, 4], kind=kind, average=True)
    want = losses.preference_loss(x, None, [1, -1, -1, 2], [0, 2, 4], kind=kind, average=True)
    for k in got:
        assert np.array_equal(got[k], want[k]) and np.isfinite(got[k]).all()


def test_an_infinite_margin_without_smoothing():
    out = losses.preference_loss(np.zeros((2, 4)), None, [1, 1], [0, 1, 2],
                                 ref_logp=[-np.inf, -1.0])
    assert out["margin"][0] == np.inf and out["loss"][0] == 0 and np.all(out["grad"] == 0)


def test_a_zero_advantage_takes_any_ratio():
    out = losses.policy_loss(np.zeros((2, 4)), None, [1, 1], old_logp=[-np.inf, -2000.0],
                             advantage=[0.0, -0.0])
    assert np.all(out["loss"] == 0) and np.all(out["grad"] == 0)
