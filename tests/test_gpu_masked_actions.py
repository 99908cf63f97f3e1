"""Actions that a mask has taken out count as none, in the policy loss and in
both lines of a pair; and infinite margins and zero advantages leave no NaN."""

import numpy as np
import pytest

import gpu_util
import learn_gpu as lg
import loss_util as lu
from metalfish_amd import backend

pytestmark = pytest.mark.gpu

# A vocabulary for each kernel, and lists (vocabulary, moves).
SHAPES = {"wave": (200, 0), "waves": (1858, 0), "loop": (40009, 0), "streamed": (70001, 0),
          "list": (1858, 12), "long-list": (1858, 150)}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


def _rows(rng, shape, n):
    vocab, moves = SHAPES[shape]
    x = rng.normal(size=(n, vocab)) * 2
    lists = [list(rng.choice(vocab, moves, replace=False)) for _ in range(n)] if moves else None
    actions = np.array([int(m[3]) for m in lists]) if moves else rng.integers(0, vocab, n)
    return x, lists, actions


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_policy_loss(dev, shape, dtype):
    rng = np.random.default_rng(1)
    x, lists, actions = _rows(rng, shape, 5)
    for b in (0, 2, 3):
        x[b, actions[b]] = -np.inf
    ref = x + 0.3 * rng.normal(size=x.shape)
    none = actions.copy()
    none[[0, 2, 3]] = -1
    old = np.array([-np.inf, -2.0, -np.inf, -3.0, -4.0], np.float32)
    kw = dict(old_logp=old, advantage=np.array([1.0, 1, -1, 1, -1]), kl_coef=0.2, entropy_coef=0.1)
    for r in (None, ref):
        more = dict(kw, ref=r) if r is not None else dict(kw, kl_coef=0.0)
        got = lg.policy(lg.Batch(dev, x, dtype, lists, actions), **more)
        want = lg.policy(lg.Batch(dev, x, dtype, lists, none), **more)
        for k, v in got.items():
            assert np.isfinite(v).all(), k
            assert np.array_equal(v, want[k]), k
        assert np.all(got["logp"][[0, 2, 3]] == 0) and np.all(got["logp"][[1, 4]] < 0)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind,average", [("sigmoid", False), ("hinge", True), ("square", True)])
def test_preference_loss(dev, shape, dtype, kind, average):
    rng = np.random.default_rng(2)
    off = [0, 2, 5, 6, 9]
    x, lists, actions = _rows(rng, shape, 9)
    hidden = [1, 3, 5, 8]          # in chosen and rejected lines, one a line's only row
    for b in hidden:
        x[b, actions[b]] = -np.inf
    none = actions.copy()
    none[hidden] = -1
    ref = (rng.normal(size=9) - 4).astype(np.float32)
    ref[3] = -np.inf
    kw = dict(kind=kind, average=average, beta=0.3)
    got = lg.preference(lg.Batch(dev, x, dtype, lists, actions), off, ref, **kw)
    want = lg.preference(lg.Batch(dev, x, dtype, lists, none), off, ref, **kw)
    for k, v in got.items():
        assert np.isfinite(v).all(), k
        assert np.array_equal(v, want[k]), k
    assert np.all(got["logp"][hidden] == 0) and np.all(got["grad"][hidden] == 0)


@pytest.mark.parametrize("listed", [True, False])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
def test_infinite_margins(dev, kind, listed):
    """A reference that would never have played a move: +inf where that is the
    preferred line's, with nothing left to learn; -inf in the other."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=(4, 60))
    lists = [list(range(2, 20))] * 4 if listed else None
    ref = np.array([-np.inf, -2, -2, -np.inf], np.float32)
    got = lg.preference(lg.Batch(dev, x, "f32", lists, [5, 6, 7, 8]), [0, 1, 2, 3, 4], ref,
                        kind=kind, beta=0.5)
    assert list(got["margin"]) == [np.inf, -np.inf]
    assert got["loss"][1] == np.inf
    if kind != "square":
        assert got["loss"][0] == 0 and np.all(got["grad"][:2] == 0)
        assert np.isfinite(got["grad"][2:]).all() and np.any(got["grad"][2:] != 0)
    else:
        assert got["loss"][0] == np.inf


@pytest.mark.parametrize("shape", SHAPES)
def test_a_zero_advantage_is_no_surrogate(dev, shape):
    """Whatever the ratio: its overflow times 0 is 0."""
    rng = np.random.default_rng(4)
    x, lists, actions = _rows(rng, shape, 5)
    old = np.array([-200.0, -np.inf, -5.0, 3e38, -1e30], np.float32)
    for low, high in ((0.2, 0.2), (np.inf, np.inf)):
        batch = lg.Batch(dev, x, "f32", lists, actions)
        got = lg.policy(batch, old_logp=old, advantage=np.array([0.0, 0.0, 0.0, 0.0, -0.0]),
                        clip_low=low, clip_high=high)
        assert np.all(got["loss"] == 0) and np.all(got["grad"] == 0)
        assert np.all(got["logp"] < 0)
