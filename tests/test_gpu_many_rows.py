"""Every output is written anew by each call: more rows than one launch takes,
and pairs in one launch and in three, each from outputs that hold a pattern."""

import numpy as np
import pytest

import gpu_util
import learn_gpu as lg
import loss_util as lu
from metalfish_amd import backend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


@pytest.mark.parametrize("listed", [True, False])
def test_rows_of_several_launches(dev, listed):
    """More rows than one launch takes (2^21)."""
    rows = (1 << 21) + 5
    rng = np.random.default_rng(2)
    x = rng.standard_normal((rows, 2), dtype=np.float32)
    d_x, d_a = dev.put(x), dev.put((np.arange(rows) % 2).astype(np.int32))
    logp = lg.Column(dev, rows)
    grad = lg.Padded(dev, np.full((rows, 2), lg.SENTINEL["f32"]), "f32")
    kw = {}
    if listed:
        kw = dict(d_move_offsets=dev.put((2 * np.arange(rows + 1)).astype(np.int32)),
                  d_move_indices=dev.put(np.tile(np.array([0, 1], np.int16), rows)),
                  n_moves=2 * rows)
    r = backend.policy_rows(d_x, rows, 2, d_actions=d_a, **kw)
    backend.policy_loss_device(r, d_advantage=dev.put(np.ones(rows, np.float32)),
                               d_logp=logp.ptr, d_grad=grad.ptr)
    dev.sync()
    at = np.arange(rows) % 2
    d = (x[:, 1] - x[:, 0]).astype(np.float64) * np.where(at, 1, -1)
    want = -np.logaddexp(0, -d)
    # ln S is below 1, |z| below 12: the bounds of loss_util at K = 86; p(1 -
    # p) of the gradient twice that.
    limit = 2 * lu.U * (4 * 12 + 86 + 5 * 12 + 4)
    np.testing.assert_allclose(logp.get(), want, rtol=0, atol=limit)
    g = grad.get().astype(np.float64)
    np.testing.assert_allclose(g[np.arange(rows), at], -(1 - np.exp(want)), rtol=0, atol=2 * limit)
    np.testing.assert_allclose(g.sum(1), 0, rtol=0, atol=2 * limit)


@pytest.mark.parametrize("lists", [True, False])
def test_pairs_of_empty_sequences_without_a_row(dev, lists):
    loss, margin = lg.Column(dev, 2), lg.Column(dev, 2)
    kw = dict(d_move_offsets=dev.put(np.zeros(1, np.int32))) if lists else {}
    rows = backend.policy_rows(None, 0, 10, **kw)
    backend.preference_loss_device(rows, 2, dev.put(np.zeros(5, np.int32)), d_loss=loss.ptr,
                                   d_margin=margin.ptr, d_grad=dev.alloc(64))
    dev.sync()
    np.testing.assert_allclose(loss.get(), np.log(2.0), rtol=2 ** -23)
    assert np.all(margin.get() == 0)
