"""mfh_preference_loss_device against the 64-bit oracle: kinds, types, move
lists and whole rows, sequences of no, one and many rows, rows outside the
sequences, rows without an action, weights, and both gradients against the
formula.  Bounds: ``loss_util``."""

import numpy as np
import pytest

import gpu_util
import learn_gpu as lg
import loss_util as lu
from metalfish_amd import backend
from oracle import losses

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


def check(batch, off, got, ref_logp=None, weight=None, **kw):
    want = losses.preference_loss(batch.values, batch.moves, batch.actions, off, temp=batch.temp,
                                  ref_logp=ref_logp, weight=weight, **kw)
    beta, kind, average = kw.get("beta", 0.1), kw.get("kind", "sigmoid"), kw.get("average", False)
    k = lu.additions(batch.vocab, batch.moves is not None)
    bounds = {b: lu.Bounds(losses.Row(batch.values[b],
                                      None if batch.moves is None else batch.moves[b],
                                      batch.actions[b], batch.temp), k)
              for b in range(off[0], off[-1])}
    for i in range((len(off) - 1) // 2):
        w = 1.0 if weight is None else float(weight[i])
        # The sums are in 64 bits: the error of D is that of its terms.
        err, counts = 0.0, []
        for j in (2 * i, 2 * i + 1):
            acted = [b for b in range(off[j], off[j + 1]) if bounds[b].row.acted]
            counts.append(max(1, len(acted)) if average else 1)
            err += sum(bounds[b].logp for b in acted) / counts[-1]
        err += lu.U * 1e-3
        h, diff = want["margin"][i], want["margin"][i] / beta
        lu.close(got["margin"][i], want["margin"][i], beta * err + 2 * lu.U * abs(h))
        # Slopes by D: at most beta (sigmoid, hinge) or 2 |D - 1 / (2 beta)|;
        # their own change with D: beta^2 / 4, 0 off the kink, 2.
        if kind == "square":
            first, second = 2 * abs(diff - 0.5 / beta), 2.0
        else:
            first, second = beta, beta * beta / 4 if kind == "sigmoid" else 0.0
        lu.close(got["loss"][i], want["loss"][i],
                 w * (first * err + second * err * err) + 2 * lu.U * want["loss"][i])
        for s, j in enumerate((2 * i, 2 * i + 1)):
            for b in range(off[j], off[j + 1]):
                bd = bounds[b]
                lu.close(got["logp"][b], want["logp"][b], bd.logp if bd.row.acted else 0.0)
                if "grad" not in got:
                    continue
                c = want["coef"][b]
                if c == 0.0:
                    assert np.all(got["grad"][b] == 0)
                    continue
                rel = w * second * err / counts[s] / abs(c) + 4 * lu.U
                lu.close(got["grad"][b], want["grad"][b], bd.grad(1.0 / batch.temp, c, rel),
                         batch.dtype)
    outside = [b for b in range(batch.rows) if b < off[0] or b >= off[-1]]
    keep = lu.from_bits(lg.SENTINEL[batch.dtype], batch.dtype)
    assert np.all(got["logp"][outside] == float(lg.SENTINEL["f32"]))
    if "grad" in got:
        assert np.all(got["grad"][outside] == keep)


def _batch(dev, rng, lengths, vocab, dtype, listed, lead=0, tail=0, temp=1.0, pad=0):
    off = list(np.concatenate([[0], np.cumsum(lengths)]) + lead)
    rows = int(off[-1] + tail)
    x = rng.normal(size=(rows, vocab)) * 2
    moves = [list(rng.choice(vocab, size=int(rng.integers(1, min(60, vocab) + 1)), replace=False))
             for _ in range(rows)] if listed else None
    actions = np.array([int(m[0]) for m in moves]) if listed else rng.integers(0, vocab, rows)
    actions[rng.random(rows) < 0.15] = -1
    batch = lg.Batch(dev, x, dtype, moves, actions, temp, pad)
    ref = (rng.normal(size=rows) * 0.5 - 3).astype(np.float32)
    weight = rng.uniform(0.5, 1.5, len(lengths) // 2).astype(np.float32)
    if len(weight) > 2:
        weight[1] = 0.0
    return batch, [int(v) for v in off], ref, weight


LENGTHS = ([1, 1], [0, 3, 4, 0, 0, 0, 1, 2], [5, 64, 65, 1, 300, 257, 2, 2], [1] * 40)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("listed", [True, False])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_lines_of_moves(dev, dtype, listed, lengths):
    rng = np.random.default_rng(len(lengths))
    batch, off, ref, weight = _batch(dev, rng, lengths, 1858, dtype, listed, lead=2, tail=3, pad=1)
    kw = dict(beta=0.2, label_smoothing=0.05)
    got = lg.preference(batch, off, ref, weight, **kw)
    check(batch, off, got, ref, weight, **kw)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
@pytest.mark.parametrize("average", [False, True])
def test_kinds(dev, kind, average):
    rng = np.random.default_rng(3)
    batch, off, ref, weight = _batch(dev, rng, [3, 4, 0, 7, 12, 1, 30, 31], 200, "f32", False)
    for beta in (0.05, 1.5):
        kw = dict(kind=kind, average=average, beta=beta)
        got = lg.preference(batch, off, ref, weight, **kw)
        check(batch, off, got, ref, weight, **kw)
        got = lg.preference(batch, off, None, None, grad=False, **kw)
        check(batch, off, got, None, None, **kw)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("vocab", [1, 65, 4097, 32000, 70001])
def test_vocabularies(dev, dtype, vocab):
    rng = np.random.default_rng(vocab)
    batch, off, ref, weight = _batch(dev, rng, [2, 1, 3, 4], vocab, dtype, False, lead=1, tail=1,
                                     temp=0.8)
    got = lg.preference(batch, off, ref, weight, beta=0.3)
    check(batch, off, got, ref, weight, beta=0.3)


@pytest.mark.parametrize("dtype,vocab", [("f32", 20003), ("bf16", 45001)])
def test_more_long_rows_than_the_card_runs_at_once(dev, dtype, vocab):
    rng = np.random.default_rng(vocab)
    lengths = [40, 50, 0, 3, 100, 120, 130, 57]
    off = [int(v) for v in np.concatenate([[0], np.cumsum(lengths)]) + 3]
    rows = off[-1] + 260
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * 2
    actions = rng.integers(0, vocab, rows)
    actions[10:30] = -1
    x[40, 5:] = -np.inf
    actions[40] = 2
    batch = lg.Batch(dev, x, dtype, None, actions)
    ref = (rng.normal(size=rows) * 0.5 - 10).astype(np.float32)
    weight = np.array([1.0, 0.0, 0.5, 1.0], np.float32)
    got = lg.preference(batch, off, ref, weight, beta=0.02)
    check(batch, off, got, ref, weight, beta=0.02)


@pytest.mark.parametrize("pairs,most", [(1, 1), (3, 8), (512, 2), (513, 2), (40, 16), (700, 5)])
def test_numbers_of_pairs(dev, pairs, most):
    """Both sides of the rule that takes a few short pairs in one launch."""
    rng = np.random.default_rng(pairs)
    lengths = list(rng.integers(0, most + 1, 2 * pairs))
    batch, off, ref, weight = _batch(dev, rng, lengths, 300, "f32", True, lead=1, tail=2)
    kw = dict(beta=0.3, label_smoothing=0.1)
    got = lg.preference(batch, off, ref, weight, **kw)
    check(batch, off, got, ref, weight, **kw)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("vocab", [2048, 4288, 32768])
def test_short_pairs_of_wide_lists(dev, dtype, vocab):
    """The one launch's LDS at its largest."""
    rng = np.random.default_rng(vocab)
    batch, off, ref, weight = _batch(dev, rng, [1, 2, 3, 4], vocab, dtype, True)
    got = lg.preference(batch, off, ref, weight, beta=0.3)
    check(batch, off, got, ref, weight, beta=0.3)


def test_pairs_of_empty_sequences_without_a_row(dev):
    loss, margin = lg.Column(dev, 2), lg.Column(dev, 2)
    for lists in ({}, dict(d_move_offsets=dev.put(np.zeros(1, np.int32)))):
        rows = backend.policy_rows(None, 0, 10, **lists)
        backend.preference_loss_device(rows, 2, dev.put(np.zeros(5, np.int32)), d_loss=loss.ptr,
                                       d_margin=margin.ptr, d_grad=dev.alloc(64))
        dev.sync()
        np.testing.assert_allclose(loss.get(), np.log(2.0), rtol=2 ** -23)
        assert np.all(margin.get() == 0)


def test_far_margins_do_not_overflow(dev):
    """h = +-1e4: the loss is |h| or 0, the gradient full or none."""
    x = np.zeros((4, 8))
    batch = lg.Batch(dev, x, "f32", None, [1, 2, 3, 4])
    ref = np.array([1e4, 0, -1e4, 0], np.float32)
    off = [0, 1, 2, 3, 4]
    got = lg.preference(batch, off, ref, None, beta=1.0)
    check(batch, off, got, ref, None, beta=1.0)
    assert got["loss"][1] == 0.0 and np.all(got["grad"][2:] == 0)


def test_masked_rows_and_nan_stay_in_their_pair(dev):
    rng = np.random.default_rng(4)
    x = rng.normal(size=(8, 30))
    x[0] = -np.inf                      # nothing left: as if it had no action
    x[5, 3] = np.nan
    batch = lg.Batch(dev, x, "f32", None, [1, 2, 3, 4, 5, 6, 7, 8])
    off = [0, 2, 4, 6, 8]
    got = lg.preference(batch, off, None, None, beta=0.5)
    assert np.isfinite(got["loss"][0]) and np.isnan(got["loss"][1])
    assert np.all(got["grad"][0] == 0) and got["logp"][0] == 0
    assert np.isnan(got["grad"][4:]).all() and np.isfinite(got["grad"][:4]).all()
    weight = np.array([1, 0], np.float32)   # weight 0 takes the pair out
    again = lg.preference(batch, off, None, weight, beta=0.5)
    assert np.all(again["grad"][4:] == 0) and again["loss"][1] == 0 and again["margin"][1] == 0
    assert np.array_equal(again["grad"][:4], got["grad"][:4])


def test_offsets_outside_the_rows_are_clamped(dev):
    rng = np.random.default_rng(5)
    x = rng.normal(size=(5, 30))
    batch = lg.Batch(dev, x, "f32", None, [1, 2, 3, 4, 5])
    got = lg.preference(batch, [-7, 2, 1 << 30], None, None)
    check(batch, [0, 2, 5], got)


@pytest.mark.parametrize("dtype", lu.TYPES)
def test_gradient_in_place_and_outputs_left_out(dev, dtype):
    rng = np.random.default_rng(6)
    for listed, vocab in ((True, 1858), (False, 1858), (False, 70001)):
        batch, off, ref, weight = _batch(dev, rng, [2, 3, 1, 2], vocab, dtype, listed, lead=1,
                                         tail=1, pad=2)
        a = lg.preference(batch, off, ref, weight)
        n = lg.preference(batch, off, ref, weight, grad=False)
        b = lg.preference(batch, off, ref, weight, in_place=True)
        for k in ("loss", "margin", "logp"):
            assert np.array_equal(a[k], b[k]) and np.array_equal(a[k], n[k])
        inside = slice(off[0], off[-1])
        assert np.array_equal(a["grad"][inside], b["grad"][inside])
        assert np.array_equal(b["grad"][0], batch.values[0])       # rows outside: the logits still


def test_same_bits_on_any_stream(dev):
    rng = np.random.default_rng(7)
    batch, off, ref, weight = _batch(dev, rng, list(rng.integers(0, 40, 60)), 1858, "bf16", True)
    first = lg.preference(batch, off, ref, weight)
    for stream in (None, dev.stream(), dev.stream()):
        again = lg.preference(batch, off, ref, weight, stream=stream)
        assert all(np.array_equal(first[k], again[k]) for k in first)


def test_gradient_against_differences(dev):
    """The device's own loss, differenced along random directions."""
    rng = np.random.default_rng(8)
    lengths = [3, 5, 2, 4]
    batch, off, ref, weight = _batch(dev, rng, lengths, 50, "f32", False)
    kw = dict(beta=2.0)
    grad = lg.preference(batch, off, ref, weight, **kw)["grad"]
    for trial in range(4):
        way = rng.normal(size=batch.values.shape)
        way /= np.linalg.norm(way)
        step = 2.0 ** -5
        sides = []
        for s in (1, -1):
            moved = lg.Batch(dev, batch.values + s * step * way, "f32", None, batch.actions)
            sides.append(lg.preference(moved, off, ref, weight, grad=False, **kw)["loss"].sum())
        slope = (sides[0] - sides[1]) / (2 * step)
        # Third derivatives of a sum of log-softmaxes in a unit direction are
        # below 2, of the loss below 2 beta^3 = 16: 16 step^2 / 6 = 2.7e-3;
        # rounding: 1e-6 times losses near 10 over 2 step = 1.6e-4.
        assert abs(slope - float(np.sum(grad * way))) < 3e-3, trial
