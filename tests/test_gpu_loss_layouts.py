"""The losses on layouts and calls that their other tests leave out: the
gradient over the reference, strides of each array's own, rows of millions of
columns, long rows in a captured graph, preference weights of any size, and
lists in pairs of unlike lengths.  Each against the same rows laid out plainly
(the same bits) or against the 64-bit oracle."""

import numpy as np
import pytest

import gpu_util
import learn_gpu as lg
import loss_util as lu
from metalfish_amd import backend
from oracle import losses

pytestmark = pytest.mark.gpu

# A vocabulary for each kernel, and lists (vocabulary, moves).
SHAPES = {"wave": (200, 0), "waves": (1858, 0), "eight": (24001, 0), "loop": (40009, 0),
          "streamed": (70001, 0), "list": (1858, 12), "long-list": (1858, 150)}
LOWEST = {"f32": -float(np.finfo(np.float32).max), "f16": -65504.0,
          "bf16": -float(lu.from_bits(np.uint16(0x7F7F), "bf16"))}
KW = dict(kl_coef=0.3, entropy_coef=0.1, clip_low=0.2, clip_high=0.3)


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


def _rows(rng, shape, dtype):
    """Near and far rows, masked ones, and one of weight 0."""
    vocab, moves = SHAPES[shape]
    x = rng.normal(size=(8, vocab)) * 2
    ref = x + 0.3 * rng.normal(size=x.shape)
    ref[1] -= 500.0                                 # a constant away
    ref[2, ::3] = LOWEST[dtype]                     # far apart, KL beyond 88
    x[3, 1::2] = ref[3, 1::2] = -np.inf
    x[4] = np.nan
    ref[5] = LOWEST[dtype]
    x[6] = -np.inf
    lists = [list(rng.choice(vocab, moves, replace=False)) for _ in range(8)] if moves else None
    actions = np.array([int(m[2]) for m in lists]) if moves else rng.integers(0, vocab, 8)
    weight = np.array([1, 2, 0.5, 1, 0, 1, 1, 1], np.float32)
    return x, ref, lists, actions, dict(advantage=rng.normal(size=8).astype(np.float32),
                                        weight=weight)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradient_over_the_logits_and_over_the_reference(dev, shape, dtype):
    rng = np.random.default_rng(1)
    x, ref, lists, actions, sc = _rows(rng, shape, dtype)
    batch = lg.Batch(dev, x, dtype, lists, actions, pad=3)
    apart = lg.policy(batch, ref=ref, **sc, **KW)
    scalars = {"d_" + k: lg.f32(dev, v) for k, v in sc.items()}
    for over in ("logits", "reference"):
        batch = lg.Batch(dev, x, dtype, lists, actions, pad=3)
        r = batch.like(ref)
        grad = batch.x if over == "logits" else r
        cols = {k: lg.Column(dev, 8) for k in ("loss", "logp", "kl", "entropy")}
        backend.policy_loss_device(batch.desc, d_ref_logits=r.ptr, ref_stride=r.stride,
                                   d_grad=grad.ptr, grad_stride=grad.stride, **scalars,
                                   **{"d_" + k: c.ptr for k, c in cols.items()}, **KW)
        dev.sync()
        for k, c in cols.items():
            assert np.array_equal(c.get().astype(np.float64), apart[k], equal_nan=True), (over, k)
        got = lu.from_bits(grad.get(), dtype)
        assert np.array_equal(got, apart["grad"], equal_nan=True), over


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_strides_of_their_own(dev, shape, dtype):
    """Logits, reference and gradient each with another stride and start."""
    rng = np.random.default_rng(2)
    x, ref, lists, actions, sc = _rows(rng, shape, dtype)
    plain = lg.policy(lg.Batch(dev, x, dtype, lists, actions), ref=ref, **sc, **KW)
    batch = lg.Batch(dev, x, dtype, lists, actions, pad=5, shift=1)
    r = lg.Padded(dev, lu.to_bits(ref, dtype), dtype, 2, 3)
    grad = lg.Padded(dev, np.full(x.shape, lg.SENTINEL[dtype]), dtype, 12, 6)
    cols = {k: lg.Column(dev, 8) for k in ("loss", "kl")}
    backend.policy_loss_device(batch.desc, d_ref_logits=r.ptr, ref_stride=r.stride,
                               d_grad=grad.ptr, grad_stride=grad.stride,
                               **{"d_" + k: lg.f32(dev, v) for k, v in sc.items()},
                               **{"d_" + k: c.ptr for k, c in cols.items()}, **KW)
    dev.sync()
    for k, c in cols.items():
        assert np.array_equal(c.get().astype(np.float64), plain[k], equal_nan=True)
    assert np.array_equal(lu.from_bits(grad.get(), dtype), plain["grad"], equal_nan=True)
    batch.x.get(), r.get()


@pytest.mark.parametrize("dtype,vocab", [("f32", 3_000_001), ("bf16", 2_000_003)])
def test_millions_of_columns(dev, dtype, vocab):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, vocab), dtype=np.float32) * 2
    ref = x + 0.3 * rng.standard_normal((2, vocab), dtype=np.float32)
    actions = np.array([vocab - 1, 5])
    adv = np.array([1.0, -0.5], np.float32)
    batch = lg.Batch(dev, x, dtype, None, actions)
    got = lg.policy(batch, ref=ref, advantage=adv, **KW)
    refv = lu.from_bits(lu.to_bits(ref, dtype), dtype)
    want = losses.policy_loss(batch.values, None, actions, advantage=adv, ref=refv, **KW)
    k = lu.additions(vocab, False)
    for b in range(2):
        row = losses.Row(batch.values[b], None, actions[b], 1.0, refv[b])
        bd = lu.Bounds(row, k)
        kl = bd.kl()[0]
        lu.close(got["logp"][b], want["logp"][b], bd.logp)
        lu.close(got["entropy"][b], want["entropy"][b], bd.entropy)
        lu.close(got["kl"][b], want["kl"][b], kl)
        lu.close(got["grad"][b], want["grad"][b],
                 bd.grad(1.0, want["slope"][b], bd.logp + 8 * lu.U, 0.3, 0.1), dtype)


@pytest.mark.parametrize("shape", SHAPES)
def test_captured_and_replayed_on_new_logits(dev, shape):
    """Both losses in a graph, replayed between eager calls."""
    rng = np.random.default_rng(4)
    x, ref, lists, actions, sc = _rows(rng, shape, "bf16")
    batch = lg.Batch(dev, x, "bf16", lists, actions)
    r, scalars = batch.like(ref), {"d_" + k: lg.f32(dev, v) for k, v in sc.items()}
    seq = dev.put(np.array([0, 3, 4, 6, 8], np.int32))
    need = backend.preference_loss_workspace_bytes(8)
    ws, stream = dev.alloc(need), dev.stream()
    side = [dict(kl=lg.Column(dev, 8), grad=batch.blank(), margin=lg.Column(dev, 2),
                 pref=batch.blank()) for _ in range(2)]

    def run(out, s):
        backend.policy_loss_device(batch.desc, d_ref_logits=r.ptr, ref_stride=r.stride,
                                   d_kl=out["kl"].ptr, d_grad=out["grad"].ptr,
                                   grad_stride=out["grad"].stride, stream=s, **scalars, **KW)
        backend.preference_loss_device(batch.desc, 2, seq, d_margin=out["margin"].ptr,
                                       d_grad=out["pref"].ptr, grad_stride=out["pref"].stride,
                                       d_workspace=ws, workspace_bytes=need, stream=s)

    launch = dev.capture(stream, lambda: run(side[0], stream))
    for turn in range(4):
        moved = np.where(np.isfinite(x), x + 0.2 * rng.normal(size=x.shape), x)
        moved[4] = 1.0 + turn
        flat = batch.x.flat.copy()
        batch.x.view(flat)[:, :batch.vocab] = lu.to_bits(moved, "bf16")
        dev.write(batch.x.base, flat)
        launch()
        dev.sync(stream)
        run(side[1], None)
        dev.sync()
        for k in side[0]:
            a, b = side[0][k].get(), side[1][k].get()
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), (turn, k)
        assert np.any(side[0]["pref"].get() != 0)


@pytest.mark.parametrize("shape", SHAPES)
def test_preference_weights_of_any_size(dev, shape):
    """Loss scales and negative weights: the gradient of the pair of weight 1,
    times them."""
    rng = np.random.default_rng(5)
    vocab, moves = SHAPES[shape]
    weight = np.array([1.0, 65536.0, 2.0 ** 60, -2.0, 2.0 ** -30], np.float32)
    one = rng.normal(size=(3, vocab))
    x = np.tile(one, (5, 1))
    m = [list(rng.choice(vocab, moves, replace=False)) for _ in range(3)] if moves else None
    lists = m * 5 if moves else None
    a = np.array([int(v[1]) for v in m]) if moves else rng.integers(0, vocab, 3)
    off = list(np.concatenate([[0], np.cumsum([1, 2] * 5)]))
    got = lg.preference(lg.Batch(dev, x, "f32", lists, np.tile(a, 5)), off, None, weight, beta=0.3)
    want = losses.preference_loss(one, m, a, [0, 1, 3], beta=0.3)
    k = lu.additions(vocab, bool(moves))
    bd = [lu.Bounds(losses.Row(one[b].astype(np.float32), m[b] if moves else None, a[b]), k)
          for b in range(3)]
    err = sum(b.logp for b in bd) + lu.U
    for i, w in enumerate(weight.astype(np.float64)):
        lu.close(got["loss"][i] / w, want["loss"][0], 0.3 * err + 4 * lu.U * want["loss"][0])
        for b in range(3):
            c = abs(want["coef"][b])
            lu.close(got["grad"][3 * i + b] / w, want["grad"][b],
                     bd[b].grad(1.0, c, 0.3 * 0.3 / 4 * err / c + 4 * lu.U))


@pytest.mark.parametrize("lengths", [[40, 30, 1, 1, 2, 1, 0, 1, 1, 1] * 2, [200, 1] + [1, 0] * 40])
@pytest.mark.parametrize("average", [False, True])
def test_one_long_line_among_short_ones(dev, lengths, average):
    """On both sides of the rule that takes few rows a pair in one launch: more
    rows behind the last sequence give the same bits."""
    rng = np.random.default_rng(6)
    off = [int(v) for v in np.concatenate([[0], np.cumsum(lengths)])]
    pairs = len(lengths) // 2
    rows = max(off[-1], 8 * pairs) + 1
    vocab = 300
    x = rng.normal(size=(rows, vocab))
    lists = [list(rng.choice(vocab, int(rng.integers(1, 40)), replace=False)) for _ in range(rows)]
    actions = np.array([int(m[0]) for m in lists])
    actions[rng.random(rows) < 0.2] = -1
    ref = (rng.normal(size=rows) - 3).astype(np.float32)
    sides = []
    for n in (off[-1], rows):
        batch = lg.Batch(dev, x[:n], "f32", lists[:n], actions[:n])
        sides.append(lg.preference(batch, off, ref[:n], beta=0.2, average=average))
    want = losses.preference_loss(x, lists, actions, off, beta=0.2, average=average, ref_logp=ref)
    np.testing.assert_allclose(sides[0]["margin"], want["margin"], rtol=0, atol=241 * 0.2 * 3e-6)
    for k in sides[0]:
        n = off[-1] if k in ("logp", "grad") else pairs
        a, b = sides[0][k][:n], sides[1][k][:n]
        # Sums over 8 waves and over one or four differ by 2^-52.
        if k == "logp":
            assert np.array_equal(a, b)
        else:
            np.testing.assert_allclose(a, b, rtol=2 ** -22, atol=2 ** -100)
