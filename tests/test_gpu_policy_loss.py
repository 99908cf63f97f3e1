"""mfh_policy_loss_device against the 64-bit oracle: types, vocabularies
around every size a kernel takes, strides and alignments, move lists with
none, one, repeated and outside entries, masks, temperatures, weights, and
which outputs are asked for.  Bounds: ``loss_util``."""

import ctypes

import numpy as np
import pytest

import gpu_util
import learn_gpu as lg
import loss_util as lu
from metalfish_amd import backend
from oracle import losses

pytestmark = pytest.mark.gpu

CLIP = dict(clip_low=0.2, clip_high=0.3)


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


def _scalars(rng, batch, ref, spread=0.15):
    """old_logp near the policy's own and off the clip's borders, advantages,
    weights (one of them 0)."""
    rows = batch.rows
    own = losses.policy_loss(batch.values, batch.moves, batch.actions, temp=batch.temp)["logp"]
    move = rng.normal(size=rows) * spread
    for border in (np.log(0.8), np.log(1.3)):
        near = np.abs(move - border) < 1e-3
        move[near] = border + 2e-3
    weight = rng.uniform(0.5, 1.5, rows)
    if rows > 2:
        weight[rows // 2] = 0.0
    return dict(old_logp=(own - move).astype(np.float32),
                advantage=rng.normal(size=rows).astype(np.float32),
                weight=weight.astype(np.float32))


def check(batch, got, ref=None, kl_coef=0.0, entropy_coef=0.0, old_logp=None, advantage=None,
          weight=None, rows=None):
    """Every output of `got` against the oracle."""
    refv = None if ref is None else lu.from_bits(lu.to_bits(ref, batch.dtype), batch.dtype)
    if kl_coef == 0.0 and "kl" not in got:
        refv = None
    want = losses.policy_loss(batch.values, batch.moves, batch.actions, temp=batch.temp,
                              old_logp=old_logp, advantage=advantage, weight=weight, ref=refv,
                              kl_coef=kl_coef, entropy_coef=entropy_coef, **CLIP)
    k = lu.additions(batch.vocab, batch.moves is not None)
    for b in range(batch.rows) if rows is None else rows:
        w = 1.0 if weight is None else float(weight[b])
        if w == 0.0:
            for v in got.values():
                assert np.all(v[b] == 0), b
            continue
        row = losses.Row(batch.values[b], None if batch.moves is None else batch.moves[b],
                         None if batch.actions is None else batch.actions[b], batch.temp,
                         None if refv is None else refv[b])
        bd = lu.Bounds(row, k)
        if row.empty:
            for v in got.values():
                assert np.all(v[b] == 0), b
            continue
        logp = bd.logp if row.acted else 0.0
        lu.close(got["logp"][b], want["logp"][b], logp)
        lu.close(got["entropy"][b], want["entropy"][b], bd.entropy)
        kl = 0.0
        if refv is not None:
            kl = bd.kl()[0]
            if "kl" in got:
                lu.close(got["kl"][b], want["kl"][b], kl)
        # rho = exp(logp - old): the error of logp, the difference's rounding,
        # and 2 ulp of the exponential and the products.
        dist = 0.0 if old_logp is None else abs(row.logp - float(old_logp[b]))
        slope_rel = logp + lu.U * (dist + 8)
        surrogate = 0.0
        if advantage is not None and row.acted:
            rho = 1.0 if old_logp is None else np.exp(row.logp - float(old_logp[b]))
            surrogate = min(rho, 1.3) * abs(float(advantage[b])) * slope_rel if want["slope"][b] \
                == 0.0 else abs(want["slope"][b] / w) * slope_rel
        total = surrogate + kl_coef * kl + entropy_coef * bd.entropy
        sizes = kl_coef * abs(row.kl) + entropy_coef * abs(row.entropy) + abs(want["loss"][b] / w)
        lu.close(got["loss"][b], want["loss"][b], 2 * w * (total + 4 * lu.U * sizes))
        if "grad" in got:
            lu.close(got["grad"][b], want["grad"][b],
                     bd.grad(w / batch.temp, want["slope"][b] / w, slope_rel, kl_coef,
                             entropy_coef), batch.dtype)


def _run_and_check(dev, rng, x, dtype, moves, actions, with_ref=True, temp=1.0, pad=0, shift=0,
                   noise=0.4, coefs=(0.3, 0.1), **kw):
    batch = lg.Batch(dev, x, dtype, moves, actions, temp, pad, shift)
    ref = x + noise * rng.normal(size=x.shape) if with_ref else None
    scalars = _scalars(rng, batch, ref)
    kl_coef = coefs[0] if with_ref else 0.0
    got = lg.policy(batch, ref=ref, kl_coef=kl_coef, entropy_coef=coefs[1], **scalars, **CLIP, **kw)
    check(batch, got, ref, kl_coef, coefs[1], **scalars)
    return batch, got


# Around each number of columns that a kernel variant holds (powers of two
# times 64 lanes), the policy's 1858 and the raw map's 4288, and one value.
VOCABS = (1, 2, 3, 63, 65, 255, 257, 511, 513, 1023, 1025, 1858, 2047, 2049, 4095, 4097, 4288, 8191,
          8193, 16383, 16385, 32767, 32769, 65535, 65537, 100003)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_whole_rows(dev, dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 7 if vocab < 5000 else 3
    x = rng.normal(size=(rows, vocab)) * 2
    actions = rng.integers(0, vocab, rows)
    actions[0], actions[-1] = 0, vocab - 1
    for with_ref in (True, False):
        _run_and_check(dev, rng, x, dtype, None, actions, with_ref, pad=vocab % 5, shift=vocab % 3)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("rows", [1, 2, 255, 3001])
def test_whole_rows_of_the_policy(dev, dtype, rows):
    rng = np.random.default_rng(rows)
    x = rng.normal(size=(rows, 1858)) * 2
    batch = lg.Batch(dev, x, dtype, None, rng.integers(0, 1858, rows))
    ref = x + 0.3 * rng.normal(size=x.shape)
    sc = _scalars(rng, batch, ref)
    got = lg.policy(batch, ref=ref, kl_coef=0.2, entropy_coef=0.05, **sc, **CLIP)
    check(batch, got, ref, 0.2, 0.05, **sc, rows=range(0, rows, max(1, rows // 60)))


@pytest.mark.parametrize("dtype,vocab", [("f32", 20003), ("f32", 28001), ("bf16", 40009),
                                         ("bf16", 65535), ("f16", 50021)])
@pytest.mark.parametrize("in_place", [False, True])
def test_more_long_rows_than_the_card_runs_at_once(dev, dtype, vocab, in_place):
    """Rows that a workgroup takes one after another, the next one's logits
    loaded ahead: among them rows of weight 0 (with NaN), rows with nothing
    left, masked rows, rows far below their reference, and the last row."""
    rng = np.random.default_rng(vocab)
    rows = 600
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * 2
    ref = x + 0.3 * rng.standard_normal((rows, vocab), dtype=np.float32)
    actions = rng.integers(0, vocab, rows)
    actions[5], actions[300] = vocab - 1, -1
    special = {1: "masked", 3: "empty", 257: "masked", 258: "far", 259: "nan", 400: "empty",
               511: "masked", 513: "far", 599: "masked"}
    weight = rng.uniform(0.5, 1.5, rows).astype(np.float32)
    for b, kind in special.items():
        actions[b] = 7
        if kind == "masked":
            x[b, 100:] = ref[b, 100:] = -np.inf
        elif kind == "empty":
            x[b] = -np.inf
        elif kind == "far":
            x[b, 50:60] -= 90.0
        else:
            x[b], weight[b] = np.nan, 0.0
    weight[[2, 255, 598]] = 0.0
    batch = lg.Batch(dev, x, dtype, None, actions, pad=vocab % 3)
    sc = dict(advantage=rng.normal(size=rows).astype(np.float32), weight=weight)
    got = lg.policy(batch, ref=ref, kl_coef=0.3, entropy_coef=0.1, in_place=in_place, **sc, **CLIP)
    some = sorted({0, 5, 256, 300, 512, 597, 2, 255, 598, *special, *range(20, 600, 97)})
    refv = lu.from_bits(lu.to_bits(ref[some], dtype), dtype)
    part = lg.Batch.__new__(lg.Batch)
    part.dev, part.dtype, part.moves, part.temp = dev, dtype, None, 1.0
    part.values, part.actions = batch.values[some], actions[some]
    part.rows, part.vocab = len(some), vocab
    check(part, {k: v[some] for k, v in got.items()}, refv, 0.3, 0.1,
          advantage=sc["advantage"][some], weight=weight[some])


def test_rows_of_several_launches(dev):
    """More rows than one launch takes (2^21)."""
    rows = (1 << 21) + 5
    rng = np.random.default_rng(2)
    x = rng.standard_normal((rows, 2), dtype=np.float32)
    d_x, d_a = dev.put(x), dev.put((np.arange(rows) % 2).astype(np.int32))
    logp, grad = lg.Column(dev, rows), dev.put(np.zeros_like(x))
    adv = dev.put(np.ones(rows, np.float32))
    off = dev.put((2 * np.arange(rows + 1)).astype(np.int32))
    idx = dev.put(np.tile(np.array([0, 1], np.int16), rows))
    d = (x[:, 1] - x[:, 0]).astype(np.float64) * np.where(np.arange(rows) % 2, 1, -1)
    want = -np.logaddexp(0, -d)
    for kw in ({}, dict(d_move_offsets=off, d_move_indices=idx, n_moves=2 * rows)):
        r = backend.policy_rows(d_x, rows, 2, d_actions=d_a, **kw)
        backend.policy_loss_device(r, d_advantage=adv, d_logp=logp.ptr, d_grad=grad)
        dev.sync()
        got = logp.get()
        # ln S is below 1, |z| below 12: the bounds of loss_util at K = 86.
        np.testing.assert_allclose(got, want, rtol=0, atol=2 * lu.U * (4 * 12 + 86 + 5 * 12 + 4))
        g = dev.get(grad, x)
        at = np.arange(rows) % 2
        np.testing.assert_allclose(g[np.arange(rows), at], -(1 - np.exp(want)), rtol=0, atol=4e-5)
        assert np.isfinite(g).all()


def _lists(rng, rows, vocab, most=60):
    out = []
    for b in range(rows):
        n = (0, 1, 2, 64, 65, 218, 256)[b] if b < 7 else int(rng.integers(1, most))
        out.append(list(rng.choice(vocab, size=min(n, vocab), replace=False)))
    if rows > 8:
        m = out[7]
        out[7] = [m[0], m[0], min(vocab, 32767), -1, -7, -32768] + m[:3] + [m[0]]  # repeated, outside
    return out


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1858, 0), (8, 5, 1), (300, 1858, 0), (40, 1858, 7),
                                            (20, 2048, 0), (20, 2049, 3), (12, 4288, 1),
                                            (12, 32768, 0), (9, 1, 0)])
def test_move_lists(dev, dtype, rows, vocab, pad):
    rng = np.random.default_rng(rows + vocab)
    x = rng.normal(size=(rows, vocab)) * 2
    moves = _lists(rng, rows, vocab)
    actions = np.array([int(m[-1]) if m else -1 for m in moves])
    for with_ref in (True, False):
        _run_and_check(dev, rng, x, dtype, moves, actions, with_ref, pad=pad)


def test_more_moves_than_a_row_has_are_cut_at_256(dev):
    rng = np.random.default_rng(5)
    x = rng.normal(size=(2, 1858))
    full = list(rng.choice(1858, 300, replace=False))
    batch = lg.Batch(dev, x, "f32", [full, [4, 5]], [full[0], 5])
    got = lg.policy(batch, advantage=[1.0, 1.0], **CLIP)
    batch.moves = [full[:256], [4, 5]]
    check(batch, got, advantage=[1.0, 1.0])


def test_offsets_outside_their_array_are_clamped(dev):
    x = np.random.default_rng(6).normal(size=(4, 20))
    batch = lg.Batch(dev, x, "f32", [[1, 2], [3], [4, 5, 6], [7]], [1, 3, 4, 7])
    dev.write(batch.desc.d_move_offsets, np.array([-5, 2, 3, 1 << 30, 2], np.int32))
    batch.moves = [[1, 2], [3], [4, 5, 6, 7], []]
    got = lg.policy(batch, advantage=np.ones(4), **CLIP)
    check(batch, got, advantage=np.ones(4))


@pytest.mark.parametrize("vocab", [40, 1858, 9001, 70001])
@pytest.mark.parametrize("dtype", lu.TYPES)
def test_masks_and_far_logits(dev, dtype, vocab):
    """Masks of -inf and of the type's lowest value, a row with nothing left,
    a row of lowest values alone, one entry far above the rest, and NaN and
    infinities in rows of weight 0."""
    rng = np.random.default_rng(vocab + 1)
    lowest = {"f32": -np.finfo(np.float32).max, "f16": -65504.0,
              "bf16": -float(lu.from_bits(np.uint16(0x7F7F), "bf16"))}[dtype]
    x = rng.normal(size=(8, vocab)) * 3
    ref = x + 0.3 * rng.normal(size=x.shape)
    hide = rng.random(vocab) < 0.8
    hide[3] = False
    x[0, hide] = ref[0, hide] = -np.inf
    x[1, hide] = lowest
    ref[1, hide] = lowest
    x[2] = ref[2] = -np.inf
    x[3] = ref[3] = lowest
    x[4, 3] = 60.0
    x[5, ::2] = np.nan
    ref[5, 1::2] = np.inf
    x[6, hide] = -np.inf          # masked in the policy, open in the reference
    x[7, hide] = lowest
    ref[7, hide] = -np.inf
    actions = np.full(8, 3)
    weight = np.array([1, 1, 1, 1, 1, 0, 1, 1], np.float32)
    batch = lg.Batch(dev, x, dtype, None, actions)
    sc = dict(advantage=rng.normal(size=8).astype(np.float32), weight=weight)
    got = lg.policy(batch, ref=ref, kl_coef=0.5, entropy_coef=0.1, **sc, **CLIP)
    check(batch, got, ref, 0.5, 0.1, **sc)


@pytest.mark.parametrize("vocab", [1858, 4288, 12000, 33000])
def test_finite_masks_whole_waves_wide_and_large_weights(dev, vocab):
    """Masks of the lowest value that cover all of a wave's columns, at
    temperatures and weights where their products overflow."""
    rng = np.random.default_rng(vocab + 2)
    lowest = -np.finfo(np.float32).max
    x = rng.normal(size=(6, vocab)) * 3
    ref = x + 0.3 * rng.normal(size=x.shape)
    x[0, 5:] = lowest
    x[1, :-3] = ref[1, :-3] = lowest
    x[2, 40:] = ref[2, 40:] = -np.inf
    x[3, 100:] = lowest
    ref[3, 100:] = -np.inf
    ref[4, 700:] = lowest
    x[4, 700:] = -1e4
    actions = np.array([1, vocab - 1, 3, 50, 20, 9])
    for temp, weight in ((1.0, 1.0), (4.0, 1.0), (4.0, 3e3), (0.3, 1e3)):
        batch = lg.Batch(dev, x, "f32", None, actions, temp)
        sc = dict(advantage=rng.normal(size=6).astype(np.float32),
                  weight=np.full(6, weight, np.float32))
        got = lg.policy(batch, ref=ref, kl_coef=0.2, entropy_coef=0.1, **sc, **CLIP)
        check(batch, got, ref, 0.2, 0.1, **sc)
        got = lg.policy(batch, entropy_coef=0.5, **sc, **CLIP)
        check(batch, got, None, 0.0, 0.5, **sc)


@pytest.mark.parametrize("vocab", [1858, 12000, 33000, 140000])
def test_weights_of_any_size(dev, vocab):
    """Loss scales, negative weights, and ones near the ends of the range."""
    rng = np.random.default_rng(vocab + 3)
    x = rng.normal(size=(6, vocab)) * 2
    ref = x + 0.3 * rng.normal(size=x.shape)
    weight = np.array([65536.0, -2.5, 1e-20, 3e30, -1e-9, 1.0], np.float32)
    lists = [list(range(5, 45))] * 6 if vocab == 1858 else None
    for moves in (None, lists) if lists else (None,):
        batch = lg.Batch(dev, x, "f32", moves, np.full(6, 9))
        sc = dict(advantage=rng.normal(size=6).astype(np.float32), weight=weight)
        got = lg.policy(batch, ref=ref, kl_coef=0.2, entropy_coef=0.1, **sc, **CLIP)
        for b in range(6):   # each row on its own scale
            part = lg.Batch.__new__(lg.Batch)
            part.dtype, part.moves, part.temp = "f32", None if moves is None else [moves[b]], 1.0
            part.values, part.actions = batch.values[b:b + 1], batch.actions[b:b + 1]
            part.rows, part.vocab = 1, vocab
            scale = 2.0 ** -np.round(np.log2(abs(float(weight[b]))))
            w = np.array([float(weight[b]) * scale])
            mine = {k: v[b:b + 1] * (scale if k in ("loss", "grad") else 1.0)
                    for k, v in got.items()}
            sign = np.sign(w[0])
            mine["loss"], mine["grad"] = mine["loss"] * sign, mine["grad"] * sign
            check(part, mine, ref[b:b + 1], 0.2, 0.1, advantage=sc["advantage"][b:b + 1],
                  weight=w * sign)


def test_masked_entries_of_move_lists(dev):
    rng = np.random.default_rng(8)
    x = rng.normal(size=(4, 1858))
    ref = x + 0.2 * rng.normal(size=x.shape)
    moves = [list(range(10)), list(range(70)), [5, 6], list(range(100, 130))]
    x[0, [1, 4]] = ref[0, [1, 4]] = -np.inf
    x[1, 10:70] = ref[1, 10:70] = -np.inf
    x[2, [5, 6]] = -np.inf
    x[3, :100] = np.nan           # not among the moves: not read
    ref[3, 130:] = np.inf
    for dtype in lu.TYPES:
        batch = lg.Batch(dev, x, dtype, moves, [0, 3, 5, 101])
        got = lg.policy(batch, ref=ref, kl_coef=0.5, entropy_coef=0.1, advantage=np.ones(4), **CLIP)
        check(batch, got, ref, 0.5, 0.1, advantage=np.ones(4))


def test_nan_and_infinity_show(dev):
    """A NaN or +inf logit that counts makes its row's outputs NaN, no other's."""
    x = np.zeros((4, 100))
    x[1, 7], x[2, 50] = np.nan, np.inf
    for moves in (None, [[1, 2], [7, 8], [50, 3], [4, 5]]):
        batch = lg.Batch(dev, x, "f32", moves, [1, 8, 3, 4])
        got = lg.policy(batch, advantage=np.ones(4), entropy_coef=0.1, **CLIP)
        for k in ("loss", "logp", "entropy"):
            assert list(np.isnan(got[k])) == [False, True, True, False], (k, got[k])
        assert np.isnan(got["grad"][1, 7]) and np.isnan(got["grad"][2, 50])
        assert np.isfinite(got["grad"][[0, 3]]).all()


def test_a_reference_without_what_the_policy_plays_is_infinitely_far(dev):
    x = np.zeros((2, 50))
    ref = x.copy()
    ref[0, 10] = -np.inf
    batch = lg.Batch(dev, x, "f32", None, [1, 1])
    got = lg.policy(batch, ref=ref, kl_coef=0.0, advantage=np.ones(2), grad=False, **CLIP)
    assert got["kl"][0] == np.inf and got["kl"][1] == 0.0


@pytest.mark.parametrize("temp", [0.25, 0.7, 2.2, 30.0])
def test_temperatures(dev, temp):
    rng = np.random.default_rng(9)
    x = rng.normal(size=(20, 1858)) * 3
    moves = _lists(rng, 20, 1858)
    actions = np.array([int(m[0]) if m else -1 for m in moves])
    for dtype in ("f32", "bf16"):
        _run_and_check(dev, rng, x, dtype, moves, actions, temp=temp)
        _run_and_check(dev, rng, x, dtype, None, actions, temp=temp)


def test_near_policies_have_a_small_divergence(dev):
    """KL of policies 1e-3 apart (about 5e-7): a difference of log-sum-exps
    near 8 would be off by 1e-6."""
    rng = np.random.default_rng(10)
    x = rng.normal(size=(9, 1858))
    for moves in (None, _lists(rng, 9, 1858)):
        actions = np.full(9, -1)
        batch = lg.Batch(dev, x, "f32", moves, actions)
        ref = x + 1e-3 * rng.normal(size=x.shape)
        got = lg.policy(batch, ref=ref, kl_coef=1.0, **CLIP)
        check(batch, got, ref, 1.0)
        assert np.all(got["kl"] >= 0)
    got = lg.policy(batch, ref=batch.values, kl_coef=1.0, **CLIP)
    assert np.all(got["kl"] == 0) and np.all(got["grad"] == 0)


def test_actions_that_are_none(dev):
    """-1, one outside the vocabulary, one that is no move of the row, and no
    actions at all: no surrogate, the other terms stay."""
    rng = np.random.default_rng(11)
    x = rng.normal(size=(6, 64))
    moves = [[1, 2, 3]] * 6
    for m in (moves, None):
        for actions in ([-1, 64, 1 << 30, -(1 << 31), 1, 3], None):
            batch = lg.Batch(dev, x, "f32", m, actions)
            got = lg.policy(batch, advantage=np.ones(6), entropy_coef=0.3, **CLIP)
            check(batch, got, None, 0.0, 0.3, advantage=np.ones(6))
    batch = lg.Batch(dev, x, "f32", moves, [4, 5, 6, 7, 1, 0])
    got = lg.policy(batch, advantage=np.ones(6), **CLIP)
    check(batch, got, advantage=np.ones(6))
    assert list(got["loss"] != 0) == [False] * 4 + [True, False]


def test_outputs_can_be_left_out(dev):
    """Any subset gives the same bits as all together."""
    rng = np.random.default_rng(12)
    for vocab, moves in ((1858, True), (300, False), (40001, False), (90001, False)):
        x = rng.normal(size=(5, vocab))
        lists = [list(range(3, 40))] * 5 if moves else None
        batch = lg.Batch(dev, x, "f32", lists, [5] * 5)
        ref = x + 0.3 * rng.normal(size=x.shape)
        sc = _scalars(rng, batch, ref)
        kw = dict(ref=ref, kl_coef=0.3, entropy_coef=0.1, **sc, **CLIP)
        full = lg.policy(batch, **kw)
        for outputs, grad in (((), True), (("loss",), False), (("kl",), False), (("logp",), False),
                              (("entropy", "kl"), True), (("loss",), True), ((), False)):
            got = lg.policy(batch, outputs=outputs, grad=grad, **kw)
            for k, v in got.items():
                assert np.array_equal(v, full[k]), (vocab, outputs, k)
        # kl without a coefficient leaves the loss alone.
        kw["kl_coef"] = 0.0
        a, b = lg.policy(batch, **kw), lg.policy(batch, **dict(kw, ref=None))
        assert np.array_equal(a["kl"], full["kl"])
        for k in ("loss", "grad", "logp", "entropy"):
            lu.close(a[k], b[k], 4 * lu.U * np.abs(b[k]))


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("vocab,moves", [(1858, True), (1858, False), (30011, False),
                                         (80001, False)])
def test_gradient_in_place(dev, dtype, vocab, moves):
    rng = np.random.default_rng(13)
    x = rng.normal(size=(6, vocab))
    lists = [sorted(rng.choice(vocab, 30, replace=False)) for _ in range(6)] if moves else None
    actions = [m[0] for m in lists] if moves else [7] * 6
    batch = lg.Batch(dev, x, dtype, lists, actions, pad=3)
    ref = x + 0.3 * rng.normal(size=x.shape)
    sc = _scalars(rng, batch, ref)
    kw = dict(ref=ref, kl_coef=0.3, entropy_coef=0.1, **sc, **CLIP)
    apart = lg.policy(batch, **kw)
    same = lg.policy(batch, in_place=True, **kw)
    for k in apart:
        assert np.array_equal(apart[k], same[k]), k


def test_open_clips_and_own_log_probabilities(dev):
    """Infinite bounds never clip; without old log-probabilities rho is 1."""
    rng = np.random.default_rng(14)
    x = rng.normal(size=(8, 1858))
    batch = lg.Batch(dev, x, "f32", None, rng.integers(0, 1858, 8))
    adv = rng.normal(size=8).astype(np.float32)
    own = losses.policy_loss(batch.values, None, batch.actions)["logp"]
    old = (own + rng.normal(size=8) * 2).astype(np.float32)
    got = lg.policy(batch, old_logp=old, advantage=adv, clip_low=np.inf, clip_high=np.inf)
    rho = np.exp(got["logp"] - old)
    np.testing.assert_allclose(got["loss"], -rho * adv, rtol=1e-5)  # 2^-24 times |logp| ~ 10, x 8
    got = lg.policy(batch, advantage=adv, **CLIP)
    assert np.array_equal(got["loss"], -adv.astype(np.float64))
    check(batch, got, advantage=adv)


def test_same_bits_every_time_and_on_any_stream(dev):
    rng = np.random.default_rng(15)
    x = rng.normal(size=(500, 1858))
    moves = _lists(rng, 500, 1858)
    actions = [int(m[0]) if m else -1 for m in moves]
    s = [dev.stream(), dev.stream()]
    for m in (moves, None):
        batch = lg.Batch(dev, x, "bf16", m, actions)
        ref = x + 0.3 * rng.normal(size=x.shape)
        kw = dict(ref=ref, kl_coef=0.3, entropy_coef=0.1, **_scalars(rng, batch, ref), **CLIP)
        first = lg.policy(batch, **kw)
        for stream in (None, s[0], s[1]):
            again = lg.policy(batch, stream=stream, **kw)
            assert all(np.array_equal(first[k], again[k]) for k in first)


def test_rows_beyond_two_gigabytes_apart(dev):
    """Offsets that pass 32 bits: three rows 1.2 G elements apart."""
    stride = 1_200_000_000
    hip = dev.hip
    base = dev.alloc((2 * stride + 64) * 2)
    rng = np.random.default_rng(16)
    x = lu.to_bits(rng.normal(size=(3, 64)), "bf16")
    for b in range(3):
        dev.write(base + b * stride * 2, x[b])
    rows = backend.policy_rows(base, 3, 64, dtype="bf16", stride=stride,
                               d_actions=dev.put(np.array([1, 2, 63], np.int32)))
    logp = lg.Column(dev, 3)
    grad = dev.put(np.zeros((3, 64), np.uint16))
    backend.policy_loss_device(rows, d_advantage=dev.put(np.ones(3, np.float32)), d_logp=logp.ptr,
                               d_grad=grad)
    dev.sync()
    want = losses.policy_loss(lu.from_bits(x, "bf16"), None, [1, 2, 63], advantage=np.ones(3))
    np.testing.assert_allclose(logp.get(), want["logp"], rtol=1e-5)
    got = lu.from_bits(dev.get(grad, np.zeros((3, 64), np.uint16)), "bf16")
    np.testing.assert_allclose(got, want["grad"], rtol=2 ** -8 + 1e-5, atol=1e-6)
    assert hip is not None


def test_host_memory_is_refused(dev):
    """Checked on the host: nothing is launched."""
    x = np.zeros((2, 8), np.float32)
    out = np.zeros(2, np.float32)
    rows = backend.policy_rows(x.ctypes.data, 2, 8)
    with pytest.raises(RuntimeError, match="d_logits is not device memory"):
        backend.policy_loss_device(rows, d_loss=dev.put(out))
    rows = backend.policy_rows(dev.put(x), 2, 8)
    with pytest.raises(RuntimeError, match="d_loss is not device memory"):
        backend.policy_loss_device(rows, d_loss=out.ctypes.data)
    with pytest.raises(RuntimeError, match="ordinal out of range"):
        backend.policy_loss_device(backend.policy_rows(dev.put(x), 2, 8, device=64),
                                   d_loss=dev.put(out))
    assert isinstance(rows, ctypes.Structure)
