"""KL of the policy loss where the policy and its reference are far apart:
divergences beyond 88 nats, finite masks in the reference, weights of any
size, references a constant away, and KL watched without a coefficient.  On
whole rows of one wave, of several, in the loop and streamed, and on lists.

Bounds: ``loss_util``'s, with u = d - E_p d off by 3 roundings of what d is
formed from, and for KL of 1 and more as an error of the logarithm: the
relative errors of the terms p exp(-u), weighted by their shares q."""

import numpy as np
import pytest

import gpu_util
import learn_gpu as lg
import loss_util as lu
from metalfish_amd import backend
from oracle import losses

pytestmark = pytest.mark.gpu

LOWEST = {"f32": -float(np.finfo(np.float32).max), "f16": -65504.0,
          "bf16": -float(lu.from_bits(np.uint16(0x7F7F), "bf16"))}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


class Bounds(lu.Bounds):
    def kl(self):
        row, p, temp = self.row, self.row.p, self.row.temp
        on = p > 0
        with np.errstate(all="ignore"):
            raw = row.v - row.r
            zx, zy = (row.v - np.max(row.v)) / temp, (row.r - np.max(row.r)) / temp
            mean_raw = float(np.sum(np.where(on, p * raw, 0.0)))
            # Far references are taken relative to both maxima.
            apart = abs(mean_raw) > 64
            d = np.where(on, zx - zy if apart else raw / temp, 0.0)
            size = np.abs(d) + (np.where(on, np.abs(zx) + np.abs(zy), 0.0) if apart else 0.0)
            mean = float(np.sum(p * d))
            u = np.where(on, d - mean, 0.0)
            off_mean = float(np.sum(p * (np.abs(d) * (self.rel_p + (self.k + 7) * lu.U) +
                                         3 * lu.U * size)))
            off_u = 3 * lu.U * size + lu.U * np.abs(u) + off_mean
            q = np.exp(row.lq)
            offset = 0.0 if apart else abs(np.max(row.v) - np.max(row.r)) / temp
            rel = np.where(on, self.rel_p + off_u + lu.U * (self.k + 14 + 4 * np.abs(u)),
                           off_mean + lu.U * (self.k + 14 + 8 * np.abs(zy)
                                              + 8 * (offset + abs(mean))))
            rel = np.where(q > 0, rel, 0.0)
            if row.kl >= 1:
                bound = float(np.sum(q * rel)) + 3 * lu.U * offset
            else:
                grow = np.exp(np.minimum(-u, 700.0))
                phi = np.maximum(grow - 1 + u, 0.0)
                terms = p * (phi * (self.rel_p + (self.k + 10) * lu.U) + np.abs(1 - grow) * off_u +
                             grow * off_u ** 2 +
                             np.where(np.abs(u) < 0.2, 0.0,
                                      4 * lu.U * (grow * (1 + np.abs(u)) + 1 + np.abs(u))))
                bound = float(np.sum(np.where(on, terms, 3 * q * rel)))
        return 2 * (self.p_mass(bound) + 4 * lu.U * abs(row.kl)), off_u, np.abs(u)

    def p_mass(self, bound):
        # p below 2^-126 is 0 on the device, at u > -40 with exp(-u) < 2^58; the
        # oracle's logarithms of sums near 1 are off by 2^-53 a step.
        return bound + self.row.p.size * 2.0 ** -68 + 2.0 ** -50

    def grad(self, scale, slope, slope_rel, kl_coef=0.0, entropy_coef=0.0):
        """The same, with what such p miss in the means, and the oracle's own
        rounding (2^-53 a step) of ln p - ln q - KL."""
        row, p = self.row, self.row.p
        on = p > 0
        with np.errstate(all="ignore"):
            known = super().grad(scale, slope, slope_rel, kl_coef, entropy_coef)
            far = abs(kl_coef) * np.max(np.where(on, np.abs(row.v - row.r), 0.0)) / row.temp + \
                abs(entropy_coef) * np.max(np.where(on, np.abs(self.z), 0.0))
            own = p * np.where(on, np.abs(row.lp) + np.abs(row.lq) + abs(row.kl), 0.0)
        return known + abs(scale) * (row.spread(p * far * p.size * 2.0 ** -125) +
                                     row.spread(own * 2.0 ** -50))


def check(batch, got, ref, kl_coef, entropy_coef=0.0, weight=None):
    """KL, loss and gradient of every row, without a surrogate."""
    refv = lu.from_bits(lu.to_bits(ref, batch.dtype), batch.dtype)
    k = lu.additions(batch.vocab, batch.moves is not None)
    for b in range(batch.rows):
        w = 1.0 if weight is None else float(weight[b])
        row = losses.Row(batch.values[b], None if batch.moves is None else batch.moves[b], None,
                         batch.temp, refv[b])
        bd = Bounds(row, k)
        kl = bd.kl()[0]
        lu.close(got["kl"][b], row.kl, kl)
        want = kl_coef * row.kl - entropy_coef * row.entropy
        total = kl_coef * kl + entropy_coef * bd.entropy
        sizes = kl_coef * abs(row.kl) + entropy_coef * abs(row.entropy) + abs(want)
        lu.close(got["loss"][b], w * want, 2 * abs(w) * (total + 4 * lu.U * sizes))
        grad = kl_coef * row.grad_kl() - entropy_coef * row.grad_entropy()
        lu.close(got["grad"][b], w * grad,
                 bd.grad(w / batch.temp, 0.0, 0.0, kl_coef, entropy_coef), batch.dtype)


# A vocabulary for each kernel: one wave, four, eight, the loop, streamed, and
# lists of a few and of more than 64 moves (vocabulary, moves).
SHAPES = {"wave": (256, 0), "waves": (1858, 0), "eight": (12000, 0), "loop": (20003, 0),
          "streamed": (33001, 0), "list": (1858, 12), "long-list": (1858, 150)}


def _rows(rng, shape, dtype, n, far=-50.0):
    """n rows of entries `far` below 0 in policy and reference alike, and five
    columns among the entries, the first and the last of the row with them."""
    vocab, moves = SHAPES[shape]
    if dtype != "f32" and vocab > 4096:
        vocab *= 2
    x = np.full((n, vocab), far)
    at = np.concatenate([[0, vocab - 1], 1 + rng.choice(vocab - 2, 3, replace=False)])
    lists = None
    if moves:
        more = np.setdiff1d(np.arange(1, vocab - 1), at)
        lists = [list(at) + list(rng.choice(more, moves - 5, replace=False)) for _ in range(n)]
    return x, x.copy(), at, lists


@pytest.mark.parametrize("shape", SHAPES)
def test_small_weights_leave_kl_alone(dev, shape):
    """Entries far below the maximum whose reference is not so far: their
    terms are of p exp(-u) with p near 2^-100 and exp(-u) near 2^85."""
    rng = np.random.default_rng(1)
    weight = np.array([1.0, 1e-3, -1e-6, 1e-9, 1e-20, 2.0], np.float32)
    for below, ref_below in ((70.0, 11.0), (75.0, 16.0), (95.0, 30.0)):
        x, ref, at, lists = _rows(rng, shape, "f32", len(weight), -below)
        ref[:] = -ref_below
        x[:, at[2]] = ref[:, at[2]] = 0.0
        batch = lg.Batch(dev, x, "f32", lists, None)
        got = lg.policy(batch, ref=ref, weight=weight, kl_coef=0.3, entropy_coef=0.1)
        assert np.all(got["kl"] > 0)
        check(batch, got, ref, 0.3, 0.1, weight)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_kl_without_a_coefficient_leaves_the_gradient_alone(dev, shape, dtype):
    """The reference lacks entries that the policy has: KL is infinite, and
    neither loss nor gradient holds it."""
    rng = np.random.default_rng(2)
    x, ref, at, lists = _rows(rng, shape, dtype, 4)
    x[:] = rng.normal(size=x.shape)
    ref[:] = x + 0.3 * rng.normal(size=x.shape)
    ref[0, at[0]] = -np.inf
    ref[1, at[1:3]] = -np.inf
    ref[2] = -np.inf
    action = int(at[3])
    batch = lg.Batch(dev, x, dtype, lists, [action] * 4)
    kw = dict(advantage=np.ones(4), entropy_coef=0.1)
    got, want = lg.policy(batch, ref=ref, **kw), lg.policy(batch, **kw)
    assert np.all(got["kl"][:3] == np.inf) and np.isfinite(got["kl"][3])
    for k in ("loss", "logp", "entropy"):
        lu.close(got[k], want[k], 4 * lu.U * np.abs(want[k]))
    # The same sums in another order, and one rounding more.
    lu.close(got["grad"], want["grad"], 16 * lu.U * np.abs(want["grad"]).max(), dtype)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("temp", [0.3, 0.7, 1.0])
def test_entries_masked_in_the_reference_alone(dev, shape, dtype, temp):
    """The reference masked by the type's lowest value at every other column,
    where the policy is far below its maximum, but finite."""
    rng = np.random.default_rng(3)
    x, ref, at, lists = _rows(rng, shape, dtype, 3)
    x[:] = rng.normal(size=x.shape)
    ref[:] = x + 0.3 * rng.normal(size=x.shape)
    for b, below in enumerate((-1e4, -300.0, -6e4)):
        x[b, 1::2], ref[b, 1::2] = below, LOWEST[dtype]
    batch = lg.Batch(dev, x, dtype, lists, None, temp)
    got = lg.policy(batch, ref=ref, kl_coef=0.3, entropy_coef=0.1)
    assert all(np.isfinite(v).all() for v in got.values())
    check(batch, got, ref, 0.3, 0.1)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("temp", [0.7, 1.0, 3.0])
def test_divergences_of_any_size(dev, shape, dtype, temp):
    """Masks of the reference where p is of order 1, and references that
    prefer by far what the policy does not."""
    rng = np.random.default_rng(4)
    x, ref, at, lists = _rows(rng, shape, dtype, 9)
    x[:, at[:3]] = ref[:, at[:3]] = 0.0
    ref[0, at[0]] = -1e4
    ref[1, at[2]] = LOWEST[dtype]
    ref[2, at[1]] = 200.0
    ref[3, at[1]] = 90.0
    ref[4, at[1]] = 50.0
    ref[5, at[0]] = -300.0
    ref[6, at[4]] = 130.0            # where the policy has about nothing
    ref[7, at[:2]] = -1e4
    x[8, at[:3]], ref[8, at[:3]] = (30.0, 0.0, -30.0), (-30.0, 1.0, 31.0)
    batch = lg.Batch(dev, x, dtype, lists, None, temp)
    got = lg.policy(batch, ref=ref, kl_coef=0.3, entropy_coef=0.1)
    assert all(np.isfinite(v).all() for v in got.values())
    check(batch, got, ref, 0.3, 0.1)


@pytest.mark.parametrize("shape", SHAPES)
def test_large_weights_leave_kl_alone(dev, shape):
    rng = np.random.default_rng(5)
    weight = np.array([1.0, 65536.0, 2.0 ** 39, 2.0 ** 60, -2.0 ** 90, 2.0 ** 41], np.float32)
    for far in (130.0, 45.0, 28.0, 1e4):
        x, ref, at, lists = _rows(rng, shape, "f32", len(weight))
        x[:, at[:2]] = ref[:, at[:2]] = 0.0
        ref[:, at[1]] = far
        batch = lg.Batch(dev, x, "f32", lists, None)
        got = lg.policy(batch, ref=ref, weight=weight, kl_coef=0.3, entropy_coef=0.1)
        check(batch, got, ref, 0.3, 0.1, weight)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_several_entries_of_the_lowest_value(dev, shape, dtype):
    """Their differences add up beyond the 32-bit range; KL, two thirds of one
    of them, does not."""
    rng = np.random.default_rng(6)
    x, ref, at, lists = _rows(rng, shape, dtype, 2)
    x[:, at[:3]] = ref[:, at[:3]] = 0.0
    ref[0, at[:2]] = LOWEST[dtype]
    x[1, at] = ref[1, at] = 0.0
    ref[1, at[:4]] = LOWEST[dtype]
    batch = lg.Batch(dev, x, dtype, lists, None)
    got = lg.policy(batch, ref=ref, kl_coef=0.3, entropy_coef=0.1)
    assert all(np.isfinite(v).all() for v in got.values())
    check(batch, got, ref, 0.3, 0.1)


@pytest.mark.parametrize("dtype", lu.TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("temp", [0.7, 1.0])
def test_references_a_constant_away(dev, shape, dtype, temp):
    """Softmax does not see a constant: a reference of lowest values alone is
    uniform, one 3e4 lower or higher the same policy as without."""
    rng = np.random.default_rng(7)
    x, ref, at, lists = _rows(rng, shape, dtype, 4)
    x[:] = rng.normal(size=x.shape)
    ref[:] = x + 0.5 * rng.normal(size=x.shape)
    ref[0] = LOWEST[dtype]
    ref[1] -= 3e4
    ref[2] += 3e4
    ref[3], x[3] = ref[3] + 100.0, x[3] - 100.0
    batch = lg.Batch(dev, x, dtype, lists, None, temp)
    got = lg.policy(batch, ref=ref, kl_coef=0.3, entropy_coef=0.1)
    check(batch, got, ref, 0.3, 0.1)
    n = batch.vocab if lists is None else len(lists[0])
    uniform = np.log(n) - got["entropy"][0]
    assert abs(got["kl"][0] - uniform) < 1e-4 * np.log(n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_products_that_leave_the_range_on_the_way(dev, shape, dtype):
    """Masks of the lowest value where p is 1/3, with weights and coefficients
    whose product with KL or u is within the range only in the end."""
    rng = np.random.default_rng(8)
    weight = np.array([1e-4, 1e-12, 0.5, 1e-30], np.float32)
    for temp, kl_coef, w in ((1.0, 3.0, weight), (1.0, 0.05, weight * np.float32(32))):
        x, ref, at, lists = _rows(rng, shape, dtype, 4)
        x[:, at[:3]] = ref[:, at[:3]] = 0.0
        ref[:, at[0]] = LOWEST[dtype]
        ref[:2, at[1]] = LOWEST[dtype]
        batch = lg.Batch(dev, x, dtype, lists, None, temp)
        got = lg.policy(batch, ref=ref, weight=w, kl_coef=kl_coef, entropy_coef=0.1)
        assert np.isfinite(got["kl"]).all() and np.isfinite(got["grad"]).all()
        check(batch, got, ref, kl_coef, 0.1, w)
