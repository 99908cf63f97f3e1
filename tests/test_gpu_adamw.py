"""AdamW over many tensors on the device: 32-bit states and codes to the bit,
weights against the 64-bit formula."""

import numpy as np
import pytest

import gpu_util
import layer_util as lu
from metalfish_amd import backend
from oracle import layers

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


class Tensor:
    def __init__(self, dev, rng, count, eight, param_dtype="f32", grad_dtype="f32", copy_dtype=None,
                 lr_scale=1.0, weight_decay=0.0, fresh=False, grad=None):
        self.eight, self.count, self.lr_scale, self.decay = eight, count, lr_scale, weight_decay
        self.param = lu.values(rng, count, param_dtype, 0.03)
        self.grad = lu.values(rng, count, grad_dtype, 1e-3) if grad is None else grad
        m = np.zeros(count, np.float32) if fresh else (1e-4 * rng.normal(size=count)).astype(np.float32)
        v = np.zeros(count, np.float32) if fresh else \
            (1e-7 * 10.0 ** rng.uniform(-4, 0, count)).astype(np.float32)
        d = {"param": lu.Flat(dev, self.param, param_dtype), "grad": lu.Flat(dev, self.grad, grad_dtype)}
        if eight:
            (mc, ms), (vc, vs) = layers.encode_m(m), layers.encode_v(v)
            if fresh:
                ms, vs = 0 * ms, 0 * vs
            d.update(m=lu.Flat(dev, mc, "u8"), v=lu.Flat(dev, vc, "u8"), m_scale=lu.Flat(dev, ms),
                     v_scale=lu.Flat(dev, vs))
            m, v = layers.decode_m(mc, ms), layers.decode_v(vc, vs)
        else:
            d.update(m=lu.Flat(dev, m), v=lu.Flat(dev, v))
        if copy_dtype:
            d["copy"] = lu.Flat(dev, np.zeros(count), copy_dtype)
        self.m, self.v, self.d = m, v, d
        self.desc = {**{k: a.p for k, a in d.items()}, "count": count, "param_dtype": param_dtype,
                     "grad_dtype": grad_dtype, "lr_scale": lr_scale, "weight_decay": weight_decay}
        if copy_dtype:
            self.desc["copy_dtype"] = copy_dtype

    def check(self, lr, step, beta1, beta2, eps, factor=1.0, bits=None):
        """One step from what the tensor held, every output; the new state is
        what the next step starts from."""
        lr = lr * self.lr_scale
        m, v = layers.states_after(self.grad, self.m, self.v, beta1, beta2, factor)
        want, _, _ = layers.adamw(self.param, self.grad, self.m, self.v, step, lr, beta1, beta2, eps,
                                  self.decay, factor)
        # A rounding each: decay's factor, its product, the step's size, square
        # root, its factor, eps, sum, quotient, product, difference, and 6 u of
        # the states; bits of m that cancel are u of |beta1 m| + |(1 - beta1) g|.
        up = np.abs(want - self.param * (1 - lr * self.decay))
        raw = beta1 * np.abs(self.m) + (1 - beta1) * np.abs(self.grad) * factor
        lost = up * raw / np.where(m != 0, np.abs(m).astype(np.float64), np.inf)
        tol = 4 * lu.U * np.abs(want) + 12 * lu.U * (up + lost)
        got = self.d["param"].get()
        lu.check(got, want, tol + lu.rounding(want, self.d["param"].dtype), "param")
        if "copy" in self.d:
            host = lu.to_bits(got, self.d["copy"].dtype)
            assert np.array_equal(self.d["copy"].bits(), host), "copy"
        if self.eight:
            for name, (code, scale) in (("m", layers.encode_m(m, bits)), ("v", layers.encode_v(v, bits))):
                assert np.array_equal(self.d[name].bits(), code), name
                assert np.array_equal(self.d[name + "_scale"].bits(), scale), name
                if name == "m":
                    m = layers.decode_m(code, scale)
                else:
                    v = layers.decode_v(code, scale)
        else:
            assert np.array_equal(self.d["m"].bits(), m) and np.array_equal(self.d["v"].bits(), v)
        self.param, self.m, self.v = got, m, v
        self.d["grad"].bits()


def places(tensors):
    """The first place in the set of each tensor."""
    at, out = 0, []
    for t in tensors:
        out.append(at)
        at += -(-t.count // layers.BLOCK) * layers.BLOCK
    return out


def steps(dev, tensors, eight, n=2, lr=1e-3, beta1=0.9, beta2=0.98, eps=1e-7, first=5,
          stochastic=False, seed=11, **kw):
    s = backend.AdamWSet([t.desc for t in tensors], state_bits=8 if eight else 32)
    factor = kw.pop("factor", 1.0)
    for k in range(n):
        step = first + k
        s.step_device(lr, step, beta1=beta1, beta2=beta2, eps=eps, stochastic=stochastic, seed=seed,
                      **kw)
        dev.sync()
        for t, at in zip(tensors, places(tensors)):
            bits = layers.random_bits(seed, step, at + np.arange(t.count)) if stochastic else None
            t.check(lr, step, beta1, beta2, eps, factor, bits)
    s.close()


COUNTS = (1, 3, 4, 255, 256, 257, 1023, 1025, 4095, 4096, 4097, 9000, 20000)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("param,grad,copy", [("f32", "f32", None), ("f32", "bf16", "bf16"),
                                             ("f32", "f16", "f16"), ("bf16", "bf16", None),
                                             ("f16", "f32", "f32"), ("bf16", "f16", "f32")])
def test_sizes_and_types(dev, param, grad, copy, eight):
    rng = np.random.default_rng(1)
    tensors = [Tensor(dev, rng, n, eight, param, grad, copy, lr_scale=1 + n % 3, weight_decay=0.01 * (n % 2))
               for n in COUNTS]
    steps(dev, tensors, eight)


@pytest.mark.parametrize("past", [False, True])
@pytest.mark.parametrize("stochastic", [False, True])
def test_codes_to_the_bit(dev, stochastic, past):
    """Three steps each from the codes of the one before; small sets and those
    past the caches."""
    rng = np.random.default_rng(2)
    tensors = [Tensor(dev, rng, n, True, grad_dtype="bf16", weight_decay=0.1) for n in (5000, 300, 70001)]
    if past:
        tensors.append(Tensor(dev, rng, 12_000_001, True))
    steps(dev, tensors, True, n=3, stochastic=stochastic)


def test_large_sets_in_32_bits(dev):
    rng = np.random.default_rng(3)
    steps(dev, [Tensor(dev, rng, 5_000_003, False), Tensor(dev, rng, 77, False)], False)


@pytest.mark.parametrize("eight", [False, True])
def test_first_step_from_nothing(dev, eight):
    """Fresh states are zeros: the first update is lr times the sign."""
    rng = np.random.default_rng(4)
    t = Tensor(dev, rng, 1000, eight, fresh=True)
    before = t.param.copy()
    steps(dev, [t], eight, n=1, first=1, beta2=0.999, eps=1e-12)
    assert np.all(np.abs(before - t.param - 1e-3 * np.sign(t.grad)) < 2e-6)


@pytest.mark.parametrize("eight", [False, True])
def test_a_gradient_of_zero(dev, eight):
    rng = np.random.default_rng(5)
    t = Tensor(dev, rng, 600, eight, fresh=True, grad=np.zeros(600), weight_decay=0.5)
    before = t.param.copy()
    steps(dev, [t], eight, n=2, first=1)
    # Decayed twice, a rounding each time.
    assert np.all(np.abs(t.param - before * (1 - 5e-4) ** 2) <= 4 * lu.U * np.abs(before))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e-9, 1e6, 1e15])
def test_gradients_of_any_size(dev, size, eight):
    rng = np.random.default_rng(6)
    g = lu.from_bits(lu.to_bits(size * rng.normal(size=3000), "f32"), "f32")
    t = Tensor(dev, rng, 3000, eight, grad=g.astype(np.float64), fresh=True)
    # eps 0: the quotient is m over the root of v, whatever their size, but
    # where v itself is below fp32 (gradients of 1e-30: both are 0).
    if size < 1e-20:
        steps(dev, [t], eight, n=2, first=1)
    else:
        steps(dev, [t], eight, n=2, first=1, eps=0.0 if size > 1e-10 else 1e-12)


@pytest.mark.parametrize("eight", [False, True])
def test_clipped_by_the_sum_of_squares(dev, eight):
    """Both calls of a step: the norm of a gradient set, and the step that reads it."""
    rng = np.random.default_rng(7)
    tensors = [Tensor(dev, rng, n, eight, grad_dtype="bf16") for n in (3000, 17, 9001)]
    grads = backend.GradSet([(t.d["grad"].p, None, t.count, "bf16") for t in tensors])
    sumsq = dev.put(np.zeros(1))
    grads.norm_device(sumsq, dev.alloc(grads.workspace_bytes), grads.workspace_bytes)
    dev.sync()
    total = dev.get(sumsq, np.zeros(1))[0]
    assert abs(total - sum((t.grad ** 2).sum() for t in tensors)) < 1e-12 * total
    for max_norm, grad_scale in ((0.5 * np.sqrt(total), 1.0), (2 * np.sqrt(total), 1.0),
                                 (0.25 * np.sqrt(total), 0.5), (float("inf"), 0.125), (0.0, 1.0)):
        max_norm = float(np.float32(max_norm))
        steps(dev, tensors, eight, n=1, d_sumsq=sumsq, max_norm=max_norm, grad_scale=grad_scale,
              factor=layers.clip_factor(total, max_norm, grad_scale))


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_skipping_sums_that_are_not_finite(dev, bad, eight):
    rng = np.random.default_rng(8)
    t = Tensor(dev, rng, 5000, eight, copy_dtype="bf16")
    held = {k: a.bits() for k, a in t.d.items()}
    s = backend.AdamWSet([t.desc], state_bits=8 if eight else 32)
    s.step_device(1e-3, 3, d_sumsq=dev.put(np.array([bad])), max_norm=1.0, skip_nonfinite=True)
    dev.sync()
    assert all(np.array_equal(held[k], a.bits()) for k, a in t.d.items())
    s.step_device(1e-3, 3, d_sumsq=dev.put(np.array([1.0])), max_norm=1.0, skip_nonfinite=True)
    dev.sync()
    assert not np.array_equal(held["param"], t.d["param"].bits())


def test_a_gradient_that_is_not_finite_spoils_its_block(dev):
    rng = np.random.default_rng(9)
    for bad in (np.nan, np.inf):
        g = lu.values(rng, 1000, "f32", 1e-3)
        g[300] = bad
        t = Tensor(dev, rng, 1000, True, grad=g)
        s = backend.AdamWSet([t.desc], state_bits=8)
        s.step_device(1e-3, 3)
        dev.sync()
        assert np.array_equal(~np.isfinite(t.d["m_scale"].get()), [False, True, False, False])
        assert np.array_equal(~np.isfinite(t.d["v_scale"].get()), [False, True, False, False])
        fine = np.isfinite(t.d["param"].get())
        assert not fine[300] and np.all(np.delete(fine, 300))
        s.step_device(1e-3, 4)
        dev.sync()
        fine = np.isfinite(t.d["param"].get())
        assert not fine[256:512].any() and fine[:256].all() and fine[512:].all()


def test_rate_and_step_on_the_device(dev):
    rng = np.random.default_rng(10)
    a, b = Tensor(dev, rng, 5000, True), None
    rng = np.random.default_rng(10)
    b = Tensor(dev, rng, 5000, True)
    sa, sb = (backend.AdamWSet([t.desc], state_bits=8) for t in (a, b))
    d_lr, d_step = dev.put(np.zeros(1, np.float32)), dev.put(np.zeros(1, np.int64))
    for step in (1, 2, 77, 100000):
        lr = float(np.float32(1e-3 / step ** 0.5))
        dev.write(d_lr, np.array([lr], np.float32))
        dev.write(d_step, np.array([step], np.int64))
        sa.step_device(lr, step, stochastic=True, seed=5)
        sb.step_device(9.0, 1, stochastic=True, seed=5, d_lr=d_lr, d_step=d_step)
        dev.sync()
        for k in ("m", "v", "m_scale", "v_scale"):
            assert np.array_equal(a.d[k].bits(), b.d[k].bits()), (step, k)
        # The device's logarithms differ from the host's in the last bits of 64.
        assert np.all(np.abs(a.d["param"].get() - b.d["param"].get()) <= 1e-7 * lr + 2 ** -23 * 0.2)


def test_stochastic_states_follow_a_falling_gradient(dev):
    """v falls by a thousandth a step: rounded to nearest it would stay."""
    n, rounds = 4096, 2000
    rng = np.random.default_rng(12)
    g = np.full(n, 1e-3)
    g[::256] = 0.1  # each block's largest, whose scale the others do not share
    kept = {}
    for stochastic in (False, True):
        t = Tensor(dev, rng, n, True, fresh=True, grad=lu.from_bits(lu.to_bits(g, "f32"), "f32"))
        s = backend.AdamWSet([t.desc], state_bits=8)
        s.step_device(0.0, 1, beta2=0.0)  # v = g^2
        small = np.where(np.arange(n) % 256 == 0, 0.1, 0.0).astype(np.float32)
        dev.write(t.d["grad"].p, small)
        for step in range(2, 2 + rounds):
            s.step_device(0.0, step, beta2=0.999, stochastic=stochastic, seed=3)
        dev.sync()
        v = layers.decode_v(t.d["v"].bits(), t.d["v_scale"].bits())
        kept[stochastic] = v[np.arange(n) % 256 != 0].mean() / 1e-6
    want = 0.999 ** rounds  # 0.135
    # 4080 values: the mean of codes whose steps are an eighth of the value.
    assert abs(kept[True] - want) < 0.1 * want and kept[False] > 0.9


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("eps", [1e-300, 1e-45, 1e-40, 2.0 ** -126])
def test_weights_without_gradients_stay_under_a_tiny_eps(dev, eps, eight):
    """0 / eps is 0, however small eps is above 0 (rows that no batch has met)."""
    rng = np.random.default_rng(15)
    t = Tensor(dev, rng, 700, eight, fresh=True, grad=np.zeros(700), weight_decay=0.5)
    steps(dev, [t], eight, n=2, first=1, eps=eps)


def test_steps_that_are_refused(dev):
    rng = np.random.default_rng(13)
    t = Tensor(dev, rng, 300, False)
    s = backend.AdamWSet([t.desc])
    ok = dev.put(np.ones(1))
    nan = float("nan")
    for kw in (dict(lr=-1.0), dict(lr=nan), dict(lr=float("inf")), dict(step=0), dict(step=-3),
               dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=nan), dict(eps=-1e-8),
               dict(eps=nan), dict(grad_scale=0.0), dict(grad_scale=-1.0), dict(grad_scale=nan),
               dict(grad_scale=1e39), dict(lr=1e39),
               dict(max_norm=-1.0, d_sumsq=ok), dict(max_norm=nan, d_sumsq=ok),
               dict(skip_nonfinite=True), dict(d_sumsq=ok + 4), dict(d_lr=ok + 2), dict(d_step=ok + 4),
               dict(d_sumsq=t.d["grad"].p), dict(d_lr=t.d["param"].p + 4), dict(d_step=t.d["m"].p),
               dict(d_sumsq=np.ones(1).ctypes.data)):
        kw = dict(dict(lr=1e-3, step=1), **kw)
        with pytest.raises(RuntimeError, match=r"failed \(-1\): mfh_adamw_step"):
            s.step_device(kw.pop("lr"), kw.pop("step"), **kw)
    raw = backend.MfhAdamwStep(1e-3, 0.9, 0.99, 1e-8, 1.0, 1, None, None, None, 1.0, 0, 2, 0)
    import ctypes
    assert backend.lib().mfh_adamw_step_device(s._h, ctypes.addressof(raw), None) == -1
    raw.stochastic, raw.skip_nonfinite = 0, 2
    assert backend.lib().mfh_adamw_step_device(s._h, ctypes.addressof(raw), None) == -1
    dev.sync()
    assert np.array_equal(t.d["param"].get(), t.param)
    with pytest.raises(RuntimeError, match="not device memory"):
        backend.AdamWSet([dict(t.desc, grad=np.ones(300, np.float32).ctypes.data)])
    empty = backend.AdamWSet([])
    empty.step_device(1e-3, 1)
    dev.sync()
