"""The layers of a training step as a learner uses them: forward, backward,
the gradients' norm and the update of the same weights, one after another on a
stream, captured into a graph, from two threads."""

import threading

import numpy as np
import pytest

import gpu_util
import layer_util as lu
from metalfish_amd import backend
from oracle import layers

pytestmark = pytest.mark.gpu

LINES, TOKENS, HEADS, DIM = 3, 64, 4, 32
WIDTH, ROWS = HEADS * DIM, LINES * TOKENS
EPS, LR, MAX_NORM = 1e-3, 1e-2, 0.5


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


class Learner:
    """Queries from a layer norm's rows, keys and values given, a bias shared by
    the lines; trained are the norm's weights and the bias."""

    def __init__(self, dev, seed, dtype="bf16", eight=True):
        rng = np.random.default_rng(seed)
        self.dev, self.dtype = dev, dtype
        data = lambda *shape: lu.values(rng, shape, dtype)  # noqa: E731
        self.x, self.res = data(ROWS, WIDTH), data(ROWS, WIDTH)
        self.k, self.v, self.dout = (data(LINES, TOKENS, HEADS, DIM) for _ in range(3))
        self.w = {"gamma": lu.values(rng, WIDTH, "f32", 0.1, 1.0),
                  "beta": lu.values(rng, WIDTH, "f32", 0.1),
                  "bias": lu.values(rng, (1, HEADS, TOKENS, TOKENS), "f32", 0.5)}
        put = lambda t, dt=dtype: lu.Flat(dev, t, dt)  # noqa: E731
        d = {n: put(getattr(self, n)) for n in ("x", "res", "k", "v", "dout")}
        d.update({n: put(t, "f32") for n, t in self.w.items()})
        d.update({"d" + n: put(0 * t, "f32") for n, t in self.w.items()})
        d.update({n: put(0 * self.x) for n in ("y", "out", "dy", "dx", "dres")})
        d.update({n: put(0 * self.k) for n in ("dk", "dv")})
        d.update(mean=put(np.zeros(ROWS), "f32"), rstd=put(np.zeros(ROWS), "f32"),
                 lse=put(np.zeros(LINES * HEADS * TOKENS), "f32"))
        self.d = d
        tensors = []
        for n, t in self.w.items():
            blocks = -(-t.size // 256)
            state = {"m": dev.put(np.zeros(t.size, np.uint8 if eight else np.float32)),
                     "v": dev.put(np.zeros(t.size, np.uint8 if eight else np.float32))}
            if eight:
                state.update(m_scale=dev.put(np.zeros(blocks, np.float32)),
                             v_scale=dev.put(np.zeros(blocks, np.float32)))
            tensors.append(dict(state, param=d[n].p, grad=d["d" + n].p, count=t.size,
                                weight_decay=0.01 if n == "bias" else 0.0))
        self.adam = backend.AdamWSet(tensors, state_bits=8 if eight else 32)
        self.grads = backend.GradSet([(d["d" + n].p, None, t.size, "f32") for n, t in self.w.items()])
        self.norm = backend.norm_rows(d["x"].p, ROWS, WIDTH, dtype=dtype, d_residual=d["res"].p,
                                      alpha=0.5, d_gamma=d["gamma"].p, d_beta=d["beta"].p, eps=EPS)
        self.attention = backend.attention_problem(
            d["y"].p, d["k"].p, d["v"].p, LINES, HEADS, TOKENS, TOKENS, DIM, dtype=dtype,
            causal=True, d_bias=d["bias"].p, bias_strides=(0, TOKENS * TOKENS, TOKENS))
        need = max(backend.layer_norm_workspace_bytes(ROWS, WIDTH),
                   backend.attention_backward_workspace_bytes(self.attention),
                   backend.attention_forward_workspace_bytes(self.attention),
                   self.grads.workspace_bytes)
        self.ws, self.need = dev.alloc(need), need
        self.sumsq, self.d_step = dev.put(np.zeros(1)), dev.put(np.ones(1, np.int64))

    def step(self, stream):
        d, ws = self.d, dict(d_workspace=self.ws, workspace_bytes=self.need, stream=stream)
        backend.layer_norm_device(self.norm, d["y"].p, d_mean=d["mean"].p, d_rstd=d["rstd"].p,
                                  stream=stream)
        backend.attention_forward_device(self.attention, d["out"].p, d_lse=d["lse"].p, **ws)
        backend.attention_backward_device(self.attention, d["out"].p, d["lse"].p, d["dout"].p,
                                          d_dq=d["dy"].p, d_dk=d["dk"].p, d_dv=d["dv"].p,
                                          d_dbias=d["dbias"].p, **ws)
        backend.layer_norm_backward_device(self.norm, d["dy"].p, d["mean"].p, d["rstd"].p,
                                           d_dx=d["dx"].p, d_dresidual=d["dres"].p,
                                           d_dgamma=d["dgamma"].p, d_dbeta=d["dbeta"].p, **ws)
        self.grads.norm_device(self.sumsq, self.ws, self.need, stream=stream)
        self.adam.step_device(LR, 1, d_step=self.d_step, d_sumsq=self.sumsq, max_norm=MAX_NORM,
                              skip_nonfinite=True, stochastic=True, seed=9, stream=stream)

    def at_step(self, t):
        self.dev.write(self.d_step, np.array([t], np.int64))

    def outputs(self):
        return {n: a.bits() for n, a in self.d.items()}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_step_stage_by_stage(dev, dtype):
    l = Learner(dev, 1, dtype, eight=False)
    stream = dev.stream()
    l.step(stream)
    dev.sync(stream)
    got = {n: a.get() for n, a in l.d.items()}
    alpha = 0.5
    w = l.w
    want = layers.layer_norm(l.x, l.res, alpha, w["gamma"], w["beta"], float(np.float32(EPS)))
    tol = lu.norm_bounds(l.x, l.res, alpha, w["gamma"], w["beta"], EPS, want, dtype)
    for n in ("y", "mean", "rstd"):
        lu.check(got[n].reshape(want[n].shape), want[n], tol[n], n)
    q = got["y"].reshape(LINES, TOKENS, HEADS, DIM)
    scale = float(np.float32(DIM ** -0.5))
    want = layers.attention_backward(q, l.k, l.v, l.dout, scale, w["bias"], True)
    tol = lu.attention_bounds(q, l.k, l.v, scale, w["bias"], want, dtype, l.dout)
    ds = want["dbias"]
    want["dbias"], tol["dbias"] = ds.sum(0), tol["dbias"].sum(0) + 3 * lu.U * np.abs(ds).sum(0)
    for n, name in (("out", "out"), ("dy", "dq"), ("dk", "dk"), ("dv", "dv"), ("dbias", "dbias"),
                    ("lse", "lse")):
        lu.check(got[n].reshape(want[name].shape), want[name], tol[name], name)
    dy = got["dy"].reshape(ROWS, WIDTH)
    want = layers.layer_norm_backward(l.x, dy, got["mean"], got["rstd"], l.res, alpha, w["gamma"])
    tol = lu.norm_backward_bounds(l.x, l.res, alpha, w["gamma"], dy, got["mean"], got["rstd"], want,
                                  dtype)
    for n, name in (("dx", "dx"), ("dres", "dresidual"), ("dgamma", "dgamma"), ("dbeta", "dbeta")):
        lu.check(got[n].reshape(want[name].shape), want[name], tol[name], name)
    total = sum((got["d" + n] ** 2).sum() for n in w)
    assert abs(dev.get(l.sumsq, np.zeros(1))[0] - total) <= 1e-12 * total and total > MAX_NORM ** 2
    factor = layers.clip_factor(total, MAX_NORM)
    for n, t in w.items():
        g = got["d" + n].reshape(t.shape)
        p, _, _ = layers.adamw(t, g, 0 * g, 0 * g, 1, LR, weight_decay=0.01 if n == "bias" else 0.0,
                               factor=factor)
        # Of the update (LR at most): 16 roundings, where eps does not matter.
        big = np.abs(g) * factor > 1e-4
        off = np.abs(got[n].reshape(t.shape) - p)
        assert np.all(off[big] <= (2 ** -20 * LR + 2 * lu.U * np.abs(p))[big])
        assert np.all(off <= LR * 1e-2)


def test_a_captured_step_trains_as_the_eager_one(dev):
    """The same weights after each of five steps, on new inputs each, the
    step's number read on the device."""
    a, b = Learner(dev, 2), Learner(dev, 2)
    stream = dev.stream()
    launch = dev.capture(stream, lambda: a.step(stream))
    rng = np.random.default_rng(3)
    first = a.outputs()
    for t in range(1, 6):
        x = lu.to_bits(rng.normal(size=ROWS * WIDTH), "bf16")
        for l in (a, b):
            dev.write(l.d["x"].p, x)
            l.d["x"].flat[4:4 + x.size] = x
            l.at_step(t)
        launch()
        dev.sync(stream)
        b.step(None)
        dev.sync()
        got, want = a.outputs(), b.outputs()
        assert all(np.array_equal(got[n], want[n]) for n in want), t
    assert all(not np.array_equal(first[n], got[n]) for n in ("gamma", "beta", "bias"))


def test_two_threads_on_streams_of_their_own(dev):
    sides, want = [Learner(dev, 4), Learner(dev, 5)], []
    for seed in (4, 5):
        l = Learner(dev, seed)
        for t in range(1, 11):
            l.at_step(t)
            l.step(None)
            dev.sync()
        want.append(l.outputs())
    streams, errors = [dev.stream(), dev.stream()], []

    def work(l, s):
        try:
            for t in range(1, 11):
                dev.sync(s)
                l.at_step(t)
                l.step(s)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(sides, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    dev.sync()
    assert not errors
    for l, w in zip(sides, want):
        got = l.outputs()
        assert all(np.array_equal(got[n], w[n]) for n in w)
