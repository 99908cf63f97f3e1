"""Attention with much work, where rows and keys run in kernels of their own and
a wave has two sets of columns: the few lines that a 64-bit oracle can do, many
times over, so that every line of a call is checked."""

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


LINES = 4  # that differ


class Many:
    """`batch` lines, of which each is one of the first LINES."""

    def __init__(self, dev, batch, heads, kv_heads, q_len, k_len, dim, dtype, causal=False,
                 lengths=False, seed=0, order="bthd", bias_dtype=None, shared=()):
        rng = np.random.default_rng(seed)
        assert batch % LINES == 0
        self.dev, self.dtype, self.batch, self.heads, self.causal = dev, dtype, batch, heads, causal
        self.q, self.dout = (lu.values(rng, (LINES, q_len, heads, dim), dtype) for _ in range(2))
        self.k, self.v = (lu.values(rng, (LINES, k_len, kv_heads, dim), dtype) for _ in range(2))
        self.scale = float(np.float32(dim ** -0.5))
        self.lengths = (None, None)
        if lengths:
            self.lengths = ([q_len, 0, 1, (q_len + 1) // 2], [k_len, 5, k_len - 1, 2 * k_len // 3])
        self.order = order
        self.d = {n: self._heads(getattr(self, n)) for n in ("q", "k", "v", "dout")}
        self.out = self._heads(self.q, fill=True)
        self.lse = lu.Flat(dev, np.full(batch * heads * q_len, -7.0))
        ptr = lambda a: None if a is None else dev.put(  # noqa: E731
            np.tile(np.asarray(a, np.int32), batch // LINES))
        self.bias, kw = None, {}
        if bias_dtype:
            shape = [1 if i in shared else n for i, n in enumerate((LINES, heads, q_len, k_len))]
            self.bias, self.shared = lu.values(rng, shape, bias_dtype), shared
            every = self.bias if 0 in shared else np.tile(self.bias, (batch // LINES, 1, 1, 1))
            self.d_bias = lu.Flat(dev, every, bias_dtype)
            self.dbias = lu.Flat(dev, np.full(every.shape, -3.0), bias_dtype)
            steps = [heads * q_len * k_len, q_len * k_len, k_len]
            if 1 in shared:
                steps[0] = q_len * k_len
            kw = dict(d_bias=self.d_bias.p, bias_dtype=bias_dtype,
                      bias_strides=[0 if i in shared else n for i, n in enumerate(steps)])
        self.p = backend.attention_problem(
            self.d["q"].p, self.d["k"].p, self.d["v"].p, batch, heads, q_len, k_len, dim,
            dtype=dtype, kv_heads=kv_heads, scale=self.scale, causal=causal,
            q_strides=self.d["q"].strides, k_strides=self.d["k"].strides,
            v_strides=self.d["v"].strides, d_q_lengths=ptr(self.lengths[0]),
            d_k_lengths=ptr(self.lengths[1]), **kw)

    def _heads(self, t, fill=False):
        shape = (self.batch, *t.shape[1:])
        data = None if fill else np.tile(t, (self.batch // LINES, 1, 1, 1))
        return lu.Heads(self.dev, shape, self.dtype, data, order=self.order)

    def _one(self, t, name):
        """The first LINES of an output, of which all others are copies."""
        t = t.reshape(self.batch // LINES, LINES, *t.shape[1:])
        assert np.array_equal(t, np.broadcast_to(t[:1], t.shape)), name
        return t[0]

    def forward(self):
        need = backend.attention_forward_workspace_bytes(self.p)
        ws, end = lu.workspace(self.dev, need)
        backend.attention_forward_device(self.p, self.out.p, self.out.strides, d_lse=self.lse.p,
                                         d_workspace=ws, workspace_bytes=need)
        self.dev.sync()
        end()
        lse = self.lse.get().reshape(self.batch, self.heads, -1)
        return self._one(self.out.get(), "out"), self._one(lse, "lse")

    def backward(self, only=("dq", "dk", "dv", "dbias")):
        g = {n: self._heads(getattr(self, n[1:]), fill=True) for n in only if n != "dbias"}
        need = backend.attention_backward_workspace_bytes(self.p)
        ws, end = lu.workspace(self.dev, need)
        kw = {"d_" + n: g[n].p for n in g}
        kw.update({n + "_strides": g[n].strides for n in g})
        biased = self.bias is not None and "dbias" in only
        if biased:
            kw["d_dbias"] = self.dbias.p
        backend.attention_backward_device(
            self.p, self.out.p, self.lse.p, self.d["dout"].p, out_strides=self.out.strides,
            dout_strides=self.d["dout"].strides, d_workspace=ws, workspace_bytes=need, **kw)
        self.dev.sync()
        end()
        got = {n: self._one(g[n].get(), n) for n in g}
        if biased:
            t = self.dbias.get().reshape(-1, *self.bias.shape[1:])
            got["dbias"] = t if 0 in self.shared else self._one(t, "dbias")
        return got

    def check(self):
        args = (self.q, self.k, self.v)
        want = layers.attention_backward(*args, self.dout, self.scale, self.bias, self.causal,
                                         *self.lengths)
        tol = lu.attention_bounds(*args, self.scale, self.bias, want, self.dtype, self.dout)
        if self.bias is not None:
            # Sums over all that share it: as many additions in a row, of all copies.
            ds, over = want["dbias"], tuple(self.shared)
            copies = self.batch // LINES if 0 in over else 1
            n = copies * np.prod([ds.shape[i] for i in over]) if over else 0
            want["dbias"] = copies * ds.sum(over, keepdims=True)
            tol["dbias"] = copies * (tol["dbias"].sum(over, keepdims=True)
                                     + n * lu.U * np.abs(ds).sum(over, keepdims=True))
            tol["dbias"] += lu.rounding(want["dbias"], self.d_bias.dtype)
        out, lse = self.forward()
        lu.check(out, want["out"], tol["out"], "out")
        lu.check(lse, want["lse"], tol["lse"], "lse")
        every = self.backward()
        for n in every:
            lu.check(every[n], want[n], tol[n], n)
        for n in every:
            assert np.array_equal(self.backward(only=(n,))[n], every[n]), n


# Two sets of columns from 1024 workgroups of 128 rows (keys) on, for heads of 32
# and, in 16 bits, of 64; rows and keys in one launch up to 4096 workgroups, 1024 for
# heads above 64.
SHAPES = {
    # Two sets on both sides, of every type.
    "both-wide": dict(batch=32, heads=16, kv_heads=16, q_len=150, k_len=140, dim=32),
    # Two sets in 16 bits; fp32 has one, and more workgroups than go together.
    "wide-or-apart": dict(batch=48, heads=16, kv_heads=16, q_len=150, k_len=140, dim=64),
    "large-heads-apart": dict(batch=16, heads=16, kv_heads=16, q_len=150, k_len=140, dim=120),
    # Two sets on one side (fp32 of 56: on none, and apart).
    "rows-wide": dict(batch=128, heads=8, kv_heads=2, q_len=150, k_len=140, dim=24),
    "rows-wide-56": dict(batch=176, heads=8, kv_heads=2, q_len=150, k_len=140, dim=56),
    "keys-wide": dict(batch=32, heads=16, kv_heads=16, q_len=70, k_len=300, dim=40),
    # One tile of keys, read once; more keys than rows see.
    "one-tile-of-keys": dict(batch=64, heads=16, kv_heads=16, q_len=200, k_len=60, dim=32),
    # Eight heads to a row tile's 64 rows.
    "short-queries": dict(batch=128, heads=64, kv_heads=8, q_len=9, k_len=200, dim=32),
}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", ["plain", "causal", "ragged", "causal-ragged"])
@pytest.mark.parametrize("name", SHAPES)
def test_much_work(dev, name, mask, dtype):
    order = "bhtd" if mask == "causal" else "bthd"
    Many(dev, **SHAPES[name], dtype=dtype, causal=mask.startswith("causal"),
         lengths=mask.endswith("ragged"), seed=len(name), order=order).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bias_dtype", ["f32", "f16"])
def test_much_work_with_a_bias(dev, bias_dtype, dtype):
    Many(dev, **SHAPES["both-wide"], dtype=dtype, bias_dtype=bias_dtype, seed=5).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shared", [(0,), (0, 1)])
@pytest.mark.parametrize("q_len,k_len", [(64, 64), (40, 70)])
def test_a_bias_that_many_lines_share(dev, q_len, k_len, shared, dtype):
    Many(dev, 300, 4, 4, q_len, k_len, 32, dtype, causal=q_len == 40, lengths=True,
         bias_dtype="f32", shared=shared, seed=6).check()
