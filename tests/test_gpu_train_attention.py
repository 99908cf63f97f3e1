"""Attention with its gradients on the device against the 64-bit formulas."""

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


class Case:
    """One attention on the device, run forward and backward, every output
    held to its bound."""

    def __init__(self, dev, batch, heads, q_len, k_len, dim, dtype, kv_heads=None, causal=False,
                 bias=None, bias_dtype="f32", shared=(), q_lengths=None, k_lengths=None,
                 order="bthd", gap=0, shift=0, scale=None, seed=0, q_scale=1.0, spoil=False):
        rng = np.random.default_rng(seed)
        self.dev, self.dtype, self.causal = dev, dtype, causal
        self.kv, self.heads = kv_heads or heads, heads
        self.q = lu.values(rng, (batch, q_len, heads, dim), dtype, q_scale)
        self.k, self.v = (lu.values(rng, (batch, k_len, self.kv, dim), dtype) for _ in range(2))
        self.dout = lu.values(rng, self.q.shape, dtype)
        self.scale = float(np.float32(dim ** -0.5 if scale is None else scale))
        self.lengths = (q_lengths, k_lengths)
        lay = dict(order=order, gap=gap, shift=shift)
        self.d = {n: lu.Heads(dev, getattr(self, n).shape, dtype, getattr(self, n), **lay)
                  for n in ("q", "k", "v", "dout")}
        if spoil:  # what lies behind a length is never read
            for n, lens in (("q", q_lengths), ("dout", q_lengths), ("k", k_lengths), ("v", k_lengths)):
                t = self.d[n]
                mask = np.zeros(t.shape, bool)
                for b, m in enumerate(lens):
                    mask[b, m:] = True
                t.raw(mask, lu.NAN[dtype])
        self.out = lu.Heads(dev, self.q.shape, dtype, **lay)
        self.lse = lu.Flat(dev, np.full((batch, heads, q_len), -7.0))
        self.bias, kw = None, {}
        if bias is not None:
            full = [batch, heads, q_len, k_len]
            shape = [1 if i in shared else n for i, n in enumerate(full)]
            if isinstance(bias, str):
                self.bias = lu.values(rng, shape, bias_dtype)
            else:
                b = np.broadcast_to(bias, shape).astype(np.float32).reshape(-1)
                self.bias = lu.from_bits(lu.to_bits(b, bias_dtype), bias_dtype).astype(
                    np.float64).reshape(shape)
            self.d_bias = lu.Flat(dev, self.bias, bias_dtype)
            steps = [int(np.prod(shape[1:])), int(np.prod(shape[2:])), k_len]
            steps = [0 if i in shared else s for i, s in enumerate(steps)]
            kw = dict(d_bias=self.d_bias.p, bias_dtype=bias_dtype, bias_strides=steps)
            self.dbias = lu.Flat(dev, np.full(shape, -3.0), bias_dtype)
            self.shared = shared
        ptr = lambda a: None if a is None else dev.put(np.asarray(a, np.int32))  # noqa: E731
        self.p = backend.attention_problem(
            self.d["q"].p, self.d["k"].p, self.d["v"].p, batch, heads, q_len, k_len, dim,
            dtype=dtype, kv_heads=self.kv, scale=self.scale, causal=causal,
            q_strides=self.d["q"].strides, k_strides=self.d["k"].strides,
            v_strides=self.d["v"].strides, d_q_lengths=ptr(q_lengths),
            d_k_lengths=ptr(k_lengths), **kw)
        self.lay = lay

    def oracle(self):
        return (self.q, self.k, self.v), (self.scale, self.bias, self.causal, *self.lengths)

    def forward(self, stream=None):
        need = backend.attention_forward_workspace_bytes(self.p)
        ws, end = lu.workspace(self.dev, need)
        backend.attention_forward_device(self.p, self.out.p, self.out.strides, d_lse=self.lse.p,
                                         d_workspace=ws, workspace_bytes=need, stream=stream)
        self.dev.sync(stream)
        end()
        return self.out.get(), self.lse.get().reshape(self.q.shape[0], self.heads, -1)

    def backward(self, stream=None, only=("dq", "dk", "dv", "dbias")):
        g = {n: lu.Heads(self.dev, getattr(self, n[1:]).shape, self.dtype, **self.lay)
             for n in ("dq", "dk", "dv")}
        need = backend.attention_backward_workspace_bytes(self.p)
        ws, end = lu.workspace(self.dev, need)
        kw = {}
        for n in ("dq", "dk", "dv"):
            kw["d_" + n] = g[n].p if n in only else None
            kw[n + "_strides"] = g[n].strides
        if self.bias is not None and "dbias" in only:
            kw["d_dbias"] = self.dbias.p
        backend.attention_backward_device(
            self.p, self.out.p, self.lse.p, self.d["dout"].p, out_strides=self.out.strides,
            dout_strides=self.d["dout"].strides, d_workspace=ws, workspace_bytes=need,
            stream=stream, **kw)
        self.dev.sync(stream)
        end()
        got = {n: g[n].get() for n in ("dq", "dk", "dv") if n in only}
        if "d_dbias" in kw:
            got["dbias"] = self.dbias.get().reshape(self.bias.shape)
        return got

    def check(self):
        (q, k, v), rest = self.oracle()
        want = layers.attention_backward(q, k, v, self.dout, *rest)
        tol = lu.attention_bounds(q, k, v, self.scale, self.bias, want, self.dtype, self.dout)
        out, lse = self.forward()
        lu.check(out, want["out"], tol["out"], "out")
        lu.check(lse, want["lse"], tol["lse"], "lse")
        got = self.backward()
        if self.bias is not None:
            over = tuple(i for i in self.shared)
            tol["dbias"] = tol["dbias"].sum(over, keepdims=True) * 1.0
            n = np.prod([want["dbias"].shape[i] for i in over]) if over else 1
            tol["dbias"] += n * lu.U * np.abs(want["dbias"]).sum(over, keepdims=True)
            want["dbias"] = want["dbias"].sum(over, keepdims=True)
            tol["dbias"] += lu.rounding(want["dbias"], self.d_bias.dtype)
        for n in got:
            lu.check(got[n], want[n], tol[n], n)
        return got


DTYPES = ("f32", "bf16", "f16")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [(1, 1), (1, 64), (64, 1), (3, 5), (15, 17), (64, 64),
                                         (63, 65), (65, 63), (130, 70), (33, 200)])
def test_lengths(dev, q_len, k_len, dtype):
    Case(dev, 2, 3, q_len, k_len, 32, dtype, seed=q_len).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 48, 56, 64, 72, 96, 120, 128])
def test_head_sizes(dev, dim, dtype):
    Case(dev, 2, 2, 40, 71, dim, dtype, seed=dim, bias="random").check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (6, 2), (9, 3)])
@pytest.mark.parametrize("q_len,k_len", [(1, 130), (5, 40), (50, 50), (100, 65)])
def test_shared_heads(dev, heads, kv_heads, q_len, k_len, dtype):
    Case(dev, 2, heads, q_len, k_len, 24, dtype, kv_heads=kv_heads, causal=q_len != 5, seed=heads).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [(1, 1), (7, 7), (64, 64), (65, 65), (129, 129), (20, 90),
                                         (90, 20), (200, 64), (1, 77)])
def test_causal(dev, q_len, k_len, dtype):
    """Queries before the first key see nothing."""
    Case(dev, 1, 2, q_len, k_len, 40, dtype, causal=True, seed=k_len).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("order", ["bthd", "bhtd"])
def test_ragged_lines(dev, causal, order, dtype):
    """What lies behind a line's length is never read; its gradients are 0."""
    Case(dev, 5, 4, 100, 90, 32, dtype, kv_heads=2, causal=causal, q_lengths=[100, 0, 1, 64, 37],
         k_lengths=[90, 13, 0, 64, 65], order=order, spoil=True, bias="random").check()


@pytest.mark.parametrize("bias_dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [(64, 64), (57, 61), (100, 90), (70, 203), (5, 900)])
def test_a_bias_of_what_is_not_seen_has_no_effect(dev, q_len, k_len, bias_dtype):
    """NaN there: behind the lengths and right of the diagonal."""
    m, n = [q_len, 1, q_len - 2], [k_len, k_len - 3, 9]
    rng = np.random.default_rng(14)
    ok = np.stack([layers.seen(q_len, k_len, a, b, True) for a, b in zip(m, n)])[:, None]
    bias = np.where(ok, rng.normal(size=(3, 2, q_len, k_len)), 0.0)
    for dtype in DTYPES:
        c = Case(dev, 3, 2, q_len, k_len, 32, dtype, bias=bias, bias_dtype=bias_dtype, causal=True,
                 q_lengths=m, k_lengths=n)
        unseen = np.broadcast_to(~ok, bias.shape).reshape(-1)
        at = c.d_bias.lead + np.flatnonzero(unseen)
        c.d_bias.flat[at] = lu.NAN[bias_dtype]
        dev.write(c.d_bias.base, c.d_bias.flat)
        got = c.check()
        assert not got["dbias"].reshape(-1)[unseen].any()


def test_lengths_outside_their_arrays_are_clamped(dev):
    Case(dev, 3, 2, 20, 30, 16, "f32", q_lengths=[50, -4, 20], k_lengths=[31, 5, -1]).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap,shift", [(8, 0), (1, 1), (3, 5)])
def test_strides_and_alignments(dev, gap, shift, dtype):
    for order in ("bthd", "bhtd"):
        Case(dev, 2, 4, 30, 70, 32, dtype, kv_heads=2, order=order, gap=gap, shift=shift,
             bias="random", bias_dtype=dtype).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias_dtype", DTYPES)
@pytest.mark.parametrize("shared", [(), (0,), (1,), (0, 1)])
def test_biases(dev, shared, bias_dtype, dtype):
    """One of each head and line, or shared: its gradient is the sum."""
    Case(dev, 3, 4, 64, 64, 32, dtype, bias="random", bias_dtype=bias_dtype, shared=shared).check()
    Case(dev, 2, 4, 35, 67, 16, dtype, kv_heads=2, bias="random", bias_dtype=bias_dtype,
         shared=shared, causal=True).check()


@pytest.mark.parametrize("bias_dtype", DTYPES)
@pytest.mark.parametrize("k_len", [1, 3, 7, 8, 9, 12, 15, 17, 63, 65, 70, 129, 134, 333])
def test_rows_of_a_bias_that_end_inside_a_vector(dev, k_len, bias_dtype):
    """Alone and side by side in memory; the last row's end is the array's."""
    for n, dtype in enumerate(DTYPES):
        for shared, q_len in (((), 20), ((), 64), ((0, 1), 33)):
            Case(dev, 2, 2, q_len, k_len, 32, dtype, bias="random", bias_dtype=bias_dtype,
                 shared=shared, seed=k_len + n, causal=n == 1).check()


@pytest.mark.parametrize("q_len,k_len", [(70, 521), (1021, 139)])
@pytest.mark.parametrize("bias_dtype", DTYPES)
def test_two_sets_of_columns_with_an_odd_bias(dev, q_len, k_len, bias_dtype):
    for dtype in ("bf16", "f16"):
        Case(dev, 8, 16, q_len, k_len, 32, dtype, kv_heads=16, bias="random", bias_dtype=bias_dtype,
             k_lengths=[k_len, 1, 77, 0, 64, 138, 130, k_len - 1], seed=k_len).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [24, 64, 120])
@pytest.mark.parametrize("batch,heads,kv_heads,q_len,k_len", [
    (1, 1, 1, 1, 65), (3, 5, 5, 66, 66), (2, 8, 2, 130, 70), (1, 2, 1, 900, 65), (5, 4, 4, 65, 700),
    (9, 8, 8, 70, 129), (1, 3, 3, 1100, 1100)])
def test_rows_and_keys_in_one_launch(dev, batch, heads, kv_heads, q_len, k_len, dim, dtype):
    """Little work without a bias: odd numbers of lines and tiles, either side split,
    lengths; an output does not depend on which others are asked for."""
    rng = np.random.default_rng(q_len + k_len)
    for causal in (False, True):
        lengths = {}
        if causal and batch > 1:
            lengths = dict(q_lengths=rng.integers(0, q_len + 1, batch),
                           k_lengths=rng.integers(0, k_len + 1, batch))
        c = Case(dev, batch, heads, q_len, k_len, dim, dtype, kv_heads=kv_heads, causal=causal,
                 seed=dim, **lengths)
        every = c.check()
        for n in every:
            assert np.array_equal(c.backward(only=(n,))[n], every[n]), n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len,bias", [(1, 1, None), (7, 1, None), (64, 1, "random"),
                                              (1, 64, None)])
def test_a_query_of_one_key_has_gradients_of_exactly_0(dev, q_len, k_len, bias, dtype):
    """p is 1 and delta the same dp: nothing is left of their difference."""
    k_lengths = [1, 0, 1]
    c = Case(dev, 3, 4, q_len, k_len, 32, dtype, bias=bias, k_lengths=k_lengths, seed=3)
    got = c.check()
    assert not any(got[n].any() for n in got if n != "dv") and got["dv"].any()


def test_a_bias_shared_by_queries(dev):
    c = Case(dev, 2, 2, 20, 70, 16, "f32", bias="random", shared=(2,))
    (q, k, v), rest = c.oracle()
    want = layers.attention_backward(q, k, v, c.dout, *rest)
    tol = lu.attention_bounds(q, k, v, c.scale, c.bias, want, "f32", c.dout)
    out, lse = c.forward()
    lu.check(out, want["out"], tol["out"])
    for n, got in c.backward(only=("dq", "dk", "dv")).items():
        lu.check(got, want[n], tol[n], n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,k_len", [(64, 64), (40, 150)])
def test_masks_by_the_bias(dev, q_len, k_len, dtype):
    """-inf takes a key out, a row of them gives zeros, a row of the lowest
    value is uniform."""
    rng = np.random.default_rng(8)
    bias = np.where(rng.random((1, 2, q_len, k_len)) < 0.4, -np.inf, rng.normal(size=(1, 2, q_len, k_len)))
    bias[0, 0, 3] = -np.inf
    bias[0, 1, :, 5] = -np.inf
    bias[0, 1, 7] = np.float32(np.finfo(np.float32).min)
    c = Case(dev, 1, 2, q_len, k_len, 32, dtype, bias=bias)
    c.check()
    out, lse = c.forward()
    assert lse[0, 0, 3] == -np.inf and not out[0, 3, 0].any()
    assert np.abs(out[0, 7, 1] - c.v[0, :, 1].mean(0)).max() < 0.05


LOWEST = {"f32": float(np.finfo(np.float32).min), "bf16": -(2.0 - 2.0 ** -7) * 2.0 ** 127,
          "f16": -65504.0}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias_dtype,mask", [("f32", LOWEST["f32"]), ("f32", -1e9), ("f32", -1e4),
                                             ("f32", 1e9), ("bf16", LOWEST["bf16"]),
                                             ("f16", LOWEST["f16"])])
@pytest.mark.parametrize("q_len,k_len,shared", [(64, 64, ()), (40, 150, ()), (9, 1200, ()),
                                                (70, 65, (0,)), (33, 64, (1,))])
def test_rows_that_a_finite_mask_takes_whole(dev, q_len, k_len, shared, bias_dtype, mask, dtype):
    """A row with the same large bias on every key is uniform over them, in its
    gradients too, though ln(keys) is less than a rounding of its log-sum-exp.

    Their queries are 0, so each score is the mask's value itself and p = 1 / keys
    but for the sum's and the exponential's roundings: the bounds are those of the
    same rows with a bias of 0."""
    rng = np.random.default_rng(12)
    rows = [0, 5, q_len - 1]
    shape = [1 if i in shared else n for i, n in enumerate((2, 2, q_len, k_len))]
    bias = rng.normal(size=shape)
    bias[:, :, rows] = mask
    c = Case(dev, 2, 2, q_len, k_len, 32, dtype, bias=bias, bias_dtype=bias_dtype, shared=shared)
    c.q[:, rows] = 0.0
    c.d["q"] = lu.Heads(dev, c.q.shape, dtype, c.q)
    c.p.q.p = c.d["q"].p
    (q, k, v), rest = c.oracle()
    want = layers.attention_backward(q, k, v, c.dout, *rest)
    plain = c.bias.copy()
    plain[:, :, rows] = 0.0
    flat = layers.attention(q, k, v, c.scale, plain)
    tol = lu.attention_bounds(q, k, v, c.scale, plain, {**want, "lse": flat["lse"]}, dtype, c.dout)
    out, _ = c.forward()
    lu.check(out, want["out"], tol["out"], "out")
    got = c.backward()
    n = np.prod([want["dbias"].shape[i] for i in shared]) if shared else 1
    tol["dbias"] = tol["dbias"].sum(shared, keepdims=True) + n * lu.U * np.abs(
        want["dbias"]).sum(shared, keepdims=True)
    want["dbias"] = want["dbias"].sum(shared, keepdims=True)
    tol["dbias"] += lu.rounding(want["dbias"], bias_dtype)
    for name in got:
        lu.check(got[name], want[name], tol[name], name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dev, dtype):
    # Scores of +-500: one key of each row holds nearly all of it.
    Case(dev, 1, 2, 70, 70, 64, dtype, q_scale=60.0, seed=4).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len", [1, 3, 17])
@pytest.mark.parametrize("dim", [32, 128])
def test_few_queries_over_many_keys(dev, q_len, dim, dtype):
    """The long axis is split, forward and backward."""
    c = Case(dev, 1, 4, q_len, 1500, dim, dtype, kv_heads=2, causal=True, seed=q_len)
    assert backend.attention_forward_workspace_bytes(c.p) > 0
    c.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_keys_under_many_queries(dev, dtype):
    Case(dev, 1, 2, 1500, 20, 64, dtype, seed=2, bias="random").check()
    Case(dev, 2, 2, 700, 9, 32, dtype, seed=2, q_lengths=[700, 1], k_lengths=[9, 4]).check()


def test_no_keys_and_no_queries(dev):
    c = Case(dev, 2, 2, 5, 0, 16, "f32")
    out, lse = c.forward()
    assert not out.any() and np.all(lse == -np.inf)
    assert not c.backward()["dq"].any()
    c = Case(dev, 2, 2, 0, 5, 16, "bf16")
    c.forward()
    got = c.backward()
    assert not got["dk"].any() and not got["dv"].any()


@pytest.mark.parametrize("dtype,q_len,k_len", [("bf16", 64, 64), ("f32", 64, 64), ("bf16", 200, 300),
                                               ("f16", 2, 3000)])
def test_the_same_bits_every_run_and_each_output_alone(dev, dtype, q_len, k_len):
    c = Case(dev, 2, 4, q_len, k_len, 32, dtype, bias="random", bias_dtype=dtype)
    out, lse = c.forward()
    a = c.backward()
    for _ in range(2):
        o, ls = c.forward()
        assert np.array_equal(o, out) and np.array_equal(ls, lse)
        b = c.backward()
        assert all(np.array_equal(a[n], b[n]) for n in a)
    for n in a:
        assert np.array_equal(c.backward(only=(n,))[n], a[n]), n


def test_parts_of_one_array(dev):
    """q, k and v and their gradients as columns of one row a token."""
    rng = np.random.default_rng(9)
    b, t, h, d = 2, 64, 4, 32
    x = lu.values(rng, (b, t, 3, h, d), "bf16")
    dout = lu.values(rng, (b, t, h, d), "bf16")
    qkv = dev.put(lu.to_bits(x.reshape(-1), "bf16"))
    grads = lu.Flat(dev, np.zeros(x.size), "bf16")
    s = (t * 3 * h * d, 3 * h * d, d)
    p = backend.attention_problem(qkv, qkv + 2 * h * d, qkv + 4 * h * d, b, h, t, t, d,
                                  dtype="bf16", q_strides=s, k_strides=s, v_strides=s)
    out = dev.put(np.zeros(dout.size, np.uint16))
    lse = dev.put(np.zeros(b * h * t, np.float32))
    backend.attention_forward_device(p, out, d_lse=lse)
    need = backend.attention_backward_workspace_bytes(p)
    backend.attention_backward_device(
        p, out, lse, dev.put(lu.to_bits(dout.reshape(-1), "bf16")), d_dq=grads.p,
        d_dk=grads.p + 2 * h * d, d_dv=grads.p + 4 * h * d, dq_strides=s, dk_strides=s,
        dv_strides=s, d_workspace=dev.alloc(need), workspace_bytes=need)
    dev.sync()
    q, k, v = (x[:, :, i] for i in range(3))
    scale = float(np.float32(d ** -0.5))
    want = layers.attention_backward(q, k, v, dout, scale)
    tol = lu.attention_bounds(q, k, v, scale, None, want, "bf16", dout)
    got = grads.get().reshape(x.shape)
    for i, n in enumerate(("dq", "dk", "dv")):
        lu.check(got[:, :, i], want[n], tol[n], n)


def test_a_long_cache_beyond_32_bits(dev):
    """Keys whose elements lie more than 2^31 apart."""
    rng = np.random.default_rng(10)
    k_len, dim, token = 70, 32, 1 << 25
    k, v = lu.values(rng, (1, k_len, 1, dim), "bf16"), lu.values(rng, (1, k_len, 1, dim), "bf16")
    q, dout = lu.values(rng, (1, 4, 1, dim), "bf16"), lu.values(rng, (1, 4, 1, dim), "bf16")
    far = dev.alloc(2 * (k_len * token))
    host = np.zeros(3 * dim, np.uint16)
    for j in range(k_len):  # keys and values side by side in each token
        host[:dim] = lu.to_bits(k[0, j, 0], "bf16")
        host[dim:2 * dim] = lu.to_bits(v[0, j, 0], "bf16")
        dev.write(far + 2 * j * token, host[:2 * dim])
    st = (0, token, 0)
    d_q, d_do = (dev.put(lu.to_bits(t.reshape(-1), "bf16")) for t in (q, dout))
    p = backend.attention_problem(d_q, far, far + 2 * dim, 1, 1, 4, k_len, dim, dtype="bf16",
                                  k_strides=st, v_strides=st)
    out, lse = dev.put(np.zeros(4 * dim, np.uint16)), dev.put(np.zeros(4, np.float32))
    backend.attention_forward_device(p, out, d_lse=lse)
    need = backend.attention_backward_workspace_bytes(p)
    backend.attention_backward_device(p, out, lse, d_do, d_dk=far + 4 * dim, dk_strides=st,
                                      d_workspace=dev.alloc(need), workspace_bytes=need)
    dev.sync()
    scale = float(np.float32(dim ** -0.5))
    want = layers.attention_backward(q, k, v, dout, scale)
    tol = lu.attention_bounds(q, k, v, scale, None, want, "bf16", dout)
    got = lu.from_bits(dev.get(out, np.zeros(4 * dim, np.uint16)), "bf16").reshape(q.shape)
    lu.check(got, want["out"], tol["out"])
    dk = np.stack([lu.from_bits(dev.get(far + 4 * dim + 2 * j * token, host[:dim]), "bf16")
                   for j in range(k_len)]).reshape(k.shape)
    lu.check(dk, want["dk"], tol["dk"])


@pytest.mark.parametrize("case", [
    dict(q_len=3, k_len=1500, kv_heads=2, causal=True, q_lengths=[3, 1], k_lengths=[1500, 900]),
    dict(q_len=700, k_len=9), dict(q_len=200, k_len=300, bias="random", shared=(0,), causal=True),
    dict(q_len=64, k_len=64, bias="random")])
def test_captured_calls_give_what_eager_ones_do(dev, case):
    """Replayed on new inputs each, with eager calls of the same problem between."""
    c = Case(dev, 2, 4, dim=32, dtype="bf16", **case)
    p, n = c.p, max(backend.attention_backward_workspace_bytes(c.p),
                    backend.attention_forward_workspace_bytes(c.p))
    grads = [lu.Heads(dev, t.shape, "bf16") for t in (c.q, c.k, c.v)]
    ws = [dict(d_workspace=dev.alloc(n), workspace_bytes=n) for _ in range(2)]
    if c.bias is not None:
        for w in ws:
            w["d_dbias"] = c.dbias.p

    def call(w, stream):
        f = {k: w[k] for k in ("d_workspace", "workspace_bytes")}
        backend.attention_forward_device(p, c.out.p, d_lse=c.lse.p, stream=stream, **f)
        backend.attention_backward_device(p, c.out.p, c.lse.p, c.d["dout"].p, d_dq=grads[0].p,
                                          d_dk=grads[1].p, d_dv=grads[2].p, stream=stream, **w)

    def outputs():
        every = [c.out.get(), c.lse.bits()] + [g.get() for g in grads]
        return every + ([c.dbias.bits()] if c.bias is not None else [])

    stream = dev.stream()
    launch = dev.capture(stream, lambda: call(ws[0], stream))
    rng = np.random.default_rng(21)
    seen = []
    for _ in range(4):
        c.d["q"].flat[c.d["q"].at] = lu.to_bits(rng.normal(size=c.q.size), "bf16").reshape(c.q.shape)
        dev.write(c.d["q"].base, c.d["q"].flat)
        launch()
        dev.sync(stream)
        got = outputs()
        call(ws[1], None)
        dev.sync()
        assert all(np.array_equal(a, b) for a, b in zip(got, outputs()))
        seen.append(got[0])
    assert not any(np.array_equal(a, b) for a, b in zip(seen, seen[1:]))


def test_host_memory_is_refused(dev):
    c = Case(dev, 1, 1, 4, 4, 8, "f32")
    host = np.zeros(32, np.float32)
    with pytest.raises(RuntimeError, match="not device memory"):
        backend.attention_forward_device(c.p, host.ctypes.data)
