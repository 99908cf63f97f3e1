"""Queries that see nothing and what lies behind a line's end, where the line's
own values are not finite: outputs and gradients of exactly 0."""

import numpy as np
import pytest

import gpu_util
import layer_util as lu
from metalfish_amd import backend
from test_gpu_train_attention import Case
from test_gpu_train_attention_much import Many

pytestmark = pytest.mark.gpu
INF, NAN = np.inf, np.nan


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


def _put(t, where, value):
    """Elements of a lu.Heads by a boolean mask."""
    t.raw(where, lu.to_bits(np.float32([value]), t.dtype)[0])


def _spoil(c, value):
    """Not finite: one element of a key and of a value that is seen, and of dout of
    a query that sees something, of every line and head."""
    for n in ("k", "v", "dout"):
        t = c.d[n]
        at = np.zeros(t.shape, bool)
        at[:, 0, :, 3] = True
        _put(t, at, value)


def _check(c, dead, behind, lse, out, got):
    """dead: [line, head, query] that see nothing, behind: [line, key]."""
    rows = dead.transpose(0, 2, 1)
    assert dead.any() and np.all(lse[dead] == -INF)
    assert not out[rows].any()
    assert not got["dq"][rows].any()
    for n in ("dk", "dv"):
        assert not got[n][behind].any(), n
    if "dbias" in got and not c.shared:
        assert not got["dbias"][dead].any()


DTYPES = ("f32", "bf16", "f16")
# Squares; rows and keys in one launch; apart, with a bias; rows and keys split.
SHAPES = [(64, 64, None), (64, 64, "random"), (57, 40, "random"), (150, 140, None),
          (150, 140, "random"), (3, 900, None), (900, 20, None), (3, 3000, None)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("q_len,k_len,bias", SHAPES)
def test_behind_the_lengths(dev, q_len, k_len, bias, value, dtype):
    m, n = [q_len, 1, max(1, q_len - 2)], [k_len, max(1, k_len - 5), 1]
    c = Case(dev, 3, 4, q_len, k_len, 32, dtype, kv_heads=4 if bias else 2, bias=bias,
             q_lengths=m, k_lengths=n)
    _spoil(c, value)
    out, lse = c.forward()
    dead = np.broadcast_to((np.arange(q_len) >= np.array(m)[:, None])[:, None], lse.shape)
    _check(c, dead, np.arange(k_len) >= np.array(n)[:, None], lse, out, c.backward())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("q_len,k_len", [(64, 30), (200, 140), (900, 20)])
def test_before_the_first_key(dev, q_len, k_len, value, dtype):
    """More queries than keys, causal: the first see nothing."""
    c = Case(dev, 2, 2, q_len, k_len, 32, dtype, causal=True)
    at = np.zeros(c.q.shape, bool)
    at[:, -1, :, 3] = True
    _put(c.d["dout"], at, value)
    for n in ("k", "v"):
        at = np.zeros(c.k.shape, bool)
        at[:, 0, :, 3] = True
        _put(c.d[n], at, value)
    out, lse = c.forward()
    dead = np.broadcast_to(np.arange(q_len) < q_len - k_len, lse.shape)
    _check(c, dead, np.zeros((2, k_len), bool), lse, out, c.backward())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("q_len,k_len,shared", [(64, 64, ()), (70, 90, ()), (3, 900, ()),
                                                (64, 64, (0,)), (70, 90, (0,))])
def test_rows_that_the_bias_takes_out(dev, q_len, k_len, shared, value, dtype):
    """A row of -inf; a value of the line is not finite."""
    bias = np.random.default_rng(3).normal(size=[1 if i in shared else n for i, n in
                                                 enumerate((2, 2, q_len, k_len))])
    bias[:, :, 1] = -INF
    c = Case(dev, 2, 2, q_len, k_len, 32, dtype, bias=bias, shared=shared)
    at = np.zeros(c.v.shape, bool)
    at[:, 0, :, 3] = True
    _put(c.d["v"], at, value)
    out, lse = c.forward()
    got = c.backward()
    dead = np.zeros(lse.shape, bool)
    dead[:, :, 1] = True
    _check(c, dead, np.zeros((2, k_len), bool), lse, out, got)
    assert not got["dbias"][:, :, 1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,bias_dtype", [(32, None), (64, None), (32, "f32"), (32, "bf16")])
def test_with_much_work(dev, dim, bias_dtype, dtype):
    c = Many(dev, 48, 16, 16, 150, 140, dim, dtype, lengths=True, bias_dtype=bias_dtype)
    for n in ("k", "v", "dout"):
        at = np.zeros(c.d[n].shape, bool)
        at[:, 0, :, 3] = True
        _put(c.d[n], at, INF)
    # All copies alike: NaN equals nothing, so outputs of dead places alone.
    c._one = lambda t, name: t
    out, lse = c.forward()
    got = c.backward()
    m, n = (np.tile(a, 12) for a in c.lengths)
    dead = np.broadcast_to((np.arange(150) >= m[:, None])[:, None], lse.shape)
    _check(c, dead, np.arange(140) >= n[:, None], lse, out, got)
