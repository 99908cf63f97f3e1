"""Layer norm and its gradients on the device against the 64-bit formulas."""

import numpy as np
import pytest

import gpu_util
import layer_util as lu
import learn_gpu as lg
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


def _padded(dev, x, dtype, pad, shift):
    return lg.Padded(dev, lu.to_bits(x.reshape(-1), dtype).reshape(x.shape), dtype, pad, shift)


def _get(a):
    return lu.from_bits(a.get().reshape(-1), a.dtype).astype(np.float64).reshape(a.shape)


def run(dev, rows, width, dtype, residual=True, alpha=0.43, affine=True, eps=1e-3, pad=0, shift=0,
        seed=0, in_place=False, x=None, scale=1.5):
    """Forward and backward on the device, every output against its bound."""
    rng = np.random.default_rng(seed)
    x = lu.values(rng, (rows, width), dtype, scale, 0.5) if x is None else x
    r = lu.values(rng, (rows, width), dtype) if residual else None
    dy = lu.values(rng, (rows, width), dtype)
    gamma = lu.values(rng, width, "f32", 0.3, 1.0) if affine else None
    beta = lu.values(rng, width, "f32", 0.3) if affine else None
    alpha = float(np.float32(alpha))
    eps = float(np.float32(eps))
    dx, dr = _padded(dev, x, dtype, pad, shift), None
    if residual:
        dr = _padded(dev, r, dtype, pad + 3 if pad else 0, shift)
    blank = lambda: lg.Padded(dev, np.full((rows, width), lg.SENTINEL[dtype]), dtype, pad, shift)  # noqa: E731
    y = dx if in_place else blank()
    d_gamma = None if gamma is None else lu.Flat(dev, gamma)
    d_beta = None if beta is None else lu.Flat(dev, beta)
    mean, rstd = lg.Column(dev, rows), lg.Column(dev, rows)
    desc = lambda: backend.norm_rows(  # noqa: E731
        dx.ptr, rows, width, dtype=dtype, x_stride=dx.stride, d_residual=dr.ptr if dr else None,
        residual_stride=dr.stride if dr else None, alpha=alpha,
        d_gamma=d_gamma.p if d_gamma else None, d_beta=d_beta.p if d_beta else None, eps=eps)
    backend.layer_norm_device(desc(), y.ptr, y_stride=y.stride, d_mean=mean.ptr, d_rstd=rstd.ptr)
    dev.sync()
    want = layers.layer_norm(x, r, alpha, gamma, beta, eps)
    tol = lu.norm_bounds(x, r, alpha, gamma, beta, eps, want, dtype)
    got = {"y": _get(y), "mean": mean.get().astype(np.float64), "rstd": rstd.get().astype(np.float64)}
    for k in got:
        lu.check(got[k], want[k], tol[k], k)
    if in_place:  # x is gone
        dx = _padded(dev, x, dtype, pad, shift)
    ddy = _padded(dev, dy, dtype, pad + 1 if pad else 0, shift)
    need = backend.layer_norm_workspace_bytes(rows, width)
    ws, ws_end = lu.workspace(dev, need)
    d_dx = ddy if in_place else blank()
    d_dr = (dr if in_place else blank()) if residual else None
    dg, db = lg.Column(dev, width), lg.Column(dev, width)
    backend.layer_norm_backward_device(
        desc(), ddy.ptr, mean.ptr, rstd.ptr, d_dx=d_dx.ptr,
        d_dresidual=d_dr.ptr if d_dr else None, d_dgamma=dg.ptr, d_dbeta=db.ptr,
        dy_stride=ddy.stride, dx_stride=d_dx.stride,
        dresidual_stride=d_dr.stride if d_dr else None, d_workspace=ws, workspace_bytes=need)
    dev.sync()
    m, s = got["mean"], got["rstd"]
    want = layers.layer_norm_backward(x, dy, m, s, r, alpha, gamma)
    tol = lu.norm_backward_bounds(x, r, alpha, gamma, dy, m, s, want, dtype)
    back = {"dx": _get(d_dx), "dgamma": dg.get(), "dbeta": db.get()}
    if residual:
        back["dresidual"] = _get(d_dr)
    for k in back:
        lu.check(back[k], want[k], tol[k], k)
    ws_end()
    return got, back


# Every lane count and its borders: 16, 64, 256, 1024 lanes, rows read again.
WIDTHS = (1, 3, 8, 63, 64, 65, 127, 129, 256, 500, 511, 513, 1023, 1024, 1025, 2047, 4096, 4099,
          8191, 16383, 16384, 16385, 20001, 32768, 40001)


@pytest.mark.parametrize("dtype", lu.HALF)
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(dev, width, dtype):
    run(dev, 5, width, dtype, residual=width % 2 == 0, seed=width)


@pytest.mark.parametrize("dtype", lu.HALF)
@pytest.mark.parametrize("rows,width", [(1, 256), (2, 96), (4, 1024), (7, 33), (64, 256),
                                        (2050, 40), (2100, 300), (9001, 16), (3001, 1024),
                                        (700, 2500)])
def test_rows(dev, rows, width, dtype):
    run(dev, rows, width, dtype, seed=rows)


@pytest.mark.parametrize("dtype", lu.HALF)
@pytest.mark.parametrize("width", [5, 60, 257, 1030, 5000, 17001])
def test_strides_and_alignments(dev, width, dtype):
    run(dev, 6, width, dtype, pad=5, shift=3, seed=width)
    run(dev, 6, width, dtype, pad=1, shift=1, residual=False, affine=False, alpha=1.0)


@pytest.mark.parametrize("dtype", lu.HALF)
@pytest.mark.parametrize("width", [40, 320, 1024, 3001, 17000])
def test_in_place(dev, width, dtype):
    a, b = run(dev, 9, width, dtype, seed=3)
    c, d = run(dev, 9, width, dtype, seed=3, in_place=True)
    assert all(np.array_equal(a[k], c[k]) for k in a)
    assert all(np.array_equal(b[k], d[k]) for k in b)


@pytest.mark.parametrize("dtype", lu.HALF)
@pytest.mark.parametrize("rows,width", [(140_001, 3), (70_001, 40), (20_003, 250), (4_500, 513),
                                        (4_100, 2048), (4_100, 2049)])
def test_more_rows_than_the_workgroups_have(dev, rows, width, dtype):
    """Both sides of every number of workgroups; nothing behind the workspace."""
    run(dev, rows, width, dtype, seed=width)


@pytest.mark.parametrize("width", [5, 40, 1030])
def test_rows_beyond_32_bits(dev, width):
    """Three rows 2^30 elements apart, every array's row in columns of one buffer."""
    rng = np.random.default_rng(8)
    rows, stride, at = 3, 1 << 30, 2048
    x, r, dy = (lu.values(rng, (rows, width), "bf16") for _ in range(3))
    far = dev.alloc(2 * ((rows - 1) * stride + 8 * at))

    def row(k, i):
        return far + 2 * (i * stride + k * at)

    for k, t in enumerate((x, r, dy)):
        for i in range(rows):
            dev.write(row(k, i), lu.to_bits(t[i], "bf16"))
    stats = [dev.put(np.zeros(rows, np.float32)) for _ in range(2)]
    p = backend.norm_rows(row(0, 0), rows, width, dtype="bf16", x_stride=stride,
                          d_residual=row(1, 0), residual_stride=stride, alpha=0.5)
    backend.layer_norm_device(p, row(3, 0), y_stride=stride, d_mean=stats[0], d_rstd=stats[1])
    backend.layer_norm_backward_device(p, row(2, 0), *stats, d_dx=row(4, 0), d_dresidual=row(5, 0),
                                       dy_stride=stride, dx_stride=stride, dresidual_stride=stride)
    dev.sync()

    def get(k):
        host = np.zeros(width, np.uint16)
        return np.stack([lu.from_bits(dev.get(row(k, i), host), "bf16") for i in range(rows)])

    eps = float(np.float32(1e-3))
    want = layers.layer_norm(x, r, 0.5, None, None, eps)
    tol = lu.norm_bounds(x, r, 0.5, None, None, eps, want, "bf16")
    lu.check(get(3), want["y"], tol["y"], "y")
    mean, rstd = (dev.get(d, np.zeros(rows, np.float32)).astype(np.float64) for d in stats)
    want = layers.layer_norm_backward(x, dy, mean, rstd, r, 0.5, None)
    tol = lu.norm_backward_bounds(x, r, 0.5, None, dy, mean, rstd, want, "bf16")
    lu.check(get(4), want["dx"], tol["dx"], "dx")
    lu.check(get(5), want["dresidual"], tol["dresidual"], "dresidual")


def test_large_means_keep_their_variance(dev):
    # The variance is 1e-6 of the mean's square: a difference of mean squares
    # would hold no digit of it.
    rng = np.random.default_rng(5)
    x = lu.values(rng, (8, 1024), "f32", 1.0, 1000.0)
    got, _ = run(dev, 8, 1024, "f32", residual=False, alpha=1.0, x=x, eps=1e-5)
    assert np.all(np.abs(got["rstd"] - 1) < 0.1)


def test_constant_rows_and_zero_alpha(dev):
    x = np.full((4, 320), 3.0)
    got, back = run(dev, 4, 320, "f32", residual=False, alpha=1.0, x=x, affine=False)
    assert np.all(got["y"] == 0) and np.all(np.isfinite(back["dx"]))
    _, back = run(dev, 4, 320, "bf16", alpha=0.0)
    assert np.all(back["dx"] == 0)


@pytest.mark.parametrize("dtype", lu.HALF)
@pytest.mark.parametrize("width", [48, 700, 3000, 18000])
def test_a_row_that_is_not_finite_spoils_only_itself(dev, width, dtype):
    rng = np.random.default_rng(6)
    x = lu.values(rng, (4, width), dtype)
    bits = lu.to_bits(x.reshape(-1), dtype).reshape(x.shape)
    bits[1, width // 2] = lu.NAN[dtype]
    dx, dy = dev.put(bits), dev.put(lu.to_bits(x.reshape(-1), dtype).reshape(x.shape))
    y, mean, rstd = dev.put(bits), dev.put(np.zeros(4, np.float32)), dev.put(np.zeros(4, np.float32))
    r = backend.norm_rows(dx, 4, width, dtype=dtype)
    backend.layer_norm_device(r, y, d_mean=mean, d_rstd=rstd)
    g = dev.put(bits)
    backend.layer_norm_backward_device(r, dy, mean, rstd, d_dx=g)
    dev.sync()
    for a in (y, g):
        v = lu.from_bits(dev.get(a, bits).reshape(-1), dtype).reshape(4, width)
        assert np.all(np.isnan(v[1])) and np.all(np.isfinite(v[[0, 2, 3]]))


def test_no_rows_give_sums_of_zero(dev):
    dg, db = lg.Column(dev, 70), lg.Column(dev, 70)
    backend.layer_norm_backward_device(backend.norm_rows(None, 0, 70), None, None, None,
                                       d_dgamma=dg.ptr, d_dbeta=db.ptr)
    dev.sync()
    assert not dg.get().any() and not db.get().any()


@pytest.mark.parametrize("width", [300, 17000])
def test_each_output_alone(dev, width):
    """An output does not depend on which others are asked for."""
    rng = np.random.default_rng(7)
    rows = 37
    x, dy = (dev.put(rng.normal(size=(rows, width)).astype(np.float32)) for _ in range(2))
    stats = [dev.put(np.zeros(rows, np.float32)) for _ in range(2)]
    r = backend.norm_rows(x, rows, width, d_residual=dy, alpha=0.5)
    backend.layer_norm_device(r, None, d_mean=stats[0], d_rstd=stats[1])
    need = backend.layer_norm_workspace_bytes(rows, width)
    ws = dev.alloc(need)
    like = {"d_dx": (rows, width), "d_dresidual": (rows, width), "d_dgamma": width, "d_dbeta": width}

    def call(names):
        out = {n: dev.put(np.zeros(like[n], np.float32)) for n in names}
        backend.layer_norm_backward_device(r, dy, *stats, d_workspace=ws, workspace_bytes=need, **out)
        dev.sync()
        return {n: dev.get(p, np.zeros(like[n], np.float32)) for n, p in out.items()}

    every = call(list(like))
    for n in like:
        assert np.array_equal(call([n])[n], every[n]) and every[n].any()
    again = call(list(like))
    assert all(np.array_equal(every[n], again[n]) for n in like)


def test_host_memory_and_other_streams_are_refused(dev):
    x = np.zeros((4, 64), np.float32)
    d = dev.put(x)
    with pytest.raises(RuntimeError, match="not device memory"):
        backend.layer_norm_device(backend.norm_rows(d, 4, 64), x.ctypes.data)
    with pytest.raises(RuntimeError, match=r"failed \(-1\)|failed \(-4\)"):
        backend.layer_norm_device(backend.norm_rows(d, 4, 64, device=backend.device_count()),
                                  dev.put(x))
