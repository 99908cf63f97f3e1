"""Clipping where max_norm / norm leaves the 32-bit range: gradients that have
all but overflowed against a small norm.  Bounds: three roundings of a product
(factor, product, store), as for any other factor."""

import numpy as np
import pytest

import gpu_util
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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("count", [5, 4096, 16384 * 3 + 1])
@pytest.mark.parametrize("max_norm", [1e-2, 1e-7, 1.0, 0.7e30])
def test_tiny_factors(dev, dtype, count, max_norm):
    rng = np.random.default_rng(count)
    v = np.clip(rng.normal(size=count), -3, 3) * 1e38
    v[::3] = rng.normal(size=v[::3].size)       # small ones beside
    bits = lu.to_bits(v, dtype)
    values = lu.from_bits(bits, dtype)
    src, dst = dev.put(bits), dev.put(np.zeros_like(bits))
    s = backend.GradSet([(src, dst, count, dtype)])
    ws, sumsq = dev.alloc(s.workspace_bytes), dev.put(np.zeros(1))
    norm, (want,) = losses.clip([values], max_norm)
    s.clip_device(max_norm, None, ws, s.workspace_bytes)
    dev.sync()
    lu.close(lu.from_bits(dev.get(dst, bits), dtype), want, 3 * lu.U * np.abs(want), dtype)
    dev.write(dst, np.zeros_like(bits))
    s.norm_device(sumsq, ws, s.workspace_bytes)
    s.scale_device(sumsq, max_norm)
    dev.sync()
    assert abs(np.sqrt(dev.get(sumsq, np.zeros(1))[0]) - norm) <= 2 ** -40 * norm
    lu.close(lu.from_bits(dev.get(dst, bits), dtype), want, 3 * lu.U * np.abs(want), dtype)
    s.close()
