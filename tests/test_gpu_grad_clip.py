"""mfh_grad_set_* / mfh_grad_norm_device / mfh_grad_scale_device /
mfh_grad_clip_device against 64-bit sums: types, sizes around the chunks,
addresses at any element, in place and apart, norm only, large and small
values, infinities and NaN, graphs and shared sets.

Bounds: squares and sums are 64-bit (relative 2^-53 per step, at most 2^27
steps: below 2^-26 of the norm, and chains are far shorter); the factor
max_norm / norm rounds to 32 bits (2^-24), its product with a gradient again
(2^-24), and the store to the type's half step."""

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


class Grads:
    """Tensors (values, dtype) in one device array, each at an odd place with
    a pattern around, and their copies as destinations."""

    def __init__(self, dev, tensors, where="apart"):
        self.dev, self.where = dev, where
        self.parts, at = [], 16
        for j, (v, dtype) in enumerate(tensors):
            bits = lu.to_bits(v, dtype)
            es = bits.itemsize
            at = (at + es - 1) // es * es
            self.parts.append((at, bits, dtype))
            at += (bits.size + 1 + j % 3) * es
        self.host = np.full(at + 16, 0xA7, np.uint8)
        for p, bits, _ in self.parts:
            raw = bits.view(np.uint8).reshape(-1)
            self.host[p:p + raw.size] = raw
        self.src = dev.put(self.host)
        self.blank = np.full(self.host.size, 0x3C, np.uint8)
        self.dst = self.src if where == "same" else dev.put(self.blank)
        self.values = [lu.from_bits(b, d) for _, b, d in self.parts]
        self.set = backend.GradSet(self.tensors())
        self.ws = dev.put(np.full(self.set.workspace_bytes + 64, 0x5A, np.uint8))
        self.norm = dev.put(np.full(3, -1, np.float32))

    def tensors(self):
        return [(self.src + p if b.size else None,
                 None if self.where == "none" or not b.size else self.dst + p, b.size, d)
                for p, b, d in self.parts]

    def clip(self, max_norm, stream=None, check_ws=True):
        self.set.clip_device(max_norm, self.norm + 4, self.ws, self.set.workspace_bytes,
                             stream=stream)
        return self.read(stream, check_ws)

    def read(self, stream=None, check_ws=True):
        self.dev.sync(stream)
        n = self.dev.get(self.norm, np.zeros(3, np.float32))
        assert n[0] == -1 and n[2] == -1
        if check_ws:
            w = self.dev.get(self.ws, np.zeros(self.set.workspace_bytes + 64, np.uint8))
            assert np.all(w[-64:] == 0x5A)
        got = self.dev.get(self.dst, self.host)
        out, rest = [], got.copy()
        before = self.host if self.where == "same" else self.blank
        for p, b, d in self.parts:
            size = b.size * b.itemsize
            out.append(lu.from_bits(got[p:p + size].copy().view(b.dtype), d))
            rest[p:p + size] = before[p:p + size]
        assert np.array_equal(rest, before), "wrote outside"
        return float(n[1]), out


def check(g, max_norm, norm, out):
    want_norm, want = losses.clip(g.values, max_norm)
    assert abs(norm - want_norm) <= 2 * 2.0 ** -24 * want_norm
    for (_, _, d), a, b in zip(g.parts, out, want):
        lu.close(a, b, 3 * lu.U * np.abs(b), d)


SIZES = (0, 1, 2, 3, 7, 8, 9, 255, 1023, 4096, 16383, 16384, 16385, 40001)


@pytest.mark.parametrize("where", ["apart", "same"])
@pytest.mark.parametrize("dtype", lu.TYPES + ("mixed",))
def test_many_tensors(dev, dtype, where):
    rng = np.random.default_rng(1)
    tensors = [(rng.normal(size=n) * 4.0 ** (i % 4 - 2), lu.TYPES[i % 3] if dtype == "mixed"
                else dtype) for i, n in enumerate(SIZES + SIZES[::-1])]
    for max_norm in (1.0, 1e6, 0.0):
        g = Grads(dev, tensors, where)
        norm, out = g.clip(max_norm)
        check(g, max_norm, norm, out)
        if max_norm == 1e6:   # below: bit for bit
            assert all(np.array_equal(a, b) for a, b in zip(out, g.values))


@pytest.mark.parametrize("count", [1, 5, 1024 * 16384 // 4, 1025 * 16384 + 3])
def test_one_tensor(dev, count):
    rng = np.random.default_rng(2)
    g = Grads(dev, [(rng.standard_normal(count, dtype=np.float32), "f32")])
    norm, out = g.clip(0.5)
    check(g, 0.5, norm, out)


def test_no_tensors_and_empty_ones(dev):
    for tensors in ([], [(np.zeros(0), "f32"), (np.zeros(0), "bf16")]):
        g = Grads(dev, tensors)
        assert g.clip(1.0)[0] == 0.0
    g = Grads(dev, [(np.zeros(100), "f32")])
    norm, out = g.clip(0.0)
    assert norm == 0.0 and np.all(out[0] == 0)


def test_norm_only(dev):
    rng = np.random.default_rng(3)
    g = Grads(dev, [(rng.normal(size=5000), "bf16"), (rng.normal(size=77), "f32")], "none")
    norm, _ = g.clip(1e-3)
    assert abs(norm - losses.clip(g.values, 1.0)[0]) <= 2 ** -23 * norm
    assert np.array_equal(dev.get(g.src, g.host), g.host)


def test_far_apart_values(dev):
    """Squares beyond 32-bit range both ways, and small beside large."""
    rng = np.random.default_rng(4)
    for scale in (1e30, 1e-30):
        g = Grads(dev, [(rng.normal(size=1000) * scale, "f32"), (rng.normal(size=10) * scale, "bf16")])
        norm, out = g.clip(1e-3 * scale)
        check(g, 1e-3 * scale, norm, out)
    g = Grads(dev, [(np.array([3e8]), "f32"), (np.full(100000, 1.0), "f32")])
    norm, out = g.clip(1.0)
    check(g, 1.0, norm, out)


def test_infinities_and_nan(dev):
    """An infinite norm: every finite gradient 0, the infinite ones NaN; a NaN
    goes everywhere."""
    for bad, rest in ((np.inf, 0.0), (np.nan, np.nan)):
        for dtype in lu.TYPES:
            g = Grads(dev, [(np.array([1.0, bad, -2.0]), dtype), (np.ones(9), "f32")])
            norm, out = g.clip(1.0)
            assert np.array_equal(norm, abs(bad), equal_nan=True)
            assert np.isnan(out[0][1])
            assert np.array_equal(out[1], np.full(9, rest), equal_nan=True)
    g = Grads(dev, [(np.array([1.0, np.inf]), "f32")])
    norm, out = g.clip(np.inf)          # nothing to clip to
    assert norm == np.inf and out[0][1] == np.inf and out[0][0] == 1.0


def test_norm_and_scale_apart_make_the_clip(dev):
    """Two shards' sums added by the caller, then one factor for both."""
    rng = np.random.default_rng(5)
    parts = [[(rng.normal(size=30000), "f32"), (rng.normal(size=11), "f16")],
             [(rng.normal(size=20000), "bf16")]]
    shards = [Grads(dev, p) for p in parts]
    sums = []
    for s in shards:
        d = dev.put(np.zeros(1, np.float64))
        s.set.norm_device(d, s.ws, s.set.workspace_bytes)
        dev.sync()
        sums.append(dev.get(d, np.zeros(1))[0])
    total = dev.put(np.array([sum(sums)]))
    want_norm, want = losses.clip(shards[0].values + shards[1].values, 2.0)
    assert abs(np.sqrt(sum(sums)) - want_norm) <= 2 ** -50 * want_norm * 4
    got = []
    for s in shards:
        s.set.scale_device(total, 2.0)
        dev.sync()
        flat = dev.get(s.dst, s.host)
        got += [lu.from_bits(flat[p:p + b.size * b.itemsize].copy().view(b.dtype), d)
                for p, b, d in s.parts]
    dts = [d for s in shards for _, _, d in s.parts]
    for a, b, d in zip(got, want, dts):
        lu.close(a, b, 3 * lu.U * np.abs(b), d)


def test_one_source_into_two_destinations(dev):
    rng = np.random.default_rng(6)
    v = rng.normal(size=1000).astype(np.float32)
    src, a, b = dev.put(v), dev.put(v * 0), dev.put(v * 0)
    s = backend.GradSet([(src, a, 1000, "f32"), (src, b, 1000, "f32")])
    ws = dev.alloc(s.workspace_bytes)
    norm = dev.put(np.zeros(1, np.float32))
    s.clip_device(1.0, norm, ws, s.workspace_bytes)
    dev.sync()
    want_norm, want = losses.clip([v, v], 1.0)
    for p in (a, b):
        lu.close(dev.get(p, v), want[0], 3 * lu.U * np.abs(want[0]))
    assert abs(dev.get(norm, np.zeros(1, np.float32))[0] - want_norm) < 1e-6 * want_norm


def test_one_set_on_two_streams_with_workspaces_of_their_own(dev):
    rng = np.random.default_rng(7)
    g = Grads(dev, [(rng.normal(size=300000), "f32")], "none")
    streams = [dev.stream(), dev.stream()]
    ws = [dev.alloc(g.set.workspace_bytes) for _ in streams]
    norms = [dev.put(np.zeros(1, np.float32)) for _ in streams]
    for _ in range(5):
        for s, w, n in zip(streams, ws, norms):
            g.set.clip_device(1.0, n, w, g.set.workspace_bytes, stream=s)
    dev.sync()
    a, b = (dev.get(n, np.zeros(1, np.float32))[0] for n in norms)
    assert a == b == np.float32(losses.clip(g.values, 1.0)[0])


def test_same_bits_every_time(dev):
    rng = np.random.default_rng(8)
    tensors = [(rng.normal(size=n), "bf16") for n in (100000, 7, 33333)]
    first = Grads(dev, tensors).clip(0.1)
    again = Grads(dev, tensors).clip(0.1)
    assert first[0] == again[0]
    assert all(np.array_equal(a, b) for a, b in zip(first[1], again[1]))


def test_refusals_with_a_device(dev):
    g = Grads(dev, [(np.ones(10), "f32")])
    with pytest.raises(RuntimeError, match="workspace is too small"):
        g.set.clip_device(1.0, g.norm, g.ws, g.set.workspace_bytes - 1)
    with pytest.raises(RuntimeError, match="max_norm"):
        g.set.clip_device(-1.0, g.norm, g.ws, g.set.workspace_bytes)
    with pytest.raises(RuntimeError, match="max_norm"):
        g.set.clip_device(float("nan"), g.norm, g.ws, g.set.workspace_bytes)
    with pytest.raises(RuntimeError, match="null argument"):
        g.set.clip_device(1.0, g.norm, None, 1 << 20)
    with pytest.raises(RuntimeError, match="aligned"):
        g.set.clip_device(1.0, g.norm + 1, g.ws, g.set.workspace_bytes)
    with pytest.raises(RuntimeError, match="aligned"):
        g.set.norm_device(g.norm + 4, g.ws, g.set.workspace_bytes)
    host = np.zeros(64)
    with pytest.raises(RuntimeError, match="d_workspace is not device memory"):
        g.set.clip_device(1.0, g.norm, host.ctypes.data, 512)
    with pytest.raises(RuntimeError, match="src is not device memory"):
        backend.GradSet([(host.ctypes.data, None, 4, "f32")])
    g.set.close()
    with pytest.raises(RuntimeError, match="null argument"):
        g.set.clip_device(1.0, g.norm, g.ws, 1 << 12)


def test_a_norm_in_the_workspace_is_refused(dev):
    """Refused on the host; right behind the workspace it is taken."""
    g = Grads(dev, [(np.full(9000, 2.0), "f32")])
    n = g.set.workspace_bytes
    for at in (0, 4, n - 4):
        with pytest.raises(RuntimeError, match="d_norm lies in the workspace"):
            g.set.clip_device(1.0, g.ws + at, g.ws, n)
    g.set.clip_device(1.0, g.ws + n, g.ws, n)
    dev.sync()
    got = dev.get(g.ws + n, np.zeros(1, np.float32))[0]
    assert got == np.float32(2.0 * np.sqrt(9000.0))


def test_the_standing_streams(dev):
    """hipStreamLegacy and hipStreamPerThread, by their handles."""
    rng = np.random.default_rng(12)
    tensors = [(rng.normal(size=n), "f32") for n in (5000, 77)]
    want = Grads(dev, tensors).clip(0.1)
    for stream in (1, 2):
        g = Grads(dev, tensors)
        g.set.clip_device(0.1, g.norm, g.ws, g.set.workspace_bytes, stream=stream)
        dev.sync()
        assert dev.get(g.norm, np.zeros(1, np.float32))[0] == want[0]
