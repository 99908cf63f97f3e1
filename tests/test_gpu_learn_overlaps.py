"""Calls that would write into another of their arrays are refused, on the
host and before any launch; arrays side by side and in the gaps between rows
are taken."""

import numpy as np
import pytest

import gpu_util
from metalfish_amd import backend

pytestmark = pytest.mark.gpu

N, VOCAB, STRIDE, MOVES = 6, 20, 32, 12


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if backend.device_count() < 1:
        pytest.fail("GPU tests need an MI355X; none visible")


@pytest.fixture
def dev():
    d = gpu_util.DeviceBuffers()
    yield d
    d.free()


class Arena:
    """One allocation, all arrays of a call in it, 4 KiB apart, and 4 KiB
    before the first."""

    def __init__(self, dev, names):
        self.dev, self.bytes = dev, 4096 * (len(names) + 1)
        self.base = dev.put(np.zeros(self.bytes, np.uint8))
        self.at = {k: self.base + 4096 * (i + 1) for i, k in enumerate(names)}

    def put(self, name, values):
        self.dev.write(self.at[name], values)

    def unchanged(self, before):
        return np.array_equal(self.dev.get(self.base, before), before)


def _rows(a):
    return backend.policy_rows(a["logits"], N, VOCAB, stride=STRIDE, d_move_offsets=a["offsets"],
                               d_move_indices=a["indices"], n_moves=MOVES, d_actions=a["actions"])


ROWS = ("logits", "offsets", "indices", "actions")
POLICY_IN = ROWS + ("old_logp", "advantage", "weight", "ref_logits")
POLICY_OUT = ("loss", "logp", "kl", "entropy", "grad")
SIZES = {"logits": 4 * (STRIDE * (N - 1) + VOCAB), "offsets": 4 * (N + 1), "indices": 2 * MOVES}


def _policy(a):
    backend.policy_loss_device(
        _rows(a), ref_stride=STRIDE, grad_stride=STRIDE, kl_coef=0.1,
        **{"d_" + k: a[k] for k in POLICY_IN[4:] + POLICY_OUT})


PREFERENCE_IN = ROWS + ("seq_offsets", "ref_logp", "weight")
PREFERENCE_OUT = ("loss", "margin", "logp", "grad", "workspace")


def _preference(a, pairs=2):
    need = backend.preference_loss_workspace_bytes(N)
    backend.preference_loss_device(
        _rows(a), pairs, a["seq_offsets"], d_ref_logp=a["ref_logp"], d_weight=a["weight"],
        d_loss=a["loss"], d_margin=a["margin"], d_logp=a["logp"], d_grad=a["grad"],
        grad_stride=STRIDE, d_workspace=a["workspace"], workspace_bytes=need)


def _fill(arena):
    arena.put("offsets", np.arange(0, MOVES + 1, 2).astype(np.int32))
    arena.put("indices", np.arange(MOVES).astype(np.int16))
    if "seq_offsets" in arena.at:
        arena.put("seq_offsets", np.array([0, 1, 3, 4, 6], np.int32))


def _sizes(name, call):
    big = ("logits", "ref_logits", "grad")
    if name in big:
        return SIZES["logits"]
    if name == "workspace":
        return 8 * N
    if name == "seq_offsets":
        return 20
    if call is _preference and name in ("weight", "loss", "margin"):
        return 8
    return SIZES.get(name, 4 * N)


@pytest.mark.parametrize("call,ins,outs", [(_policy, POLICY_IN, POLICY_OUT),
                                           (_preference, PREFERENCE_IN, PREFERENCE_OUT)])
def test_every_output_in_every_other_array(dev, call, ins, outs):
    arena = Arena(dev, ins + outs)
    _fill(arena)
    call(arena.at)      # apart: taken
    dev.sync()
    before = dev.get(arena.base, np.zeros(arena.bytes, np.uint8))
    for out in outs:
        for other in ins + outs:
            if other == out:
                continue
            start = arena.at[other]
            # The other's first bytes, its last ones, and from before it.
            places = [start, start + _sizes(other, call) - 8, start - _sizes(out, call) + 8]
            for place in places:
                if out == "grad" and other in ("logits", "ref_logits") and place == start:
                    continue        # in place
                place -= place % (8 if out == "workspace" else 4)
                moved = dict(arena.at, **{out: place})
                with pytest.raises(RuntimeError, match="overlaps"):
                    call(moved)
    dev.sync()
    assert arena.unchanged(before)


def test_arrays_in_the_gaps_between_rows(dev):
    """Twelve columns lie between two rows: room for the losses, by bytes."""
    arena = Arena(dev, POLICY_IN + POLICY_OUT)
    _fill(arena)
    gap = 4 * VOCAB
    moved = dict(arena.at, loss=arena.at["grad"] + gap, logp=arena.at["logits"] + gap + 8,
                 kl=arena.at["logits"] + 4 * STRIDE + gap + 24)
    _policy(moved)
    dev.sync()
    for k, by in (("loss", 28), ("logp", -12), ("kl", 4)):
        with pytest.raises(RuntimeError, match="overlaps"):
            _policy(dict(moved, **{k: moved[k] + by}))
    touching = dict(arena.at, loss=arena.at["logp"] + 4 * N, entropy=arena.at["logp"] - 4 * N)
    _policy(touching)
    dev.sync()


def test_sums_in_the_gradients(dev):
    g = dev.put(np.ones(4096, np.float32))
    s = backend.GradSet([(g + 64, g + 64, 1000, "f32"), (g + 8192, g + 12288, 100, "f32")])
    ws, out = dev.alloc(s.workspace_bytes), dev.alloc(64)
    n = s.workspace_bytes
    for at in (g + 64, g + 4056, g + 8192, g + 8584, g + 12288):
        with pytest.raises(RuntimeError, match="in a gradient"):
            s.clip_device(1.0, at, ws, n)
        with pytest.raises(RuntimeError, match="in a gradient"):
            s.norm_device(at, ws, n)
        with pytest.raises(RuntimeError, match="in a gradient"):
            s.scale_device(at, 1.0)
        with pytest.raises(RuntimeError, match="in a gradient"):
            s.clip_device(1.0, out, at, n)
        with pytest.raises(RuntimeError, match="in a gradient"):
            s.norm_device(out, at, n)
    dev.sync()
    assert np.all(dev.get(g, np.zeros(4096, np.float32)) == 1.0)
    # Between and behind the tensors of one buffer.
    for at in (g + 48, g + 4064, g + 8600, g + 12688):
        s.norm_device(at, ws, n)
        s.scale_device(at, 1e9)
    s.clip_device(1e9, g + 4072, ws, n)
    dev.sync()
    assert dev.get(g + 4072, np.zeros(1, np.float32))[0] == np.float32(np.sqrt(1100.0))
    s.close()


def test_inputs_may_share_memory(dev):
    """The policy as its own reference."""
    arena = Arena(dev, POLICY_IN + POLICY_OUT)
    _fill(arena)
    arena.put("weight", np.ones(N, np.float32))
    _policy(dict(arena.at, ref_logits=arena.at["logits"], advantage=arena.at["old_logp"]))
    dev.sync()
    assert np.all(dev.get(arena.at["kl"], np.zeros(N, np.float32)) == 0)
