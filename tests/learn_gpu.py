"""Calls of the losses on device buffers for the GPU tests, with everything
around an output filled with a pattern that must stay."""

import numpy as np

import loss_util as lu
from metalfish_amd import backend

SENTINEL = {"f32": np.float32(-77.25), "f16": np.float16(-77.25), "bf16": np.uint16(0xC29B)}


class Padded:
    """Rows of a device array with `pad` columns behind and one row before
    and after, all holding a pattern."""

    def __init__(self, dev, values, dtype, pad=0, shift=0):
        rows, cols = values.shape
        self.dev, self.dtype, self.shape = dev, dtype, (rows, cols)
        self.stride, self.lead = cols + pad, cols + pad + shift
        flat = np.full(self.lead + rows * self.stride + cols + 8, SENTINEL[dtype])
        self.view(flat)[:, :cols] = values
        self.flat = flat
        self.base = dev.put(flat)
        self.ptr = self.base + self.lead * flat.itemsize

    def view(self, flat):
        rows, _ = self.shape
        return flat[self.lead:self.lead + rows * self.stride].reshape(rows, self.stride)

    def get(self):
        """The rows; fails if anything around them changed."""
        flat = self.dev.get(self.base, self.flat)
        got = self.view(flat)[:, :self.shape[1]].copy()
        self.view(flat)[:, :self.shape[1]] = self.view(self.flat)[:, :self.shape[1]]
        assert np.array_equal(flat.view(np.uint8), self.flat.view(np.uint8)), "wrote outside"
        return got


class Column:
    """A float32 output of n values with a pattern around."""

    def __init__(self, dev, n):
        self.dev, self.n = dev, n
        self.flat = np.full(n + 8, SENTINEL["f32"])
        self.base = dev.put(self.flat)
        self.ptr = self.base + 16

    def get(self):
        flat = self.dev.get(self.base, self.flat)
        got = flat[4:4 + self.n].copy()
        flat[4:4 + self.n] = SENTINEL["f32"]
        assert np.all(flat == SENTINEL["f32"]), "wrote outside"
        return got


class Batch:
    """Logits with move lists and actions on the device."""

    def __init__(self, dev, x, dtype, moves, actions, temp=1.0, pad=0, shift=0):
        self.dev, self.dtype, self.moves, self.actions, self.temp = dev, dtype, moves, actions, temp
        bits = lu.to_bits(x, dtype)
        self.values = lu.from_bits(bits, dtype)  # as the device sees them
        self.rows, self.vocab = bits.shape
        self.pad, self.shift = pad, shift
        self.x = Padded(dev, bits, dtype, pad, shift)
        kw = {}
        if moves is not None:
            off, idx = lu.move_lists(moves)
            kw = dict(d_move_offsets=dev.put(off), n_moves=idx.size,
                      d_move_indices=dev.put(idx) if idx.size else None)
        if actions is not None:
            kw["d_actions"] = dev.put(np.asarray(actions, np.int32))
        self.desc = backend.policy_rows(self.x.ptr, self.rows, self.vocab, dtype=dtype,
                                        stride=self.x.stride, softmax_temp=temp, **kw)

    def like(self, values):
        return Padded(self.dev, lu.to_bits(values, self.dtype), self.dtype, self.pad, self.shift)

    def blank(self):
        """An output of the same shape, all pattern."""
        return Padded(self.dev, np.full((self.rows, self.vocab), SENTINEL[self.dtype]), self.dtype,
                      self.pad, self.shift)


def f32(dev, a):
    return None if a is None else dev.put(np.asarray(a, np.float32))


def policy(batch, ref=None, old_logp=None, advantage=None, weight=None, grad=True, in_place=False,
           stream=None, outputs=("loss", "logp", "kl", "entropy"), **kw):
    """Runs mfh_policy_loss_device; {"loss", ..., "grad"} in float64."""
    dev = batch.dev
    cols = {k: Column(dev, batch.rows) for k in outputs if k != "kl" or ref is not None}
    r = None if ref is None else batch.like(ref)
    g = (batch.x if in_place else batch.blank()) if grad else None
    backend.policy_loss_device(
        batch.desc, d_old_logp=f32(dev, old_logp), d_advantage=f32(dev, advantage),
        d_weight=f32(dev, weight), d_ref_logits=None if r is None else r.ptr,
        ref_stride=None if r is None else r.stride, d_grad=None if g is None else g.ptr,
        grad_stride=None if g is None else g.stride, stream=stream,
        **{"d_" + k: c.ptr for k, c in cols.items()}, **kw)
    dev.sync(stream)
    out = {k: c.get().astype(np.float64) for k, c in cols.items()}
    if g is not None:
        out["grad"] = lu.from_bits(g.get(), batch.dtype)
    if not in_place:
        batch.x.get()
    if r is not None:
        r.get()
    return out


def preference(batch, seq_offsets, ref_logp=None, weight=None, grad=True, in_place=False,
               stream=None, **kw):
    dev = batch.dev
    pairs = (len(seq_offsets) - 1) // 2
    cols = {"loss": Column(dev, pairs), "margin": Column(dev, pairs),
            "logp": Column(dev, batch.rows)}
    g = (batch.x if in_place else batch.blank()) if grad else None
    need = backend.preference_loss_workspace_bytes(batch.rows)
    ws = dev.put(np.full(need + 64, 0x5A, np.uint8))
    backend.preference_loss_device(
        batch.desc, pairs, dev.put(np.asarray(seq_offsets, np.int32)), d_ref_logp=f32(dev, ref_logp),
        d_weight=f32(dev, weight), d_grad=None if g is None else g.ptr,
        grad_stride=None if g is None else g.stride, d_workspace=ws, workspace_bytes=need,
        stream=stream, **{"d_" + k: c.ptr for k, c in cols.items()}, **kw)
    dev.sync(stream)
    assert np.all(dev.get(ws, np.zeros(need + 64, np.uint8))[need:] == 0x5A)
    out = {k: c.get().astype(np.float64) for k, c in cols.items()}
    if g is not None:
        out["grad"] = lu.from_bits(g.get(), batch.dtype)
    return out
