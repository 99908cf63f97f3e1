"""Error bounds and device arrays for the tests of the training layers.

The bounds count roundings of the 32-bit arithmetic, u = 2^-24 each, to first
order, and are doubled for what is left out (second order, constants).

Layer norm, a row of n values, sums of K additions in a row (a lane's own, the
tree's, the waves'; 40, and n / 1024 more for rows longer than the registers):

* h = residual + alpha x: e_h = u (|alpha x| + |h|).
* mean: e_m = u K mean|h| + mean e_h + u |mean|; the variance about it: relative
  error 2 (max e_h + e_m) rstd + (K + 4) u; rstd half of that and 3 u.
* n = (h - mean) rstd: e_n = rstd (e_h + e_m + u |h - mean|) + |n| rel(rstd) + u |n|.
* y: |gamma| e_n + 2 u (|n gamma| + |beta|), and half a step of y's type.
* backward, from given mean and rstd: e_n = rstd (e_h + u |h - mean|) + u |n|;
  w: u |w|; a = mean w: (K + 3) u mean|w|; b = mean w n: (K + 4) u mean|w n| + mean |w|
  e_n; dh: rstd (2 u |w| + e_a + |n| e_b + |b| e_n + 3 u |n b| + 3 u |a|) + 2 u |dh|.
* sums over R rows: sum |dy| e_n + (R' + 2) u sum |dy n|, R' additions in a row.

Attention, head size d, k keys; scores on the matrix unit add up d products in
any order:

* e_s = scale (d + 4) u sum|q||k| + 3 u |s|.
* p = exp(s - m): relative e_p = 2 max e_s + u (4 max|s - m| + 8) (the exponent's
  constant, product and difference; the exponential's ulp); the sum of k of them
  (k + 8) u more.  lse: e_s + (k + 12) u + 2 u |lse|.
* with 16 bits each p is rounded before the product: h, half a step, and fp16
  leaves 2^-25 of what lies below 2^-14.
* out = sum p v: sum p |v| (e_p + h + 2 (k + 8) u) + k 2^-25 max|v| (fp16), then half
  a step.
* backward: p from the kernel's lse, relative e_p + e_lse; delta = dout . out: sum
  |dout| e_out + (d + 4) u sum|dout||out|; dp: (d + 4) u sum|dout||v|; dS = p (dp -
  delta): p (e_p |dp - delta| + e_dp + e_delta) + 2 u |dS|, rounded to 16 bits: h
  |dS| + 2^-25 (fp16); dq = scale sum dS k: the errors of dS against |k|, (keys + 8) u
  of the sum of magnitudes, half a step; dk, dv alike over the rows.
"""

import numpy as np

from learn_gpu import SENTINEL
from loss_util import HALF, TINY, U, from_bits, to_bits  # noqa: F401

NAN = {"f32": np.float32(np.nan), "f16": np.float16(np.nan), "bf16": np.uint16(0x7FC1)}


def values(rng, shape, dtype, scale=1.0, shift=0.0):
    """Random values as the device sees them, float64."""
    x = (shift + scale * rng.normal(size=shape)).astype(np.float32)
    return from_bits(to_bits(x.reshape(-1), dtype), dtype).astype(np.float64).reshape(shape)


def check(got, want, tol, what=""):
    """got within tol of want, NaN and infinities where want has them."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.where(fine, 0, got), np.where(fine, 0, want), equal_nan=True), what
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)), 0)
    tol = np.broadcast_to(tol, off.shape)
    worst = np.unravel_index(np.argmax(off - tol), off.shape) if off.size else ()
    assert np.all(off <= tol), (what, worst, off[worst], tol[worst], want[worst])


def rounding(want, dtype):
    return HALF[dtype] * np.abs(want) + TINY[dtype]


def _depth(width):
    return 40 + width // 1024


def norm_bounds(x, residual, alpha, gamma, beta, eps, want, dtype):
    h = alpha * x if residual is None else residual + alpha * x
    k = _depth(x.shape[1])
    e_h = U * (np.abs(alpha * x) + np.abs(h))
    e_m = U * k * np.abs(h).mean(1) + e_h.mean(1) + U * np.abs(want["mean"])
    rel = (e_h.max(1) + e_m) * want["rstd"] + (k + 8) * U
    c, rstd = h - want["mean"][:, None], want["rstd"][:, None]
    n = c * rstd
    e_n = rstd * (e_h + e_m[:, None] + U * np.abs(c)) + np.abs(n) * (rel[:, None] + U)
    g = np.ones(x.shape[1]) if gamma is None else gamma
    b = np.zeros(x.shape[1]) if beta is None else beta
    e_y = np.abs(g) * e_n + 2 * U * (np.abs(n * g) + np.abs(b))
    return {"mean": 2 * e_m + TINY["f32"], "rstd": 2 * rel * want["rstd"],
            "y": 2 * e_y + rounding(want["y"], dtype)}


def norm_backward_bounds(x, residual, alpha, gamma, dy, mean, rstd, want, dtype):
    h = alpha * x if residual is None else residual + alpha * x
    k = _depth(x.shape[1])
    c, r = h - mean[:, None], rstd[:, None]
    n = c * r
    e_n = r * (U * (np.abs(alpha * x) + np.abs(h)) + U * np.abs(c)) + U * np.abs(n)
    w = dy * (1.0 if gamma is None else gamma)
    a, b = w.mean(1)[:, None], (w * n).mean(1)[:, None]
    e_a = (k + 3) * U * np.abs(w).mean(1)[:, None]
    e_b = (k + 4) * U * np.abs(w * n).mean(1)[:, None] + (np.abs(w) * e_n).mean(1)[:, None]
    e = r * (2 * U * np.abs(w) + e_a + np.abs(n) * e_b + np.abs(b) * e_n
             + 3 * U * np.abs(n * b) + 3 * U * np.abs(a)) + 2 * U * np.abs(want["dresidual"])
    rows = x.shape[0] // min(max(x.shape[0], 1), 64) + 64
    return {"dresidual": 2 * e + rounding(want["dresidual"], dtype),
            "dx": 2 * (abs(alpha) * e + U * np.abs(want["dx"])) + rounding(want["dx"], dtype),
            "dgamma": 2 * ((np.abs(dy) * e_n).sum(0) + (rows + 2) * U * np.abs(dy * n).sum(0))
            + TINY["f32"],
            "dbeta": 2 * (rows + 2) * U * np.abs(dy).sum(0) + TINY["f32"]}


def _by_head(t, heads):
    return np.repeat(t, heads // t.shape[2], axis=2).transpose(0, 2, 1, 3)


def attention_bounds(q, k, v, scale, bias, want, dtype, dout=None):
    """Of out and lse, and with dout (want from attention_backward) of the gradients."""
    heads, kv, d = q.shape[2], k.shape[2], q.shape[3]
    b, tk = k.shape[0], k.shape[1]
    if tk == 0 or q.shape[1] == 0 or b == 0:
        return {n: np.zeros(np.shape(want[n])) for n in want}
    half = 0.0 if dtype == "f32" else HALF[dtype]
    low = 2.0 ** -25 if dtype == "f16" else 0.0
    Q, K, V = (np.nan_to_num(_by_head(t, heads)) for t in (q, k, v))
    p, lse = want["p"], np.where(np.isfinite(want["lse"]), want["lse"], 0.0)
    kt = K.transpose(0, 1, 3, 2)
    mag = np.abs(Q) @ np.abs(kt) * abs(scale)
    s = Q @ kt * scale
    if bias is not None:
        s = s + np.broadcast_to(bias, s.shape)
    on = p > 0
    s_on = np.where(on, s, 0.0)
    e_s = np.where(on, (d + 4) * U * mag + 3 * U * np.abs(s_on), 0.0).max(3)
    far = np.where(on, np.abs(s_on - lse[..., None]), 0.0).max(3) + np.log(tk + 1.0)
    e_p = 2 * e_s + U * (4 * far + 8)
    e_lse = e_s + (tk + 12) * U + 2 * U * np.abs(lse)
    e_out = (p @ np.abs(V)) * (e_p + half + 2 * (tk + 8) * U)[..., None]
    e_out = 2 * e_out + tk * low * np.abs(V).max(2, keepdims=True)
    O = _by_head(want["out"], heads)
    e_out = e_out + rounding(O, dtype)
    back = lambda t: t.transpose(0, 2, 1, 3)  # noqa: E731
    tol = {"out": back(e_out), "lse": 2 * e_lse + 2 * (tk + 8) * U}
    if dout is None:
        return tol
    D = np.nan_to_num(_by_head(dout, heads))
    e_delta = (np.abs(D) * e_out).sum(3) + (d + 4) * U * np.abs(D * O).sum(3)
    e_dp = (d + 4) * U * (np.abs(D) @ np.abs(V).transpose(0, 1, 3, 2))
    dp = D @ V.transpose(0, 1, 3, 2)
    ds = want["dbias"]
    base = np.abs(dp - (D * O).sum(3, keepdims=True))
    rel = (e_p + 2 * tol["lse"])[..., None]
    e_ds = 2 * p * (rel * base + e_dp + e_delta[..., None]) + 4 * U * np.abs(ds)
    e_in = e_ds + half * np.abs(ds) + low * (p > 0)
    tq = q.shape[1]
    group = heads // kv
    sums = lambda t: t.reshape(b, kv, group, tk, d).sum(2).transpose(0, 2, 1, 3)  # noqa: E731
    dq = (e_in + (tk + 8) * U * np.abs(ds)) @ np.abs(K) * abs(scale)
    e_k = e_in + (tq * group + 8) * U * np.abs(ds)
    dk = sums(e_k.transpose(0, 1, 3, 2) @ np.abs(Q)) * abs(scale)
    e_v = p * (rel + half + (tq * group + 8) * U) + low * (p > 0)
    dv = sums(e_v.transpose(0, 1, 3, 2) @ np.abs(D))
    tol.update(dq=2 * back(dq) + rounding(want["dq"], dtype),
               dk=2 * dk + rounding(want["dk"], dtype), dv=2 * dv + rounding(want["dv"], dtype),
               dbias=2 * e_ds)
    return tol


class Heads:
    """[batch, tokens, heads, dim] on the device with gaps that hold a pattern:
    order "bthd" or "bhtd", `gap` elements behind each innermost row, `shift`
    before all.  `fill`: what the elements hold at first (outputs)."""

    def __init__(self, dev, shape, dtype, data=None, order="bthd", gap=0, shift=0, fill=None):
        b, t, h, d = shape
        self.dev, self.dtype, self.shape = dev, dtype, shape
        row = d + gap
        self.strides = (t * h * row, h * row, row) if order == "bthd" else (t * h * row, row, t * row)
        size = shift + b * t * h * row + 8
        self.flat = np.full(size, SENTINEL[dtype])
        self.at = (shift + np.arange(b)[:, None, None, None] * self.strides[0]
                   + np.arange(t)[None, :, None, None] * self.strides[1]
                   + np.arange(h)[None, None, :, None] * self.strides[2] + np.arange(d))
        if data is not None:
            self.flat[self.at] = to_bits(np.asarray(data).reshape(-1), dtype).reshape(shape)
        elif fill is not None:
            self.flat[self.at] = fill
        self.base = dev.put(self.flat)
        self.p = self.base + shift * self.flat.itemsize

    def raw(self, mask, value):
        """Overwrites elements (by a boolean mask of the shape) on the device."""
        self.flat[self.at[mask]] = value
        self.dev.write(self.base, self.flat)

    def get(self):
        flat = self.dev.get(self.base, self.flat)
        got = flat[self.at].copy()
        flat[self.at] = self.flat[self.at]
        assert np.array_equal(flat.view(np.uint8), self.flat.view(np.uint8)), "wrote outside"
        return from_bits(got.reshape(-1), self.dtype).astype(np.float64).reshape(self.shape)


class Flat:
    """A one-dimensional array with a pattern around it."""

    def __init__(self, dev, data, dtype="f32"):
        bits = data if dtype == "u8" else to_bits(np.asarray(data).reshape(-1), dtype)
        self.dev, self.dtype, self.n = dev, dtype, bits.size
        mark = np.uint8(0xA5) if dtype == "u8" else SENTINEL[dtype]
        self.lead = 16 if dtype == "u8" else 4
        self.flat = np.full(self.n + 2 * self.lead, mark)
        self.flat[self.lead:self.lead + self.n] = bits.reshape(-1)
        self.base = dev.put(self.flat)
        self.p = self.base + self.lead * self.flat.itemsize

    def bits(self):
        flat = self.dev.get(self.base, self.flat)
        got = flat[self.lead:self.lead + self.n].copy()
        flat[self.lead:self.lead + self.n] = self.flat[self.lead:self.lead + self.n]
        assert np.array_equal(flat.view(np.uint8), self.flat.view(np.uint8)), "wrote outside"
        return got

    def get(self):
        return from_bits(self.bits(), self.dtype).astype(np.float64)


def workspace(dev, need):
    """`need` bytes with a pattern behind: (address, a check that it stayed)."""
    host = np.full(need + 256, 0x5A, np.uint8)
    p = dev.put(host)

    def check_end():
        assert np.all(dev.get(p, host)[need:] == 0x5A), "wrote behind the workspace"
    return p, check_end
