"""Element types, move lists and error bounds for the tests of the losses.

The bounds count roundings of the 32-bit arithmetic, u = 2^-24 each
(relative), for one row with z_k = (x_k - max) / T, p = softmax(z):

* z: x is exact; the difference, 1 / T and the product round: 3 u |z|.
* e = exp2(z log2 e): the constant and the product add 2 u |z| to the
  exponent, the exponential 1 ulp = 2 u: relative 5 u |z| + 2 u.
* S: K additions in a row at most (a lane's own, the tree's, the waves'):
  relative K u plus the p-weighted error of e, (5 E|z| + 2) u.  1 / S and the
  product with it round once each.  So p is off by rel_p = u (5 |z| + 5 E|z| +
  K + 8) relative.
* ln S: the relative error of S, plus 2 u |ln S| for the logarithm.
* ln p_a = z_a - ln S: 3 u |z_a| + the error of ln S + u |ln p_a|.
* E_p f: sum p |f| (rel_p + error of f + (K + 4) u).
* exp(-u) - 1 + u: 4 u (exp(-u) + 1 + |u|) for its roundings (argument
  included: 2 u |u| exp(-u)), |1 - exp(-u)| times the error of u, and the
  relative error of p.
Every bound is doubled: products of the terms above (second order) and the
few roundings of the coefficients are within that.
"""

import numpy as np

U = 2.0 ** -24
TYPES = ("f32", "bf16", "f16")
# Half a step relative to the value, and half of the smallest step.
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}


def to_bits(x, dtype):
    """Values as the device array of ``dtype`` (uint16 bits for bf16)."""
    x = np.asarray(x, dtype=np.float32)
    if dtype == "f32":
        return x.copy()
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(a, dtype):
    if dtype == "bf16":
        return (np.asarray(a).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(a).astype(np.float64)


def move_lists(lists):
    """(offsets int32, indices int16) of per-row lists of columns."""
    off = np.zeros(len(lists) + 1, np.int32)
    off[1:] = np.cumsum([len(m) for m in lists])
    idx = np.concatenate([np.asarray(m, np.int16) for m in lists]) if off[-1] else \
        np.zeros(0, np.int16)
    return off, idx.astype(np.int16)


def additions(vocab, moves):
    """K above."""
    return 4 + 6 if moves else max(64, vocab // 1024 + 8) + 6 + 16


class Bounds:
    """Error bounds of one row's quantities from its oracle ``Row``."""

    def __init__(self, row, k):
        self.row, self.k = row, k
        if row.empty:
            return
        p = row.p
        on = p > 0
        with np.errstate(invalid="ignore"):
            z = np.where(on, (row.v - np.max(row.v)) / row.temp, 0.0)
        self.z = z
        mean_abs = float(np.sum(p * np.abs(z)))
        log_s = float(np.log(1.0 / np.max(p)))
        self.rel_p = U * (5 * np.abs(z) + 5 * mean_abs + k + 8)
        self.log_s = U * (k + 5 * mean_abs + 2) + 2 * U * log_s
        za = abs(row.logp + log_s) if row.acted else 0.0
        self.logp = 2 * (3 * U * za + self.log_s + U * abs(row.logp))
        self.mean_z = float(np.sum(p * np.abs(z) * (self.rel_p + (k + 9) * U)))
        self.entropy = 2 * (self.log_s + self.mean_z + U * abs(row.entropy))

    def kl(self):
        """(bound of KL, of u, |u|)."""
        row, p = self.row, self.row.p
        on = p > 0
        with np.errstate(invalid="ignore"):
            d = np.where(on, (row.v - row.r) / row.temp, 0.0)
        mean = float(np.sum(p * d))
        u = np.where(on, d - mean, 0.0)
        off_u = 3 * U * np.abs(d) + U * np.abs(u) + \
            float(np.sum(p * np.abs(d) * (self.rel_p + (self.k + 7) * U)))
        grow = np.exp(np.minimum(-u, 700.0))
        phi = np.maximum(grow - 1 + u, 0.0)
        small = np.abs(u) < 0.2
        # An error d of u moves the term by (1 - exp(-u)) d + exp(-u') d^2 / 2
        # with u' within d of u (Taylor): the second part counts where u is 0,
        # as in a row of one entry; exp(-u') <= 2 exp(-u) for d < 0.69.
        terms = p * (phi * (self.rel_p + (self.k + 10) * U) + np.abs(1 - grow) * off_u +
                     grow * off_u ** 2 +
                     np.where(small, 0.0, 4 * U * (grow * (1 + np.abs(u)) + 1 + np.abs(u))))
        return 2 * (float(np.sum(terms)) + 4 * U * abs(row.kl)), off_u, np.abs(u)

    def grad(self, scale, slope, slope_rel, kl_coef=0.0, entropy_coef=0.0):
        """Bound of scale (slope (1[a] - p) + p (kl u + entropy (z - mean)))
        over the entries, spread over the row."""
        row = self.row
        if row.empty:
            return np.zeros(row.vocab)
        p = row.p
        part = abs(slope) * (row.delta * (slope_rel + 4 * U) +
                             p * (self.rel_p + slope_rel + 4 * U))
        total = abs(slope) * (row.delta + p) * 4 * U
        if kl_coef:
            _, off_u, u = self.kl()
            part = part + abs(kl_coef) * p * (u * (self.rel_p + 6 * U) + off_u)
            total = total + abs(kl_coef) * p * u * 4 * U
        if entropy_coef:
            mean = float(np.sum(p * self.z))
            zc = np.abs(self.z - mean)
            part = part + abs(entropy_coef) * p * (
                zc * (self.rel_p + 6 * U) + 3 * U * np.abs(self.z) + self.mean_z)
            total = total + abs(entropy_coef) * p * zc * 4 * U
        # p below 2^-126 is 0 on the device.
        return abs(scale) * (2 * row.spread(part + total) + 2.0 ** -125 * 64)


def close(got, want, bound, dtype="f32"):
    """|got - want| within the bound, and one rounding to ``dtype``."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    bound = np.asarray(bound, np.float64)
    limit = bound + (np.abs(want) + bound) * HALF[dtype] + TINY[dtype]
    off = np.abs(got - want)
    bad = ~(off <= limit)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], off[bad][:4],
                           np.broadcast_to(limit, off.shape)[bad][:4])
