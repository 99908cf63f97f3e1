"""CPU ORACLE of the losses on policy logits and of the gradient clipping --
TEST INFRASTRUCTURE ONLY.

Written from the definitions in 64 bits, row by row: log-softmax over a row's
entries, the clipped policy loss with KL and entropy, the paired preference
loss, and the scaling of gradients to a largest norm.  The reference has no
counterpart; ``tests/test_losses_oracle.py`` pins the gradients against
central differences and the values against closed forms.
"""

from __future__ import annotations

import numpy as np


def _entries(x, columns):
    """Logits of the listed columns; 0 for one outside the row."""
    k = np.asarray(columns, dtype=np.int64)
    inside = (k >= 0) & (k < x.size)
    return np.where(inside, x[np.where(inside, k, 0)], 0.0), k, inside


def log_softmax(v):
    """ln softmax; None if no entry is above -inf (or there is none)."""
    if v.size == 0 or not np.any(v != -np.inf):
        return None
    m = np.max(v)
    with np.errstate(invalid="ignore"):
        z = v - m
    return z - np.log(np.sum(np.exp(z)))


class Row:
    """Softmax of one row over its entries (``columns``: None for all)."""

    def __init__(self, x, columns, action, temp=1.0, ref=None):
        x = np.asarray(x, dtype=np.float64)
        self.vocab = x.size
        cols = np.arange(x.size) if columns is None else columns
        v, self.k, self.inside = _entries(x, cols)
        self.v, self.temp = v, temp
        self.lp = log_softmax(v / temp)
        self.empty = self.lp is None
        # An action that is masked is none of the row's entries.
        self.acted = (not self.empty and action is not None and 0 <= action < x.size
                      and bool(np.any((self.k == action) & (v != -np.inf))))
        self.logp = 0.0
        self.delta = np.zeros(self.k.size)
        if self.acted:
            first = int(np.argmax(self.k == action))
            self.delta[first] = 1.0
            self.logp = self.lp[first]
        if self.empty:
            self.p = np.zeros(self.k.size)
            self.entropy = self.kl = 0.0
            return
        self.p = np.exp(self.lp)
        on = self.p > 0
        self.entropy = -np.sum(self.p[on] * self.lp[on])
        self.kl = 0.0
        if ref is not None:
            self.r = _entries(np.asarray(ref, dtype=np.float64), cols)[0]
            self.lq = log_softmax(self.r / temp)
            if self.lq is None:  # no reference entry left: infinitely far
                self.lq = np.full(self.k.size, -np.inf)
            with np.errstate(invalid="ignore"):
                self.kl = np.sum(self.p[on] * (self.lp[on] - self.lq[on]))

    def spread(self, g):
        """A gradient of the entries as one of the whole row."""
        out = np.zeros(self.vocab)
        np.add.at(out, self.k[self.inside], g[self.inside])
        return out

    def grad_logp(self):
        return self.spread((self.delta - self.p) / self.temp) if self.acted \
            else np.zeros(self.vocab)

    def grad_entropy(self):
        if self.empty:
            return np.zeros(self.vocab)
        lp = np.where(self.p > 0, self.lp, 0.0)
        return self.spread(-self.p * (lp + self.entropy) / self.temp)

    def grad_kl(self):
        if self.empty:
            return np.zeros(self.vocab)
        with np.errstate(invalid="ignore"):
            diff = np.where(self.p > 0, self.lp - self.lq - self.kl, 0.0)
        return self.spread(self.p * diff / self.temp)


def policy_loss(logits, moves, actions, *, temp=1.0, old_logp=None, advantage=None, weight=None,
                ref=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0):
    """mfh_policy_loss_device in 64 bits: {"loss", "logp", "kl", "entropy",
    "grad", "slope"} (slope: the loss' derivative by ln p of the action)."""
    logits = np.asarray(logits, dtype=np.float64)
    rows, vocab = logits.shape
    out = {k: np.zeros(rows) for k in ("loss", "logp", "kl", "entropy", "slope")}
    out["grad"] = np.zeros((rows, vocab))
    for b in range(rows):
        w = 1.0 if weight is None else float(weight[b])
        if w == 0.0:
            continue
        r = Row(logits[b], None if moves is None else moves[b],
                None if actions is None else int(actions[b]), temp,
                None if ref is None else ref[b])
        loss, slope = 0.0, 0.0
        if r.acted and advantage is not None:
            a = float(advantage[b])
            rho = 1.0 if old_logp is None else np.exp(r.logp - float(old_logp[b]))
            if a != 0.0:  # without an advantage no ratio counts, however large
                plain = rho * a
                bounded = min(max(rho, 1.0 - clip_low), 1.0 + clip_high) * a
                loss, slope = (-bounded, 0.0) if bounded < plain else (-plain, -plain)
        g = slope * r.grad_logp()
        if kl_coef:
            loss += kl_coef * r.kl
            g = g + kl_coef * r.grad_kl()
        if entropy_coef:
            loss -= entropy_coef * r.entropy
            g = g - entropy_coef * r.grad_entropy()
        out["loss"][b], out["logp"][b] = w * loss, r.logp
        out["kl"][b], out["entropy"][b] = r.kl, r.entropy
        out["slope"][b], out["grad"][b] = w * slope, w * g
    return out


def preference_loss(logits, moves, actions, seq_offsets, *, temp=1.0, kind="sigmoid", beta=0.1,
                    label_smoothing=0.0, average=False, ref_logp=None, weight=None):
    """mfh_preference_loss_device in 64 bits: {"loss", "margin", "logp",
    "grad", "coef"}; rows outside the sequences are NaN in logp and grad."""
    logits = np.asarray(logits, dtype=np.float64)
    off = np.asarray(seq_offsets, dtype=np.int64)
    pairs = (off.size - 1) // 2
    rows, vocab = logits.shape
    out = {"loss": np.zeros(pairs), "margin": np.zeros(pairs), "logp": np.full(rows, np.nan),
           "grad": np.full((rows, vocab), np.nan), "coef": np.zeros(rows)}
    for i in range(pairs):
        w = 1.0 if weight is None else float(weight[i])
        seqs, sums, counts = [], [], []
        for j in (2 * i, 2 * i + 1):
            seq = [(b, Row(logits[b], None if moves is None else moves[b], int(actions[b]), temp))
                   for b in range(off[j], off[j + 1])]
            got = [r.logp - (0.0 if ref_logp is None else float(ref_logp[b]))
                   for b, r in seq if r.acted]
            seqs.append(seq)
            counts.append(len(got))
            sums.append(sum(got) / (max(1, len(got)) if average else 1))
        diff = sums[0] - sums[1]
        h = beta * diff
        if kind == "sigmoid":
            e = label_smoothing
            loss = (1 - e) * np.logaddexp(0.0, -h) + (e * np.logaddexp(0.0, h) if e else 0.0)
            sig = np.exp(-np.logaddexp(0.0, -h))
            slope = beta * (e * sig - (1 - e) * np.exp(-np.logaddexp(0.0, h)))
        elif kind == "hinge":
            loss, slope = max(0.0, 1.0 - h), -beta if h < 1.0 else 0.0
        else:
            loss, slope = (diff - 0.5 / beta) ** 2, 2.0 * (diff - 0.5 / beta)
        out["loss"][i], out["margin"][i] = (w * loss, h) if w else (0.0, 0.0)
        for s, seq in enumerate(seqs):
            for b, r in seq:
                c = (w * slope * (1 - 2 * s) / (max(1, counts[s]) if average else 1)
                     if w and r.acted else 0.0)
                out["logp"][b], out["coef"][b] = r.logp, c
                out["grad"][b] = c * r.grad_logp() if c else 0.0
    return out


def clip(tensors, max_norm):
    """The norm of all tensors together, and each scaled by min(1, max_norm /
    norm), in 64 bits."""
    tensors = [np.asarray(t, dtype=np.float64) for t in tensors]
    norm = np.sqrt(sum(float(np.sum(t * t)) for t in tensors))
    scale = 1.0 if norm <= max_norm else max_norm / norm
    return norm, [t * scale for t in tensors]
