"""Layer norm, attention and AdamW from their definitions, in 64 bits with
numpy: what the kernels of a training step are compared with.  No counterpart
in the reference (it evaluates nets, it does not train them)."""

import numpy as np


def layer_norm(x, residual=None, alpha=1.0, gamma=None, beta=None, eps=1e-3):
    """{"y", "mean", "rstd"} of rows residual + alpha x."""
    h = alpha * x if residual is None else residual + alpha * x
    mean = h.mean(1)
    rstd = 1 / np.sqrt(((h - mean[:, None]) ** 2).mean(1) + eps)
    y = (h - mean[:, None]) * rstd[:, None]
    y = y * (1.0 if gamma is None else gamma) + (0.0 if beta is None else beta)
    return {"y": y, "mean": mean, "rstd": rstd}


def layer_norm_backward(x, dy, mean, rstd, residual=None, alpha=1.0, gamma=None):
    """{"dx", "dresidual", "dgamma", "dbeta"} from the forward pass's statistics."""
    h = alpha * x if residual is None else residual + alpha * x
    n = (h - mean[:, None]) * rstd[:, None]
    w = dy * (1.0 if gamma is None else gamma)
    dh = rstd[:, None] * (w - w.mean(1)[:, None] - n * (w * n).mean(1)[:, None])
    return {"dx": alpha * dh, "dresidual": dh, "dgamma": (dy * n).sum(0), "dbeta": dy.sum(0)}


def seen(q_len, k_len, m, n, causal):
    """[q_len, k_len]: which keys a query of a line of m queries and n keys sees."""
    i, j = np.arange(q_len)[:, None], np.arange(k_len)[None]
    ok = (i < m) & (j < n)
    return ok & (j <= i + n - m) if causal else ok


def attention(q, k, v, scale, bias=None, causal=False, q_lengths=None, k_lengths=None):
    """q [b, tq, hq, d], k and v [b, tk, hk, d], bias broadcast to [b, hq, tq,
    tk]: {"out", "lse", "p"}, p [b, hq, tq, tk]."""
    b, tq, hq, _ = q.shape
    tk, hk = k.shape[1], k.shape[2]
    out, lse = np.zeros(q.shape), np.full((b, hq, tq), -np.inf)
    p = np.zeros((b, hq, tq, tk))
    full = None if bias is None else np.broadcast_to(bias, (b, hq, tq, tk))
    for i in range(b):
        m = tq if q_lengths is None else min(max(int(q_lengths[i]), 0), tq)
        n = tk if k_lengths is None else min(max(int(k_lengths[i]), 0), tk)
        ok = seen(tq, tk, m, n, causal)
        for h in range(hq):
            kv = h // (hq // hk)
            if not ok.any():
                continue
            s = np.full((tq, tk), -np.inf)
            s[:m, :n] = q[i, :m, h] @ k[i, :n, kv].T * scale
            if full is not None:
                s[:m, :n] += full[i, h, :m, :n]
            s = np.where(ok, s, -np.inf)
            top = s.max(1)
            some = top > -np.inf
            e = np.where(some[:, None], np.exp(s - np.where(some, top, 0.0)[:, None]), 0.0)
            total = e.sum(1)
            lse[i, h, some] = top[some] + np.log(total[some])
            p[i, h, some] = e[some] / total[some, None]
            out[i, :, h] = p[i, h, :, :n] @ v[i, :n, kv]
    return {"out": out, "lse": lse, "p": p}


def attention_backward(q, k, v, dout, scale, bias=None, causal=False, q_lengths=None,
                       k_lengths=None):
    """{"dq", "dk", "dv", "dbias" [b, hq, tq, tk], "ds"}."""
    f = attention(q, k, v, scale, bias, causal, q_lengths, k_lengths)
    b, tq, hq, _ = q.shape
    tk, hk = k.shape[1], k.shape[2]
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    ds = np.zeros((b, hq, tq, tk))
    for i in range(b):
        m = tq if q_lengths is None else min(max(int(q_lengths[i]), 0), tq)
        n = tk if k_lengths is None else min(max(int(k_lengths[i]), 0), tk)
        ok = seen(tq, tk, m, n, causal)
        rows = ok.any(1)
        for h in range(hq):
            kv = h // (hq // hk)
            p, do = f["p"][i, h][:, :n], np.where(rows[:, None], dout[i, :, h], 0.0)
            dp = do @ v[i, :n, kv].T
            delta = (p * dp).sum(1)
            g = p * (dp - delta[:, None])
            ds[i, h, :, :n] = g
            dq[i, :, h] = g @ k[i, :n, kv] * scale
            dk[i, :n, kv] += g[:m].T @ q[i, :m, h] * scale
            dv[i, :n, kv] += p.T @ do
    return {"dq": dq, "dk": dk, "dv": dv, "dbias": ds, **f}


def adamw(param, grad, m, v, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0,
          factor=1.0):
    """(param, m, v) after step number `step`, in 64 bits."""
    g = np.asarray(grad, np.float64) * factor
    m = beta1 * np.asarray(m, np.float64) + (1 - beta1) * g
    v = beta2 * np.asarray(v, np.float64) + (1 - beta2) * g * g
    p = np.asarray(param, np.float64)
    update = m / (1 - beta1 ** step) / (np.sqrt(v / (1 - beta2 ** step)) + eps)
    return p * (1 - lr * weight_decay) - lr * update, m, v


def clip_factor(sumsq, max_norm, grad_scale=1.0):
    norm = grad_scale * np.sqrt(np.float64(sumsq))
    return grad_scale if norm <= max_norm else grad_scale * (max_norm / norm)


# ---- States in 8 bits: fp32 arithmetic, each operation rounded by itself ----

BLOCK = 256
F = np.float32


def _values(lowest, codes):
    """Values of codes of three bits of mantissa, smallest normal 2^lowest."""
    c = np.arange(codes, dtype=np.float64)
    e = np.maximum(c // 8, 1)
    return ((c - 8 * (e - 1)) * 2.0 ** (e + lowest - 4)).astype(F)


M_VALUES = np.concatenate([_values(-6, 128), -_values(-6, 128)])
M_VALUES[[127, 255]] = np.nan
V_VALUES = _values(-14, 256)


def random_bits(seed, step, place):
    """uint32 for each place in the set."""
    with np.errstate(over="ignore"):
        key = np.uint64((seed + step * 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF)
        key ^= key >> np.uint64(29)
        low, high = np.uint32(key & np.uint64(0xFFFFFFFF)), np.uint32(key >> np.uint64(32))
        x = (np.asarray(place).astype(np.uint32) ^ low) * np.uint32(0x9E3779B1)
        x ^= x >> np.uint32(15)
        x = x * np.uint32(0xBB67AE85) + high
        x ^= x >> np.uint32(13)
        x = x * np.uint32(0x6A09E667)
        return x ^ (x >> np.uint32(16))


def _codes(x, lowest, most, extra):
    """Codes of fp32 x >= 0: nearest, ties to even, or with `extra` (16 bits)
    up with the probability of the part cut off.  Below the normal range a code
    is a multiple of the smallest, and twenty bits behind the point are kept."""
    x = x.astype(np.float64)
    e = np.where(x > 0, np.maximum(np.frexp(x)[1] - 1, lowest), lowest)
    q = np.rint(np.ldexp(x, 3 - e + 20)) / 2.0 ** 20
    q = np.rint(q) if extra is None else np.floor(q + extra / 65536.0)
    return np.minimum((e - lowest) * 8 + q.astype(np.int64), most)


def _blocks(n):
    return np.arange(n) // BLOCK


def _scale(x, largest, least):
    n = -(-x.size // BLOCK)
    most = np.zeros(n, F)
    np.maximum.at(most, _blocks(x.size), np.abs(x))
    return np.maximum(most * F(1 / largest), F(least))


def encode_m(m, bits=None):
    m = m.astype(F)
    scale = _scale(m, 448.0, 2.0 ** -100)
    x = m * (F(1) / scale)[_blocks(m.size)]
    code = _codes(np.abs(x), -6, 0x7E, None if bits is None else bits & np.uint32(0xFFFF))
    return (code | np.where(x < 0, 0x80, 0)).astype(np.uint8), scale


def encode_v(v, bits=None):
    v = v.astype(F)
    scale = _scale(v, 122880.0, 2.0 ** -120)
    x = v * (F(1) / scale)[_blocks(v.size)]
    code = _codes(x, -14, 0xFF, None if bits is None else bits >> np.uint32(16))
    return np.maximum(code, (v > 0).astype(np.int64)).astype(np.uint8), scale


def decode_m(code, scale):
    return M_VALUES[code] * scale[_blocks(code.size)]


def decode_v(code, scale):
    return V_VALUES[code] * scale[_blocks(code.size)]


def states_after(grad, m, v, beta1, beta2, factor):
    """m and v in fp32, each product and sum rounded by itself."""
    g = grad.astype(F) * F(factor)
    m = m * F(beta1) + g * F(1 - beta1)
    return m, v * F(beta2) + (g * g) * F(1 - beta2)
