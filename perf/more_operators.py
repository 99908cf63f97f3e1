"""The operators of a training step between the losses and the next weights
whose speed is measured.

A program that trains the framework's nets has the gradient of the logits from
the losses, and needs the layers' backward passes and the update:

* ``norm`` / ``norm-back``: layer norm of ``residual + alpha x`` with its
  statistics, and the gradients of everything that went in;
* ``attend`` / ``attend-back``: attention with an additive bias (the nets'
  smolgen), which keeps a row's log-sum-exp, and its backward pass, which forms
  the probabilities again from it;
* ``adamw``: one AdamW step over all weights of a net, gradients clipped to a
  norm on the way, states in 32 bits or in 8 (blocks of 256 values with a
  scale each).
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
# The nets' LayerNorm and the residual weight of a 15-layer body.
EPS, ALPHA = 1e-3, (2.0 * 15) ** -0.25
BETA1, BETA2, ADAM_EPS = 0.9, 0.98, 1e-7
BLOCK = 256
SEED = 0x5EED5EED12345
# Most values of one drawn norm, most pairs of query and key, most weights.
MOST_VALUES, MOST_PAIRS, MOST_WEIGHTS = 16_777_216, 33_554_432, 159_000_000


def _norm(op, rows, width, dtype="bf16", residual=True, name=None):
    case = {"op": op, "rows": rows, "width": width, "dtype": dtype, "residual": residual}
    return case if name is None else {"name": name, **case}


def _attend(op, batch, heads, q_len, k_len, dim, dtype="bf16", kv_heads=None, causal=False,
            ragged=False, bias=False, name=None):
    """``bias``: one for every pair of every head of every position."""
    case = {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads or heads,
            "q_len": q_len, "k_len": k_len, "dim": dim, "dtype": dtype, "causal": causal,
            "ragged": ragged, "bias": bias}
    return case if name is None else {"name": name, **case}


def _adamw(width, layers, ffn, dtype="f32", state=32, smolgen=True, copy=False, stochastic=False,
           name=None):
    """``dtype``: the matrices' gradients; weights are in 32 bits, ``copy``:
    with a bf16 copy of the matrices for the next forward pass."""
    case = {"op": "adamw", "width": width, "layers": layers, "ffn": ffn, "dtype": dtype,
            "state": state, "smolgen": smolgen, "copy": copy, "stochastic": stochastic}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # A batch of 256 positions in a body of width 1024.
        _norm("norm", 16384, 1024, name="norm-body-bf16"),
        # One position's squares in the small network: latency.
        _norm("norm-back", 64, 256, "f32", name="norm-back-small"),
        # The batch's backward pass.
        _norm("norm-back", 16384, 1024, name="norm-back-body-bf16"),
        # Odd long rows of another model, without a residual.
        _norm("norm-back", 2053, 5003, "f16", False, name="norm-back-odd-f16"),
        # The batch's attention over 64 squares with a bias from smolgen.
        _attend("attend", 256, 32, 64, 64, 32, bias=True, name="attend-squares-bf16"),
        # A few new tokens of one long line: the keys are the long axis.
        _attend("attend", 1, 16, 3, 20011, 64, kv_heads=4, causal=True, name="attend-line-bf16"),
        # Four positions of the small network in 32 bits: latency.
        _attend("attend-back", 4, 8, 64, 64, 32, "f32", name="attend-back-small"),
        # The batch's attention, backward, with the bias's gradient.
        _attend("attend-back", 256, 32, 64, 64, 32, bias=True, name="attend-back-squares-bf16"),
        # Ragged lines of tokens, heads sharing keys.
        _attend("attend-back", 4, 16, 1021, 1021, 64, kv_heads=4, causal=True, ragged=True,
                name="attend-back-lines-bf16"),
        # The small network's weights.
        _adamw(256, 2, 512, smolgen=False, name="adamw-small"),
        # The benchmark's network: bf16 gradients, a bf16 copy, states in 8 bits.
        _adamw(1024, 15, 1536, "bf16", 8, copy=True, stochastic=True, name="adamw-large-8bit"),
        # The same with gradients and states in 32 bits.
        _adamw(1024, 15, 1536, name="adamw-large"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "norm-back", "norm-back", "attend", "attend-back", "attend-back",
                     "attend-back", "adamw", "adamw"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op.startswith("norm"):
        width = _spread(rng, 16, 20000)
        return _norm(op, _spread(rng, 1, min(50000, MOST_VALUES // width)), width, dtype,
                     rng.random() < 0.6)
    if op == "adamw":
        width = 64 * rng.randint(1, 16)
        case = _adamw(width, rng.randint(1, 15), 32 * rng.randint(2, max(2, 3 * width // 64)),
                      dtype, rng.choice((8, 32)), rng.random() < 0.5, rng.random() < 0.5)
        case["stochastic"] = case["state"] == 8 and rng.random() < 0.5
        while sum(_sizes(case)) > MOST_WEIGHTS:
            case["layers"] -= 1
        return case
    if rng.random() < 0.5:
        heads = rng.choice((4, 8, 16, 24, 32))
        return _attend(op, _spread(rng, 1, 256 * 32 // heads), heads, 64, 64, 32, dtype,
                       bias=rng.random() < 0.6)
    kv_heads = rng.choice((1, 2, 4))
    heads, dim = kv_heads * rng.choice((1, 3, 4)), rng.choice((32, 64, 96, 128))
    k_len = _spread(rng, 1, 20000 if op == "attend" else 4000)
    q_len = k_len if rng.random() < 0.6 else rng.randint(1, min(k_len, 40))
    if q_len * k_len * heads > MOST_PAIRS // 2:
        q_len = max(1, MOST_PAIRS // 2 // (k_len * heads))
    most = max(1, min(64, MOST_PAIRS // (2 * q_len * k_len * heads)))
    if dtype == "f32":
        most = max(1, most // 4)
    return _attend(op, _spread(rng, 1, most), heads, q_len, k_len, dim, dtype, kv_heads,
                   rng.random() < 0.6, q_len == k_len and rng.random() < 0.5)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


# ---- Layer norm ---------------------------------------------------------


def _prepare_norm(case, g):
    rows, width, dt = case["rows"], case["width"], DTYPES[case["dtype"]]
    s = {"case": case, "x": (0.5 + 1.5 * _randn(g, rows, width)).to(dt),
         "gamma": 1 + 0.1 * _randn(g, width), "beta": 0.1 * _randn(g, width),
         "residual": _randn(g, rows, width).to(dt) if case["residual"] else None}
    s["mean"], s["rstd"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    if case["op"] == "norm":
        s["y"] = torch.empty_like(s["x"])
        return s
    h = _sum(s)
    s["mean"] = h.mean(1)
    s["rstd"] = 1 / torch.sqrt((h - s["mean"][:, None]).square().mean(1) + EPS)
    s["dy"] = _randn(g, rows, width).to(dt)
    s["dx"] = torch.empty_like(s["x"])
    s["dresidual"] = torch.empty_like(s["x"]) if case["residual"] else None
    s["dgamma"], s["dbeta"] = torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
    return s


def _sum(s):
    if s["residual"] is None:
        return s["x"].float()
    return s["residual"].float() + ALPHA * s["x"].float()


def _plain_norm(s):
    h, dt = _sum(s), s["x"].dtype
    if s["case"]["op"] == "norm":
        mean = h.mean(1, keepdim=True)
        c = h - mean
        rstd = 1 / torch.sqrt(c.square().mean(1, keepdim=True) + EPS)
        return {"y": (c * rstd * s["gamma"] + s["beta"]).to(dt), "mean": mean[:, 0],
                "rstd": rstd[:, 0]}
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xh = (h - s["mean"][:, None]) * rstd
    w = dy * s["gamma"]
    dh = rstd * (w - w.mean(1, keepdim=True) - xh * (w * xh).mean(1, keepdim=True))
    out = {"dgamma": (dy * xh).sum(0), "dbeta": dy.sum(0)}
    if s["residual"] is None:
        return {**out, "dx": dh.to(dt)}
    return {**out, "dx": (ALPHA * dh).to(dt), "dresidual": dh.to(dt)}


def _own_norm(backend, s, stream):
    c = s["case"]
    rows = backend.norm_rows(
        s["x"].data_ptr(), c["rows"], c["width"], dtype=c["dtype"],
        d_residual=_address(s["residual"]), alpha=ALPHA if c["residual"] else 1.0,
        d_gamma=s["gamma"].data_ptr(), d_beta=s["beta"].data_ptr(), eps=EPS)
    if c["op"] == "norm":
        backend.layer_norm_device(rows, s["y"].data_ptr(), d_mean=s["mean"].data_ptr(),
                                  d_rstd=s["rstd"].data_ptr(), stream=stream)
        return {k: s[k] for k in ("y", "mean", "rstd")}
    backend.layer_norm_backward_device(
        rows, s["dy"].data_ptr(), s["mean"].data_ptr(), s["rstd"].data_ptr(),
        d_dx=s["dx"].data_ptr(), d_dresidual=_address(s["dresidual"]),
        d_dgamma=s["dgamma"].data_ptr(), d_dbeta=s["dbeta"].data_ptr(),
        d_workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(),
        stream=stream)
    out = {k: s[k] for k in ("dx", "dgamma", "dbeta")}
    return {**out, "dresidual": s["dresidual"]} if c["residual"] else out


def _exact_norm(s):
    x = s["x"].double().requires_grad_()
    r = None if s["residual"] is None else s["residual"].double().requires_grad_()
    gamma, beta = (s[k].double().requires_grad_() for k in ("gamma", "beta"))
    h = x if r is None else r + ALPHA * x
    y = torch.nn.functional.layer_norm(h, h.shape[1:], gamma, beta, EPS)
    if s["case"]["op"] == "norm":
        var = h.var(1, unbiased=False)
        return {"y": y.detach(), "mean": h.mean(1).detach(),
                "rstd": (var + EPS).rsqrt().detach()}
    names = ["dx", "dgamma", "dbeta"] + ([] if r is None else ["dresidual"])
    of = [x, gamma, beta] + ([] if r is None else [r])
    return dict(zip(names, torch.autograd.grad(y, of, s["dy"].double())))


# ---- Attention ----------------------------------------------------------


def _lengths(case):
    """Tokens of each line; a case's own, so that its shapes are."""
    r = torch.Generator().manual_seed(1000 * case["batch"] + case["q_len"])
    n = torch.randint(1, case["q_len"] + 1, (case["batch"],), generator=r)
    n[0] = case["q_len"]
    return n


def _prepare_attend(case, g):
    b, hq, hk, tq, tk, d = (case[k] for k in ("batch", "heads", "kv_heads", "q_len", "k_len",
                                              "dim"))
    dt, dev = DTYPES[case["dtype"]], "cuda"
    s = {"case": case, "q": _randn(g, b, tq, hq, d).to(dt), "k": _randn(g, b, tk, hk, d).to(dt),
         "v": _randn(g, b, tk, hk, d).to(dt), "scale": 1 / math.sqrt(d), "bias": None,
         "lengths": _lengths(case).int().to(dev) if case["ragged"] else None}
    if case["bias"]:
        s["bias"] = _randn(g, b, hq, tq, tk).to(dt)
    s["out"], s["lse"] = torch.empty_like(s["q"]), torch.empty(b, hq, tq, device=dev)
    if case["op"] == "attend-back":
        # What the forward pass left.
        f = _plain_attend(s)
        s["out"], s["lse"] = f["out"].contiguous(), f["lse"].contiguous()
        s["dout"] = _randn(g, b, tq, hq, d).to(dt)
        for name in ("q", "k", "v"):
            s["d" + name] = torch.empty_like(s[name])
        if s["bias"] is not None:
            s["dbias"] = torch.empty_like(s["bias"])
    return s


def _by_head(t, heads):
    """[batch, tokens, heads, dim] as [batch, heads, tokens, dim] in 32 bits,
    shared heads repeated."""
    t = t.float().transpose(1, 2)
    return t.repeat_interleave(heads // t.shape[1], 1).contiguous()


def _seen(s):
    """Which keys each query sees, or None: all."""
    c, ok = s["case"], None
    q, k = torch.arange(c["q_len"], device="cuda"), torch.arange(c["k_len"], device="cuda")
    if c["causal"]:
        # The last query sees the last key (of a ragged line: its last token).
        ok = (k[None] <= q[:, None] + (c["k_len"] - c["q_len"]))[None, None]
    if s["lengths"] is not None:
        n = s["lengths"].long()[:, None, None, None]
        inside = (q[:, None] < n) & (k[None] < n)
        ok = inside if ok is None else ok & inside
    return ok


def _scores(s, q, k):
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    if s["bias"] is not None:
        x = x + s["bias"].float()
    ok = _seen(s)
    return x if ok is None else torch.where(ok, x, -math.inf)


def _plain_attend(s):
    heads = s["case"]["heads"]
    x = _scores(s, _by_head(s["q"], heads), _by_head(s["k"], heads))
    m = x.amax(3, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(x - m)
    total = e.sum(3, keepdim=True)
    out = torch.matmul(e, _by_head(s["v"], heads)) / torch.where(total == 0, 1.0, total)
    return {"out": out.transpose(1, 2).to(s["q"].dtype), "lse": (m + torch.log(total))[..., 0]}


def _shared(s, t):
    """A gradient per head as one per shared head, in the inputs' type."""
    b, _, n, d = t.shape
    return t.view(b, s["case"]["kv_heads"], -1, n, d).sum(2).transpose(1, 2).to(s["q"].dtype)


def _plain_attend_back(s):
    heads = s["case"]["heads"]
    q, k, v, o, do = (_by_head(s[n], heads) for n in ("q", "k", "v", "out", "dout"))
    x = _scores(s, q, k)
    lse = s["lse"][..., None]
    p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse))
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(3, keepdim=True))
    dq = torch.matmul(ds, k) * s["scale"]
    back = lambda t, u: torch.matmul(t.transpose(2, 3).contiguous(), u)  # noqa: E731
    out = {"dq": dq.transpose(1, 2).to(s["q"].dtype), "dk": _shared(s, back(ds, q) * s["scale"]),
           "dv": _shared(s, back(p, do))}
    if s["bias"] is not None:
        out["dbias"] = ds.to(s["bias"].dtype)
    return out


def _own_problem(backend, s):
    c = s["case"]
    return backend.attention_problem(
        s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), c["batch"], c["heads"],
        c["q_len"], c["k_len"], c["dim"], dtype=c["dtype"], kv_heads=c["kv_heads"],
        scale=s["scale"], causal=c["causal"], d_bias=_address(s["bias"]),
        bias_dtype=c["dtype"], d_q_lengths=_address(s["lengths"]),
        d_k_lengths=_address(s["lengths"]))


def _own_attend(backend, s, stream):
    ws = {"d_workspace": s["workspace"].data_ptr(), "workspace_bytes": s["workspace"].numel(),
          "stream": stream}
    problem = _own_problem(backend, s)
    if s["case"]["op"] == "attend":
        backend.attention_forward_device(problem, s["out"].data_ptr(), d_lse=s["lse"].data_ptr(),
                                         **ws)
        return {"out": s["out"], "lse": s["lse"]}
    backend.attention_backward_device(
        problem, s["out"].data_ptr(), s["lse"].data_ptr(), s["dout"].data_ptr(),
        d_dq=s["dq"].data_ptr(), d_dk=s["dk"].data_ptr(), d_dv=s["dv"].data_ptr(),
        d_dbias=_address(s.get("dbias")), **ws)
    return {k: s[k] for k in ("dq", "dk", "dv", "dbias") if k in s}


def _exact_attend(s):
    c = s["case"]
    if _pairs(c) * c["batch"] > 400_000_000:
        return None
    q, k, v = (s[n].double().requires_grad_() for n in ("q", "k", "v"))
    each = c["heads"] // c["kv_heads"]
    bias = None if s["bias"] is None else s["bias"].double().requires_grad_()
    qh = q.permute(0, 2, 1, 3)
    kh, vh = (t.permute(0, 2, 1, 3)[:, :, None].expand(-1, -1, each, -1, -1).flatten(1, 2)
              for t in (k, v))
    x = (qh * s["scale"]) @ kh.mT.contiguous()
    if bias is not None:
        x = x + bias
    ok = torch.ones(c["q_len"], c["k_len"], dtype=torch.bool, device="cuda")
    if c["causal"]:
        ok = ok.tril(c["k_len"] - c["q_len"])
    ok = ok.expand(c["batch"], 1, -1, -1).clone()
    if s["lengths"] is not None:
        for i, n in enumerate(s["lengths"].tolist()):
            ok[i, :, n:] = False
            ok[i, :, :, n:] = False
    none = ~ok.any(3, keepdim=True)
    x = x.masked_fill(~(ok | none), -math.inf)
    p = torch.softmax(x, 3).masked_fill(none, 0.0)
    out = (p @ vh).permute(0, 2, 1, 3)
    if c["op"] == "attend":
        lse = torch.logsumexp(x, 3).masked_fill(none[..., 0], -math.inf)
        return {"out": out.detach(), "lse": lse.detach()}
    names = ["dq", "dk", "dv"] + ([] if bias is None else ["dbias"])
    of = [q, k, v] + ([] if bias is None else [bias])
    return dict(zip(names, torch.autograd.grad(out, of, s["dout"].double())))


def _pairs(case):
    """Pairs of query and key that one head computes, over the batch."""
    def one(tq, tk):
        if not case["causal"]:
            return tq * tk
        first = max(0, tq - tk)  # queries before it see nothing
        n = tq - first
        return n * (tk - tq) + sum(range(first + 1, tq + 1)) if n else 0
    if case["ragged"]:
        return sum(one(int(n), int(n)) for n in _lengths(case)) / case["batch"]
    return one(case["q_len"], case["k_len"])


# ---- AdamW --------------------------------------------------------------


def _sizes(case):
    """Values of each weight tensor of a network of this shape."""
    e, f, squares, heads = case["width"], case["ffn"], 64, case["width"] // 32
    sizes = [squares * 16 * squares * 12, squares * 16, e * 128, e, e, e, e * squares, e * squares,
             f * e, f, e * f, e, e, e]
    if case["smolgen"]:
        sizes.append(squares * squares * 256)
    for _ in range(case["layers"]):
        sizes += [e * e, e] * 4
        if case["smolgen"]:
            sizes += [32 * e, 256 * squares * 32, 256, heads * 256 * 256, heads * 256, 256, 256,
                      heads * 256, heads * 256]
        sizes += [e, e, f * e, f, e * f, e, e, e]
    sizes += [e * e, e] * 3 + [4 * e, 32 * e, 32, 128 * squares * 32, 128, 384, 3]
    return sizes


def _prepare_adamw(case, g):
    """Two flat buffers, as trainers keep them: the matrices, with a decay,
    and the vectors, without.  Each tensor begins on a whole block; what lies
    between tensors is zero and stays so."""
    s = {"case": case, "step": 100, "lr": 1e-3, "max_norm": 1.0, "flat": {}}
    sizes = _sizes(case)
    for kind in ("matrices", "vectors"):
        mine = [n for n in sizes if (n >= 4096) == (kind == "matrices")]
        starts, total = [], 0
        for n in mine:
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        live = torch.zeros(total, dtype=torch.bool, device="cuda")
        for at, n in zip(starts, mine):
            live[at:at + n] = True
        gdt = DTYPES[case["dtype"] if kind == "matrices" else "f32"]
        f = {"param": 0.03 * _randn(g, total) * live, "decay": 0.01 if kind == "matrices" else 0.0,
             "grad": (1e-3 * _randn(g, total) * live).to(gdt),
             "tensors": list(zip(starts, mine))}
        m = 1e-4 * _randn(g, total) * live
        v = 1e-7 * (0.1 + torch.rand(total, device="cuda", generator=g)) * live
        if case["state"] == 8:
            f["m"], f["m_scale"] = _to_m_codes(m, None)
            f["v"], f["v_scale"] = _to_v_codes(v, None)
        else:
            f["m"], f["v"] = m, v
        if case["copy"] and kind == "matrices":
            f["copy"] = f["param"].bfloat16()
        s["flat"][kind] = f
    grads = [f["grad"] for f in s["flat"].values()]
    s["sumsq"] = sum(t.double().square().sum() for t in grads).reshape(1)
    return s


def _bits(case, step, count):
    """32 random bits of each value, from the seed, the step and its place."""
    mask = 0xFFFFFFFF
    key = (SEED + step * 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF
    key ^= key >> 29
    at = torch.arange(count, device="cuda")
    x = ((at ^ (key & mask)) * 0x9E3779B1) & mask
    x ^= x >> 15
    x = (x * 0xBB67AE85 + (key >> 32)) & mask
    x ^= x >> 13
    x = (x * 0x6A09E667) & mask
    return x ^ (x >> 16)


def _to_code(x, lowest, most, extra):
    """Codes of three bits of mantissa of non-negative values; ``lowest``: the
    exponent of the smallest normal one.  Nearest, ties to even, or with
    ``extra`` (16 random bits) up with the probability of the part cut off."""
    e = (torch.frexp(x).exponent - 1).clamp(min=lowest)
    q = torch.ldexp(x.double(), 3 - e)
    q = torch.round(q * 2.0 ** 20) / 2.0 ** 20
    q = torch.round(q) if extra is None else torch.floor(q + extra / 65536.0)
    return ((e - lowest) * 8 + q.long()).clamp(max=most)


def _scaled(x, largest, least):
    """Blocks over their scales: largest code for a block's largest value."""
    scale = (x.abs().view(-1, BLOCK).amax(1) * (1 / largest)).clamp(min=least)
    return (x.view(-1, BLOCK) * (1 / scale)[:, None]).view(-1), scale


def _to_m_codes(m, bits):
    x, scale = _scaled(m, 448.0, 2.0 ** -100)
    code = _to_code(x.abs(), -6, 0x7E, None if bits is None else bits & 0xFFFF)
    return (code | ((x < 0).long() << 7)).to(torch.uint8), scale


def _to_v_codes(v, bits):
    x, scale = _scaled(v, 122880.0, 2.0 ** -120)
    code = _to_code(x, -14, 0xFF, None if bits is None else bits >> 16)
    return code.clamp(min=(v > 0).long()).to(torch.uint8), scale


def _of_v_codes(code, scale):
    c = torch.arange(256, device="cuda", dtype=torch.float64)
    e = (c // 8).clamp(min=1)
    table = ((c - 8 * (e - 1)) * 2.0 ** (e - 18)).float()
    return (table[code.int()].view(-1, BLOCK) * scale[:, None]).view(-1)


def _of_m_codes(code, scale):
    x = code.view(torch.float8_e4m3fn).float()
    return (x.view(-1, BLOCK) * scale[:, None]).view(-1)


def _outputs(s):
    """Everything a step changes.  What is held in 8 bits as the codes'
    values, next to the scales: the first moment's codes are e4m3."""
    out = {}
    for kind, f in s["flat"].items():
        out[kind] = {k: f[k] for k in ("param", "m", "v", "m_scale", "v_scale", "copy") if k in f}
        if s["case"]["state"] == 8:
            out[kind]["m"] = f["m"].view(torch.float8_e4m3fn)
    return out


def _plain_adamw(s):
    c, step, lr = s["case"], s["step"], s["lr"]
    norm = s["sumsq"].sqrt()
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0).float()
    rbc2 = 1 / math.sqrt(1 - BETA2 ** step)
    size = lr / (1 - BETA1 ** step)
    at = 0
    for f in s["flat"].values():
        eight = c["state"] == 8
        m = _of_m_codes(f["m"], f["m_scale"]) if eight else f["m"]
        v = _of_v_codes(f["v"], f["v_scale"]) if eight else f["v"]
        g = f["grad"].float() * scale
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + (g * g) * (1 - BETA2)
        f["param"].copy_(f["param"] * (1 - lr * f["decay"])
                         - size * (m / (torch.sqrt(v) * rbc2 + ADAM_EPS)))
        if eight:
            bits = _bits(c, step, at + g.numel())[at:] if c["stochastic"] else None
            for name, (code, sc) in (("m", _to_m_codes(m, bits)), ("v", _to_v_codes(v, bits))):
                f[name].copy_(code)
                f[name + "_scale"].copy_(sc)
        else:
            f["m"].copy_(m)
            f["v"].copy_(v)
        if "copy" in f:
            f["copy"].copy_(f["param"])
        at += g.numel()
    s["step"] += 1
    return _outputs(s)


def _own_set(backend, s):
    eight, tensors, at = s["case"]["state"] == 8, [], 0
    for f in s["flat"].values():
        gdt = {v: k for k, v in DTYPES.items()}[f["grad"].dtype]
        for b, n in f["tensors"]:
            # The update runs over the whole flat buffers, padding included, as
            # the plain form's does (its encoding gives a padding's states codes
            # above 0, and those change with every step).
            n = -(-n // BLOCK) * BLOCK
            t = {"param": f["param"][b:].data_ptr(), "grad": f["grad"][b:].data_ptr(),
                 "m": f["m"][b:].data_ptr(), "v": f["v"][b:].data_ptr(), "count": n,
                 "grad_dtype": gdt, "weight_decay": f["decay"]}
            if eight:
                t["m_scale"] = f["m_scale"][b // BLOCK:].data_ptr()
                t["v_scale"] = f["v_scale"][b // BLOCK:].data_ptr()
            if "copy" in f:
                t["copy"], t["copy_dtype"] = f["copy"][b:].data_ptr(), "bf16"
            tensors.append(t)
    return backend.AdamWSet(tensors, state_bits=s["case"]["state"])


def _own_adamw(s, stream):
    s["set"].step_device(s["lr"], s["step"], beta1=BETA1, beta2=BETA2, eps=ADAM_EPS,
                         d_sumsq=s["sumsq"].data_ptr(), max_norm=s["max_norm"],
                         stochastic=s["case"]["stochastic"], seed=SEED, stream=stream)
    s["step"] += 1
    return _outputs(s)


def _exact_adamw(s):
    """Weights and 32-bit states; codes depend on each rounding before them."""
    c, step, lr = s["case"], s["step"], s["lr"]
    factor = min(1.0, s["max_norm"] / float(s["sumsq"].sqrt()))
    out = {}
    for kind, f in s["flat"].items():
        if c["state"] == 8:
            m = f["m"].view(torch.float8_e4m3fn).double().view(-1, BLOCK)
            m = (m * f["m_scale"].double()[:, None]).view(-1)
            code = f["v"].long()
            e, low = code >> 3, (code & 7).double()
            v = torch.where(e > 0, (8 + low) * 2.0 ** (e.double() - 18), low * 2.0 ** -17)
            v = (v.view(-1, BLOCK) * f["v_scale"].double()[:, None]).view(-1)
        else:
            m, v = f["m"].double(), f["v"].double()
        g = f["grad"].double() * factor
        m = torch.lerp(g, m, BETA1)
        v = torch.lerp(g * g, v, BETA2)
        p = f["param"].double()
        update = (m / (1 - BETA1 ** step)) / ((v / (1 - BETA2 ** step)).sqrt() + ADAM_EPS)
        p = p - lr * (update + f["decay"] * p)
        out[kind] = {"param": p, "copy": p if "copy" in f else None}
        if c["state"] == 32:
            out[kind].update(m=m, v=v)
        else:
            out[kind].update(m_scale=m.abs().view(-1, BLOCK).amax(1) / 448,
                             v_scale=v.view(-1, BLOCK).amax(1) / 122880)
    return out


# -------------------------------------------------------------------------


def _address(t):
    return None if t is None else t.data_ptr()


def _prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, g)
    return _prepare_norm(case, g) if case["op"].startswith("norm") else _prepare_attend(case, g)


def prepare(case, seed):
    s = _prepare(case, seed)
    if own:
        from metalfish_amd import backend
        if case["op"] == "adamw":
            s["set"] = _own_set(backend, s)
        else:
            if case["op"] == "attend":
                need = backend.attention_forward_workspace_bytes(_own_problem(backend, s))
            elif case["op"] == "attend-back":
                need = backend.attention_backward_workspace_bytes(_own_problem(backend, s))
            else:
                need = backend.layer_norm_workspace_bytes(case["rows"], case["width"])
            s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        from metalfish_amd import backend
        stream = torch.cuda.current_stream().cuda_stream
        if op == "adamw":
            return _own_adamw(state, stream)
        return (_own_norm if op.startswith("norm") else _own_attend)(backend, state, stream)
    if op == "adamw":
        return _plain_adamw(state)
    if op.startswith("norm"):
        return _plain_norm(state)
    return _plain_attend(state) if op == "attend" else _plain_attend_back(state)


def work(case):
    op = case["op"]
    if op == "adamw":
        # Weights and states read and written, gradients read, the copy written.
        total = 0
        for n in _sizes(case):
            big = n >= 4096
            total += n * (8 + (BYTES[case["dtype"]] if big else 4)
                          + (2 if big and case["copy"] else 0)
                          + (16 if case["state"] == 32 else 4 + 16 / BLOCK))
        return {"bytes": total, "flops": 15 * sum(_sizes(case))}
    es = BYTES[case["dtype"]]
    if op.startswith("norm"):
        n, more = case["rows"] * case["width"], 1 if case["residual"] else 0
        if op == "norm":
            return {"bytes": n * es * (2 + more) + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": n * es * (3 + 2 * more) + 8 * case["rows"], "flops": 16 * n}
    b, hq, hk, d = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    rows = [(int(n), int(n)) for n in _lengths(case)] if case["ragged"] \
        else [(case["q_len"], case["k_len"])] * b
    nq, nk = sum(r[0] for r in rows) * hq, sum(r[1] for r in rows) * hk
    biased = b * hq * case["q_len"] * case["k_len"] * es if case["bias"] else 0
    pairs = _pairs(case) * b * hq
    if op == "attend":
        return {"bytes": (2 * nq + 2 * nk) * d * es + 4 * nq + biased, "flops": 4 * d * pairs}
    return {"bytes": (4 * nq + 4 * nk) * d * es + 4 * nq + 2 * biased, "flops": 10 * d * pairs}


def exact(case, seed):
    """From the definitions, in 64 bits, gradients by differentiation."""
    s = _prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    return _exact_norm(s) if case["op"].startswith("norm") else _exact_attend(s)
