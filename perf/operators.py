"""The operators of learning from the network's answers whose speed is measured.

A program that trains a policy on self-play holds the logits of a batch of
positions on the GPU, next to the move lists that the prior softmax reads, and
needs three things there:

* ``policy``: the clipped policy loss of the moves played, with a divergence
  from a reference policy and an entropy term, per position, and its gradient
  with respect to the logits;
* ``preference``: the loss of pairs of lines (one preferred to the other) by
  their log-probability ratios against a reference policy, and its gradient;
* ``clip``: the global norm of all weight gradients, and the gradients scaled
  down to a largest norm.

Logits are rows over a vocabulary (1858 moves for this framework's networks).
With ``moves`` a row's softmax runs over its legal moves alone, as in the
priors call; without, over the whole row.  A row's weight of 0 takes it out; a
position without moves (mate, stalemate) contributes nothing.
"""

import math

import torch

own = False

POLICY = 1858
MAX_MOVES = 60
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CLIP_LOW, CLIP_HIGH = 0.2, 0.25
KL_COEF, ENTROPY_COEF = 0.05, 0.01
BETA, SMOOTHING = 0.1, 0.05
# Most logits of one drawn call, and most gradients.
MOST_LOGITS = 75_000_000
MOST_GRADS = 159_000_000


def _policy(rows, vocab=POLICY, dtype="f32", moves=True, kl=True, temp=1.0, name=None):
    case = {"op": "policy", "rows": rows, "vocab": vocab, "dtype": dtype, "moves": moves, "kl": kl,
            "temp": temp}
    return case if name is None else {"name": name, **case}


def _preference(pairs, plies, vocab=POLICY, dtype="f32", moves=True, name=None):
    case = {"op": "preference", "pairs": pairs, "plies": plies, "vocab": vocab, "dtype": dtype,
            "moves": moves}
    return case if name is None else {"name": name, **case}


def _clip(width, layers, ffn, dtype="f32", smolgen=True, max_norm=1.0, name=None):
    case = {"op": "clip", "width": width, "layers": layers, "ffn": ffn, "dtype": dtype,
            "smolgen": smolgen, "max_norm": max_norm}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # One game's last positions, as they come in: latency.
        _policy(16, name="policy-16"),
        # An ordinary step of a self-play learner.
        _policy(1024, name="policy-1024"),
        # A large odd batch under mixed precision, no reference policy, a
        # warmer softmax.
        _policy(20011, dtype="bf16", kl=False, temp=1.5, name="policy-20011-bf16"),
        # The whole vocabulary of moves (an unmasked policy), with a reference.
        _policy(4099, moves=False, name="policy-4099-whole"),
        # A long odd vocabulary of tokens.
        _policy(1500, vocab=50021, dtype="bf16", moves=False, name="policy-1500-long-bf16"),
        # Six positions, a better and a worse move each: latency.
        _preference(6, 1, name="preference-6-moves"),
        # Pairs of lines of up to 60 plies.
        _preference(128, 60, name="preference-128-lines"),
        # Pairs of texts over a token vocabulary.
        _preference(16, 200, vocab=32000, dtype="bf16", moves=False,
                    name="preference-16-texts-bf16"),
        # The gradients of the small network of tests.
        _clip(256, 2, 512, smolgen=False, name="clip-small"),
        # A middle network trained in fp16 with scaled losses.
        _clip(512, 8, 768, dtype="f16", name="clip-middle-f16"),
        # The benchmark's network, bf16 matrices.
        _clip(1024, 15, 1536, dtype="bf16", name="clip-large-bf16"),
        # The same in 32 bits.
        _clip(1024, 15, 1536, name="clip-large"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("policy", "policy", "preference", "clip"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "clip":
        width = 64 * rng.randint(1, 16)
        ffn = 32 * rng.randint(2, max(2, 3 * width // 64))
        smolgen = rng.random() < 0.5
        layers = rng.randint(1, 15)
        case = _clip(width, layers, ffn, dtype, smolgen, rng.choice((0.5, 1.0, 1e9)))
        while sum(_sizes(case)) > MOST_GRADS:
            case["layers"] -= 1
        return case
    moves = rng.random() < 0.6
    vocab = POLICY if moves or rng.random() < 0.3 else _spread(rng, 33, 60000)
    most = min(20000, MOST_LOGITS // vocab)
    if op == "policy":
        return _policy(_spread(rng, 1, most), vocab, dtype, moves, rng.random() < 0.6,
                       rng.choice((1.0, 1.0, 0.7, 2.2)))
    plies = _spread(rng, 1, 200)
    return _preference(_spread(rng, 1, max(1, most // (2 * plies))), plies, vocab, dtype, moves)


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


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _move_lists(rows, vocab, g):
    """Legal moves of each row: int32 offsets [rows + 1], int16 indices, and
    how many each row has.  One position in fifty is over and has none."""
    dev = "cuda"
    n = (32 + 9 * torch.randn(rows, device=dev, generator=g)).round().long().clamp(1, MAX_MOVES)
    n[torch.rand(rows, device=dev, generator=g) < 0.02] = 0
    order = torch.rand(rows, vocab, device=dev, generator=g).topk(MAX_MOVES, dim=1).indices
    keep = torch.arange(MAX_MOVES, device=dev) < n[:, None]
    offsets = torch.zeros(rows + 1, dtype=torch.int32, device=dev)
    offsets[1:] = n.cumsum(0)
    return offsets, order[keep].to(torch.int16), n


def _rows(case, rows, g):
    """Logits, move lists and the moves played (policy indices, -1 where a
    position has none)."""
    dev, vocab = "cuda", case["vocab"]
    x = (2 * torch.randn(rows, vocab, device=dev, generator=g)).to(DTYPES[case["dtype"]])
    s = {"case": case, "rows": rows, "vocab": vocab, "temp": case.get("temp", 1.0), "logits": x,
         "offsets": None, "indices": None, "max_moves": 0}
    if case["moves"]:
        s["offsets"], s["indices"], n = _move_lists(rows, vocab, g)
        s["max_moves"] = MAX_MOVES
        pick = (torch.rand(rows, device=dev, generator=g) * n).long()
        at = (s["offsets"][:-1] + pick).clamp(max=max(0, s["indices"].numel() - 1))
        a = s["indices"][at].int() if s["indices"].numel() else torch.zeros(rows, device=dev).int()
        s["actions"] = torch.where(n > 0, a, -1)
    else:
        s["actions"] = torch.randint(0, vocab, (rows,), device=dev, generator=g).int()
    return s


def _log_probs(s):
    """Log-probabilities in 64 bits of the moves played (0 where none), for
    inputs that come from an earlier state of the policy."""
    out = torch.zeros(s["rows"], dtype=torch.float64, device="cuda")
    step = max(1, 40_000_000 // s["vocab"])
    for b in range(0, s["rows"], step):
        e = min(s["rows"], b + step)
        x = s["logits"][b:e].double() / s["temp"]
        if s["offsets"] is not None:
            x = x.masked_fill(~_allowed(s, b, e), -math.inf)
        a = s["actions"][b:e].long()
        lp = x.gather(1, a.clamp(min=0)[:, None])[:, 0] - x.logsumexp(1)
        out[b:e] = torch.where(a >= 0, lp, 0.0)
    return out


def _allowed(s, b, e):
    """Which of rows b to e's columns are legal moves."""
    off = s["offsets"][b:e + 1].long()
    row = torch.repeat_interleave(torch.arange(e - b, device="cuda"), off[1:] - off[:-1])
    ok = torch.zeros(e - b, s["vocab"], dtype=torch.bool, device="cuda")
    ok[row, s["indices"][off[0]:off[-1]].long()] = True
    return ok


def _prepare_policy(case, g):
    rows, dev = case["rows"], "cuda"
    s = _rows(case, rows, g)
    # The policy has moved a little since the moves were played; no ratio sits
    # on a border of the clip, where the gradient jumps.
    move = 0.2 * torch.randn(rows, device=dev, generator=g, dtype=torch.float64)
    for border in (math.log1p(-CLIP_LOW), math.log1p(CLIP_HIGH)):
        near = (move - border).abs() < 1e-3
        move[near] = border + 2e-3
    s["old_logp"] = (_log_probs(s) - move).float()
    s["advantage"] = torch.randn(rows, device=dev, generator=g)
    weight = 0.5 + torch.rand(rows, device=dev, generator=g)
    weight[torch.rand(rows, device=dev, generator=g) < 0.05] = 0.0
    s["weight"] = weight
    s["ref"] = None
    if case["kl"]:
        noise = 0.3 * torch.randn(rows, s["vocab"], device=dev, generator=g)
        s["ref"] = (s["logits"].float() + noise).to(s["logits"].dtype)
    s["out"] = {k: torch.empty(rows, device=dev) for k in ("loss", "logp", "entropy")}
    if case["kl"]:
        s["out"]["kl"] = torch.empty(rows, device=dev)
    s["out"]["grad"] = torch.empty_like(s["logits"])
    return s


def _lengths(case):
    """Plies of each line; a case's own, so that its shapes are."""
    r = torch.Generator().manual_seed(1000 * case["pairs"] + case["plies"])
    return torch.randint(1, case["plies"] + 1, (2 * case["pairs"],), generator=r)


def _prepare_preference(case, g):
    pairs, dev, n = case["pairs"], "cuda", _lengths(case)
    offsets = torch.zeros(2 * pairs + 1, dtype=torch.int32)
    offsets[1:] = n.cumsum(0)
    rows = int(offsets[-1])
    s = _rows(case, rows, g)
    s["pairs"] = pairs
    s["seq_offsets"] = offsets.to(dev)
    # What leads up to a line (a prompt) is not judged.
    s["actions"][torch.rand(rows, device=dev, generator=g) < 0.1] = -1
    drift = 0.3 * torch.randn(rows, device=dev, generator=g)
    s["ref_logp"] = (_log_probs(s) + drift).float()
    s["weight"] = 0.5 + torch.rand(pairs, device=dev, generator=g)
    s["out"] = {"loss": torch.empty(pairs, device=dev), "margin": torch.empty(pairs, device=dev),
                "logp": torch.empty(rows, device=dev), "grad": torch.empty_like(s["logits"])}
    return s


def _prepare_clip(case, g):
    dev, sizes = "cuda", _sizes(case)
    # Matrices in the case's type, vectors in 32 bits; each kind in one flat
    # buffer, as trainers keep them.
    low = case["dtype"]
    kinds = [low if n >= 4096 else "f32" for n in sizes]
    s = {"case": case, "src": {}, "dst": {}, "tensors": [], "max_norm": case["max_norm"]}
    for kind in sorted(set(kinds)):
        total = sum(n for n, k in zip(sizes, kinds) if k == kind)
        s["src"][kind] = torch.randn(total, device=dev, generator=g).to(DTYPES[kind])
        s["dst"][kind] = torch.empty_like(s["src"][kind])
    at = {kind: 0 for kind in s["src"]}
    scales = torch.rand(len(sizes), generator=torch.Generator().manual_seed(int(g.initial_seed())))
    for n, kind, u in zip(sizes, kinds, scales.tolist()):
        src = s["src"][kind][at[kind]:at[kind] + n]
        src *= 0.02 * 4.0 ** u
        s["tensors"].append((src, s["dst"][kind][at[kind]:at[kind] + n], kind))
        at[kind] += n
    s["norm"] = torch.empty(1, device=dev)
    return s


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "policy":
        s = _prepare_policy(case, g)
    elif case["op"] == "preference":
        s = _prepare_preference(case, g)
    else:
        s = _prepare_clip(case, g)
    if own:
        from metalfish_amd import backend
        if case["op"] == "clip":
            s["set"] = backend.GradSet([(a.data_ptr(), b.data_ptr(), a.numel(), kind)
                                        for a, b, kind in s["tensors"]])
            need = s["set"].workspace_bytes
        elif case["op"] == "preference":
            need = backend.preference_loss_workspace_bytes(s["rows"])
        else:
            need = 0
        s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return s


def _address(t):
    return None if t is None else t.data_ptr()


def _own_rows(backend, s):
    return backend.policy_rows(
        s["logits"].data_ptr(), s["rows"], s["vocab"], dtype=s["case"]["dtype"],
        d_move_offsets=_address(s["offsets"]), d_move_indices=_address(s["indices"]),
        n_moves=0 if s["indices"] is None else s["indices"].numel(),
        d_actions=s["actions"].data_ptr(), softmax_temp=s["temp"])


def _own_run(s):
    from metalfish_amd import backend
    stream = torch.cuda.current_stream().cuda_stream
    op = s["case"]["op"]
    if op == "clip":
        s["set"].clip_device(s["max_norm"], s["norm"].data_ptr(), s["workspace"].data_ptr(),
                             s["workspace"].numel(), stream=stream)
        return {"norm": s["norm"], "grads": s["dst"]}
    out = s["out"]
    if op == "policy":
        backend.policy_loss_device(
            _own_rows(backend, s), d_old_logp=s["old_logp"].data_ptr(),
            d_advantage=s["advantage"].data_ptr(), d_weight=s["weight"].data_ptr(),
            d_ref_logits=_address(s["ref"]), clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
            kl_coef=KL_COEF if s["ref"] is not None else 0.0, entropy_coef=ENTROPY_COEF,
            d_loss=out["loss"].data_ptr(), d_logp=out["logp"].data_ptr(),
            d_kl=_address(out.get("kl")), d_entropy=out["entropy"].data_ptr(),
            d_grad=out["grad"].data_ptr(), stream=stream)
        return out
    backend.preference_loss_device(
        _own_rows(backend, s), s["pairs"], s["seq_offsets"].data_ptr(), kind="sigmoid", beta=BETA,
        label_smoothing=SMOOTHING, d_ref_logp=s["ref_logp"].data_ptr(),
        d_weight=s["weight"].data_ptr(), d_loss=out["loss"].data_ptr(),
        d_margin=out["margin"].data_ptr(), d_logp=out["logp"].data_ptr(),
        d_grad=out["grad"].data_ptr(), d_workspace=s["workspace"].data_ptr(),
        workspace_bytes=s["workspace"].numel(), stream=stream)
    return out


def _entries(s):
    """Each row's softmax entries: logits in 32 bits, their columns (None:
    all), which of them count, and which is the move played."""
    a = s["actions"].long()[:, None]
    if s["offsets"] is None:
        x = s["logits"].float()
        return x, None, None, torch.arange(s["vocab"], device="cuda") == a
    off = s["offsets"].long()
    j = torch.arange(s["max_moves"], device="cuda")
    ok = j < (off[1:] - off[:-1])[:, None]
    at = torch.where(ok, off[:-1, None] + j, 0)
    k = torch.where(ok, s["indices"][at].long(), 0)
    x = s["logits"].gather(1, k).float()
    return x, k, ok, (k == a) & ok


def _softmax(x, ok, temp):
    """z = (x - max) / temperature, ln sum exp z, and the probabilities; zeros where a row has
    no entry."""
    if ok is not None:
        x = torch.where(ok, x, -math.inf)
    m = x.amax(1, keepdim=True)
    z = (x - torch.where(m == -math.inf, 0.0, m)) / temp
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    total = torch.where(total == 0, 1.0, total)
    z = z if ok is None else torch.where(ok, z, 0.0)
    return z, torch.log(total)[:, 0], e / total


def _spread_out(s, g, k, ok):
    """A gradient of the entries as a gradient of the whole logits, rounded
    once."""
    if k is not None:
        whole = torch.zeros(s["rows"], s["vocab"], device="cuda")
        g = whole.scatter_add_(1, k, torch.where(ok, g, 0.0))
    return g.to(s["logits"].dtype)


def _plain_policy(s):
    x, k, ok, played = _entries(s)
    z, log_sum, p = _softmax(x, ok, s["temp"])
    acted = played.any(1)
    logp = torch.where(acted, torch.where(played, z, 0.0).sum(1) - log_sum, 0.0)
    ratio = torch.exp(logp - s["old_logp"])
    adv = torch.where(acted, s["advantage"], 0.0)
    plain, clipped = ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
    loss = -torch.minimum(plain, clipped)
    g = torch.where(plain <= clipped, -plain, 0.0)
    grad = g[:, None] * (played.float() - p)
    mean_z = (p * z).sum(1)
    entropy = log_sum - mean_z
    loss = loss - ENTROPY_COEF * entropy
    grad += ENTROPY_COEF * p * (z - mean_z[:, None])
    live = s["weight"] != 0
    out = {"logp": torch.where(live, logp, 0.0), "entropy": torch.where(live, entropy, 0.0)}
    if s["ref"] is not None:
        y = s["ref"] if k is None else s["ref"].gather(1, k)
        d = (x - y.float()) / s["temp"]
        u = d - (p * d).sum(1, keepdim=True)
        # ln E_p exp(-u) with E_p u = 0: no two nearly equal terms cancel.
        kl = torch.log1p((p * (torch.expm1(-u) + u)).sum(1))
        loss = loss + KL_COEF * kl
        grad += KL_COEF * p * u
        out["kl"] = torch.where(live, kl, 0.0)
    out["loss"] = torch.where(live, s["weight"] * loss, 0.0)
    out["grad"] = _spread_out(s, (s["weight"] / s["temp"])[:, None] * grad, k, ok)
    return out


def _plain_preference(s):
    x, k, ok, played = _entries(s)
    z, log_sum, p = _softmax(x, ok, s["temp"])
    acted = played.any(1)
    logp = torch.where(acted, torch.where(played, z, 0.0).sum(1) - log_sum, 0.0)
    ratio = torch.where(acted, logp.double() - s["ref_logp"].double(), 0.0)
    run = torch.cat([ratio.new_zeros(1), ratio.cumsum(0)])[s["seq_offsets"].long()]
    total = (run[1:] - run[:-1]).view(-1, 2)
    h = BETA * (total[:, 0] - total[:, 1])
    softplus = lambda v: torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    loss = s["weight"] * ((1 - SMOOTHING) * softplus(-h) + SMOOTHING * softplus(h))
    sig = 1 / (1 + torch.exp(-h))
    c = s["weight"] * BETA * (sig - (1 - SMOOTHING))
    seq = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["seq_offsets"][1:].long(), seq, right=True)
    c = torch.stack([c, -c], 1).reshape(-1)[seq].float()
    c = torch.where(acted, c, 0.0)[:, None] / s["temp"]
    return {"loss": loss.float(), "margin": h.float(), "logp": logp,
            "grad": _spread_out(s, c * (played.float() - p), k, ok)}


def _plain_clip(s):
    # On the flat buffers: a few passes, whatever the number of tensors.
    total = sum(v.float().square().sum(dtype=torch.float64) for v in s["src"].values())
    norm = total.sqrt().reshape(1)
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0).float()
    return {"norm": norm.float(), "grads": {k: (v.float() * scale).to(v.dtype)
                                            for k, v in s["src"].items()}}


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    if op == "policy":
        return _plain_policy(state)
    return _plain_preference(state) if op == "preference" else _plain_clip(state)


def work(case):
    if case["op"] == "clip":
        # Every gradient read once and written once.
        sizes = _sizes(case)
        moved = sum(n * (BYTES[case["dtype"]] if n >= 4096 else 4) for n in sizes)
        return {"bytes": 2 * moved, "flops": 3 * sum(sizes)}
    es, vocab = BYTES[case["dtype"]], case["vocab"]
    if case["op"] == "policy":
        rows, read, flops = case["rows"], 2 if case["kl"] else 1, 20 if case["kl"] else 12
    else:
        rows, read, flops = int(_lengths(case).sum()), 1, 6
    if case["moves"]:
        # About 32 moves a row: index and logits read; the whole gradient row
        # written.
        entries = 32 * rows
        return {"bytes": rows * (vocab * es + 36) + entries * (2 + read * es),
                "flops": entries * flops}
    return {"bytes": rows * (vocab * es * (read + 1) + 32), "flops": rows * vocab * flops}


def _masked_log_softmax(s, x):
    """log_softmax in 64 bits over the legal moves, -inf elsewhere, 0 in rows
    that have none."""
    if s["offsets"] is None:
        return torch.log_softmax(x / s["temp"], 1), None
    ok = _allowed(s, 0, s["rows"])
    none = ~ok.any(1, keepdim=True)
    lp = torch.log_softmax((x / s["temp"]).masked_fill(~(ok | none), -math.inf), 1)
    return lp.masked_fill(~ok, 0.0), ok


def exact(case, seed):
    """From the definitions, in 64 bits, gradients by differentiation."""
    g = _generator(seed)
    if case["op"] == "clip":
        s = _prepare_clip(case, g)
        norm = torch.linalg.vector_norm(
            torch.stack([torch.linalg.vector_norm(a.double()) for a, _, _ in s["tensors"]]))
        scale = min(1.0, case["max_norm"] / float(norm))
        return {"norm": norm.reshape(1), "grads": {k: v.double() * scale
                                                   for k, v in s["src"].items()}}
    s = _prepare_policy(case, g) if case["op"] == "policy" else _prepare_preference(case, g)
    x = s["logits"].double().requires_grad_()
    lp, ok = _masked_log_softmax(s, x)
    a = s["actions"].long()
    logp = torch.where(a >= 0, lp.gather(1, a.clamp(min=0)[:, None])[:, 0], 0.0)
    if case["op"] == "preference":
        w = s["weight"].double()
        r = torch.where(a >= 0, logp - s["ref_logp"].double(), 0.0)
        bounds = s["seq_offsets"].tolist()
        totals = torch.stack([r[b:e].sum() for b, e in zip(bounds, bounds[1:])]).view(-1, 2)
        h = BETA * (totals[:, 0] - totals[:, 1])
        sig = torch.nn.functional.logsigmoid
        loss = -w * ((1 - SMOOTHING) * sig(h) + SMOOTHING * sig(-h))
        grad, = torch.autograd.grad(loss.sum(), x)
        return {"loss": loss.detach(), "margin": h.detach(), "logp": logp.detach(), "grad": grad}
    w = s["weight"].double()
    p = lp.exp() if ok is None else torch.where(ok, lp.exp(), 0.0)
    ratio, adv = torch.exp(logp - s["old_logp"].double()), s["advantage"].double()
    gain = torch.minimum(ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
    entropy = -(p * lp).sum(1)
    loss = torch.where(a >= 0, -gain, 0.0) - ENTROPY_COEF * entropy
    out = {"logp": logp, "entropy": entropy}
    if s["ref"] is not None:
        lq, _ = _masked_log_softmax(s, s["ref"].double())
        out["kl"] = (p * (lp - lq)).sum(1)
        loss = loss + KL_COEF * out["kl"]
    grad, = torch.autograd.grad((w * loss).sum(), x)
    out = {k: torch.where(w != 0, v, 0.0).detach() for k, v in out.items()}
    return {**out, "loss": (w * loss).detach(), "grad": grad}
