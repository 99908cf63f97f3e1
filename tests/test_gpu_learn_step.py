"""The losses and the clipping as a learner uses them: on a net's own logits
and move lists, together, captured into a graph, from two threads."""

import threading

import numpy as np
import pytest

import gpu_util
import learn_gpu as lg
import loss_util as lu
from metalfish_amd import backend, synth
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


def test_a_learning_step_on_a_nets_answers(dev):
    """Self-play's data flow: the net's logits and priors from
    mfh_net_eval_priors_device, then both losses on the same device arrays,
    a step of a per-move bias and a temperature scale fitted on top of the net
    (gradients of logits * s + b), clipped together.  Every stage against the
    64-bit oracle on the logits that the net gave."""
    n = 24
    spec = synth.SPECS["cpu_plumbing"]
    net = backend.create_network(spec, synth.make_weights(spec, seed=0), max_batch=n, device=0)
    planes, legal = synth.playout_positions(n, seed=5)
    masks, values = backend.pack_planes(planes)
    moves = [[int(k) for k in m if k >= 0] for m in legal]
    off, idx = lu.move_lists(moves)
    d_off, d_idx = dev.put(off), dev.put(idx)
    logits, priors = lg.Padded(dev, np.zeros((n, 1858), np.float32), "f32"), lg.Column(dev, idx.size)
    stream = dev.stream()
    net.eval_priors_device(n, dev.put(masks), dev.put(values), d_off, d_idx, 1.0, logits.ptr,
                           priors.ptr, dev.put(np.zeros((n, 3), np.float32)), stream)
    rng = np.random.default_rng(1)
    actions = np.array([m[int(rng.integers(len(m)))] if m else -1 for m in moves], np.int32)
    adv = rng.normal(size=n).astype(np.float32)
    rows = backend.policy_rows(logits.ptr, n, 1858, d_move_offsets=d_off, d_move_indices=d_idx,
                               n_moves=idx.size, d_actions=dev.put(actions))
    logp, loss = lg.Column(dev, n), lg.Column(dev, n)
    grad = lg.Padded(dev, np.zeros((n, 1858), np.float32), "f32")
    backend.policy_loss_device(rows, d_advantage=dev.put(adv), entropy_coef=0.02, d_loss=loss.ptr,
                               d_logp=logp.ptr, d_grad=grad.ptr, stream=stream)
    # Halves of the positions as lines: the first better than the second.
    seq = [0, n // 4, n // 2, n // 2 + n // 4, n]
    pref_grad = lg.Padded(dev, np.zeros((n, 1858), np.float32), "f32")
    need = backend.preference_loss_workspace_bytes(n)
    margin = lg.Column(dev, 2)
    backend.preference_loss_device(rows, 2, dev.put(np.array(seq, np.int32)), beta=0.2,
                                   d_ref_logp=logp.ptr, d_margin=margin.ptr, d_grad=pref_grad.ptr,
                                   d_workspace=dev.alloc(need), workspace_bytes=need,
                                   stream=stream)
    dev.sync(stream)
    x = logits.get().astype(np.float64)
    pr = priors.get()
    assert np.all(np.isfinite(pr))
    want = losses.policy_loss(x, moves, actions, advantage=adv, entropy_coef=0.02)
    assert np.all(want["logp"] <= 0)
    # 2^-24 times the roundings of loss_util for rows of 60 moves at most and
    # |z| below 20: 5 * 20 * 2 + 40 below 256.
    np.testing.assert_allclose(logp.get(), want["logp"], rtol=0, atol=256 * lu.U * 4)
    np.testing.assert_allclose(loss.get(), want["loss"], rtol=0, atol=256 * lu.U * 8)
    g = grad.get().astype(np.float64)
    np.testing.assert_allclose(g, want["grad"], rtol=0, atol=256 * lu.U * 8)
    # The reference is the policy itself: margin 0, the gradient at ln 2.
    got_margin = margin.get()
    assert np.all(np.abs(got_margin) < 1e-5)
    wantp = losses.preference_loss(x, moves, actions, seq, beta=0.2, ref_logp=want["logp"])
    gp = pref_grad.get().astype(np.float64)
    np.testing.assert_allclose(gp, wantp["grad"], rtol=0, atol=256 * lu.U * 8)
    # Gradients of the bias and the scale, clipped together in place.
    total = g + gp
    gb, gs = total.sum(0).astype(np.float32), np.array([(total * x).sum()], np.float32)
    d_b, d_s = dev.put(gb), dev.put(gs)
    grads = backend.GradSet([(d_b, d_b, gb.size, "f32"), (d_s, d_s, 1, "f32")])
    norm = lg.Column(dev, 1)
    grads.clip_device(0.25, norm.ptr, dev.alloc(grads.workspace_bytes), grads.workspace_bytes,
                      stream=stream)
    dev.sync(stream)
    want_norm, clipped = losses.clip([gb, gs], 0.25)
    assert abs(norm.get()[0] - want_norm) <= 2 ** -23 * want_norm
    for p, w in ((d_b, clipped[0]), (d_s, clipped[1])):
        lu.close(dev.get(p, w.astype(np.float32)), w, 3 * lu.U * np.abs(w))
    net.close()


def _setup(dev, rng, rows=96, vocab=1858, dtype="bf16"):
    moves = [sorted(rng.choice(vocab, size=int(rng.integers(1, 50)), replace=False))
             for _ in range(rows)]
    moves[3] = []
    actions = np.array([int(m[0]) if m else -1 for m in moves], np.int32)
    x = lu.to_bits(rng.normal(size=(rows, vocab)) * 2, dtype)
    y = lu.to_bits(lu.from_bits(x, dtype) + 0.3 * rng.normal(size=(rows, vocab)), dtype)
    off, idx = lu.move_lists(moves)
    d = dict(x=dev.put(x), y=dev.put(y), adv=dev.put(rng.normal(size=rows).astype(np.float32)),
             seq=dev.put(np.arange(0, rows + 1, rows // 4).astype(np.int32)),
             loss=dev.put(np.zeros(rows, np.float32)), kl=dev.put(np.zeros(rows, np.float32)),
             g=dev.put(np.zeros_like(x)), g2=dev.put(np.zeros_like(x)),
             margin=dev.put(np.zeros(2, np.float32)), norm=dev.put(np.zeros(1, np.float32)),
             out=dev.put(np.zeros_like(x)))
    d["rows"] = backend.policy_rows(d["x"], rows, vocab, dtype=dtype, d_move_offsets=dev.put(off),
                                    d_move_indices=dev.put(idx), n_moves=idx.size,
                                    d_actions=dev.put(actions))
    d["need"] = backend.preference_loss_workspace_bytes(rows)
    d["ws"] = dev.alloc(d["need"])
    d["set"] = backend.GradSet([(d["g"], d["out"], x.size // 2, dtype),
                                (d["g2"], d["out"] + 2 * (x.size // 2), x.size // 2, dtype)])
    d["cws"] = dev.alloc(d["set"].workspace_bytes)
    d["host"] = x
    return d


def _step(d, stream):
    backend.policy_loss_device(d["rows"], d_advantage=d["adv"], d_ref_logits=d["y"], kl_coef=0.1,
                               entropy_coef=0.01, d_loss=d["loss"], d_kl=d["kl"], d_grad=d["g"],
                               stream=stream)
    backend.preference_loss_device(d["rows"], 2, d["seq"], d_margin=d["margin"], d_grad=d["g2"],
                                   d_workspace=d["ws"], workspace_bytes=d["need"], stream=stream)
    d["set"].clip_device(0.05, d["norm"], d["cws"], d["set"].workspace_bytes, stream=stream)


def _outputs(dev, d):
    n = np.zeros(d["rows"].rows, np.float32)
    return [dev.get(d["loss"], n), dev.get(d["kl"], n), dev.get(d["margin"], n[:2]),
            dev.get(d["norm"], n[:1]), dev.get(d["g"], d["host"]), dev.get(d["g2"], d["host"]),
            dev.get(d["out"], d["host"])]


def test_a_captured_step_replays_on_new_inputs(dev):
    rng = np.random.default_rng(2)
    d = _setup(dev, rng)
    stream = dev.stream()
    launch = dev.capture(stream, lambda: _step(d, stream))
    for _ in range(4):
        dev.write(d["x"], lu.to_bits(rng.normal(size=d["host"].shape) * 2, "bf16"))
        launch()
        dev.sync(stream)
        got = _outputs(dev, d)
        for p in ("g", "g2", "out"):
            dev.write(d[p], np.full_like(d["host"], 0x4242))
        _step(d, None)
        dev.sync()
        want = _outputs(dev, d)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        assert np.any(want[6] != 0) and want[3][0] > 0.05


def test_two_threads_on_streams_of_their_own(dev):
    rng = np.random.default_rng(3)
    sides = [_setup(dev, rng), _setup(dev, rng)]
    want = []
    for d in sides:
        _step(d, None)
        dev.sync()
        want.append(_outputs(dev, d))
    streams = [dev.stream(), dev.stream()]
    errors = []

    def work(d, s):
        try:
            for _ in range(20):
                _step(d, s)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(sides, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    dev.sync()
    assert not errors
    for d, w in zip(sides, want):
        assert all(np.array_equal(a, b) for a, b in zip(_outputs(dev, d), w))
