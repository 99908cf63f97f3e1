"""Entry points of the losses and the gradient clipping without a device:
what they refuse, before any device is touched, and what is nothing to do."""

import ctypes

import numpy as np
import pytest

from metalfish_amd import backend

A = 1 << 20  # stands for an address; nothing here is dereferenced


def _rows(**kw):
    d = dict(d_logits=A, rows=4, vocab=10, d_actions=A)
    d.update(kw)
    return backend.policy_rows(d.pop("d_logits"), d.pop("rows"), d.pop("vocab"), **d)


def _set(rows, **kw):
    for k, v in kw.items():
        setattr(rows, k, v)
    return rows


LISTS = dict(d_move_offsets=A, d_move_indices=A, n_moves=8)
BAD_ROWS = {
    "rows": lambda: _rows(rows=-1),
    "vocab": lambda: _rows(vocab=0, stride=4),
    "vocab-large": lambda: _rows(vocab=(1 << 30) + 1),
    "dtype": lambda: _set(_rows(), dtype=3),
    "dtype-negative": lambda: _set(_rows(), dtype=-1),
    "temperature": lambda: _rows(softmax_temp=0.0),
    "temperature-negative": lambda: _rows(softmax_temp=-1.0),
    "temperature-nan": lambda: _rows(softmax_temp=float("nan")),
    "temperature-infinite": lambda: _rows(softmax_temp=float("inf")),
    "temperature-tiny": lambda: _rows(softmax_temp=1e-40),
    "device": lambda: _rows(device=-2),
    "stride": lambda: _rows(stride=9),
    "stride-overflow": lambda: _rows(stride=1 << 61),
    "moves-negative": lambda: _rows(**dict(LISTS, n_moves=-1)),
    "moves-many": lambda: _rows(**dict(LISTS, n_moves=1 << 31)),
    "indices-alone": lambda: _rows(d_move_indices=A),
    "offsets-alone": lambda: _rows(**dict(LISTS, d_move_indices=None)),
    "lists-vocab": lambda: _rows(vocab=32769, **LISTS),
    "null-logits": lambda: _rows(d_logits=None),
    "logits-alignment": lambda: _rows(d_logits=A + 2),
    "half-alignment": lambda: _rows(d_logits=A + 1, dtype="bf16"),
    "offsets-alignment": lambda: _rows(**dict(LISTS, d_move_offsets=A + 2)),
    "indices-alignment": lambda: _rows(**dict(LISTS, d_move_indices=A + 1)),
    "actions-alignment": lambda: _rows(d_actions=A + 1),
}
BAD_POLICY = {
    "clip-low": dict(clip_low=-0.1), "clip-high": dict(clip_high=-0.1),
    "clip-nan": dict(clip_low=float("nan")),
    "kl-infinite": dict(kl_coef=float("inf"), d_ref_logits=A),
    "entropy-nan": dict(entropy_coef=float("nan")),
    "kl-without-reference": dict(kl_coef=0.1), "kl-output-without-reference": dict(d_kl=A),
    "ref-stride": dict(d_ref_logits=A, ref_stride=9),
    "ref-stride-overflow": dict(d_ref_logits=A, ref_stride=1 << 61),
    "ref-alignment": dict(d_ref_logits=A + 2), "old-alignment": dict(d_old_logp=A + 2),
    "advantage-alignment": dict(d_advantage=A + 2), "weight-alignment": dict(d_weight=A + 2),
    "loss-alignment": dict(d_loss=A + 2), "logp-alignment": dict(d_logp=A + 1),
    "kl-alignment": dict(d_ref_logits=A, d_kl=A + 3), "entropy-alignment": dict(d_entropy=A + 2),
    "grad-alignment": dict(d_grad=A + 4096 + 2), "grad-stride": dict(d_grad=A + 4096, grad_stride=9),
    "grad-stride-overflow": dict(d_grad=A + 4096, grad_stride=1 << 61),
    "grad-in-logits": dict(d_grad=A + 4), "grad-behind-in-logits": dict(d_grad=A - 4),
    "grad-other-stride": dict(d_grad=A, grad_stride=11),
    "grad-in-reference": dict(d_grad=A + 8192 + 40, d_ref_logits=A + 8192),
}
BAD_PREFERENCE = {
    "pairs": dict(pairs=-1), "pairs-many": dict(pairs=(1 << 23) + 1),
    "offsets": dict(d_seq_offsets=None), "offsets-alignment": dict(d_seq_offsets=A + 2),
    "beta": dict(beta=0.0), "beta-nan": dict(beta=float("nan")),
    "beta-infinite": dict(beta=float("inf")),
    "smoothing": dict(label_smoothing=0.6), "smoothing-negative": dict(label_smoothing=-0.1),
    "smoothing-hinge": dict(kind="hinge", label_smoothing=0.1),
    "ref-alignment": dict(d_ref_logp=A + 1), "weight-alignment": dict(d_weight=A + 2),
    "loss-alignment": dict(d_loss=A + 2), "margin-alignment": dict(d_margin=A + 2),
    "logp-alignment": dict(d_logp=A + 2), "grad-alignment": dict(d_grad=A + 4098),
    "grad-stride": dict(d_grad=A + 4096, grad_stride=9), "grad-in-logits": dict(d_grad=A + 40),
    "workspace": dict(d_workspace=None), "workspace-alignment": dict(d_workspace=A + 4),
    "workspace-small": dict(workspace_bytes=31),
}


def _invalid(call):
    with pytest.raises(RuntimeError, match=r"failed \(-1\): mfh_"):
        call()


def _preference(rows, **kw):
    d = dict(pairs=2, d_seq_offsets=A, d_workspace=A, workspace_bytes=1 << 12)
    d.update(kw)
    backend.preference_loss_device(rows, d.pop("pairs"), d.pop("d_seq_offsets"), **d)


@pytest.mark.parametrize("name", BAD_ROWS)
def test_bad_rows_are_refused(name):
    _invalid(lambda: backend.policy_loss_device(BAD_ROWS[name](), d_loss=A))
    _invalid(lambda: _preference(BAD_ROWS[name]()))


@pytest.mark.parametrize("name", BAD_POLICY)
def test_bad_policy_losses_are_refused(name):
    _invalid(lambda: backend.policy_loss_device(_rows(), **BAD_POLICY[name]))


@pytest.mark.parametrize("name", BAD_PREFERENCE)
def test_bad_preference_losses_are_refused(name):
    _invalid(lambda: _preference(_rows(), **BAD_PREFERENCE[name]))


def test_null_structs_and_bad_enums_are_refused():
    L = backend.lib()
    r, p, q = _rows(), backend.MfhPolicyLoss(), backend.MfhPreferenceLoss()
    assert L.mfh_policy_loss_device(None, ctypes.addressof(p), None) == -1
    assert L.mfh_policy_loss_device(ctypes.addressof(r), None, None) == -1
    assert L.mfh_preference_loss_device(None, ctypes.addressof(q), None) == -1
    assert L.mfh_preference_loss_device(ctypes.addressof(r), None, None) == -1
    for field, bad in (("kind", 3), ("kind", -1), ("average", 2)):
        q = backend.MfhPreferenceLoss(A, 1, None, None, 0, 0, 1.0, 0.0, A, None, None, None, 10, A,
                                      4096)
        setattr(q, field, bad)
        assert L.mfh_preference_loss_device(ctypes.addressof(r), ctypes.addressof(q), None) == -1
    n = ctypes.c_uint64(0)
    assert L.mfh_preference_loss_workspace_bytes(-1, ctypes.byref(n)) == -1
    assert L.mfh_preference_loss_workspace_bytes(5, None) == -1
    assert backend.preference_loss_workspace_bytes(5) == 40


def test_nothing_to_do_succeeds():
    backend.policy_loss_device(_rows(rows=0, d_logits=None, d_actions=None))
    _preference(_rows(), pairs=0, d_seq_offsets=None)
    _preference(_rows(rows=0, d_logits=None), pairs=0, d_seq_offsets=None, d_workspace=None,
                workspace_bytes=0)


@pytest.mark.skipif(backend.device_count() > 0, reason="a device is here")
def test_without_a_device_calls_say_so():
    with pytest.raises(RuntimeError, match=r"failed \(-4\): .*no HIP device"):
        backend.policy_loss_device(_rows(), d_loss=A)
    with pytest.raises(RuntimeError, match=r"failed \(-4\): .*no HIP device"):
        _preference(_rows())
    with pytest.raises(RuntimeError, match=r"failed \(-4\): .*no HIP device"):
        backend.GradSet([(A, A, 4, "f32")])


# Interleaved rows are apart: gradient and logits as columns of one array.
@pytest.mark.skipif(backend.device_count() > 0, reason="the addresses are made up")
def test_interleaved_rows_pass_the_overlap_check():
    with pytest.raises(RuntimeError, match=r"failed \(-4\)"):
        backend.policy_loss_device(_rows(stride=20), d_grad=A + 40, grad_stride=20, d_loss=A)
    _invalid(lambda: backend.policy_loss_device(_rows(stride=20), d_grad=A + 44, grad_stride=20))
    with pytest.raises(RuntimeError, match=r"failed \(-4\)"):
        backend.policy_loss_device(_rows(), d_grad=A, d_loss=A)  # in place


BAD_SETS = {
    "null-src": [(None, A, 4, "f32")],
    "src-alignment": [(A + 2, None, 4, "f32")],
    "dst-alignment": [(A, A + 4096 + 1, 4, "bf16")],
    "dst-in-own-src": [(A, A + 4, 4, "f32")],
    "dst-in-other-src": [(A, A, 4, "f32"), (A + 4096, A + 12, 4, "f32")],
    "dst-twice": [(A, A + 4096, 4, "f32"), (A + 64, A + 4096, 4, "f32")],
    "in-place-twice": [(A, A, 4, "f32"), (A, A, 4, "f32")],
    "dst-around-src": [(A + 64, None, 1, "f32"), (A + 8192, A, 64, "f32")],
    "too-many": [(A, None, 1 << 61, "f32")],
}


@pytest.mark.parametrize("name", BAD_SETS)
def test_bad_gradient_sets_are_refused(name):
    _invalid(lambda: backend.GradSet(BAD_SETS[name]))


@pytest.mark.skipif(backend.device_count() > 0, reason="the addresses are made up")
@pytest.mark.parametrize("tensors", [
    [(A, A, 4, "f32"), (A + 16, A + 16, 4, "f32")],           # in place, side by side
    [(A, A + 4096, 4, "f32"), (A, A + 8192, 4, "f32")],       # one src twice
    [(A, None, 4, "f32"), (A, None, 4, "f32")],
    [(A, A, 4, "f32"), (None, None, 0, "bf16")],
])
def test_sound_gradient_sets_get_as_far_as_the_device(tensors):
    with pytest.raises(RuntimeError, match=r"failed \(-4\)"):
        backend.GradSet(tensors)


def test_gradient_calls_refuse_what_they_cannot_use():
    L = backend.lib()
    h = ctypes.c_void_p()
    arr = (backend.MfhGradTensor * 1)(backend.MfhGradTensor(A, A, 4, 7))
    assert L.mfh_grad_set_create(arr, 1, -1, ctypes.byref(h)) == -1
    assert L.mfh_grad_set_create(arr, 1, -1, None) == -1
    assert L.mfh_grad_set_create(None, 1, -1, ctypes.byref(h)) == -1
    assert L.mfh_grad_set_create(arr, -1, -1, ctypes.byref(h)) == -1
    assert L.mfh_grad_set_create(arr, 1, -2, ctypes.byref(h)) == -1
    n = ctypes.c_uint64(0)
    assert L.mfh_grad_workspace_bytes(None, ctypes.byref(n)) == -1
    assert L.mfh_grad_norm_device(None, A, A, 1 << 20, None) == -1
    assert L.mfh_grad_scale_device(None, A, 1.0, None) == -1
    assert L.mfh_grad_clip_device(None, 1.0, A, A, 1 << 20, None) == -1
    L.mfh_grad_set_destroy(None)
