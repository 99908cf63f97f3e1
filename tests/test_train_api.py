"""Entry points of the training layers without a device: what they refuse,
before any device is touched, and what is nothing to do."""

import ctypes

import pytest

from metalfish_amd import backend

A = 1 << 24  # stands for an address; nothing here is dereferenced
FAR = 1 << 16
NAN, INF = float("nan"), float("inf")


def _invalid(call):
    with pytest.raises(RuntimeError, match=r"failed \(-1\): mfh_"):
        call()


def _reaches_device(call):
    """No fault of the arguments: without a device the call says so."""
    with pytest.raises(RuntimeError, match=r"failed \(-4\): .*no HIP device"):
        call()


made_up = pytest.mark.skipif(backend.device_count() > 0, reason="the addresses are made up")


# ---- Layer norm ----


def _rows(**kw):
    d = dict(d_x=A, rows=4, width=10, d_residual=A + FAR)
    d.update(kw)
    fields = {k: d.pop(k) for k in list(d) if k.startswith("set_")}
    r = backend.norm_rows(d.pop("d_x"), d.pop("rows"), d.pop("width"), **d)
    for k, v in fields.items():
        setattr(r, k[4:], v)
    return r


def _back(rows, **kw):
    d = dict(d_dy=A + 2 * FAR, d_mean=A + 3 * FAR, d_rstd=A + 4 * FAR, d_dx=A + 5 * FAR,
             d_dgamma=A + 6 * FAR, d_workspace=A + 7 * FAR, workspace_bytes=1 << 14)
    d.update(kw)
    backend.layer_norm_backward_device(rows, d.pop("d_dy"), d.pop("d_mean"), d.pop("d_rstd"), **d)


BAD_NORM = {
    "rows": dict(rows=-1), "width": dict(width=0), "width-large": dict(width=(1 << 20) + 1),
    "dtype": dict(set_dtype=3), "dtype-negative": dict(set_dtype=-1), "alpha": dict(alpha=NAN),
    "alpha-infinite": dict(alpha=INF), "eps": dict(eps=-1e-3), "eps-nan": dict(eps=NAN),
    "eps-infinite": dict(eps=INF), "device": dict(device=-2), "x": dict(d_x=None),
    "stride": dict(x_stride=9), "stride-far": dict(x_stride=1 << 60),
    "residual-stride": dict(residual_stride=9), "x-alignment": dict(d_x=A + 2),
    "half-alignment": dict(d_x=A + 1, dtype="bf16"), "residual-alignment": dict(d_residual=A + 2),
    "gamma-alignment": dict(d_gamma=A + 2), "beta-alignment": dict(d_beta=A + 1),
}


@pytest.mark.parametrize("name", BAD_NORM)
def test_bad_norm_rows_are_refused(name):
    _invalid(lambda: backend.layer_norm_device(_rows(**BAD_NORM[name]), A + 2 * FAR))
    _invalid(lambda: _back(_rows(**BAD_NORM[name])))


@pytest.mark.parametrize("kw", [dict(y_stride=9), dict(d_y=A + 4 * FAR + 2), dict(d_y=A + 4),
                                dict(d_y=A, y_stride=11), dict(d_y=A + FAR + 8),
                                dict(d_mean=A + 2), dict(d_mean=A + 8), dict(d_rstd=A + 3),
                                dict(d_mean=A + 2 * FAR, d_rstd=A + 2 * FAR + 4)])
def test_bad_norm_outputs_are_refused(kw):
    kw = dict(kw)
    _invalid(lambda: backend.layer_norm_device(_rows(), kw.pop("d_y", A + 4 * FAR), **kw))


@pytest.mark.parametrize("kw", [
    dict(d_dy=None), dict(d_mean=None), dict(d_rstd=None), dict(d_workspace=None),
    dict(workspace_bytes=319), dict(d_workspace=A + 7 * FAR + 2), dict(dy_stride=9),
    dict(dx_stride=9), dict(d_dx=A + 2), dict(d_dx=A + 40 * 4), dict(d_dx=A, d_dresidual=A),
    dict(d_dx=A, dx_stride=11), dict(d_dgamma=A + 2), dict(d_dgamma=A + 8),
    dict(d_dbeta=A + 6 * FAR + 4), dict(d_dbeta=A + 7 * FAR + 4), dict(d_dgamma=A + 3 * FAR)])
def test_bad_norm_gradients_are_refused(kw):
    if kw.get("d_dx") == A + 40 * 4:
        kw = dict(d_dx=A + 4)
    _invalid(lambda: _back(_rows(), **kw))


def test_a_gradient_of_a_residual_needs_one():
    _invalid(lambda: _back(_rows(d_residual=None), d_dresidual=A + 9 * FAR))


@made_up
def test_sound_norms_get_as_far_as_the_device():
    for y in (A, A + FAR, A + 2 * FAR):
        _reaches_device(lambda: backend.layer_norm_device(_rows(), y))
    # y as columns of the array that x is in.
    _reaches_device(lambda: backend.layer_norm_device(_rows(x_stride=20), A + 40, y_stride=20))
    for dx, dr in ((A, None), (A + FAR, A), (A + 2 * FAR, A + FAR), (A, A + 2 * FAR)):
        _reaches_device(lambda: _back(_rows(), d_dx=dx, d_dresidual=dr))
    _reaches_device(lambda: _back(_rows(rows=0, d_x=None), d_dy=None, d_mean=None, d_rstd=None))


def test_norms_with_nothing_to_do_succeed():
    backend.layer_norm_device(_rows(rows=0, d_x=None), None)
    _back(_rows(), d_dx=None, d_dgamma=None, d_workspace=None, workspace_bytes=0)
    _back(_rows(rows=0), d_dgamma=None, d_workspace=None, workspace_bytes=0)
    assert backend.layer_norm_workspace_bytes(0, 5) == 0
    assert backend.layer_norm_workspace_bytes(3, 5) >= 8 * 5 * 3
    n = ctypes.c_uint64()
    for args in ((-1, 5, ctypes.byref(n)), (1, 0, ctypes.byref(n)), (1, 5, None)):
        assert backend.lib().mfh_layer_norm_workspace_bytes(*args) == -1


# ---- Attention ----


def _problem(**kw):
    d = dict(d_q=A, d_k=A + FAR, d_v=A + 2 * FAR, batch=2, heads=4, q_len=3, k_len=5, dim=8)
    d.update(kw)
    fields = {k: d.pop(k) for k in list(d) if k.startswith("set_")}
    p = backend.attention_problem(*[d.pop(k) for k in ("d_q", "d_k", "d_v", "batch", "heads",
                                                       "q_len", "k_len", "dim")], **d)
    for k, v in fields.items():
        setattr(p, k[4:], v)
    return p


def _forward(p, **kw):
    d = dict(d_out=A + 3 * FAR, d_lse=A + 4 * FAR)
    d.update(kw)
    backend.attention_forward_device(p, d.pop("d_out"), **d)


def _grads(p, **kw):
    d = dict(d_out=A + 3 * FAR, d_lse=A + 4 * FAR, d_dout=A + 5 * FAR, d_dq=A + 6 * FAR,
             d_dk=A + 7 * FAR, d_dv=A + 8 * FAR, d_workspace=A + 9 * FAR, workspace_bytes=1 << 12)
    d.update(kw)
    backend.attention_backward_device(p, d.pop("d_out"), d.pop("d_lse"), d.pop("d_dout"), **d)


BAD_ATTENTION = {
    "batch": dict(batch=-1), "heads": dict(heads=0, kv_heads=1), "kv": dict(set_kv_heads=0),
    "group": dict(kv_heads=3), "q-len": dict(q_len=-1), "k-len": dict(k_len=-1),
    "k-long": dict(k_len=(1 << 30) + 1), "q-long": dict(q_len=(1 << 28) + 1, kv_heads=1),
    "many": dict(batch=1 << 29), "dim": dict(dim=0, scale=1.0), "dim-large": dict(dim=136), "dim-odd": dict(dim=12),
    "dtype": dict(set_dtype=3), "causal": dict(set_causal=2), "scale": dict(scale=NAN),
    "scale-infinite": dict(scale=INF), "device": dict(device=-2), "q": dict(d_q=None),
    "k": dict(d_k=None), "v": dict(d_v=None), "q-alignment": dict(d_q=A + 2),
    "k-alignment": dict(d_k=A + 1, dtype="bf16"), "stride": dict(q_strides=(-1, 32, 8)),
    "stride-far": dict(k_strides=(1 << 60, 32, 8)), "token-far": dict(v_strides=(0, 1 << 32, 8)), "lengths-alignment": dict(d_q_lengths=A + 2),
    "k-lengths-alignment": dict(d_k_lengths=A + 3),
}
BAD_BIAS = {
    "alignment": dict(d_bias=A + 10 * FAR + 2), "dtype": dict(d_bias=A + 10 * FAR, set_bias_dtype=5),
    "stride": dict(d_bias=A + 10 * FAR, bias_strides=(0, -5, 5)),
    "stride-far": dict(d_bias=A + 10 * FAR, bias_strides=(1 << 61, 15, 5)),
}


@pytest.mark.parametrize("name", BAD_ATTENTION)
def test_bad_attention_is_refused(name):
    p = _problem(**BAD_ATTENTION[name])
    _invalid(lambda: _forward(p))
    _invalid(lambda: _grads(p))
    _invalid(lambda: backend.attention_forward_workspace_bytes(p))
    _invalid(lambda: backend.attention_backward_workspace_bytes(p))


@pytest.mark.parametrize("name", BAD_BIAS)
def test_bad_biases_are_refused(name):
    _invalid(lambda: _forward(_problem(**BAD_BIAS[name])))
    _invalid(lambda: _grads(_problem(**BAD_BIAS[name])))


@pytest.mark.parametrize("kw", [
    dict(d_out=None), dict(d_out=A + 2), dict(d_out=A), dict(d_out=A + FAR + 8),
    dict(out_strides=(96, 32, 4)), dict(out_strides=(0, 32, 8)), dict(d_lse=A + 4 * FAR + 2),
    dict(d_lse=A + 3 * FAR), dict(d_lse=A + 2 * FAR + 8)])
def test_bad_attention_outputs_are_refused(kw):
    _invalid(lambda: _forward(_problem(), **kw))


@pytest.mark.parametrize("kw", [
    dict(d_out=None), dict(d_dout=None), dict(d_lse=None), dict(d_lse=A + 4 * FAR + 2),
    dict(d_dq=A), dict(d_dk=A + FAR + 4), dict(d_dv=A + 7 * FAR), dict(d_dq=A + 5 * FAR),
    dict(dk_strides=(160, 0, 8)), dict(dq_strides=(96, 32, 7)), dict(d_dbias=A + 11 * FAR),
    dict(d_workspace=None), dict(workspace_bytes=95), dict(d_workspace=A + 9 * FAR + 8),
    dict(d_workspace=A + 8 * FAR), dict(d_workspace=A + 4 * FAR)])
def test_bad_attention_gradients_are_refused(kw):
    _invalid(lambda: _grads(_problem(), **kw))


def test_bad_bias_gradients_are_refused():
    bias = dict(d_bias=A + 10 * FAR)
    for d in (A + 10 * FAR, A + 10 * FAR + 4, A + 11 * FAR + 2, A + 6 * FAR):
        _invalid(lambda: _grads(_problem(**bias), d_dbias=d))
    # One gradient for all queries, or two elements in one place.
    for strides in ((0, 5, 0), (60, 15, 4), (30, 15, 5)):
        _invalid(lambda: _grads(_problem(bias_strides=strides, **bias), d_dbias=A + 11 * FAR))


@made_up
def test_sound_attention_gets_as_far_as_the_device():
    _reaches_device(lambda: _forward(_problem()))
    _reaches_device(lambda: _grads(_problem()))
    bias = dict(d_bias=A + 10 * FAR)
    for strides in (None, (0, 15, 5), (0, 0, 5), (60, 15, 0)):
        _reaches_device(lambda: _forward(_problem(bias_strides=strides, **bias)))
        if strides is None or strides[2]:
            _reaches_device(lambda: _grads(_problem(bias_strides=strides, **bias),
                                           d_dbias=A + 11 * FAR))
    # q, k and v, and their gradients, in one array each.
    s = (5 * 96, 96, 8)
    p = _problem(d_k=A + 128, d_v=A + 256, q_len=5, q_strides=s, k_strides=s, v_strides=s)
    _reaches_device(lambda: _forward(p))
    g = A + 6 * FAR
    _reaches_device(lambda: _grads(p, d_dq=g, d_dk=g + 128, d_dv=g + 256, dq_strides=s,
                                   dk_strides=s, dv_strides=s))
    _invalid(lambda: _grads(p, d_dq=g, d_dk=g + 124, d_dv=g + 256, dq_strides=s, dk_strides=s,
                            dv_strides=s))


def test_attention_with_nothing_to_do_succeeds():
    _forward(_problem(batch=0, d_q=None, d_k=None, d_v=None), d_out=None)
    _forward(_problem(q_len=0, d_q=None), d_out=None)
    _grads(_problem(), d_dq=None, d_dk=None, d_dv=None)
    _grads(_problem(batch=0), d_out=None, d_dout=None)


def test_few_queries_over_many_keys_need_a_workspace():
    assert backend.attention_forward_workspace_bytes(_problem()) == 0
    p = _problem(d_q=A << 8, d_k=A << 9, d_v=A << 10, k_len=20000)
    n = backend.attention_forward_workspace_bytes(p)
    assert n > 0
    _invalid(lambda: _forward(p, d_out=A << 11, d_lse=A << 12))
    _invalid(lambda: _forward(p, d_out=A << 11, d_lse=A << 12, d_workspace=A << 13,
                              workspace_bytes=n - 1))


# ---- AdamW ----


def _tensor(at=0, **kw):
    d = dict(param=A + at, grad=A + at + FAR, m=A + at + 2 * FAR, v=A + at + 3 * FAR, count=10)
    d.update(kw)
    return d


EIGHT = dict(m_scale=A + 4 * FAR, v_scale=A + 5 * FAR)
BAD_SETS = {
    "param": (32, [_tensor(param=None)]), "grad": (32, [_tensor(grad=None)]),
    "m": (32, [_tensor(m=None)]), "v": (32, [_tensor(v=None)]),
    "scales-32": (32, [_tensor(**EIGHT)]), "no-scales": (8, [_tensor()]),
    "one-scale": (8, [_tensor(m_scale=A + 4 * FAR)]), "bits": (16, [_tensor()]),
    "alignment": (32, [_tensor(param=A + 2)]), "m-alignment": (32, [_tensor(m=A + 2 * FAR + 2)]),
    "scale-alignment": (8, [_tensor(**dict(EIGHT, m_scale=A + 4 * FAR + 1))]),
    "copy-alignment": (32, [_tensor(copy=A + 6 * FAR + 1, copy_dtype="bf16")]),
    "large": (32, [_tensor(count=1 << 60)]), "lr": (32, [_tensor(lr_scale=-1.0)]),
    "lr-nan": (32, [_tensor(lr_scale=NAN)]), "decay": (32, [_tensor(weight_decay=-0.1)]),
    "decay-infinite": (32, [_tensor(weight_decay=INF)]),
    "m-in-param": (32, [_tensor(m=A + 36)]), "grad-in-param": (32, [_tensor(grad=A + 36)]),
    "copy-is-param": (32, [_tensor(copy=A)]), "m-is-v": (32, [_tensor(v=A + 2 * FAR)]),
    "twice": (32, [_tensor(), _tensor()]),
    "other": (32, [_tensor(), _tensor(10 * FAR, param=A + 2 * FAR + 39)]),
    "scales": (8, [_tensor(**dict(EIGHT, v_scale=A + 4 * FAR))]),
}


@pytest.mark.parametrize("name", BAD_SETS)
def test_bad_adamw_sets_are_refused(name):
    bits, tensors = BAD_SETS[name]
    _invalid(lambda: backend.AdamWSet(tensors, state_bits=bits))


def test_unknown_types_and_keys_are_refused():
    for field in ("param_dtype", "grad_dtype", "copy_dtype"):
        t = backend.MfhAdamwTensor(A, A + FAR, A + 2 * FAR, A + 3 * FAR, None, None, A + 4 * FAR, 4,
                                   0, 0, 0, 1.0, 0.0)
        setattr(t, field, 3)
        h = ctypes.c_void_p()
        assert backend.lib().mfh_adamw_set_create(ctypes.byref(t), 1, 32, -1, ctypes.byref(h)) == -1
    with pytest.raises(ValueError, match="momentum"):
        backend.AdamWSet([_tensor(momentum=1)])
    h = ctypes.c_void_p()
    L = backend.lib()
    assert L.mfh_adamw_set_create(None, 1, 32, -1, ctypes.byref(h)) == -1
    assert L.mfh_adamw_set_create(None, -1, 32, -1, ctypes.byref(h)) == -1
    assert L.mfh_adamw_set_create(None, 0, 32, -2, ctypes.byref(h)) == -1
    assert L.mfh_adamw_set_create(None, 0, 32, -1, None) == -1
    L.mfh_adamw_set_destroy(None)


@made_up
def test_sound_adamw_sets_get_as_far_as_the_device():
    _reaches_device(lambda: backend.AdamWSet([_tensor(), _tensor(10 * FAR)]))
    _reaches_device(lambda: backend.AdamWSet([_tensor(**EIGHT)], state_bits=8))
    # One gradient for two tensors; tensors that touch.
    _reaches_device(lambda: backend.AdamWSet([_tensor(), _tensor(10 * FAR, grad=A + FAR)]))
    _reaches_device(lambda: backend.AdamWSet([_tensor(), _tensor(10 * FAR, param=A + 40)]))
    _reaches_device(lambda: backend.AdamWSet([_tensor(count=0, param=None, grad=None, m=None,
                                                      v=None)]))


def test_null_arguments_are_refused():
    L = backend.lib()
    r, g, p, a, s = _rows(), backend.MfhNormGrads(), _problem(), backend.MfhAttentionGrads(), \
        backend.MfhAdamwStep()
    at = ctypes.addressof
    h = backend.MfhHeads(A + 3 * FAR, 96, 32, 8)
    n = ctypes.c_uint64()
    assert L.mfh_layer_norm_device(None, A, 10, None, None, None) == -1
    assert L.mfh_layer_norm_backward_device(None, at(g), None) == -1
    assert L.mfh_layer_norm_backward_device(at(r), None, None) == -1
    assert L.mfh_attention_forward_device(None, at(h), None, None, 0, None) == -1
    assert L.mfh_attention_forward_device(at(p), None, None, None, 0, None) == -1
    assert L.mfh_attention_backward_device(None, at(a), None) == -1
    assert L.mfh_attention_backward_device(at(p), None, None) == -1
    assert L.mfh_attention_forward_workspace_bytes(at(p), None) == -1
    assert L.mfh_attention_backward_workspace_bytes(None, ctypes.byref(n)) == -1
    assert L.mfh_adamw_step_device(None, at(s), None) == -1
