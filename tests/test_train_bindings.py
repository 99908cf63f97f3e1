"""The Python side of the training layers: sizes that no field of the C structs
holds (no device needed)."""

import pytest

from metalfish_amd import backend

A, FAR = 1 << 24, 1 << 16  # stand for addresses
WIDE = (2 ** 32 + 8, 2 ** 31, -2 ** 31 - 1)


@pytest.mark.parametrize("size", WIDE)
def test_sizes_that_32_bits_would_cut_off_are_refused(size):
    for name in ("width", "device"):
        with pytest.raises(ValueError, match=name):
            backend.norm_rows(A, **{"rows": 4, "width": 8, name: size})
    with pytest.raises(ValueError, match="width"):
        backend.layer_norm_workspace_bytes(4, size)
    for name in ("batch", "heads", "kv_heads", "q_len", "k_len", "dim", "device"):
        kw = {"batch": 1, "heads": 2, "q_len": 3, "k_len": 5, "dim": 8, "scale": 1.0, name: size}
        with pytest.raises(ValueError, match=name):
            backend.attention_problem(A, A + FAR, A + 2 * FAR, **kw)


@pytest.mark.parametrize("dim", [0, -8])
def test_heads_without_elements_are_refused_by_the_call(dim):
    """Also where the scale is left to the head size."""
    p = backend.attention_problem(A, A + FAR, A + 2 * FAR, 1, 2, 3, 5, dim)
    with pytest.raises(RuntimeError, match="dim must be a multiple of 8"):
        backend.attention_forward_device(p, A + 3 * FAR)
    with pytest.raises(RuntimeError, match="dim must be a multiple of 8"):
        backend.attention_backward_workspace_bytes(p)
