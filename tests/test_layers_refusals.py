"""What the network layers refuse, and how: a workspace as its call, a call without a trace."""

import ctypes

import pytest


@pytest.fixture(scope="module")
def L():
    from diffrast import _lib

    return _lib


@pytest.mark.parametrize("name,args,code", [
    ("drh_linear_bytes", (1 << 31, 8, 8, 8, 8, 0), 5), ("drh_linear_bytes", (1 << 62, 8, 1 << 62, 1 << 62, 1 << 62, 0), 5),
    ("drh_linear_bytes", (8, (1 << 30) + 1, 8, 8, 8, 1), 5), ("drh_linear_bytes", (8, 8, 1 << 31, 1 << 31, 1 << 31, 1), 5),
    ("drh_linear_bytes", (100, 8, 64, 63, 64, 1), 6), ("drh_linear_bytes", (100, 8, 64, 64, 8, 1), 6),
    ("drh_linear_bytes", (100, 8, 64, 1 << 60, 64, 1), 5), ("drh_linear_backward_bytes", (1 << 31, 8, 8, 8, 8, 0, 0), 5),
    ("drh_linear_backward_bytes", (100, 8, 64, 64, 1 << 60, 1, 0), 5), ("drh_linear_backward_bytes", (100, 8, 64, -64, 64, 1, 0), 6),
    ("drh_layer_norm_backward_bytes", (1 << 31, 8, 0), 5), ("drh_layer_norm_backward_bytes", (8, 1 << 62, 0), 5),
])
def test_bytes_refuse_what_the_call_refuses(L, name, args, code):
    n = ctypes.c_uint64(77)
    assert getattr(L.lib(), name)(*args, ctypes.byref(n)) == code
    assert n.value == 77


def test_a_single_rows_stride_is_free(L):
    a, b = ctypes.c_uint64(), ctypes.c_uint64()
    for xs in (0, 64, 1 << 60, -5):
        L.check(L.lib().drh_linear_backward_bytes(1, 200, 64, xs, 64, 1, 0, ctypes.byref(a)))
        L.check(L.lib().drh_linear_backward_bytes(1, 200, 64, 64, 64, 1, 0, ctypes.byref(b)))
        assert a.value == b.value


def test_a_refused_call_ran_on_no_device(monkeypatch):
    import torch
    from diffrast import layers, torch_layer

    monkeypatch.setattr(torch_layer, "_last_device", "cpu")
    x = torch.zeros(3, 8)
    for call in (lambda: layers.layer_norm(x, torch.zeros(7)), lambda: layers.linear(x, torch.zeros(4, 7)),
                 lambda: layers.dropout(x, 1.5, seed=0)):
        with pytest.raises(ValueError):
            call()
        assert torch_layer.last_device() == "cpu"
