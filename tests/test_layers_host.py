"""What the network layers decide on the host: workspaces, and refusals that need no GPU."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from diffrast import _lib

    return _lib


def size(L, name, *args):
    n = ctypes.c_uint64()
    L.check(getattr(L.lib(), name)(*args, ctypes.byref(n)))
    return n.value


def test_workspaces_grow_with_what_they_hold(L):
    # a partial row of 2 D floats for each of the groups that a few rows need
    assert size(L, "drh_layer_norm_backward_bytes", 0, 64, 0) == 0
    assert size(L, "drh_layer_norm_backward_bytes", 1, 64, 0) == 512
    assert size(L, "drh_layer_norm_backward_bytes", 1 << 20, 1024, 1) <= 1024 * 2 * 1024 * 4
    # few rows go straight to the kernel that stages nothing
    assert size(L, "drh_linear_bytes", 1, 1500, 1024, 1024, 1024, 1) == 0
    assert size(L, "drh_linear_bytes", 64, 1501, 75, 75, 75, 2) == 0
    # rows that are not whole 16-byte chunks are copied to rows that are
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    assert size(L, "drh_linear_bytes", 1531, 1501, 75, 75, 75, 2) >= up(1531 * 80 * 2) + up(1501 * 80 * 2)
    # without an activation and with whole chunks dz is dy itself
    a = size(L, "drh_linear_backward_bytes", 4096, 1024, 1024, 1024, 1024, 1, 0)
    b = size(L, "drh_linear_backward_bytes", 4096, 1024, 1024, 1024, 1024, 1, 1)
    assert b - a == 4096 * 1024 * 2


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (65, 10, 48), (1000, 1500, 75), (16384, 4096, 1024), (16384, 1024, 4096),
                                   (100, 64, 100000), (1 << 20, 64, 64), (0, 8, 8), (8, 8, 0)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspaces_stay_within_reason(L, M, N, K, dtype):
    """Copies of the operands, dz, the bias gradient's sums, and at most 1 GB of partial products."""
    e = 4 if dtype == 0 else 2
    pads = (M * (K + 8) + N * (K + 8) + M * (N + 8)) * e + 256 * N * 4 + 4096
    assert size(L, "drh_linear_bytes", M, N, K, K, K, dtype) <= pads + 10**9
    assert size(L, "drh_linear_backward_bytes", M, N, K, K, K, dtype, 2) <= pads + 10**9


@pytest.mark.parametrize("name,args", [
    ("drh_layer_norm_backward_bytes", (-1, 8, 0)), ("drh_layer_norm_backward_bytes", (8, 0, 0)),
    ("drh_layer_norm_backward_bytes", (8, 8, 7)), ("drh_linear_bytes", (8, 0, 8, 8, 8, 0)), ("drh_linear_bytes", (8, 8, 8, 8, 8, 3)),
    ("drh_linear_backward_bytes", (8, 8, -1, 8, 8, 0, 0)), ("drh_linear_backward_bytes", (-8, 8, 8, 8, 8, 0, 0)),
])
def test_bad_sizes_are_refused(L, name, args):
    with pytest.raises(L.DiffrastError) as e:
        size(L, name, *args)
    assert e.value.code == 6


def test_no_context_no_call(L):
    f = L.lib()
    for rc in (f.drh_layer_norm(None, None, None, None, 1, 8, 8, 0, 0, 1e-5, None, None, None, None, 0),
               f.drh_linear(None, None, None, None, None, 1, 8, 8, 8, 8, 0, 0, None, None, None, 0, None, 0),
               f.drh_dropout(None, None, None, 8, 0, 0.5, 0, 0, None, None, 0)):
        assert rc == 6 and "context" in L.last_error()


def test_arguments_are_checked_before_the_device():
    from diffrast import layers

    x = torch.zeros(3, 8)
    for call in (lambda: layers.layer_norm(x, torch.zeros(7)), lambda: layers.linear(x, torch.zeros(4, 7)),
                 lambda: layers.linear(x, torch.zeros(4, 8), activation="tanh"), lambda: layers.dropout(x, 1.5, seed=0),
                 lambda: layers.dropout(x, 0.5, seed=-1)):
        with pytest.raises(ValueError):
            call()
    if not torch.cuda.is_available():
        for call in (lambda: layers.layer_norm(x), lambda: layers.linear(x, torch.zeros(4, 8)),
                     lambda: layers.dropout(x, 0.5, seed=0)):
            with pytest.raises(RuntimeError, match="no HIP device"):
                call()
