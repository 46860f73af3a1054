"""What the norms, products and optimiser step that test_layers_host.py does not hold decide on the
host: workspaces, refusals that need no GPU, and what tracers and derivatives are told."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def L():
    from diffrast import _lib

    return _lib


def size(L, name, *args):
    n = ctypes.c_uint64()
    L.check(getattr(L.lib(), name)(*args, ctypes.byref(n)))
    return n.value


def test_workspaces(L):
    # a partial row of D floats for each of the groups that a few rows need
    assert size(L, "drh_rms_norm_backward_bytes", 0, 64, 0) == 0
    assert size(L, "drh_rms_norm_backward_bytes", 1, 64, 0) == 256
    assert size(L, "drh_rms_norm_backward_bytes", 1 << 20, 1024, 1) <= 4096 * 1024 * 4
    # few rows go straight to the kernels that stage nothing
    assert size(L, "drh_gated_linear_bytes", 1, 4096, 1024, 1024, 1024, 1) == 0
    assert size(L, "drh_gated_linear_bytes", 64, 1501, 75, 75, 75, 2) == 0
    assert size(L, "drh_linear_8bit_bytes", 64, 1501, 1024, 1024, 1024, 1) == 0
    # rows that are not whole 16-byte chunks are copied to rows that are
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    assert size(L, "drh_gated_linear_bytes", 1531, 1501, 75, 75, 75, 2) >= up(1531 * 80 * 2) + up(2 * 1501 * 80 * 2)
    # the backward pass holds the gradient of both halves
    assert size(L, "drh_gated_linear_backward_bytes", 4096, 1024, 1024, 1024, 1024, 1) >= 2 * 4096 * 1024 * 2


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (65, 10, 48), (1000, 1500, 80), (16384, 4096, 1024), (100, 64, 100000), (1 << 20, 64, 64),
                                   (0, 8, 16)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspaces_stay_within_reason(L, M, N, K, dtype):
    """Copies of the operands, dz, the bias gradient's sums, and at most 1 GB of partial products."""
    e = 4 if dtype == 0 else 2
    pads = (M * (K + 8) + 2 * N * (K + 8) + M * (2 * N + 8)) * e + 512 * 2 * N * 4 + 4096
    assert size(L, "drh_gated_linear_bytes", M, N, K, K, K, dtype) <= pads + 10**9
    assert size(L, "drh_gated_linear_backward_bytes", M, N, K, K, K, dtype) <= pads + 10**9
    assert size(L, "drh_linear_8bit_bytes", M, N, K, K, K, dtype) <= 10**9 + 4096


@pytest.mark.parametrize("name,args,code", [
    ("drh_rms_norm_backward_bytes", (-1, 8, 0), 6), ("drh_rms_norm_backward_bytes", (8, 0, 0), 6),
    ("drh_rms_norm_backward_bytes", (8, 8, 7), 6), ("drh_rms_norm_backward_bytes", (1 << 31, 8, 0), 5),
    ("drh_rms_norm_backward_bytes", (8, 1 << 62, 0), 5), ("drh_gated_linear_bytes", (8, 0, 8, 8, 8, 0), 6),
    ("drh_gated_linear_bytes", (8, 8, 8, 8, 8, 3), 6), ("drh_gated_linear_bytes", (8, 1 << 62, 8, 8, 8, 0), 5),
    ("drh_gated_linear_bytes", (1 << 31, 8, 8, 8, 8, 0), 5), ("drh_gated_linear_bytes", (100, 8, 64, 63, 64, 1), 6),
    ("drh_gated_linear_bytes", (100, 1, 64, 64, 8, 1), 6), ("drh_gated_linear_backward_bytes", (8, 8, -1, 8, 8, 0), 6),
    ("drh_gated_linear_backward_bytes", (100, 8, 64, 64, 1 << 60, 1), 5), ("drh_linear_8bit_bytes", (8, 8, 8, 8, 8, 1), 6),
    ("drh_linear_8bit_bytes", (8, 8, 16, 24, 16, 1), 6), ("drh_linear_8bit_bytes", (8, 8, 16, 16, 16, 5), 6),
    ("drh_linear_8bit_bytes", (8, 8, 0, 0, 0, 1), 6), ("drh_linear_8bit_bytes", (8, 8, 16, 1 << 24, 16, 1), 5),
])
def test_bytes_refuse_what_the_call_refuses(L, name, args, code):
    n = ctypes.c_uint64(77)
    assert getattr(L.lib(), name)(*args, ctypes.byref(n)) == code
    assert n.value == 77


def test_no_context_no_call(L):
    f = L.lib()
    for rc in (f.drh_rms_norm(None, None, None, None, 1, 8, 8, 8, 0, 0, 1e-5, None, None, None, None, 0),
               f.drh_rms_norm_8bit(None, None, None, None, 1, 8, 8, 8, 0, 0, 1e-5, None, None, None, None, 0),
               f.drh_quantize_8bit(None, None, 1, 8, 8, 0, None, None, None, 0),
               f.drh_gated_linear(None, None, None, None, 1, 8, 8, 8, 8, 0, 0, None, None, None, 0, None, 0),
               f.drh_linear_8bit(None, None, None, None, None, None, None, 1, 8, 16, 16, 16, 0, 0, None, None, 0, None, 0),
               f.drh_adamw(None, None, 0, 0, 32, 0.1, 0.9, 0.9, 0.0, 0.0, 0, None, 0)):
        assert rc == 6 and "context" in L.last_error()


X = torch.ones(3, 16)
Q, S = torch.zeros(3, 16).to(E4M3), torch.ones(3)
CALLS = {
    "rms_norm": lambda L, x: L.rms_norm(x, torch.ones(16)),
    "rms_norm_residual": lambda L, x: L.rms_norm(x, None, x),
    "rms_norm_8bit": lambda L, x: L.rms_norm_8bit(x),
    "quantize_8bit": lambda L, x: L.quantize_8bit(x),
    "gated_linear": lambda L, x: L.gated_linear(x, torch.ones(8, 16)),
    "linear_8bit": lambda L, x: L.linear_8bit(Q, x[:, 0], Q, S),
}


@pytest.mark.parametrize("name", CALLS)
def test_refused_before_a_device_is_looked_for(name, monkeypatch):
    from diffrast import layers, torch_layer
    from torch.fx.experimental.proxy_tensor import make_fx

    monkeypatch.setattr(torch_layer, "_last_device", "cpu")
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        CALLS[name](layers, forward_ad.make_dual(X, X))
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(lambda x: CALLS[name](layers, x)[0], (X,), check_trace=False)
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(lambda x: CALLS[name](layers, x), tracing_mode=mode)(X)
    with pytest.raises(ValueError):
        CALLS[name](layers, X.double())
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no HIP device"):
            CALLS[name](layers, X)
    assert torch_layer.last_device() == "cpu"


def test_the_optimiser_takes_gpu_tensors_alone():
    from diffrast import optim

    t = lambda: [torch.zeros(3)]  # noqa: E731
    with pytest.raises(ValueError, match="on the GPU"):
        optim.adamw_step(t(), t(), t(), t(), torch.zeros(1, dtype=torch.int64), lr=0.1)
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.5)), dict(eps=-1.0), dict(weight_decay=float("nan")), dict(state_bits=16), dict(seed=-1)):
        with pytest.raises(ValueError):
            optim.AdamW(t(), **bad)
