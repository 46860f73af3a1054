"""The product kernel that takes any alignment and stride, with enough rows that no other does."""

import pytest
import torch

import layer_bounds as lb
from test_gpu_linear import DTYPES, IDS, compare, make, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def shifted(t, by=1):
    """t's values at an address `by` elements off a 16-byte boundary."""
    flat = torch.full((t.numel() + by,), float("nan"), dtype=t.dtype, device="cuda")
    flat[by:] = t.detach().reshape(-1)
    return flat[by:].view(t.shape)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind", lb.ACTS)
@pytest.mark.parametrize("which", ["x", "w", "g", "xwg"])
def test_misaligned_operands(layers, which, kind, dtype):
    """y from x and W, dx from dz and W, dW from dz and x: each operand off by one element, or all."""
    for M, N, K in ((300, 136, 96), (129, 64, 1032), (1030, 8, 264)):
        t = make(M, N, K, dtype, res=True)
        for k in which:
            t[k] = shifted(t[k])
            assert t[k].data_ptr() % 16
        compare(t, kind, run(layers, t, kind), f"{which} {M}x{N}x{K} {kind}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_everything_off_with_ragged_sizes(layers, dtype):
    t = make(333, 75, 101, dtype, res=True)
    for k in ("x", "w", "b", "res", "g"):
        t[k] = shifted(t[k], 3)
    compare(t, "gelu", run(layers, t, "gelu"), "all off")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strides_past_a_buffers_reach(layers, dtype):
    """Rows 2^31 bytes apart over a tile: no buffer resource spans them."""
    M, N, K = 140, 72, 80
    stride = (1 << 23) // torch.empty((), dtype=dtype).element_size() + 16
    t = make(M, N, K, dtype)
    wide = torch.empty(M, stride, dtype=dtype, device="cuda")
    wide[:, :K] = t["x"].detach()
    t["x"] = wide[:, :K]
    compare(t, "silu", run(layers, t, "silu"), "far rows")
    del wide
    t = make(M, N, K, dtype)
    wide = torch.empty(N, 4 * stride, dtype=dtype, device="cuda")
    wide[:, :K] = t["w"].detach()
    t["w"] = wide[:, :K]
    compare(t, "silu", run(layers, t, "silu"), "far weights")
