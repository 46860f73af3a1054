"""Far tails of the activations, where values and slopes are small and their relative precision is
what counts. One term a sum (x one number a row, w ones and zeros, g one number a row), so that z,
dz and the results are single values, each rounded as often as it is stored."""

import pytest
import torch

import layer_bounds as lb

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
IDS = ["bf16", "f16"]


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def one_each(layers, z, up, kind):
    """act(z) and up act'(z) through the layer, for z and up of the type under test."""
    M, K, N = z.numel(), 64, 72
    at = torch.arange(M, device="cuda")
    x = torch.zeros(M, K, dtype=z.dtype, device="cuda")
    x[at, at % K] = z
    w = torch.ones(N, K, dtype=z.dtype, device="cuda")
    g = torch.zeros(M, N, dtype=z.dtype, device="cuda")
    g[at, at % N] = up
    x.requires_grad_(True)
    y = layers.linear(x, w, activation=kind)
    (dx,) = torch.autograd.grad(y, x, g)
    return y.detach(), dx


def within(got, want, rel, what):
    err = (got.double() - want).abs() / want.abs()
    assert bool((err <= rel).all()), (what, float(err.max()) / rel)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind,low", [("silu", -20.0), ("gelu_tanh", -5.0)])
def test_slopes_keep_their_precision(layers, kind, low, dtype):
    """act' within 2^-17 and kept to 2^-11, dz rounded once, dx once."""
    z = torch.linspace(low, -4.0, 300, device="cuda").to(dtype)
    up = torch.full_like(z, 4096.0)
    _, dx = one_each(layers, z, up, kind)
    want = 4096.0 * lb.slope(kind, z.double())
    within(dx, want[:, None].expand_as(dx), 2.01 * lb.U[dtype] + 2.0**-11 + 2.0**-17, kind)
