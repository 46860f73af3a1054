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


# z down to here; beyond 2^-15 (f32: the argument's own rounding counts c^2 times) or 2^-13 (16 bits) of
# the value there is the rounding to the type alone
@pytest.mark.parametrize("dtype,low,rel", [(torch.float32, -12.0, 2.0**-15), (torch.bfloat16, -12.0, 2.0**-13),
                                           (torch.float16, -5.0, 2.0**-13)], ids=["f32", *IDS])
def test_gelus_tail(layers, dtype, low, rel):
    z = torch.linspace(low, -1.5, 300, device="cuda").to(dtype)
    up = torch.full_like(z, 4096.0)
    y, dx = one_each(layers, z, up, "gelu")
    want = lb.act("gelu", z.double())[:, None].expand_as(y)
    lb.check(y, want, rel * want.abs(), dtype, "y")
    # act' = Phi + z phi, the second term up to z^2 times the first; it is zero nowhere below -0.76
    want = 4096.0 * lb.slope("gelu", z.double())[:, None].expand_as(dx)
    within(dx[z >= -6.0], want[z >= -6.0], 2 * rel + (2.01 * lb.U[dtype] + 2.0**-11 if dtype != torch.float32 else 0.0), "dx")


@pytest.mark.parametrize("dtype", [torch.float32, *DTYPES], ids=["f32", *IDS])
@pytest.mark.parametrize("kind", lb.ACTS[1:])
def test_values_over_the_whole_range(layers, kind, dtype):
    """Every 16-bit number (of float32 as many) as z: between the bends, past them, zeros and infinities."""
    if dtype == torch.float32:
        z = (torch.arange(1 << 16, device="cuda", dtype=torch.int32) << 16).view(torch.float32)
    else:
        z = torch.arange(-(1 << 15), 1 << 15, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    z = z[~torch.isnan(z)]
    x = torch.zeros(z.numel(), 8, dtype=dtype, device="cuda")
    x[:, 0] = z
    w = torch.zeros(16, 8, dtype=dtype, device="cuda")
    w[:, 0] = 1.0
    bias = torch.zeros(16, dtype=dtype, device="cuda")
    x = x[torch.isfinite(z)]
    z = z[torch.isfinite(z)]
    y = layers.linear(x, w, bias, kind)
    want = lb.act(kind, z.double())
    want = torch.where(torch.isnan(want), z.double().clamp(min=0), want)  # the formula's own overflow
    lb.check(y, want[:, None].expand_as(y), (lb.act_error(kind, dtype)[0] * z.double().abs())[:, None].expand_as(y), dtype, kind)
