"""32-bit products whose sums have one term each, so that a result shows what the product keeps of
its two operands, whatever the length of the sum.

Products in thirds of bfloat16 drop less than 2^-21 |a b|; their six terms are added in 32 bits, with
less than 2^-23 |a b| lost at each (the matrix cores need not round to the nearest), and the result is
stored as it is: 2^-21 + 6 2^-23 < 3 2^-21. Below the normal numbers each of the six sums loses up to
their spacing, 2^-149."""

import pytest
import torch

pytestmark = pytest.mark.gpu
BOUND = 3 * 2.0**-21


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def operands(M, N, K, seed=0):
    """x with one number a row, at another k each; g with one a row, at another column; w full."""
    g = torch.Generator("cuda").manual_seed(seed + M + N + K)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    rows = torch.arange(M, device="cuda")
    at_k, at_n = (rows * 37 + 5) % K, (rows * 11 + 3) % N
    x, up = torch.zeros(M, K, device="cuda"), torch.zeros(M, N, device="cuda")
    x[rows, at_k], up[rows, at_n] = r(M), r(M)
    return x, r(N, K), up, rows, at_k, at_n


def check(got, want, what):
    err, lim = (got.double() - want).abs(), BOUND * want.abs() + 6 * 2.0**-149
    assert bool((err <= lim).all()), (what, float((err / lim).max()))


# two groups of waves on tiles of 64, one group on many of them, tiles of 128, split sums
SIZES = [(200, 136, 328), (1000, 1160, 1024), (4100, 2056, 4160), (512, 256, 8192)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("sx,sw", [(0, 0), (-108, 40), (-114, 60), (-118, 100), (-122, 60), (-125, 20), (40, -112), (60, -118),
                                   (100, -124), (-70, -70), (100, 20)])
def test_one_term_sums(layers, M, N, K, sx, sw):
    """Numbers about 2^sx times 2^sw: below 2^-111 a bfloat16 cannot hold the last of three thirds."""
    x, w, up, rows, at_k, at_n = operands(M, N, K)
    x, w = x * 2.0**sx, w * 2.0**sw
    y = layers.linear(x, w)
    check(y, x[rows, at_k].double()[:, None] * w.t()[at_k].double(), "y")
    if M <= K and K % 37:  # then another k for each row: one term in each sum of dW
        wl = w.clone().requires_grad_(True)
        (dw,) = torch.autograd.grad(layers.linear(x, wl), wl, w.t()[:1].expand(M, N).contiguous())
        want = torch.zeros(N, K, dtype=torch.float64, device="cuda")
        want[:, at_k] = w[:, 0].double()[:, None] * x[rows, at_k].double()
        check(dw, want, "dW")
    xl = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(layers.linear(xl, w), xl, up * 2.0**sx)
    check(dx, (up[rows, at_n] * 2.0**sx).double()[:, None] * w[at_n].double(), "dx")


def test_a_small_operand_beside_large_ones(layers):
    """A tile that is made again because of one tiny number is as exact for all of its others."""
    M, N, K = 1000, 1160, 1024
    x, w, _, rows, at_k, _ = operands(M, N, K)
    x[7, at_k[7]] = 1.2345678 * 2.0**-121
    w[900, 13] = 1.7654321 * 2.0**-119
    check(layers.linear(x, w), x[rows, at_k].double()[:, None] * w.t()[at_k].double(), "y")


@pytest.mark.parametrize("M,N,K", [(300, 136, 328), (1000, 1160, 1024), (512, 256, 8192)])
def test_tails_in_the_operands(layers, M, N, K):
    """Slopes down to 2^-149 among ordinary ones (GELU far below zero), softmaxes with numbers as small."""
    import layer_bounds as lb
    from test_gpu_linear import compare, make, run

    t = make(M, N, K, torch.float32, res=True)
    t["x"] *= 7.0
    assert 0 < int(((lb.slope("gelu", t["x"].double() @ t["w"].double().t()).abs() < 2.0**-115)).sum())
    compare(t, "gelu", run(layers, t, "gelu"), "gelu")
    t["x"] = torch.softmax(30 * t["x"].detach() / 7, 1)
    assert 0 < int(((t["x"] > 0) & (t["x"] < 2.0**-115)).sum())
    compare(t, None, run(layers, t, None), "softmax")
