"""How diffrast.layers.linear_8bit adds: a row with an outlier, whose large products cancel."""

import pytest
import torch

import operator_bounds as ob

pytestmark = pytest.mark.gpu


def make(M, N, K, seed):
    """Products of +-448 x 448 in two groups of eight, and else numbers of quarters up to 4: every partial
    sum is a multiple of 2^-4 below 2^19, which 32 bits hold whole."""
    g = torch.Generator("cuda").manual_seed(seed)
    small = lambda *s: torch.randint(-7, 8, s, device="cuda", generator=g) / 4.0  # noqa: E731
    x, w = small(M, K), small(N, K)
    x[:, 3] = x[:, 3 + 40] = 448.0
    w[:, 3], w[:, 3 + 40] = 448.0, -448.0
    return x, w


# few rows, tiles of 64 and 128, split sums, tiles of 256
@pytest.mark.parametrize("M,K,N", [(1, 128, 40), (20, 256, 64), (64, 1024, 33), (100, 128, 64), (100, 8192, 64), (600, 512, 600),
                                   (3900, 256, 3960)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_an_outlier_that_cancels(M, K, N, dtype):
    from diffrast import layers

    x, w = make(M, N, K, M + K)
    X, W = x.to(ob.E4M3), w.to(ob.E4M3)
    assert torch.equal(X.float(), x) and torch.equal(W.float(), w)
    y = layers.linear_8bit(X, torch.ones(M, device="cuda"), W, torch.ones(N, device="cuda"), dtype=dtype)
    want = x.double() @ w.double().t()
    if dtype == torch.float32:
        assert torch.equal(y, want.float())
    else:
        # up to 2^-10 of the terms is cut off, and the result rounded by half a step
        lost = 2.0**-10 * (x.double().abs() @ w.double().abs().t())
        assert bool(((y.double() - want).abs() <= lost + torch.finfo(dtype).eps / 2 * (want.abs() + lost)).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 1024, 4096), (64, 1024, 513), (600, 4096, 600), (3900, 1024, 3960)])
def test_normal_numbers(M, K, N, dtype):
    """Sums that are d off cross a border of their rounding, 2 e of themselves wide, with a probability of d / (2 e), and
    then differ by 2 e: sqrt(2 e d) of the norm. d is 8e-6 of it as documented; twice that here."""
    from diffrast import layers

    g = torch.Generator("cuda").manual_seed(M)
    rows = lambda n: layers.quantize_8bit(torch.randn(n, K, device="cuda", generator=g))  # noqa: E731
    ops = (*rows(M), *rows(N))
    want = layers.linear_8bit(*ops, dtype=torch.float32)
    off = (layers.linear_8bit(*ops, dtype=dtype).double() - want.to(dtype).double()).norm() / want.double().norm()
    assert float(off) <= (torch.finfo(dtype).eps * 1.6e-5) ** 0.5
