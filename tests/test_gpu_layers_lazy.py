"""Tensors whose memory is not their value: torch negates them when it reads them."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def imag(t):
    """t as the imaginary part of a conjugate: a view with the negative bit, elements two apart."""
    v = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert v.is_neg()
    return v


def neg(t):
    v = torch._neg_view(-t)
    assert v.is_neg()
    return v


CALLS = {
    "layer_norm": (((40, 24), (24,), (24,)), lambda L, x, w, b: L.layer_norm(x, w, b)),
    "linear": (((40, 24), (8, 24), (8,), (40, 8)), lambda L, x, w, b, r: L.linear(x, w, b, "silu", r)),
    "dropout": (((40, 24), (40, 24)), lambda L, x, r: L.dropout(x, 0.25, seed=1, residual=r)),
}


@pytest.mark.parametrize("make", [neg, imag])
@pytest.mark.parametrize("name", CALLS)
def test_negated_views(layers, name, make):
    shapes, call = CALLS[name]
    g = torch.Generator("cuda").manual_seed(3)
    ts = [torch.randn(*s, device="cuda", generator=g).requires_grad_(True) for s in shapes]
    y = call(layers, *ts)
    up = torch.randn(y.shape, device="cuda", generator=g)
    want = torch.autograd.grad(y, ts, up)
    for i in range(len(ts)):
        mixed = [make(t) if i == j else t for j, t in enumerate(ts)]
        z = call(layers, *mixed)
        assert bool(torch.equal(z, y)), i
        for a, b in zip(torch.autograd.grad(z, ts, up), want):
            assert bool(torch.equal(a, b)), i
    for a, b in zip(torch.autograd.grad(call(layers, *ts), ts, make(up)), want):
        assert bool(torch.equal(a, b))
