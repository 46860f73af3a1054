"""What autograd may and may not do with the network layers."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def leaves(*shapes):
    g = torch.Generator("cuda").manual_seed(len(shapes))
    return [torch.randn(*s, device="cuda", generator=g).requires_grad_(True) for s in shapes]


# name: (the inputs' shapes, the call on them)
CALLS = {
    "layer_norm": (((6, 16), (16,), (16,)), lambda L, x, w, b: L.layer_norm(x, w, b)),
    "layer_norm_plain": (((6, 16),), lambda L, x: L.layer_norm(x)),
    "linear": (((6, 16), (8, 16), (8,)), lambda L, x, w, b: L.linear(x, w, b)),
    "linear_act_residual": (((6, 16), (8, 16), (8,), (6, 8)), lambda L, x, w, b, r: L.linear(x, w, b, "gelu", r)),
    "dropout": (((6, 16),), lambda L, x: L.dropout(x, 0.25, seed=1)),
    "dropout_residual": (((6, 16), (6, 16)), lambda L, x, r: L.dropout(x, 0.25, seed=1, residual=r)),
}


@pytest.mark.parametrize("grad_requires_grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_differentiating_a_gradient_again_raises(layers, name, grad_requires_grad):
    """Mixed with a term that can be differentiated too, for each input's gradient by itself."""
    shapes, call = CALLS[name]
    ts = leaves(*shapes)
    y = call(layers, *ts)
    up = torch.ones_like(y, requires_grad=grad_requires_grad)
    want = torch.autograd.grad(y, ts, torch.ones_like(y), retain_graph=True)
    got = torch.autograd.grad(y, ts, up, create_graph=True)
    for d, w, t in zip(got, want, ts):
        assert bool(torch.equal(d.detach(), w)) and d.requires_grad
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad((d * d).sum() + t.sum(), t, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            ((d * d).sum() + t.sum()).backward(retain_graph=True)
    # without a graph of the backward pass nothing hangs on to it
    plain = torch.autograd.grad(y, ts, torch.ones_like(y))
    assert not any(d.requires_grad for d in plain)
