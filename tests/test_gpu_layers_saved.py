"""A layer keeps for its backward pass what the gradients that are wanted need: the rest may be
freed, or changed in place."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def leaf(want, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(len(shape))).to(dtype).requires_grad_(want)


def saved(call):
    """The call's result and the shapes of what it saves."""
    shapes = []

    def pack(t):
        shapes.append(tuple(t.shape))
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        return call(), sorted(shapes)


X, W, S = (6, 16), (8, 16), (6, 8)  # x, weight, slopes (and the residual)


@pytest.mark.parametrize("wanted,kind,shapes", [
    ("x", None, [W]), ("w", None, [X]), ("b", None, []), ("r", None, []), ("xw", None, [X, W]),
    ("x", "gelu", [S, W]), ("w", "gelu", [S, X]), ("b", "gelu", [S]), ("r", "gelu", []), ("xwbr", "gelu", [S, X, W]),
])
def test_linear(layers, wanted, kind, shapes):
    x, w, b, r = leaf("x" in wanted, *X), leaf("w" in wanted, *W), leaf("b" in wanted, 8), leaf("r" in wanted, *S)
    ts = dict(x=x, w=w, b=b, r=r)
    full = {k: t.detach().clone().requires_grad_(True) for k, t in ts.items()}
    up = torch.randn(*S, device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    want = dict(zip("xwbr", torch.autograd.grad(layers.linear(full["x"], full["w"], full["b"], kind, full["r"]),
                                                list(full.values()), up)))
    y, kept = saved(lambda: layers.linear(x, w, b, kind, r))
    assert kept == sorted(shapes)
    with torch.no_grad():  # what was not kept may change before the backward pass
        for k, t in ts.items():
            if tuple(t.shape) not in shapes or k in "br":
                t.fill_(7.0)
    y.backward(up)
    for k, t in ts.items():
        if k in wanted:
            assert bool(torch.equal(t.grad, want[k])), k
        else:
            assert t.grad is None


@pytest.mark.parametrize("D", [96, 9000])
@pytest.mark.parametrize("wanted", ["x", "w", "b", "wb", "xwb"])
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_layer_norm(layers, wanted, D, wdtype):
    x = leaf("x" in wanted, 20, D, dtype=torch.bfloat16)
    w, b = leaf("w" in wanted, D, dtype=wdtype), leaf("b" in wanted, D, dtype=wdtype)
    full = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    up = torch.randn(20, D, device="cuda", generator=torch.Generator("cuda").manual_seed(9)).bfloat16()
    want = torch.autograd.grad(layers.layer_norm(*full), full, up)
    y, kept = saved(lambda: layers.layer_norm(x, w, b))
    assert kept == sorted([(20, D), (2, 20)] + ([(D,)] if "x" in wanted else []))
    with torch.no_grad():
        b.fill_(7.0)
        if "x" not in wanted:
            w.fill_(7.0)
    y.backward(up)
    for k, t, d in zip("xwb", (x, w, b), want):
        assert bool(torch.equal(t.grad, d)) if k in wanted else t.grad is None, k


def test_a_frozen_layers_input_is_freed(layers):
    x0 = leaf(True, 4096, 1024)
    w = leaf(False, 8, 1024)
    before = torch.cuda.memory_allocated()
    y = layers.linear(x0 * 2.0, w)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before < x0.numel() * 4
    (d,) = torch.autograd.grad(y.sum(), x0)
    assert bool(torch.allclose(d[:1], 2 * w.sum(0), rtol=1e-5, atol=1e-5))
