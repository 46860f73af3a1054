"""What hooks hand to a layer's backward pass is checked before a kernel reads it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


CALLS = {
    "layer_norm": (((40, 24), (24,), (24,)), lambda L, x, w, b: L.layer_norm(x, w, b)),
    "linear": (((40, 24), (8, 24), (8,), (40, 8)), lambda L, x, w, b, r: L.linear(x, w, b, "silu", r)),
}


def inputs(name):
    g = torch.Generator("cuda").manual_seed(3)
    return [torch.randn(*s, device="cuda", generator=g).requires_grad_(True) for s in CALLS[name][0]]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t.half() if t.dtype == torch.float32 else t.double(),
                                    lambda t: t[:1], lambda t: t.to_sparse()], ids=["host", "type", "shape", "layout"])
def test_a_saved_tensor_that_comes_back_as_another(layers, name, which, change):
    ts, count = inputs(name), []

    def unpack(t):
        count.append(0)
        return change(t) if len(count) == which + 1 else t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = CALLS[name][1](layers, *ts)
    with pytest.raises(RuntimeError, match="saved for a layer"):
        y.sum().backward()


@pytest.mark.parametrize("name", CALLS)
def test_saved_tensors_may_be_moved_and_laid_out_anew(layers, name):
    ts = inputs(name)
    y = CALLS[name][1](layers, *ts)
    up = torch.randn(y.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    want = torch.autograd.grad(y, ts, up)

    def strided(t):  # the same values, columns first
        return t.t().contiguous().t() if t.dim() == 2 else t

    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, strided)):
        with hooks:
            y = CALLS[name][1](layers, *ts)
        for a, b in zip(torch.autograd.grad(y, ts, up), want):
            assert bool(torch.equal(a, b))


@pytest.mark.parametrize("change", [lambda t: t.half(), lambda t: t.cpu(), lambda t: t[:1]], ids=["type", "host", "shape"])
@pytest.mark.parametrize("name", CALLS)
def test_a_nodes_hook_that_changes_the_gradient(layers, name, change):
    ts = inputs(name)
    y = CALLS[name][1](layers, *ts)
    y.grad_fn.register_prehook(lambda g: (change(g[0]),))
    with pytest.raises(RuntimeError):
        y.sum().backward()
