"""What sees operators through torch's dispatcher cannot see the network layers: forward-mode
derivatives and tracers are refused, since their answers would be wrong (a derivative of zero, a
program that returns memory never written). The refusals come before a device is looked for."""

import pytest
import torch
from torch.autograd import forward_ad

from diffrast import layers

X, W, B, R = torch.ones(3, 8), torch.ones(4, 8), torch.ones(4), torch.ones(3, 4)
# name: (the inputs, the call on them)
CALLS = {
    "layer_norm": ((X, torch.ones(8), torch.ones(8)), lambda x, w, b: layers.layer_norm(x, w, b)),
    "linear": ((X, W, B, R), lambda x, w, b, r: layers.linear(x, w, b, "gelu", r)),
    "dropout": ((X, torch.ones(3, 8)), lambda x, r: layers.dropout(x, 0.5, seed=1, residual=r)),
}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    inputs, call = CALLS[name]
    for i in range(len(inputs)):
        with forward_ad.dual_level():
            ts = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(inputs)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*ts)


@pytest.mark.parametrize("name", CALLS)
def test_tracers_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    inputs, call = CALLS[name]
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(call, inputs, check_trace=False)
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(call, tracing_mode=mode)(*inputs)
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(call, pre_dispatch=True)(*inputs)


@pytest.mark.parametrize("name", CALLS)
def test_no_answer_for_wrapped_tensors(name):
    inputs, call = CALLS[name]
    first = lambda x: call(x, *inputs[1:]).sum()  # noqa: E731
    for transform in (lambda: torch.func.grad(first)(X), lambda: torch.func.vmap(first)(torch.stack([X, X])),
                      lambda: torch.func.jvp(first, (X,), (X,))):
        with pytest.raises(RuntimeError):
            transform()


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_the_same_on_the_gpu(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    inputs, call = CALLS[name]
    ts = [t.cuda() for t in inputs]
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        call(forward_ad.make_dual(ts[0], ts[0]), *ts[1:])
    first = lambda x: call(x, *ts[1:]).sum()  # noqa: E731
    for transform in (lambda: torch.jit.trace(call, ts), lambda: make_fx(call)(*ts), lambda: torch.func.grad(first)(ts[0]),
                      lambda: torch.func.vmap(first)(torch.stack([ts[0], ts[0]])),
                      lambda: torch.func.jvp(first, (ts[0],), (ts[0],))):
        with pytest.raises(RuntimeError):
            transform()
    # a backward pass is refused as well, where the forward pass was outside of the trace
    leaf = ts[0].clone().requires_grad_(True)
    y = call(leaf, *ts[1:])
    with pytest.raises(RuntimeError):
        make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True))(torch.ones_like(y))
    # and outside of them all the call is what it was
    assert bool(torch.equal(call(*ts), y.detach()))


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_compiled_and_checkpointed_programs_call_the_layers(name):
    from torch.utils.checkpoint import checkpoint

    inputs, call = CALLS[name]
    ts = [torch.rand_like(t).cuda().requires_grad_(True) for t in inputs]

    def program(f):
        for t in ts:
            t.grad = None
        y = f(*ts)
        (y * y).sum().backward()
        return [y.detach(), *[t.grad for t in ts]]

    step = lambda *a: 2 * call(*[t + 1 for t in a])  # noqa: E731
    want = program(step)
    for f in (torch.compile(step, backend="eager"), lambda *a: checkpoint(step, *a, use_reentrant=False),
              lambda *a: checkpoint(step, *a, use_reentrant=True)):
        for a, b in zip(program(f), want):
            assert bool(torch.equal(a, b))
