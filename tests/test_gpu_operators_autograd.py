"""What autograd, hooks, transforms and torch's lazy tensors may and may not do with rms_norm and
gated_linear, and with the 8-bit layers."""

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def same(a, b):
    return bool(torch.equal(a, b))


# name: (the inputs' shapes, the call on them, as a tuple of outputs)
CALLS = {
    "rms_norm": (((40, 24), (24,)), lambda L, x, w: (L.rms_norm(x, w),)),
    "rms_norm_residual": (((40, 24), (24,), (40, 24)), lambda L, x, w, r: L.rms_norm(x, w, r)),
    "gated_linear": (((40, 24), (16, 24), (16,)), lambda L, x, w, b: (L.gated_linear(x, w, b),)),
}
QUIET = {
    "rms_norm_8bit": lambda L, x: L.rms_norm_8bit(x, None, x)[1],
    "quantize_8bit": lambda L, x: L.quantize_8bit(x)[1],
    "linear_8bit": lambda L, x: L.linear_8bit(torch.zeros(3, 16, device=x.device).to(torch.float8_e4m3fn), x[:, 0],
                                              torch.zeros(8, 16, device=x.device).to(torch.float8_e4m3fn), torch.ones(8, device=x.device),
                                              dtype=torch.float32),
}


def inputs(name, grad=True):
    g = torch.Generator("cuda").manual_seed(3)
    return [torch.randn(*s, device="cuda", generator=g).requires_grad_(grad) for s in CALLS[name][0]]


def ups(outs):
    g = torch.Generator("cuda").manual_seed(4)
    return [torch.randn(o.shape, device="cuda", generator=g) for o in outs]


@pytest.mark.parametrize("grad_requires_grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_differentiating_a_gradient_again_raises(layers, name, grad_requires_grad):
    ts = inputs(name)
    outs = CALLS[name][1](layers, *ts)
    up = [u.requires_grad_(grad_requires_grad) for u in ups(outs)]
    want = torch.autograd.grad(outs, ts, [u.detach() for u in up], retain_graph=True)
    got = torch.autograd.grad(outs, ts, up, create_graph=True)
    for d, w, t in zip(got, want, ts):
        assert same(d.detach(), w) and d.requires_grad
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad((d * d).sum() + t.sum(), t, retain_graph=True)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t.half() if t.dtype == torch.float32 else t.double(), lambda t: t[:1],
                                    lambda t: t.to_sparse()], ids=["host", "type", "shape", "layout"])
def test_a_saved_tensor_that_comes_back_as_another(layers, name, which, change):
    ts, count = inputs(name), []

    def unpack(t):
        count.append(0)
        return change(t) if len(count) == which + 1 else t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        outs = CALLS[name][1](layers, *ts)
    with pytest.raises(RuntimeError, match="saved for a layer"):
        outs[0].sum().backward()


@pytest.mark.parametrize("name", CALLS)
def test_saved_tensors_may_be_moved_and_laid_out_anew(layers, name):
    ts = inputs(name)
    outs = CALLS[name][1](layers, *ts)
    up = ups(outs)
    want = torch.autograd.grad(outs, ts, up)

    def strided(t):
        if t.dim() == 2:
            return t.t().contiguous().t()
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        room[1:] = t  # not aligned
        return room[1:]

    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, strided)):
        with hooks:
            outs = CALLS[name][1](layers, *ts)
        for a, b in zip(torch.autograd.grad(outs, ts, up), want):
            assert same(a, b)


@pytest.mark.parametrize("change", [lambda t: t.half(), lambda t: t.cpu(), lambda t: t[:1]], ids=["type", "host", "shape"])
@pytest.mark.parametrize("name", CALLS)
def test_a_nodes_hook_that_changes_the_gradient(layers, name, change):
    ts = inputs(name)
    outs = CALLS[name][1](layers, *ts)
    outs[0].grad_fn.register_prehook(lambda g: (*g[:-1], change(g[-1])))
    with pytest.raises(RuntimeError):
        torch.autograd.backward(outs, ups(outs))


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_and_tracers_are_refused(layers, name):
    from torch.fx.experimental.proxy_tensor import make_fx

    ts = inputs(name, False)
    call = lambda *a: CALLS[name][1](layers, *a)[0]  # noqa: E731
    for i in range(len(ts)):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(*[forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(ts)])
    first = lambda x: call(x, *ts[1:]).sum()  # noqa: E731
    for transform in (lambda: torch.jit.trace(call, ts), lambda: make_fx(call)(*ts), lambda: torch.func.grad(first)(ts[0]),
                      lambda: torch.func.vmap(first)(torch.stack([ts[0], ts[0]])), lambda: torch.func.jvp(first, (ts[0],), (ts[0],))):
        with pytest.raises(RuntimeError):
            transform()
    leaf = ts[0].clone().requires_grad_(True)
    y = call(leaf, *ts[1:])
    with pytest.raises(RuntimeError):
        make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True))(torch.ones_like(y))


@pytest.mark.parametrize("name", QUIET)
def test_the_8_bit_layers_refuse_them_too(layers, name):
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.ones(3, 16, device="cuda")
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        QUIET[name](layers, forward_ad.make_dual(x, x))
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(lambda t: QUIET[name](layers, t), (x,), check_trace=False)
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(lambda t: QUIET[name](layers, t))(x)


@pytest.mark.parametrize("name", CALLS)
def test_compiled_and_checkpointed_programs_call_the_layers(layers, name):
    from torch.utils.checkpoint import checkpoint

    ts = inputs(name)

    def program(f):
        for t in ts:
            t.grad = None
        y = f(*ts)
        (y * y).sum().backward()
        return [y.detach(), *[t.grad for t in ts]]

    step = lambda *a: 2 * sum(o.sum() for o in CALLS[name][1](layers, *[t + 1 for t in a]))  # noqa: E731
    want = program(step)
    for f in (torch.compile(step, backend="eager"), lambda *a: checkpoint(step, *a, use_reentrant=False),
              lambda *a: checkpoint(step, *a, use_reentrant=True)):
        for a, b in zip(program(f), want):
            assert same(a, b)


def imag(t):
    """t as the imaginary part of a conjugate: a view with the negative bit, elements two apart."""
    v = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert v.is_neg()
    return v


@pytest.mark.parametrize("make", [lambda t: torch._neg_view(-t), imag])
@pytest.mark.parametrize("name", CALLS)
def test_negated_views(layers, name, make):
    ts = inputs(name)
    outs = CALLS[name][1](layers, *ts)
    up = ups(outs)
    want = torch.autograd.grad(outs, ts, up)
    for i in range(len(ts)):
        mixed = [make(t) if i == j else t for j, t in enumerate(ts)]
        z = CALLS[name][1](layers, *mixed)
        assert same(z[0], outs[0]), i
        for a, b in zip(torch.autograd.grad(z, ts, up), want):
            assert same(a, b), i
    for a, b in zip(torch.autograd.grad(CALLS[name][1](layers, *ts), ts, [make(u) for u in up]), want):
        assert same(a, b)


def test_negated_gradients_of_a_step():
    from diffrast import optim

    g = torch.randn(50, device="cuda")
    results = []
    for grad in (g, torch._neg_view(-g), imag(g)):
        p, m, v = (torch.ones(50, device="cuda") for _ in range(3))
        optim.adamw_step([p], [grad], [m], [v], torch.zeros(1, dtype=torch.int64, device="cuda"), lr=0.1)
        results.append(torch.stack([p, m, v]))
    assert same(results[0], results[1]) and same(results[0], results[2])
