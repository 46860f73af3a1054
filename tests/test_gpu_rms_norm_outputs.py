"""Which of rms_norm's outputs depend on which of its inputs."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wants", ["x", "weight", "residual", "x weight", "weight residual", ""])
def test_what_requires_a_gradient(wants, dtype):
    """The sum is no function of the weight."""
    from diffrast import layers

    g = torch.Generator("cuda").manual_seed(0)
    t = {k: torch.randn(s, device="cuda", generator=g).to(dtype) for k, s in (("x", (9, 40)), ("weight", (40,)), ("residual", (9, 40)))}
    up = [torch.randn(9, 40, device="cuda", generator=g).to(dtype) for _ in range(2)]
    whole = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    want = dict(zip(t, torch.autograd.grad(layers.rms_norm(whole["x"], whole["weight"], whole["residual"]), list(whole.values()), up)))
    for k in wants.split():
        t[k].requires_grad_(True)
    y, s = layers.rms_norm(t["x"], t["weight"], t["residual"])
    data = "x" in wants or "residual" in wants
    assert y.requires_grad == bool(wants) and s.requires_grad == data
    if wants:
        outs, ups = ([y, s], up) if data else ([y], up[:1])
        for k, d in zip(wants.split(), torch.autograd.grad(outs, [t[k] for k in wants.split()], ups)):
            assert torch.equal(d, want[k]), k


def test_a_stream_that_needs_no_gradient_is_kept_safe():
    from diffrast import layers

    x, w = torch.randn(5, 16, device="cuda"), torch.ones(16, device="cuda", requires_grad=True)
    y, s = layers.rms_norm(x, w, x)
    s += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
