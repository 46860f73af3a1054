"""The layers together as examples/amortize.py uses them: a network that answers with
triangles, trained through the rasterizer."""

import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def amortize():
    path = Path(__file__).resolve().parents[1] / "examples" / "amortize.py"
    spec = importlib.util.spec_from_file_location("amortize", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_training_lowers_the_loss(amortize):
    losses = amortize.train(60, batch=8, width=128, blocks=2, triangles=16)
    assert all(v == v for v in losses)
    assert sum(losses[-10:]) < 0.8 * sum(losses[:10]), (losses[:3], losses[-3:])


def test_same_seed_same_losses(amortize):
    kw = dict(batch=4, width=64, blocks=1, triangles=4, size=32)
    a, b = amortize.train(3, **kw), amortize.train(3, **kw)
    # the rasterizer's gradients are summed by atomics: the first loss is before any of them
    assert a[0] == b[0] and max(abs(x - y) for x, y in zip(a, b)) < 1e-3


def test_gradients_agree_with_torchs_own_layers(amortize, monkeypatch):
    """In 32 bits and without dropout, against the same network of torch's operations in 64."""
    from diffrast import layers

    net = amortize.TriangleMLP(size=32, width=64, blocks=2, triangles=5, dtype=torch.float32).cuda().eval()
    images = torch.rand(3, 3, 32, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    up = torch.randn(3, 5, 10, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    net(images).backward(up)
    got = {n: p.grad.clone() for n, p in net.named_parameters()}

    def linear(x, w, b=None, activation=None, residual=None):
        y = F.linear(x, w, b)
        y = F.gelu(y) if activation == "gelu" else y
        return y if residual is None else y + residual

    monkeypatch.setattr(layers, "linear", linear)
    monkeypatch.setattr(layers, "layer_norm", lambda x, w, b: F.layer_norm(x, x.shape[-1:], w, b, 1e-5))
    net = net.double()
    net.dtype = torch.float64
    monkeypatch.setattr(torch.Tensor, "float", lambda t: t)
    net.zero_grad()
    net(images.double()).backward(up.double())
    for n, p in net.named_parameters():
        # 32-bit sums of up to 256 terms through eight layers: 2^-24 x 256 x 8 of the gradient's norm
        err = float((got[n].double() - p.grad).norm() / p.grad.norm())
        assert err < 1.3e-4, (n, err)
