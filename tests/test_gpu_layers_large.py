"""Arrays of more than 2^31 elements: the last rows are those of a small call on them alone."""

import pytest
import torch

import layer_bounds as lb

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def fill(rows, cols, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = torch.empty(rows, cols, dtype=BF, device="cuda")
    step = max(1, (1 << 28) // cols)
    for i in range(0, rows, step):
        t[i:i + step] = torch.randn(min(step, rows - i), cols, device="cuda", generator=g).to(BF)
    return t


def test_layer_norm(layers):
    rows, D = (1 << 31) // 2048 + 1000, 2048
    x, g = fill(rows, D, 1), fill(rows, D, 2)
    w = torch.randn(D, device="cuda").to(BF)
    leaf = x.requires_grad_(True)
    y = layers.layer_norm(leaf, w)
    (dx,) = torch.autograd.grad(y, leaf, g)
    small = x.detach()[-700:].clone().requires_grad_(True)
    ys = layers.layer_norm(small, w)
    (ds,) = torch.autograd.grad(ys, small, g[-700:])
    assert bool(torch.equal(y.detach()[-700:], ys.detach())) and bool(torch.equal(dx[-700:], ds))


def test_linear(layers):
    rows, N, K = (1 << 31) // 4104 + 1000, 4104, 64
    x = fill(rows, K, 3)
    w, b = (torch.randn(N, K, device="cuda") / 8).to(BF), torch.randn(N, device="cuda").to(BF)
    leaf = x.requires_grad_(True)
    y = layers.linear(leaf, w, b, "gelu")
    g = torch.ones((), dtype=BF, device="cuda").expand_as(y)
    (dx,) = torch.autograd.grad(y, leaf, g)
    t = dict(x=x.detach()[-300:], w=w, b=b)
    want = lb.linear(t["x"], w, b, "gelu", None, g[-300:])
    lb.check(y.detach()[-300:], *want["y"], BF, "y")
    lb.check(dx[-300:], *want["dx"], BF, "dx")


def test_dropout(layers):
    n = (1 << 32) + 777
    x = torch.ones(n, dtype=BF, device="cuda")
    y = layers.dropout(x, 0.25, seed=8, offset=1)
    # the counters past 2^29 name the last elements' bits
    last = lb.philox_keep(1000, 0.25, 8, 1, first=n - 1000).cuda()
    assert bool(torch.equal(y[-1000:] != 0, last))
