"""Arrays of more than 2^31 elements: the last rows are those of a small call on them alone."""

import pytest
import torch

import operator_bounds as ob
from test_gpu_layers_large import BF, fill, give_back  # noqa: F401  (give_back: a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def test_rms_norm(layers):
    rows, D = (1 << 31) // 2048 + 1000, 2048
    x, res, g, gs = (fill(rows, D, i) for i in range(4))
    w = torch.randn(D, device="cuda").to(BF)
    q, scale, _ = layers.rms_norm_8bit(x[:, :], w, res)
    x.requires_grad_(True)
    y, s = layers.rms_norm(x, w, res)
    (dx,) = torch.autograd.grad([y, s], x, [g, gs])
    small = x.detach()[-700:].clone().requires_grad_(True)
    ys, ss = layers.rms_norm(small, w, res[-700:])
    (ds,) = torch.autograd.grad([ys, ss], small, [g[-700:], gs[-700:]])
    for a, b in ((y, ys), (s, ss), (dx, ds)):
        assert bool(torch.equal(a.detach()[-700:], b.detach()))
    qs, cs, _ = layers.rms_norm_8bit(x.detach()[-700:], w, res[-700:])
    assert bool(torch.equal(q.view(torch.uint8)[-700:], qs.view(torch.uint8))) and bool(torch.equal(scale[-700:], cs))


def test_gated_linear(layers):
    rows, N, K = (1 << 31) // 2056 + 1000, 2056, 64
    x = fill(rows, K, 3)
    w, b = (torch.randn(2 * N, K, device="cuda") / 8).to(BF), torch.randn(2 * N, device="cuda").to(BF)
    leaf = x.requires_grad_(True)
    y = layers.gated_linear(leaf, w, b)
    g = torch.ones((), dtype=BF, device="cuda").expand_as(y)
    (dx,) = torch.autograd.grad(y, leaf, g)
    want = ob.gated_linear(x.detach()[-300:], w, b, "silu", g[-300:])
    ob.check(y.detach()[-300:], *want["y"], BF, "y")
    ob.check(dx[-300:], *want["dx"], BF, "dx")


def test_linear_8bit(layers):
    rows, N, K = (1 << 31) // 4112 + 1000, 4112, 64
    x = torch.randint(0, 120, (rows, K), device="cuda", dtype=torch.uint8).view(ob.E4M3)
    w = torch.randint(0, 120, (N, K), device="cuda", dtype=torch.uint8).view(ob.E4M3)
    xs, ws = torch.rand(rows, device="cuda"), torch.rand(N, device="cuda")
    y = layers.linear_8bit(x, xs, w, ws)
    want = ob.linear_8bit(x[-300:], xs[-300:], w, ws, None, None, None, BF)
    ob.check(y[-300:], *want, BF, "y")


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(bits):
    from diffrast import optim

    n, part = (1 << 31) + 5000, 4096 + 5000
    kind = torch.float32 if bits == 32 else ob.E4M3
    p, g = fill(1, n, 1).view(-1), fill(1, n, 2).view(-1)
    m, v = (torch.zeros(n, dtype=kind, device="cuda") for _ in range(2))
    scales = [torch.zeros(-(-n // 256), device="cuda") for _ in range(2)] if bits == 8 else None
    old = p[-part:].clone()
    steps = torch.zeros(1, dtype=torch.int64, device="cuda")
    more = dict(exp_avg_scales=[scales[0]], exp_avg_sq_scales=[scales[1]]) if bits == 8 else {}
    optim.adamw_step([p], [g], [m], [v], steps, lr=0.1, **more)
    want = ob.adamw(old, g[-part:], torch.zeros_like(old), torch.zeros_like(old), 1, 0.1, 0.9, 0.999, 1e-8, 0.01)
    ob.check(p[-part:], *want["p"], BF, "p")
    if bits == 32:
        ob.check(m[-part:], *want["m"], torch.float32, "m")
    else:
        most = want["m"][0].abs().view(-1)[-(n % 256):].max() / 448
        assert abs(float(scales[0][-1]) - float(most)) <= 1e-6 * float(most)
