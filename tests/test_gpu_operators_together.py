"""rms_norm, gated_linear, the 8-bit layers and AdamW together, as examples/amortize.py uses them."""

import pytest
import torch
import torch.nn.functional as F

from test_gpu_amortize import amortize  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", ["rms", "gated"])
def test_gradients_agree_with_torchs_own_layers(amortize, monkeypatch, block):  # noqa: F811
    """In 32 bits and without dropout, against the same network of torch's operations in 64."""
    from diffrast import layers

    net = amortize.TriangleMLP(size=32, width=64, blocks=2, triangles=5, dtype=torch.float32, block=block).cuda().eval()
    images = torch.rand(3, 3, 32, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    up = torch.randn(3, 5, 10, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    net(images).backward(up)
    got = {n: p.grad.clone() for n, p in net.named_parameters()}

    def linear(x, w, b=None, activation=None, residual=None):
        y = F.linear(x, w, b)
        y = F.gelu(y) if activation == "gelu" else y
        return y if residual is None else y + residual

    def rms_norm(x, w, residual=None):
        s = x if residual is None else x + residual
        y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5) * w
        return y if residual is None else (y, s)

    def gated_linear(x, w, b):
        a, c = F.linear(x, w, b).chunk(2, -1)
        return F.silu(a) * c

    for name, f in (("linear", linear), ("rms_norm", rms_norm), ("gated_linear", gated_linear)):
        monkeypatch.setattr(layers, name, f)
    net = net.double()
    net.dtype = torch.float64
    monkeypatch.setattr(torch.Tensor, "float", lambda t: t)
    net.zero_grad()
    net(images.double()).backward(up.double())
    for n, p in net.named_parameters():
        # 32-bit sums of up to 256 terms through eight layers: 2^-24 x 256 x 8 of the gradient's norm
        err = float((got[n].double() - p.grad).norm() / p.grad.norm())
        assert err < 1.3e-4, (n, err)


@pytest.mark.parametrize("block,states", [("rms", 32), ("gated", 32), ("gated", 8), ("mlp", 8)])
def test_training_runs(amortize, block, states):  # noqa: F811
    losses = amortize.train(4, batch=4, size=32, width=64, blocks=2, triangles=4, block=block, states=states)
    assert len(losses) == 4 and all(0 <= v < 10 for v in losses)


def test_answers_in_8_bits(amortize):  # noqa: F811
    """The scenes of a network whose blocks run in 8 bits, beside its own: the products' operands are
    within 2^-4 of themselves, so a block's addition to the stream is within about an eighth of itself,
    and most of that averages out."""
    net = amortize.TriangleMLP(size=32, width=128, blocks=3, triangles=6, block="rms").cuda().eval()
    images = torch.rand(5, 3, 32, 32, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    weights = net.weights_8bit()
    got = net.answer_8bit(images, weights)
    with torch.no_grad():
        want = net(images)
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    assert float((got - want).norm() / want.norm()) < 1 / 8
    # a captured answer follows its images
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = net.answer_8bit(images, weights)
    for seed in range(3):
        images.copy_(torch.rand(images.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert bool(torch.equal(out, net.answer_8bit(images, weights)))


def test_a_captured_training_step(amortize):  # noqa: F811
    """Norm, gated feed-forward, their gradients and the optimiser's step in one graph, against the same steps
    made eagerly."""
    from diffrast import layers, optim

    def start():
        g = torch.Generator("cuda").manual_seed(1)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        leaves = [torch.ones(64, device="cuda"), 0.1 * r(256, 64), 0.1 * r(64, 128)]
        leaves = [t.requires_grad_(True) for t in leaves]
        for t in leaves:
            t.grad = torch.zeros_like(t)
        return leaves, optim.AdamW(leaves, lr=1e-2, state_bits=8, seed=3), r(40, 64), r(40, 64)

    def step(leaves, opt, x, stream):
        y, s = layers.rms_norm(x, leaves[0], residual=stream)
        h = layers.linear(layers.gated_linear(y, leaves[1]), leaves[2], residual=s)
        for t, d in zip(leaves, torch.autograd.grad((h * h).mean(), leaves)):
            t.grad.copy_(d)
        opt.step()

    a, b = start(), start()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*a)
    torch.cuda.current_stream().wait_stream(side)
    step(*b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*a)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        step(*b)
        for p, q in zip(a[0], b[0]):
            assert bool(torch.equal(p, q)), i


def chain(seed):
    """Inputs of a chain of all layers whose products are split (workspaces of partial sums), and the chain."""
    from diffrast import layers

    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g, dtype=torch.bfloat16)  # noqa: E731
    x, res, w, w8 = r(100, 2048), r(100, 2048), 0.02 * r(256, 2048), 0.1 * r(96, 128)
    q8, s8 = layers.quantize_8bit(w8)
    for t in (x, w):
        t.requires_grad_(True)

    def run():
        y, s = layers.rms_norm(x, None, residual=res)
        h = layers.gated_linear(y, w)
        gx, gw = torch.autograd.grad((h.float().square().sum() + s.float().sum()), (x, w))
        with torch.no_grad():
            a, t = layers.rms_norm_8bit(h)
            return h.detach(), gx, gw, layers.linear_8bit(a, t, q8, s8, activation="gelu")

    return run


def test_two_threads_on_two_streams():
    import threading

    runs = [chain(1), chain(2)]
    want = [f() for f in runs]
    torch.cuda.synchronize()
    wrong = [[], []]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for k in range(10):
                got = runs[i]()
                stream.synchronize()
                wrong[i] += [(k, j) for j, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a.view(torch.int16), b.view(torch.int16))]
        wrong[i].append("done")

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [["done"], ["done"]]


def test_two_captured_chains_of_one_memory_pool():
    runs = [chain(1), chain(2)]
    want = [f() for f in runs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f in runs:
            f()
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [torch.cuda.CUDAGraph() for _ in runs], []
    for k, f in enumerate(runs):
        with torch.cuda.graph(graphs[k], pool=graphs[0].pool() if k else None):
            got.append(f())
    for i in range(4):
        for graph, out, ref in zip(graphs, got, want):  # a graph's workspaces may be the other's outputs: one at a time
            graph.replay()
            torch.cuda.synchronize()
            assert all(bool(torch.equal(a.view(torch.int16), b.view(torch.int16))) for a, b in zip(out, ref)), i
        runs[i % 2]()
