"""diffrast.layers.gated_linear against its plain form in 64 bits (operator_bounds.py)."""

import pytest
import torch

import operator_bounds as ob

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def same(a, b):
    return bool(torch.equal(a, b))


def make(M, K, N, dtype, bias=True, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + M + 7 * K + 31 * N)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return dict(x=r(M, K).to(dtype), w=(r(2 * N, K) / max(K, 1) ** 0.5).to(dtype), b=(0.3 * r(2 * N)).to(dtype) if bias else None,
                g=(0.25 * r(M, N)).to(dtype))


def run(layers, t, act):
    leaves = {k: t[k] for k in ("x", "w", "b") if t[k] is not None}
    for v in leaves.values():
        v.requires_grad_(True)
    y = layers.gated_linear(t["x"], t["w"], t["b"], act)
    grads = torch.autograd.grad(y, list(leaves.values()), t["g"])
    names = {"x": "dx", "w": "dweight", "b": "dbias"}
    return {"y": y.detach(), **{names[k]: d for k, d in zip(leaves, grads)}}


def compare(t, got, act, label):
    with torch.no_grad():
        want = ob.gated_linear(t["x"], t["w"], t["b"], act, t["g"])
    for name, value in got.items():
        v, bound = want[name]
        ob.check(value.reshape(v.shape), v, bound, t["x"].dtype, f"{label} {act} {name}")


# one of each, few rows (16, 32, 64) and one more, tiles of 64, 128 and 256 with edges, odd sizes,
# long sums in parts, k below and above where 32 bits are split
SIZES = [(1, 1, 1), (1, 8, 5), (1, 1024, 64), (3, 75, 17), (16, 64, 16), (17, 200, 33), (33, 96, 130), (64, 130, 15), (65, 9, 1),
         (65, 64, 31), (129, 33, 257), (300, 1000, 130), (257, 64, 513), (200, 5000, 20), (1031, 256, 515), (2500, 72, 1290),
         (40, 48, 2100), (90, 4096, 64)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_forward_and_gradients(layers, M, K, N, dtype):
    t = make(M, K, N, dtype)
    act = ACTS[(M + N) % 5]
    compare(t, run(layers, t, act), act, f"{M}x{K}x{N}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [True, False])
def test_activations(layers, act, bias, dtype):
    for M, K, N in ((5, 80, 24), (150, 72, 100), (700, 640, 257)):
        t = make(M, K, N, dtype, bias)
        with torch.no_grad():
            t["x"][::3] *= 6  # the activations' tails
        compare(t, run(layers, t, act), act, f"{M}x{K}x{N}")


# tiles of 256 (16 bits), as many as the card has CUs, with rows, outputs and k that end inside of them
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("K,N,bias", [(1032, 1980, True), (512, 1979, False), (75, 1976, True)])
def test_large_tiles(layers, K, N, bias, dtype):
    t = make(3900, K, N, dtype, bias)
    compare(t, run(layers, t, "silu"), "silu", "large")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_values_past_float16(layers, dtype):
    """What is kept of the gate and of the other half is unbounded: y and the gradients are finite where
    a gate of 1e-3 meets 1e5."""
    M, K, N = 70, 16, 24
    x = torch.zeros(M, K, device="cuda")
    x[:, 0] = 1.0
    w = torch.zeros(2 * N, K, device="cuda")
    w[:N, 0], w[N:, 0] = 1e-3, 300.0
    x[:, 1], w[N:, 1] = 300.0, 300.0
    t = dict(x=x.to(dtype), w=w.to(dtype), b=None, g=torch.full((M, N), 2.0**-12, device="cuda").to(dtype))
    for act in (None, "relu"):
        got = run(layers, t, act)
        assert all(bool(torch.isfinite(v.float()).all()) for v in (got["y"], got["dx"]))
        compare(t, {k: got[k] for k in ("y", "dx")}, act, "large")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_infinities_and_nan_are_the_formulas(layers, dtype):
    for M, K, N in ((8, 64, 40), (200, 128, 96)):
        t = make(M, K, N, dtype, False)
        with torch.no_grad():
            t["x"][3, 5], t["x"][7, 0] = float("nan"), float("inf")
        got = run(layers, t, "silu")
        rest = [i for i in range(M) if i not in (3, 7)]
        assert bool(torch.isnan(got["y"][3]).all()) and not bool(torch.isfinite(got["y"][7].float()).any())
        sub = {**t, "x": t["x"].detach()[rest], "g": t["g"][rest]}
        compare(sub, {k: got[k][rest] for k in ("y", "dx")}, "silu", "the other rows")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views(layers, dtype):
    """Slices of columns at any element, transposed weights, more dimensions, one row's stride."""
    t = make(100, 72, 48, dtype)
    want = run(layers, t, "gelu")
    for at in (8, 1):
        wide = torch.full((100, 200), float("nan"), dtype=dtype, device="cuda")
        wide[:, at:at + 72] = t["x"].detach()
        high = torch.full((96, 100), float("nan"), dtype=dtype, device="cuda")
        high[:, at:at + 72] = t["w"].detach()
        for x, w in ((wide[:, at:at + 72], t["w"]), (t["x"], high[:, at:at + 72]), (wide[:, at:at + 72], high[:, at:at + 72])):
            v = {**t, "x": x.detach(), "w": w.detach()}
            compare(v, run(layers, v, "gelu"), "gelu", f"slice at {at}")
    v = {**t, "w": t["w"].detach().t().contiguous().t()}
    got = run(layers, v, "gelu")
    assert same(got["y"], want["y"]) and same(got["dweight"], want["dweight"])
    y = layers.gated_linear(t["x"].detach().view(5, 20, 72), t["w"], t["b"], "gelu")
    assert y.shape == (5, 20, 48) and same(y.view(100, 48), want["y"])
    one = layers.gated_linear(t["x"].detach()[3], t["w"].detach(), t["b"].detach(), "gelu")
    assert one.shape == (48,)
    far = torch.randn(3, 72, device="cuda").to(dtype).as_strided((1, 72), (1 << 40, 1))
    assert layers.gated_linear(far, t["w"].detach()).shape == (1, 48)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", [(0, 40, 24), (30, 0, 24), (0, 0, 8)])
def test_nothing_to_sum(layers, M, K, N, dtype):
    t = make(M, K, N, dtype)
    got = run(layers, t, "silu")
    assert got["y"].shape == (M, N) and got["dx"].shape == (M, K) and got["dweight"].shape == (2 * N, K)
    compare(t, got, "silu", "empty")


def test_same_bits_each_time(layers):
    for dtype, (M, K, N) in ((torch.bfloat16, (3000, 520, 264)), (torch.float32, (500, 3000, 64)), (torch.float16, (90, 4096, 64))):
        t = make(M, K, N, dtype)
        a, b = run(layers, t, "silu"), run(layers, t, "silu")
        for k in a:
            assert same(a[k], b[k]), k


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(layers, act):
    t = make(19, 57, 23, torch.float32)
    if act == "relu":  # away from its corner
        with torch.no_grad():
            t["b"][:23] = torch.where(torch.arange(23, device="cuda") % 2 == 0, 20.0, -20.0)
    got = run(layers, t, act)
    for name, key in (("x", "dx"), ("w", "dweight"), ("b", "dbias")):
        d = torch.randn(t[name].shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(2))

        def f(e):
            u = {k: t[k].detach().double() for k in ("x", "w", "b")}
            u[name] = u[name] + e * d
            z = u["x"] @ u["w"].t() + u["b"]
            return float((ob.act(act, z[:, :23]) * z[:, 23:] * t["g"].double()).sum())

        want, have = (f(1e-5) - f(-1e-5)) / 2e-5, float((got[key].double() * d).sum())
        # each gradient is a sum of up to 57 terms within 2^-18 (activations' slopes), and h^2 of the third derivative
        assert abs(have - want) <= 2.0**-12 * float((got[key].double() * d).abs().sum()) + 1e-5, name


@pytest.mark.parametrize("wanted", ["x", "w", "b", "xw", "wb"])
def test_some_gradients(layers, wanted):
    for dtype in (torch.bfloat16, torch.float32):
        t = make(130, 75, 50, dtype)
        want = dict(zip("xwb", [run(layers, t, "silu")[k] for k in ("dx", "dweight", "dbias")]))
        leaves = {k: t[k].detach().clone().requires_grad_(k in wanted) for k in "xwb"}
        shapes = []
        with torch.autograd.graph.saved_tensors_hooks(lambda s: (shapes.append(tuple(s.shape)), s)[1], lambda s: s):
            y = layers.gated_linear(leaves["x"], leaves["w"], leaves["b"])
        kept = 130 * 50 * (8 if dtype == torch.float32 else 5)
        assert sorted(shapes) == sorted([(kept,)] + ([(130, 75)] if "w" in wanted else []) + ([(100, 75)] if "x" in wanted else []))
        y.backward(t["g"])
        for k, v in leaves.items():
            assert same(v.grad, want[k]) if k in wanted else v.grad is None, k


def test_other_stream_and_cpu_tensors(layers):
    t = make(100, 264, 72, torch.bfloat16)
    want = layers.gated_linear(t["x"], t["w"], t["b"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layers.gated_linear(t["x"], t["w"], t["b"])
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want)
    y = layers.gated_linear(t["x"].cpu(), t["w"].cpu(), t["b"].cpu())
    assert y.device.type == "cpu" and same(y, want.cpu())


def test_graph_capture(layers):
    t = make(640, 200, 328, torch.bfloat16)
    for k in "xwb":
        t[k].requires_grad_(True)

    def step():
        y = layers.gated_linear(t["x"], t["w"], t["b"])
        return [y.detach(), *torch.autograd.grad(y, [t["x"], t["w"], t["b"]], t["g"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            t["x"].copy_(torch.randn_like(t["x"]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert same(a, b), i


@pytest.mark.parametrize("args,error", [
    ((torch.zeros(3, 4), torch.zeros(6, 5)), "expected x"), ((torch.zeros(3, 4), torch.zeros(5, 4)), "expected x"),
    ((torch.zeros(3, 4), torch.zeros(0, 4)), "expected x"), ((torch.zeros(()), torch.zeros(2, 1)), "expected x"),
    ((torch.zeros(3, 4), torch.zeros(6, 4), torch.zeros(3)), "bias"), ((torch.zeros(3, 4), torch.zeros(6, 4), torch.zeros(6).half()), "bias"),
    ((torch.zeros(3, 4), torch.zeros(6, 4).half()), "weight"), ((torch.zeros(3, 4), torch.zeros(6, 4), None, "tanh"), "activation"),
    ((torch.zeros(3, 4).int(), torch.zeros(6, 4).int()), "float32"),
])
def test_refusals(layers, args, error):
    with pytest.raises(ValueError, match=error):
        layers.gated_linear(*args)
