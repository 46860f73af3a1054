"""diffrast.layers.layer_norm against its plain form in 64 bits (layer_bounds.py)."""

import pytest
import torch

import layer_bounds as lb

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def same(a, b):
    return bool(torch.equal(a, b))


def make(rows, D, dtype, wdtype=None, weight=True, bias=True, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + rows + 5 * D)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    wd = wdtype or dtype
    x = r(rows, D) * (0.3 + torch.rand(D, device="cuda", generator=g)) + r(D)
    return dict(x=x.to(dtype), w=(1 + 0.1 * r(D)).to(wd) if weight else None, b=(0.1 * r(D)).to(wd) if bias else None,
                g=(0.25 * r(rows, D)).to(dtype))


def run(layers, t, eps=1e-5):
    leaves = {k: t[k] for k in ("x", "w", "b") if t[k] is not None}
    for v in leaves.values():
        v.requires_grad_(True)
    y = layers.layer_norm(t["x"], t["w"], t["b"], eps)
    grads = torch.autograd.grad(y, list(leaves.values()), t["g"])
    names = {"x": "dx", "w": "dweight", "b": "dbias"}
    return {"y": y.detach(), **{names[k]: d for k, d in zip(leaves, grads)}}


def compare(t, got, label, eps=1e-5):
    with torch.no_grad():
        want = lb.layer_norm(t["x"], t["w"], t["b"], eps, t["g"])
    for name, value in got.items():
        v, bound = want[name]
        dt = t["x"].dtype if name in ("y", "dx") else (t["w"] if t["w"] is not None else t["b"]).dtype
        lb.check(value.reshape(v.shape), v, bound, dt, f"{label} {name}")


# one element, one row, every vector width, every way a row is held (a wave, four waves, wider), odd sizes
SIZES = [(1, 1), (5, 1), (1, 64), (1, 1024), (7, 63), (33, 300), (129, 513), (1000, 75), (64, 1500), (50, 2048), (51, 2050),
         (40, 4096), (31, 5001), (20, 8192), (9, 8200), (3, 20001), (700, 8), (2100, 1030), (4099, 128)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,D", SIZES)
def test_forward_and_gradients(layers, rows, D, dtype):
    t = make(rows, D, dtype)
    compare(t, run(layers, t), f"{rows}x{D}")


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
def test_weights_in_32_bits_or_absent(layers, weight, bias, dtype):
    for D in (96, 2500, 9000):
        t = make(70, D, dtype, torch.float32, weight, bias)
        got = run(layers, t)
        assert ("dweight" in got) == weight and ("dbias" in got) == bias
        compare(t, got, f"{weight} {bias} {D}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_large_mean_does_not_cancel(layers, dtype):
    t = make(20, 768, dtype)
    with torch.no_grad():
        t["x"] += 1000.0
    compare(t, run(layers, t), "mean 1000")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_constant_rows(layers, dtype):
    """No variance: eps alone is left, and h is zero."""
    t = make(6, 200, dtype)
    with torch.no_grad():
        t["x"][:] = torch.tensor([0.0, 1.0, -3.0, 0.5, 100.0, 2.0], device="cuda")[:, None].to(dtype)
    got = run(layers, t)
    assert same(got["y"], t["b"].detach().expand(6, 200))
    assert same(got["dweight"], torch.zeros_like(got["dweight"]))
    compare(t, got, "constant")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_infinities_and_nan_stay_in_their_rows(layers, dtype):
    t = make(300, 520, dtype)
    with torch.no_grad():
        t["x"][11, 5], t["x"][200, 0] = float("nan"), float("inf")
    got = run(layers, t)
    rest = [i for i in range(300) if i not in (11, 200)]
    for i in (11, 200):
        assert bool(torch.isnan(got["y"][i]).all())
    assert bool(torch.isfinite(got["y"][rest].float()).all()) and bool(torch.isfinite(got["dx"][rest].float()).all())
    sub = {**t, "x": t["x"].detach()[rest], "g": t["g"][rest]}
    compare(sub, {"y": got["y"][rest], "dx": got["dx"][rest]}, "the other rows")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views(layers, dtype):
    """Column slices and expanded rows are read where they stand; other views are copied."""
    t = make(24, 136, dtype)
    want = run(layers, t)
    wide = torch.full((24, 300), float("nan"), dtype=dtype, device="cuda")
    for at in (8, 1):
        wide[:, at:at + 136] = t["x"].detach()
        leaf = wide.clone().requires_grad_(True)
        y = layers.layer_norm(leaf[:, at:at + 136], t["w"], t["b"])
        (d,) = torch.autograd.grad(y, leaf, t["g"])
        compare(t, {"y": y.detach(), "dx": d[:, at:at + 136]}, f"slice at {at}")
        assert not bool(d[:, :at].any()) and not bool(d[:, at + 136:].any())
    xt = t["x"].detach().t().contiguous().t()
    assert same(layers.layer_norm(xt, t["w"], t["b"]), want["y"])
    y = layers.layer_norm(t["x"].detach().view(2, 3, 4, 136), t["w"], t["b"])
    assert y.shape == (2, 3, 4, 136) and same(y.view(24, 136), want["y"])
    row = t["x"].detach()[3]
    assert same(layers.layer_norm(row.expand(5, 136), t["w"], t["b"]), want["y"][3].expand(5, 136))
    assert same(layers.layer_norm(row, t["w"], t["b"]), want["y"][3])
    # a gradient that is broadcast along the rows
    leaf = t["x"].detach().requires_grad_(True)
    g = t["g"][0].clone()
    (a,) = torch.autograd.grad(layers.layer_norm(leaf, t["w"], t["b"]), leaf, g.expand(24, 136))
    (b,) = torch.autograd.grad(layers.layer_norm(leaf, t["w"], t["b"]), leaf, g.expand(24, 136).contiguous())
    assert same(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_no_rows(layers, dtype):
    t = make(0, 40, dtype)
    got = run(layers, t)
    assert got["y"].shape == (0, 40) and got["dx"].shape == (0, 40)
    assert same(got["dweight"], torch.zeros_like(got["dweight"])) and same(got["dbias"], torch.zeros_like(got["dbias"]))


def test_same_bits_each_time(layers):
    t = make(3000, 1030, torch.bfloat16)
    a, b = run(layers, t), run(layers, t)
    for k in a:
        assert same(a[k], b[k]), k


def test_gradients_against_differences(layers):
    t = make(19, 57, torch.float32)
    got = run(layers, t)
    for name, key in (("x", "dx"), ("w", "dweight"), ("b", "dbias")):
        v = t[name].detach().double()
        d = torch.randn(v.shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(2))

        def f(s):
            u = {k: t[k].detach().double() for k in ("x", "w", "b")}
            u[name] = v + s * d
            c = u["x"] - u["x"].mean(1, keepdim=True)
            y = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * u["w"] + u["b"]
            return float((y * t["g"].double()).sum())

        want = (f(1e-4) - f(-1e-4)) / 2e-4
        have = float((got[key].double() * d).sum())
        # 2^-24 of each term's magnitude over ~1100 terms and h^2 of the third derivative
        assert abs(have - want) <= 1e-5 * float((got[key].double() * d).abs().sum()) + 1e-6, name


def test_other_stream_and_cpu_tensors(layers):
    t = make(100, 264, torch.bfloat16)
    want = layers.layer_norm(t["x"], t["w"], t["b"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layers.layer_norm(t["x"], t["w"], t["b"])
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want)
    y = layers.layer_norm(t["x"].cpu(), t["w"].cpu(), t["b"].cpu())
    assert y.device.type == "cpu" and same(y, want.cpu())


def test_graph_capture(layers):
    t = make(640, 1024, torch.bfloat16)
    for k in ("x", "w", "b"):
        t[k].requires_grad_(True)

    def step():
        y = layers.layer_norm(t["x"], t["w"], t["b"])
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
    ((torch.zeros(3, 0),), "x of shape"), ((torch.zeros(()),), "x of shape"), ((torch.zeros(3, 4), torch.zeros(5)), "weight"),
    ((torch.zeros(3, 4), None, torch.zeros(3, 4)), "bias"), ((torch.zeros(3, 4, dtype=torch.int32),), "float32"),
    ((torch.zeros(3, 4), torch.zeros(4, dtype=torch.bfloat16)), "weight"),
    ((torch.zeros(3, 4, dtype=torch.bfloat16), torch.zeros(4), torch.zeros(4, dtype=torch.bfloat16)), "bias"),
    ((torch.zeros(3, 4), None, None, -1.0), "eps"), ((torch.zeros(3, 4), None, None, float("nan")), "eps"),
])
def test_refusals(layers, args, error):
    with pytest.raises(ValueError, match=error):
        layers.layer_norm(*args)
