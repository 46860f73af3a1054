"""diffrast.layers.linear against its plain form in 64 bits (layer_bounds.py)."""

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


def make(M, N, K, dtype, bias=True, res=False, seed=0, lead=None):
    g = torch.Generator("cuda").manual_seed(seed + M + 3 * N + 7 * K)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    lead = (M,) if lead is None else lead
    return dict(x=r(*lead, K).to(dtype), w=(r(N, K) / max(K, 1) ** 0.5).to(dtype),
                b=(0.1 * r(N)).to(dtype) if bias else None, res=r(*lead, N).to(dtype) if res else None,
                g=(0.25 * r(*lead, N)).to(dtype))


def run(layers, t, kind, train=True):
    leaves = {k: t[k] for k in ("x", "w", "b", "res") if t[k] is not None}
    if train:
        for v in leaves.values():
            v.requires_grad_(True)
    y = layers.linear(t["x"], t["w"], t["b"], activation=kind, residual=t["res"])
    if not train:
        return {"y": y}
    grads = torch.autograd.grad(y, list(leaves.values()), t["g"])
    names = {"x": "dx", "w": "dweight", "b": "dbias", "res": "dres"}
    return {"y": y.detach(), **{names[k]: d for k, d in zip(leaves, grads)}}


def same(a, b):
    return bool(torch.equal(a, b))


def compare(t, kind, got, label):
    with torch.no_grad():
        want = lb.linear(t["x"].detach(), t["w"].detach(), t["b"], kind, t["res"], t["g"] if "dx" in got else None)
    for name, (value, bound) in want.items():
        if name not in got:
            continue
        lb.check(got[name].reshape(value.shape), value, bound, t["x"].dtype, f"{label} {name}")
    if "dres" in got:
        assert same(got["dres"], t["g"])


# one token; a few; ragged tiles of every kernel; widths that are and are not whole 16-byte chunks
SIZES = [(1, 10, 1), (1, 1500, 1024), (3, 1280, 75), (16, 1280, 1024), (17, 33, 31), (64, 64, 64), (65, 130, 257),
         (130, 100, 48), (257, 320, 200), (300, 1501, 75), (1000, 10, 520), (33, 2056, 1032)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_forward_and_gradients(layers, M, N, K, dtype):
    kind = lb.ACTS[(M + N + K) % 5]
    t = make(M, N, K, dtype, bias=(M + K) % 3 != 0, res=N % 2 == 0)
    compare(t, kind, run(layers, t, kind), f"{M}x{N}x{K} {kind}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind", lb.ACTS)
def test_activations(layers, kind, dtype):
    # arguments from far below to far above the activations' bends
    t = make(96, 72, 40, dtype, res=True)
    t["x"] = (t["x"].float() * torch.logspace(-3, 1.5, 96, device="cuda")[:, None]).to(dtype)
    compare(t, kind, run(layers, t, kind), str(kind))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(4100, 4104, 200), (8200, 2056, 72), (2056, 8, 4104)])
def test_large_ragged(layers, M, N, K, dtype):
    """Tiles past every edge of many whole ones, in each of the three products."""
    t = make(M, N, K, dtype, res=True)
    compare(t, "gelu", run(layers, t, "gelu"), f"{M}x{N}x{K}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(512, 256, 8192), (20000, 136, 104)])
def test_long_sums(layers, M, N, K, dtype):
    """Few outputs and a long contraction, which is split and joined."""
    t = make(M, N, K, dtype)
    compare(t, None, run(layers, t, None), f"{M}x{N}x{K}")


def test_same_bits_each_time(layers):
    t = make(700, 520, 2048, torch.bfloat16, res=True)
    a, b = run(layers, t, "silu"), run(layers, t, "silu")
    for k in a:
        assert same(a[k], b[k]), k


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views_and_leading_dimensions(layers, dtype):
    """Column slices keep their row stride, other views are copied, leading dimensions stay."""
    t = make(60, 40, 48, dtype, res=True, lead=(4, 15))
    want = run(layers, {**t}, "gelu", train=False)["y"]
    compare(t, "gelu", {"y": want}, "leading dimensions")
    wide = torch.full((60, 100), float("nan"), dtype=dtype, device="cuda")
    for at in (16, 3):
        wide[:, at:at + 48] = t["x"].detach().reshape(60, 48)
        y = layers.linear(wide[:, at:at + 48], t["w"], t["b"], "gelu", t["res"].reshape(60, 40))
        compare({**t, "x": t["x"].reshape(60, 48), "res": t["res"].reshape(60, 40)}, "gelu", {"y": y}, f"slice at {at}")
    xt = t["x"].detach().transpose(0, 1).contiguous().transpose(0, 1)
    assert same(layers.linear(xt, t["w"], t["b"], "gelu", t["res"]), want)
    wt = t["w"].detach().t().contiguous().t()
    assert same(layers.linear(t["x"], wt, t["b"], "gelu", t["res"]), want)
    one = t["x"].detach()[0, 0]
    y = layers.linear(one, t["w"], t["b"], "gelu", t["res"][0, 0])
    assert y.shape == (40,)
    compare({**t, "x": one, "res": t["res"][0, 0]}, "gelu", {"y": y}, "vector")
    # a residual and a gradient that are broadcast
    res = t["res"].detach()[:1, :1].clone().requires_grad_(True)
    y = layers.linear(t["x"], t["w"], None, None, res.expand(4, 15, 40))
    (d,) = torch.autograd.grad(y.sum(), res)
    assert same(d, torch.full_like(d, 60.0))


def test_misaligned_start(layers):
    for dtype in DTYPES:
        t = make(40, 64, 64, dtype, res=True)
        flat = torch.zeros(40 * 64 + 1, dtype=dtype, device="cuda")
        flat[1:] = t["x"].reshape(-1)
        t["x"] = flat[1:].view(40, 64)
        compare(t, "relu", run(layers, t, "relu"), "misaligned")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_empty(layers, dtype):
    t = make(0, 16, 24, dtype, res=True)
    got = run(layers, t, "gelu")
    assert got["y"].shape == (0, 16) and got["dx"].shape == (0, 24)
    assert same(got["dweight"], torch.zeros(16, 24, dtype=dtype, device="cuda"))
    assert same(got["dbias"], torch.zeros(16, dtype=dtype, device="cuda"))
    # no features: the bias alone
    t = make(5, 16, 0, dtype)
    got = run(layers, t, "relu")
    assert same(got["y"], t["b"].detach().clamp(min=0).expand(5, 16))
    assert got["dx"].shape == (5, 0) and got["dweight"].shape == (16, 0)


@pytest.mark.parametrize("kind", lb.ACTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_infinities_and_nan_stay_in_their_rows(layers, kind, dtype):
    t = make(300, 136, 64, dtype)
    x = t["x"].detach()
    x[7, 3], x[100, 0] = float("nan"), float("inf")
    got = run(layers, t, kind)
    y = got["y"].float()
    assert bool(torch.isnan(y[7]).all())
    w0 = t["w"].detach()[:, 0].float()
    assert bool((y[100][w0 > 0] == float("inf")).all())
    if kind is None:
        assert bool((y[100][w0 < 0] == -float("inf")).all())
    else:
        assert bool((y[100][w0 < 0].abs() == 0).all())
    rest = [i for i in range(300) if i not in (7, 100)]
    assert bool(torch.isfinite(y[rest]).all()) and bool(torch.isfinite(got["dx"][rest].float()).all())
    sub = {k: (v.detach()[rest] if k in ("x", "g") else v) for k, v in t.items()}
    compare(sub, kind, {"y": got["y"][rest]}, "the other rows")


def test_gradients_against_differences(layers):
    """The gradients' own definition: (f(t + h d) - f(t - h d)) / 2h along a direction d."""
    for kind in lb.ACTS:
        if kind == "relu":
            continue
        t = make(37, 29, 41, torch.float32, res=True, seed=5)
        got = run(layers, t, kind)
        for name, key in (("x", "dx"), ("w", "dweight"), ("b", "dbias")):
            v = t[name].detach().double()
            d = torch.randn(v.shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(3))
            h = 1e-4

            def f(s):
                u = {**t, name: v + s * d}
                z = u["x"].detach().double() @ u["w"].detach().double().t() + u["b"].detach().double()
                return float((lb.act(kind, z) * t["g"].double()).sum())

            want = (f(h) - f(-h)) / (2 * h)
            have = float((got[key].double() * d).sum())
            # 2^-24 of each term's magnitude over ~1500 terms and h^2 of the third derivative
            assert abs(have - want) <= 1e-5 * float((got[key].double() * d).abs().sum()) + 1e-6, (kind, name)


def test_needs_only_what_is_asked(layers):
    t = make(50, 24, 32, torch.float32)
    for want in ("x", "w", "b"):
        u = {k: v.detach().clone().requires_grad_(k == want) if v is not None and k in ("x", "w", "b") else v
             for k, v in t.items()}
        y = layers.linear(u["x"], u["w"], u["b"], "silu")
        y.backward(t["g"])
        ref = run(layers, {**t}, "silu")
        assert same(u[want].grad, ref[{"x": "dx", "w": "dweight", "b": "dbias"}[want]])
        assert all(u[k].grad is None for k in ("x", "w", "b") if k != want)


def test_other_stream_and_cpu_tensors(layers):
    t = make(200, 72, 96, torch.bfloat16, res=True)
    want = run(layers, {**t}, "gelu", train=False)["y"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layers.linear(t["x"], t["w"], t["b"], "gelu", t["res"])
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want)
    c = {k: v.detach().cpu() for k, v in t.items()}
    y = layers.linear(c["x"], c["w"], c["b"], "gelu", c["res"])
    assert y.device.type == "cpu" and same(y, want.cpu())


def test_graph_capture(layers):
    """Forward and backward in a HIP graph: every replay as the eager call on the same values."""
    t = make(520, 264, 1096, torch.bfloat16, res=True)
    for k in ("x", "w", "b", "res"):
        t[k].requires_grad_(True)
    leaves = [t["x"], t["w"], t["b"]]

    def step():
        y = layers.linear(t["x"], t["w"], t["b"], "gelu", t["res"])
        return [y.detach(), *torch.autograd.grad(y, leaves, t["g"])]

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


@pytest.mark.parametrize("change,error", [
    (dict(w=torch.zeros(4, 9)), "weight"), (dict(w=torch.zeros(8)), "weight"), (dict(b=torch.zeros(5)), "bias"),
    (dict(res=torch.zeros(3, 5)), "residual"), (dict(res=torch.zeros(2, 4)), "residual"), (dict(kind="tanh"), "activation"),
    (dict(w=torch.zeros(4, 8, dtype=torch.bfloat16)), "weight"), (dict(b=torch.zeros(4, dtype=torch.float16)), "bias"),
    (dict(x=torch.zeros(3, 8, dtype=torch.float64)), "float32"), (dict(w=torch.zeros(0, 8)), "weight"),
])
def test_refusals(layers, change, error):
    t = dict(x=torch.zeros(3, 8), w=torch.zeros(4, 8), b=torch.zeros(4), res=torch.zeros(3, 4), kind=None)
    t.update(change)
    with pytest.raises(ValueError, match=error):
        layers.linear(t["x"], t["w"], t["b"], t["kind"], t["res"])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("K", [64, 72, 96, 128, 136, 160, 192, 224, 320, 328])
def test_k_tiles_in_turn(layers, K, dtype):
    """Two groups of waves share an odd or even number of k tiles, whole or not; M in place of K in dW."""
    t = make(200, 136, K, dtype, res=True)
    compare(t, "silu", run(layers, t, "silu"), f"200x136x{K}")
    t = make(K, 136, 200, dtype)
    compare(t, None, run(layers, t, None), f"{K}x136x200")


@pytest.mark.parametrize("M,N", [(200, 136), (2100, 1160)])
def test_infinities_in_every_k_tile(layers, M, N):
    """One infinity a row, in any tile of k, alone and against one of the other sign in the next tile."""
    K = 200
    t = make(M, N, K, torch.float32, bias=False)
    x, w = t["x"].detach(), t["w"].detach()
    inf = float("inf")
    at = {3: (0,), 70: (31,), 71: (32,), 130: (101,), 190: (199,), 64: (5, 40), 127: (130, 170), M - 1: (64, 96)}
    for row, ks in at.items():
        for k in ks:
            x[row, k] = inf
    y = run(layers, t, None, train=False)["y"]
    for row, ks in at.items():
        sign = w[:, list(ks)].sign()
        want = torch.where((sign == sign[:, :1]).all(1), sign[:, 0] * inf, float("nan"))
        assert bool(torch.isclose(y[row], want, rtol=0, atol=0, equal_nan=True).all()), row
    rest = [i for i in range(M) if i not in at]
    clean = {k: v for k, v in t.items()}
    clean["x"] = x[rest].clone()
    compare(clean, None, {"y": y[rest]}, "other rows")
