"""diffrast.layers.rms_norm, rms_norm_8bit and quantize_8bit against their plain forms in 64 bits
(operator_bounds.py)."""

import pytest
import torch

import operator_bounds as ob

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


def same(a, b):
    return bool(torch.equal(a, b))


def make(rows, D, dtype, wdtype=None, weight=True, res=True, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + rows + 5 * D)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = r(rows, D) * (0.3 + torch.rand(D, device="cuda", generator=g)) + r(D)
    return dict(x=x.to(dtype), w=(1 + 0.1 * r(D)).to(wdtype or dtype) if weight else None,
                res=r(rows, D).to(dtype) if res else None, g=(0.25 * r(rows, D)).to(dtype), gs=(0.25 * r(rows, D)).to(dtype))


def run(layers, t, eps=1e-5):
    leaves = {k: t[k] for k in ("x", "w", "res") if t[k] is not None}
    for v in leaves.values():
        v.requires_grad_(True)
    r = layers.rms_norm(t["x"], t["w"], t["res"], eps)
    outs, ups = ([r], [t["g"]]) if t["res"] is None else (list(r), [t["g"], t["gs"]])
    grads = torch.autograd.grad(outs, list(leaves.values()), ups)
    names = {"x": "dx", "w": "dweight", "res": "dres"}
    got = {"y": outs[0].detach(), **{names[k]: d for k, d in zip(leaves, grads)}}
    if t["res"] is not None:
        got["sum"] = outs[1].detach()
    return got


def compare(t, got, label, eps=1e-5):
    with torch.no_grad():
        want = ob.rms_norm(t["x"], t["w"], t["res"], eps, t["g"], t["gs"] if t["res"] is not None else None)
    for name, value in got.items():
        v, bound = want["dx" if name == "dres" else name]
        dt = t["w"].dtype if name == "dweight" else t["x"].dtype
        ob.check(value.reshape(v.shape), v, bound, dt, f"{label} {name}")


# one element, one row, every vector width, every way a row is held and past them, odd sizes
SIZES = [(1, 1), (5, 1), (1, 64), (1, 1024), (7, 63), (33, 300), (129, 513), (1000, 75), (64, 1500), (50, 2048), (51, 2050),
         (40, 4096), (31, 5001), (20, 8192), (9, 8200), (7, 16384), (5, 16500), (4, 32768), (3, 32801), (700, 8), (2100, 1030), (4099, 128)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,D", SIZES)
def test_forward_and_gradients(layers, rows, D, dtype):
    for res in (True, False):
        t = make(rows, D, dtype, res=res)
        compare(t, run(layers, t), f"{rows}x{D}")


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("weight", [True, False])
def test_weight_in_32_bits_or_absent(layers, weight, dtype):
    for D in (96, 2500, 9000, 40000):
        for res in (True, False):
            t = make(70, D, dtype, torch.float32, weight, res)
            compare(t, run(layers, t), f"{weight} {res} {D}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,D", SIZES)
def test_8bit(layers, rows, D, dtype):
    t = make(rows, D, dtype)
    for w, res in ((t["w"], t["res"]), (None, None), (t["w"], None)):
        want = ob.rms_norm(t["x"], w, res, 1e-5)
        r = layers.rms_norm_8bit(t["x"], w, res)
        assert len(r) == (2 if res is None else 3)
        ob.check_8bit(r[0], r[1], *want["y"], f"{rows}x{D}")
        if res is not None:
            ob.check(r[2], *want["sum"], dtype, "sum")
            assert same(r[2], layers.rms_norm(t["x"], w, res)[1])
    q, s = layers.quantize_8bit(t["x"])
    ob.check_8bit(q, s, t["x"].double(), torch.zeros(rows, D, dtype=torch.float64, device="cuda"), "rows")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_8bit_rows_of_zeros_tiny_and_large_numbers(layers, dtype):
    big = {torch.float32: 1e37, torch.bfloat16: 1e37, torch.float16: 60000.0}[dtype]
    small = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 6e-8}[dtype]
    scale = torch.tensor([0.0, small, big, 1.0, 448.0], device="cuda", dtype=torch.float64)[:, None]
    x = (torch.linspace(-1, 1, 200, device="cuda", dtype=torch.float64) * scale).to(dtype)
    q, s = layers.quantize_8bit(x)
    ob.check_8bit(q, s, x.double(), torch.zeros(5, 200, dtype=torch.float64, device="cuda"), "rows")
    assert not bool(q[0].float().any()) and bool((s > 0).all())
    x[1, 3], x[2, 4], x[3, 5] = float("nan"), float("inf"), -float("inf")
    q, s = layers.quantize_8bit(x)
    assert bool(torch.isnan(q[1, 3].float())) and bool(torch.isnan(q[2, 4].float())) and bool(torch.isnan(q[3, 5].float()))
    bad = torch.isnan(q.float())
    assert int(bad.sum()) == 3


def test_8bit_rounds_to_nearest_even(layers):
    """A row whose scale is 1: each of e4m3's numbers, and what lies between two of them."""
    grid = torch.arange(127, dtype=torch.uint8).view(ob.E4M3).float()
    mid = (grid[1:] + grid[:-1]) / 2
    x = torch.cat([grid, mid, -grid, -mid]).cuda()
    q, s = layers.quantize_8bit(x[None])
    assert float(s[0]) == 1.0
    want = torch.cat([grid, torch.where((torch.arange(126) % 2) == 0, grid[:-1], grid[1:])])
    assert same(q[0].float().cpu(), torch.cat([want, -want]))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_of_zeros(layers, dtype):
    """eps alone is left."""
    t = make(6, 200, dtype, res=False)
    t["x"][2] = 0
    got = run(layers, t)
    assert not bool(got["y"][2].any())
    compare(t, got, "zeros")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_infinities_and_nan_stay_in_their_rows(layers, dtype):
    t = make(300, 520, dtype)
    t["x"][11, 5], t["x"][200, 0] = float("nan"), float("inf")
    got = run(layers, t)
    rest = [i for i in range(300) if i not in (11, 200)]
    assert bool(torch.isnan(got["y"][11]).all()) and bool(torch.isnan(got["y"][200, 0]))
    sub = {**t, **{k: t[k].detach()[rest] for k in ("x", "res", "g", "gs")}}
    compare(sub, {k: got[k][rest] for k in ("y", "dx", "dres", "sum")}, "the other rows")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views(layers, dtype):
    """Column slices and expanded rows are read where they stand; other views are copied."""
    t = make(24, 136, dtype)
    want = run(layers, t)
    bare = {k: t[k].detach() for k in ("x", "w", "res")}
    wide = torch.full((24, 300), float("nan"), dtype=dtype, device="cuda")
    for at in (8, 1):
        for name in ("x", "res"):
            leaf = wide.clone()
            leaf[:, at:at + 136] = bare[name]
            leaf.requires_grad_(True)
            args = {**bare, name: leaf[:, at:at + 136]}
            y, s = layers.rms_norm(args["x"], args["w"], args["res"])
            assert same(y, want["y"]) and same(s, want["sum"])
            (d,) = torch.autograd.grad([y, s], leaf, [t["g"], t["gs"]])
            assert same(d[:, at:at + 136], want["dx"]) and not bool(d[:, :at].any()) and not bool(d[:, at + 136:].any())
            if name == "x":
                q, c, s = layers.rms_norm_8bit(args["x"].detach(), args["w"], args["res"])
                q2, c2, s2 = layers.rms_norm_8bit(bare["x"], bare["w"], bare["res"])
                assert same(q.view(torch.uint8), q2.view(torch.uint8)) and same(c, c2) and same(s, s2)
    xt = bare["x"].t().contiguous().t()
    assert same(layers.rms_norm(xt, bare["w"], bare["res"])[0], want["y"])
    y, s = layers.rms_norm(bare["x"].view(2, 3, 4, 136), bare["w"], bare["res"].view(2, 3, 4, 136))
    assert y.shape == s.shape == (2, 3, 4, 136) and same(y.view(24, 136), want["y"])
    q, c = layers.rms_norm_8bit(bare["x"].view(2, 12, 136))
    assert q.shape == (2, 12, 136) and c.shape == (2, 12)
    row = bare["x"][3]
    alone = layers.rms_norm(row, bare["w"])
    assert alone.shape == (136,) and same(layers.rms_norm(row.expand(5, 136), bare["w"]), alone.expand(5, 136))
    q, c = layers.quantize_8bit(row)
    assert q.shape == (136,) and c.shape == ()
    # gradients that are broadcast along the rows
    leaf = bare["x"].requires_grad_(True)
    for gs in (t["gs"], None):
        r = layers.rms_norm(leaf, bare["w"], bare["res"] if gs is not None else None)
        outs = list(r) if gs is not None else [r]
        ups = [t["g"][0].expand(24, 136)] + ([gs[1].expand(24, 136)] if gs is not None else [])
        (a,) = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
        (b,) = torch.autograd.grad(outs, leaf, [u.contiguous() for u in ups])
        assert same(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_one_output_used(layers, dtype):
    """The gradient of y alone, and of the sum alone, which goes straight to x and residual."""
    t = make(40, 72, dtype)
    both = run(layers, t)
    y, s = layers.rms_norm(t["x"], t["w"], t["res"])
    dx, dr, dw = torch.autograd.grad(s, [t["x"], t["res"], t["w"]], t["gs"], retain_graph=True)
    assert same(dx, t["gs"]) and same(dr, t["gs"]) and not bool(dw.any())
    dx, dr, dw = torch.autograd.grad(y, [t["x"], t["res"], t["w"]], t["g"])
    assert same(dx, dr) and same(dw, both["dweight"])
    with torch.no_grad():
        want = ob.rms_norm(t["x"], t["w"], t["res"], 1e-5, t["g"])
    ob.check(dx, *want["dx"], dtype, "dx of y")


def test_the_same_tensor_twice(layers):
    x = make(30, 48, torch.float32)["x"].requires_grad_(True)
    y, s = layers.rms_norm(x, None, x)
    assert same(s, (x + x).detach())
    g = torch.randn_like(y)
    (d,) = torch.autograd.grad([y, s], x, [g, g])
    a, b = (x.detach().clone().requires_grad_(True) for _ in range(2))
    da, db = torch.autograd.grad(list(layers.rms_norm(a, None, b)), [a, b], [g, g])
    assert same(da, db) and same(d, da + db)
    # accumulated into leaves, the two gradients are two tensors
    torch.autograd.backward(list(layers.rms_norm(a, None, b)), [g, g])
    a.grad.zero_()
    assert same(b.grad, db)


def test_a_residual_stream_changed_in_place_is_noticed(layers):
    t = make(10, 32, torch.float32)
    x = t["x"].requires_grad_(True)
    y, s = layers.rms_norm(x, None, t["res"])
    with torch.no_grad():
        s += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_no_rows(layers, dtype):
    t = make(0, 40, dtype)
    got = run(layers, t)
    assert got["y"].shape == got["sum"].shape == got["dx"].shape == (0, 40) and not bool(got["dweight"].any())
    q, s = layers.rms_norm_8bit(t["x"].detach())
    assert q.shape == (0, 40) and s.shape == (0,)


def test_same_bits_each_time(layers):
    t = make(3000, 1030, torch.bfloat16)
    a, b = run(layers, t), run(layers, t)
    for k in a:
        assert same(a[k], b[k]), k


def test_gradients_against_differences(layers):
    t = make(19, 57, torch.float32)
    got = run(layers, t)
    for name, key in (("x", "dx"), ("w", "dweight"), ("res", "dres")):
        d = torch.randn(t[name].shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(2))

        def f(e):
            u = {k: t[k].detach().double() for k in ("x", "w", "res")}
            u[name] = u[name] + e * d
            s = u["x"] + u["res"]
            y = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-5) * u["w"]
            return float((y * t["g"].double()).sum() + (s * t["gs"].double()).sum())

        want, have = (f(1e-4) - f(-1e-4)) / 2e-4, float((got[key].double() * d).sum())
        # 2^-24 of each term's magnitude over ~1100 terms and h^2 of the third derivative
        assert abs(have - want) <= 1e-5 * float((got[key].double() * d).abs().sum()) + 1e-6, name


def test_other_stream_and_cpu_tensors(layers):
    t = make(100, 264, torch.bfloat16)
    want = layers.rms_norm(t["x"], t["w"], t["res"])
    codes = layers.rms_norm_8bit(t["x"], t["w"], t["res"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layers.rms_norm(t["x"], t["w"], t["res"])
    torch.cuda.current_stream().wait_stream(side)
    assert same(got[0], want[0]) and same(got[1], want[1])
    y, s = layers.rms_norm(t["x"].cpu(), t["w"].cpu(), t["res"].cpu())
    assert y.device.type == s.device.type == "cpu" and same(y, want[0].cpu()) and same(s, want[1].cpu())
    q, c, s = layers.rms_norm_8bit(t["x"].cpu(), t["w"].cpu(), t["res"].cpu())
    assert same(q.view(torch.uint8), codes[0].cpu().view(torch.uint8)) and same(c, codes[1].cpu())


def test_graph_capture(layers):
    t = make(640, 1024, torch.bfloat16)
    for k in ("x", "w", "res"):
        t[k].requires_grad_(True)

    def step():
        y, s = layers.rms_norm(t["x"], t["w"], t["res"])
        with torch.no_grad():
            q, c, _ = layers.rms_norm_8bit(t["x"], t["w"], t["res"])
        return [y.detach(), s.detach(), q.view(torch.uint8), c, *torch.autograd.grad([y, s], [t["x"], t["w"], t["res"]], [t["g"], t["gs"]])]

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


def test_8bit_has_no_gradient(layers):
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    for call in (lambda: layers.rms_norm_8bit(x), lambda: layers.quantize_8bit(x)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.parametrize("args,error", [
    ((torch.zeros(3, 0),), "x of shape"), ((torch.zeros(()),), "x of shape"), ((torch.zeros(3, 4), torch.zeros(5)), "weight"),
    ((torch.zeros(3, 4, dtype=torch.int32),), "float32"), ((torch.zeros(3, 4), torch.zeros(4, dtype=torch.bfloat16)), "weight"),
    ((torch.zeros(3, 4), None, torch.zeros(3, 5)), "residual"), ((torch.zeros(3, 4), None, torch.zeros(4)), "residual"),
    ((torch.zeros(3, 4), None, torch.zeros(3, 4, dtype=torch.float16)), "residual"),
    ((torch.zeros(3, 4), None, None, -1.0), "eps"), ((torch.zeros(3, 4), None, None, float("nan")), "eps"),
])
def test_refusals(layers, args, error):
    for f in (layers.rms_norm, layers.rms_norm_8bit):
        with pytest.raises(ValueError, match=error):
            f(*args)
