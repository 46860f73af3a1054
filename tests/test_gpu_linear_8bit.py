"""diffrast.layers.linear_8bit against its plain form in 64 bits (operator_bounds.py)."""

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


def to_8bit(t):
    s = (t.abs().amax(1) / 448).clamp(min=2.0**-126)
    return (t / s[:, None]).to(ob.E4M3), s


def make(M, K, N, dtype, bias=True, res=True, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + M + 7 * K + 31 * N)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, xs = to_8bit(r(M, K))
    w, ws = to_8bit(r(N, K) / K**0.5)
    return dict(x=x, xs=xs, w=w, ws=ws, b=(0.3 * r(N)).to(dtype) if bias else None, res=r(M, N).to(dtype) if res else None)


def run(layers, t, act, dtype):
    return layers.linear_8bit(t["x"], t["xs"], t["w"], t["ws"], t["b"], act, t["res"], dtype)


def compare(t, got, act, dtype, label):
    v, bound = ob.linear_8bit(t["x"], t["xs"], t["w"], t["ws"], t["b"], act, t["res"], dtype)
    ob.check(got.reshape(v.shape), v, bound, dtype, f"{label} {act}")


SIZES = [(1, 16, 1), (1, 1024, 4096), (2, 48, 17), (16, 128, 16), (17, 2000, 33), (33, 96, 130), (64, 4096, 15), (65, 16, 1),
         (65, 144, 31), (129, 112, 257), (300, 1008, 130), (257, 64, 513), (200, 8000, 20), (1031, 256, 515), (2500, 80, 2570),
         (40, 48, 4200), (0, 32, 8)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_products(layers, M, K, N, dtype):
    act = ACTS[(M + N) % 5]
    t = make(M, K, N, dtype)
    compare(t, run(layers, t, act, dtype), act, dtype, f"{M}x{K}x{N}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
def test_activations_bias_residual(layers, act, dtype):
    for bias in (True, False):
        for res in (True, False):
            for M, K, N in ((5, 80, 24), (150, 64, 100), (700, 640, 257)):
                t = make(M, K, N, dtype, bias, res)
                compare(t, run(layers, t, act, dtype), act, dtype, f"{M}x{K}x{N} {bias} {res}")


# tiles of 256 (16-bit outputs), as many as the card has CUs: one k tile, two and three, whole and not, an odd
# and an even number of them; widths of whole chunks and not
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("K,N", [(16, 3960), (128, 3960), (144, 3960), (256, 3960), (272, 3962), (384, 3960), (1040, 3960), (1152, 3961),
                                 (1280, 3848)])
def test_large_tiles(layers, K, N, dtype):
    for res in (True, False):
        t = make(3900, K, N, dtype, res=res)
        compare(t, run(layers, t, None, dtype), None, dtype, f"large {res}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_residual_at_any_address(layers, dtype):
    for M, K, N in ((3900, 512, 3960), (300, 512, 64), (20, 64, 40)):
        t = make(M, K, N, dtype)
        want = run(layers, t, "relu", dtype)
        room = torch.empty(M * N + 1, dtype=dtype, device="cuda")
        room[1:] = t["res"].view(-1)
        assert same(run(layers, {**t, "res": room[1:].view(M, N)}, "relu", dtype), want)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M", [1, 20, 100, 600])
def test_every_code(layers, M, dtype):
    """All of e4m3's numbers, subnormal ones among them, on both sides; NaN in one row stays in its outputs."""
    K, N = 256, 48
    g = torch.Generator().manual_seed(M)
    codes = torch.randint(0, 254, (M + N, K), generator=g, dtype=torch.int64)
    codes = (codes + (codes >= 127).long()).to(torch.uint8).cuda().view(ob.E4M3)
    t = dict(x=codes[:M], xs=torch.full((M,), 2.0**-9, device="cuda"), w=codes[M:], ws=torch.full((N,), 2.0**-4, device="cuda"), b=None,
             res=None)
    assert bool(torch.isfinite(codes.float()).all())
    compare(t, run(layers, t, None, dtype), None, dtype, "codes")
    bad = codes[M:].clone()
    bad.view(torch.uint8)[7, 3] = 0x7F
    y = run(layers, {**t, "w": bad}, None, dtype)
    assert bool(torch.isnan(y[:, 7].float()).all())
    keep = [i for i in range(N) if i != 7]
    assert same(y[:, keep], run(layers, t, None, dtype)[:, keep])


def test_sums_for_float32_are_held_in_32_bits(layers):
    """A large product among small ones, which the 8-bit instructions would cut off."""
    for M in (4, 100):
        x = torch.full((M, 128), 2.0**-6, device="cuda")
        x[:, 0] = 256.0
        w = torch.full((32, 128), 2.0**-2, device="cuda")
        w[:, 0] = 256.0
        one, ones = torch.ones(M, device="cuda"), torch.ones(32, device="cuda")
        y = layers.linear_8bit(x.to(ob.E4M3), one, w.to(ob.E4M3), ones, dtype=torch.float32)
        assert bool((y == 65536.0 + 127 * 2.0**-8).all())


def test_views_and_dimensions(layers):
    t = make(24, 96, 40, torch.bfloat16)
    want = run(layers, t, "silu", torch.bfloat16)
    for at in (16, 3):  # where it stands, and copied
        wide = torch.zeros(24, 256, dtype=torch.uint8, device="cuda")
        wide[:, at:at + 96] = t["x"].view(torch.uint8)
        high = torch.zeros(40, 160, dtype=torch.uint8, device="cuda")
        high[:, at:at + 96] = t["w"].view(torch.uint8)
        v = {**t, "x": wide.view(ob.E4M3)[:, at:at + 96], "w": high.view(ob.E4M3)[:, at:at + 96]}
        assert same(run(layers, v, "silu", torch.bfloat16), want)
    v = {**t, "x": t["x"].view(2, 3, 4, 96), "xs": t["xs"].view(2, 3, 4), "res": t["res"].view(2, 3, 4, 40)}
    y = run(layers, v, "silu", torch.bfloat16)
    assert y.shape == (2, 3, 4, 40) and same(y.view(24, 40), want)
    v = {**t, "x": t["x"][3], "xs": t["xs"][3], "res": t["res"][3]}
    assert same(run(layers, v, "silu", torch.bfloat16), want[3])


def test_with_the_norm(layers):
    """As a program that answers calls them: norm to 8 bits, product, within the rounding of both."""
    g = torch.Generator("cuda").manual_seed(5)
    for M in (1, 200):
        x, res = (torch.randn(M, 256, device="cuda", generator=g).bfloat16() for _ in range(2))
        w = torch.randn(72, 256, device="cuda", generator=g) / 16
        wq = layers.quantize_8bit(w)
        q, s, stream = layers.rms_norm_8bit(x, None, res)
        y = layers.linear_8bit(q, s, *wq, activation="gelu", residual=None)
        v, bound = ob.linear_8bit(q, s, *wq, None, "gelu", None, torch.bfloat16)
        ob.check(y, v, bound, torch.bfloat16, "with the norm")
        full = layers.linear(layers.rms_norm(x.float(), None, res.float())[0], w)
        # each operand is off by 2^-4 of its element at the most, 2^-10 of its row's largest / 448 below
        lim = 2.2 * 2.0**-4 * (layers.rms_norm(x.float(), None, res.float())[0].abs() @ w.abs().t())
        z = layers.linear_8bit(q, s, *wq, dtype=torch.float32)
        assert bool(((z - full).abs() <= lim + 1e-3).all())
        assert same(stream, (x.float() + res.float()).bfloat16())


def test_other_stream_graph_and_cpu_tensors(layers):
    t = make(300, 512, 72, torch.float16)
    call = lambda: run(layers, t, "gelu", torch.float16)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        t["xs"].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, call()), i
    on_cpu = {k: v.cpu() for k, v in t.items()}
    y = run(layers, on_cpu, "gelu", torch.float16)
    assert y.device.type == "cpu" and same(y, call().cpu())


X, S, W, V = torch.zeros(3, 32).to(ob.E4M3), torch.ones(3), torch.zeros(5, 32).to(ob.E4M3), torch.ones(5)


@pytest.mark.parametrize("args,kw,error", [
    ((torch.zeros(3, 32), S, W, V), {}, "float8"), ((X, S, torch.zeros(5, 32), V), {}, "float8"), ((X, S.half(), W, V), {}, "scales"),
    ((X, torch.ones(4), W, V), {}, "scale for each row"), ((X, S, W, torch.ones(3)), {}, "scale for each row"),
    ((X[:, :16], S, W, V), {}, "expected x"), ((X[:, :24], S, W[:, :24], V), {}, "multiples of 16"),
    ((X[:, :0], S, W[:, :0], V), {}, "multiples of 16"), ((X, S, W, V), dict(dtype=torch.float64), "output"),
    ((X, S, W, V, torch.zeros(5)), {}, "bias"), ((X, S, W, V, torch.zeros(4).bfloat16()), {}, "bias"),
    ((X, S, W, V, None, None, torch.zeros(3, 4).bfloat16()), {}, "residual"), ((X, S, W, V, None, "tanh"), {}, "activation"),
])
def test_refusals(layers, args, kw, error):
    with pytest.raises(ValueError, match=error):
        layers.linear_8bit(*args, **kw)


def test_no_gradient(layers):
    t = make(3, 32, 8, torch.float32)
    t["b"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        run(layers, t, None, torch.float32)
    with torch.no_grad():
        run(layers, t, None, torch.float32)
