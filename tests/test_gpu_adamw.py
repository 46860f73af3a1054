"""diffrast.optim against the formula in 64 bits (operator_bounds.py) and, for 8-bit states, their
rounding as drh_adamw documents it, in torch's own operations on the CPU."""

import copy

import numpy as np
import pytest
import torch

import operator_bounds as ob

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)


@pytest.fixture(scope="module")
def optim():
    from diffrast import optim

    return optim


def same(a, b):
    return bool(torch.equal(a, b))


def make(sizes, dtype, bits=32, step=3, seed=0, align=1):
    """Parameters and states of a run `step` steps old, in flat buffers with rests between them."""
    g = torch.Generator("cuda").manual_seed(seed + len(sizes))
    starts, at = [], 0
    for n in sizes:
        at = -(-at // align) * align
        starts.append(at)
        at += n
    r = lambda: torch.randn(at + 1, device="cuda", generator=g)  # noqa: E731
    spread = torch.exp(r() - 6)
    old = 1.0 if step else 0.0
    flat = dict(p=(0.05 * r()).to(dtype), g=(spread * r()).to(dtype), m=0.3 * old * spread * r(), v=old * 0.003 * (spread * r()) ** 2)
    cut = lambda t: [t[a:a + n] for a, n in zip(starts, sizes)]  # noqa: E731
    s = dict(p=cut(flat["p"]), g=cut(flat["g"]), steps=torch.full((len(sizes),), step, dtype=torch.int64, device="cuda"))
    if bits == 32:
        s["m"], s["v"] = cut(flat["m"]), cut(flat["v"])
    else:
        for k, t in (("m", flat["m"]), ("v", flat["v"].sqrt())):
            codes, scales = torch.zeros(at + 1, dtype=torch.uint8, device="cuda"), []
            for a, n in zip(starts, sizes):
                rows = torch.nn.functional.pad(t[a:a + n], (0, -n % 256)).view(-1, 256)
                c = (rows.abs().amax(1) / 448).clamp(min=2.0**-126) if len(rows) else torch.zeros(0, device="cuda")
                codes[a:a + n] = (rows / c[:, None]).to(ob.E4M3).view(torch.uint8).view(-1)[:n]
                scales.append(c)
            s[k], s[k + "s"] = cut(codes.view(ob.E4M3)), scales
    return s


def values(codes, scales, root=False):
    v = codes.double() * scales.double().repeat_interleave(256)[:codes.numel()]
    return v * v if root else v


def call(optim, s, seed=0, **more):
    kw = dict(exp_avg_scales=s["ms"], exp_avg_sq_scales=s["vs"]) if "ms" in s else {}
    optim.adamw_step(s["p"], s["g"], s["m"], s["v"], s["steps"], seed=seed, **kw, **{**HYPER, **more})


def copied(s):
    return {k: [t.clone() for t in v] if isinstance(v, list) else v.clone() for k, v in s.items()}


SIZES = [1, 3, 4, 5, 255, 256, 257, 1000, 1024, 1025, 2047, 2048, 2049, 8193, 0, 70001]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("align", [64, 1])
@pytest.mark.parametrize("step", [0, 1, 1000, 100000])
def test_32_bit_states(optim, dtype, align, step):
    s = make(SIZES, dtype, 32, step, align=align)
    old = copied(s)
    call(optim, s)
    assert bool((s["steps"] == step + 1).all())
    for i in range(len(SIZES)):
        want = ob.adamw(old["p"][i], old["g"][i], old["m"][i], old["v"][i], step + 1, 1e-3, 0.9, 0.999, 1e-8, 0.01)
        ob.check(s["p"][i], *want["p"], dtype, f"p {SIZES[i]}")
        ob.check(s["m"][i], *want["m"], torch.float32, f"m {SIZES[i]}")
        ob.check(s["v"][i], *want["v"], torch.float32, f"v {SIZES[i]}")
        assert same(s["g"][i], old["g"][i])


@pytest.mark.parametrize("hyper", [dict(betas=(0.0, 0.0)), dict(weight_decay=0.0), dict(lr=0.0), dict(eps=1e-3), dict(betas=(0.5, 0.99999)),
                                   dict(eps=0.0)])
def test_other_numbers(optim, hyper):
    s = make([700, 5], torch.float32)
    old = copied(s)
    call(optim, s, **hyper)
    h = {**HYPER, **hyper}
    for i in range(2):
        want = ob.adamw(old["p"][i], old["g"][i], old["m"][i], old["v"][i], 4, h["lr"], *h["betas"], h["eps"], h["weight_decay"])
        for k in "pmv":
            ob.check(s[k][i], *want[k], torch.float32, k)


def bits_of(n, seed, t, j):
    """The 16 random bits of each element of tensor j at step t."""
    m32, u = 0xFFFFFFFF, np.uint64
    blocks = np.arange((n + 7) // 8, dtype=u)
    c = [blocks & u(m32), blocks >> u(32), np.full_like(blocks, t & m32), np.full_like(blocks, j)]
    k = [seed & m32, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & u(m32), (a >> u(32)) ^ c[3] ^ u(k[1]), a & u(m32)]
        k = [(k[0] + 0x9E3779B9) & m32, (k[1] + 0xBB67AE85) & m32]
    words = np.stack(c, 1)
    return np.stack([words & u(0xFFFF), words >> u(16)], 2).reshape(-1)[:n].astype(np.int64)


def rounded(value, scale, bits, least, err):
    """value / scale on e4m3's grid, up where `bits` reach the upper neighbour; in 64 bits. Also
    whether the choice is clear, that is not within 2^-12 of a step (2^-24 of a quotient of up to
    sixteen steps, a hundredfold) and what the value's own error is, of the other one."""
    x = np.abs(value) / scale
    e = np.maximum(np.floor(np.log2(np.maximum(x, 2.0**-30))), -6)
    step = 2.0 ** (e - 3)
    at = x / step + bits / 65536.0
    q = np.minimum(np.floor(at) * step, 448.0)
    q = np.where(x > 0, np.maximum(q, least), 0.0)
    # near an integer from either side, or near the border of two binades
    off = 2.0**-12 + err / scale / step
    clear = (np.abs(at - np.round(at)) > off) & (np.abs(x / 2.0**e - 1) > off)
    return np.copysign(q, value), clear


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("align", [64, 1])
@pytest.mark.parametrize("step", [0, 1, 5000])
def test_8_bit_states(optim, dtype, align, step):
    s = make(SIZES, dtype, 8, step, align=align)
    old = copied(s)
    seed = 0x123456789ABCDEF
    call(optim, s, seed)
    assert bool((s["steps"] == step + 1).all())
    unclear = total = 0
    for i, n in enumerate(SIZES):
        m, v = values(old["m"][i], old["ms"][i]), values(old["v"][i], old["vs"][i], True)
        want = ob.adamw(old["p"][i], old["g"][i], m, v, step + 1, 1e-3, 0.9, 0.999, 1e-8, 0.01)
        ob.check(s["p"][i], *want["p"], dtype, f"p {n}")
        bits = bits_of(n, seed, step + 1, i)
        swapped = (bits >> 8) | ((bits & 0xFF) << 8)
        root, eroot = want["v"][0].sqrt(), 8 * ob.E * want["v"][0].sqrt() + 2.0**-74
        for k, value, err, r, least in (("m", *want["m"], bits, 0.0), ("v", root, eroot, swapped, 2.0**-9)):
            if n == 0:
                continue
            rows = lambda t: torch.nn.functional.pad(t, (0, -n % 256)).view(-1, 256)  # noqa: E731
            most = rows(value.abs()).amax(1)
            scale = (most / 448).clamp(min=ob.LEAST)
            d = (s[k + "s"][i].double() - scale).abs()
            assert bool((d <= rows(err).amax(1) / 448 + 4 * ob.E * scale).all()), (k, n)
            c = s[k + "s"][i].double().repeat_interleave(256)[:n].cpu().numpy()
            q, clear = rounded(value.cpu().numpy(), c, r, least, err.cpu().numpy())
            got = s[k][i].double().cpu().numpy()
            assert np.array_equal(got[clear], q[clear]), (k, n)
            unclear, total = unclear + int((~clear).sum()), total + n
            x = np.abs(value.cpu().numpy()) / c
            assert bool((np.abs(np.abs(got) - x) <= np.maximum(x / 8, 2.0**-9) * 1.001 + 2.0**-20).all()), (k, n)
    assert unclear < 0.02 * total


def test_rounding_is_unbiased_and_seeded(optim):
    """One state rounded with 400 seeds: the mean is the state, and a seed's rounding is its own."""
    n = 4096
    s = make([n], torch.float32, 8, 10)
    sums = {k: torch.zeros(n, dtype=torch.float64, device="cuda") for k in "mv"}
    first = None
    for seed in range(400):
        t = copied(s)
        call(optim, t, seed)
        sums["m"] += values(t["m"][0], t["ms"][0])
        sums["v"] += values(t["v"][0], t["vs"][0])
        if seed == 0:
            first = t
    again = copied(s)
    call(optim, again, 0)
    assert same(first["m"][0].view(torch.uint8), again["m"][0].view(torch.uint8)) and same(first["p"][0], again["p"][0])
    want = ob.adamw(s["p"][0], s["g"][0], values(s["m"][0], s["ms"][0]), values(s["v"][0], s["vs"][0], True), 11, 1e-3, 0.9, 0.999, 1e-8, 0.01)
    for k, exact, scale in (("m", want["m"][0], first["ms"][0]), ("v", want["v"][0].sqrt(), first["vs"][0])):
        c = scale.double().repeat_interleave(256)
        inside = exact.abs() / c >= 2.0**-9 if k == "v" else torch.ones(n, dtype=torch.bool, device="cuda")  # a root is never rounded to 0
        d = (sums[k] / 400 - exact)[inside]
        step = torch.maximum(exact.abs() / 8, c * 2.0**-9)[inside]
        # a mean of 400 roundings has a deviation of a 40th of a step at the most: six of them, over 4096 elements
        assert bool((d.abs() <= 6 / 40 * step).all())
        assert abs(float((d / step).mean())) <= 6 / 40 / 4096**0.5 + 2.0**-16


def test_8_bit_averages_follow_a_steady_gradient(optim):
    """To the nearest they would stand still after a few steps: (1 - beta2) of v is far below half a step."""
    n = 2048
    g = torch.randn(n, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    z = lambda: [torch.zeros(n, dtype=ob.E4M3, device="cuda")]  # noqa: E731
    c = lambda: [torch.zeros(n // 256, device="cuda")]  # noqa: E731
    s = dict(p=[torch.zeros(n, device="cuda")], g=[g], m=z(), v=z(), ms=c(), vs=c(), steps=torch.zeros(1, dtype=torch.int64, device="cuda"))
    steps = 2000
    for i in range(steps):
        call(optim, s, 5, weight_decay=0.0)
    v = values(s["v"][0], s["vs"][0], True) / (1 - 0.999**steps)
    ratio = (v / g.double() ** 2)[g.abs() > 0.1]
    assert 0.8 < float(ratio.median()) < 1.3 and float(ratio.min()) > 0.4
    m = (values(s["m"][0], s["ms"][0]) / g.double())[g.abs() > 0.1]
    assert 0.95 < float(m.mean()) < 1.05


def test_a_root_is_never_rounded_to_nothing(optim):
    """One large gradient in a block of tiny ones: m is divided by more than eps."""
    g = torch.full((256,), 1e-4, device="cuda")
    g[7] = 1000.0
    s = dict(p=[torch.zeros(256, device="cuda")], g=[g], m=[torch.zeros(256, dtype=ob.E4M3, device="cuda")],
             v=[torch.zeros(256, dtype=ob.E4M3, device="cuda")], ms=[torch.zeros(1, device="cuda")], vs=[torch.zeros(1, device="cuda")],
             steps=torch.zeros(1, dtype=torch.int64, device="cuda"))
    for i in range(20):
        call(optim, s, i)
        assert bool((s["v"][0].float() > 0).all())
    assert float(s["p"][0].abs().max()) < 20 * 2e-3
    s["g"][0].zero_()
    s["v"][0].zero_(), s["m"][0].zero_()
    call(optim, s)
    assert not bool(s["v"][0].float().any()) and not bool(s["m"][0].float().any())


def test_more_tensors_than_a_launch_and_steps_of_their_own(optim):
    sizes = [(37 * i) % 300 for i in range(500)]  # some of them empty
    for bits in (32, 8):
        s = make(sizes, torch.float32, bits, 0)
        s["steps"] = torch.arange(500, device="cuda", dtype=torch.int64)
        if bits == 8:
            for k in ("ms", "vs"):
                s[k] = [t.clone() for t in s[k]]
        old = copied(s)
        call(optim, s, 9)
        assert same(s["steps"], torch.arange(500, device="cuda") + 1)
        for i in (0, 1, 47, 48, 49, 95, 96, 447, 448, 499):
            m, v = (old["m"][i], old["v"][i]) if bits == 32 else (values(old["m"][i], old["ms"][i]), values(old["v"][i], old["vs"][i], True))
            want = ob.adamw(old["p"][i], old["g"][i], m, v, i + 1, 1e-3, 0.9, 0.999, 1e-8, 0.01)
            ob.check(s["p"][i], *want["p"], torch.float32, f"tensor {i}")
        if bits == 8:  # the bits of a tensor past the first launch
            alone = {k: [old[k][60]] for k in ("p", "g", "m", "v", "ms", "vs")}
            got, n = s["m"][60], sizes[60]
            want, err = (a.cpu().numpy() for a in ob.adamw(
                alone["p"][0], alone["g"][0], values(alone["m"][0], alone["ms"][0]), values(alone["v"][0], alone["vs"][0], True), 61, 1e-3,
                0.9, 0.999, 1e-8, 0.01)["m"])
            q, clear = rounded(want, s["ms"][60].double().repeat_interleave(256)[:n].cpu().numpy(), bits_of(n, 9, 61, 60), 0.0, err)
            assert np.array_equal(got.double().cpu().numpy()[clear], q[clear])


@pytest.mark.parametrize("bits", [32, 8])
def test_infinities_and_nan(optim, bits):
    s = make([600, 256], torch.bfloat16, bits)
    s["g"][0][3], s["g"][0][300] = float("nan"), float("inf")
    old = copied(s)
    call(optim, s)
    assert bool(torch.isnan(s["p"][0][[3, 300]].float()).all())
    want = ob.adamw(old["p"][1], old["g"][1], *([old["m"][1], old["v"][1]] if bits == 32 else
                    [values(old["m"][1], old["ms"][1]), values(old["v"][1], old["vs"][1], True)]), 4, 1e-3, 0.9, 0.999, 1e-8, 0.01)
    ob.check(s["p"][1], *want["p"], torch.bfloat16, "the other tensor")
    assert int(torch.isnan(s["p"][0].float()).sum()) == 2
    if bits == 8:  # in the NaN's block the other states are what they were to be
        keep = torch.arange(256, device="cuda") != 3
        assert bool(torch.isfinite(s["m"][0][:256].float()[keep]).all()) and bool(torch.isnan(s["m"][0][3].float()))
        assert bool(torch.isfinite(s["m"][0][512:].float()).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_capture_counts_on(optim, bits):
    s = make([5000, 77], torch.float32, bits, 2)
    t = copied(s)
    call(optim, s, 3)  # an eager step before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(optim, s, 3)
    call(optim, t, 3)
    for i in range(4):
        for a, b in zip(s["g"], t["g"]):
            a.copy_(torch.randn_like(a))
            b.copy_(a)
        graph.replay()
        torch.cuda.synchronize()
        call(optim, t, 3)
        assert bool((s["steps"] == 4 + i).all())
        for k in s:
            for a, b in zip(s[k], t[k]):
                assert same(a.view(torch.uint8) if a.dtype == ob.E4M3 else a, b.view(torch.uint8) if b.dtype == ob.E4M3 else b), (i, k)


def test_other_stream(optim):
    s = make([70000, 33], torch.float32)
    t = copied(s)
    call(optim, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(optim, t)
    torch.cuda.current_stream().wait_stream(side)
    for k in "pmv":
        for a, b in zip(s[k], t[k]):
            assert same(a, b)


def test_a_parameter_saved_for_a_backward_pass_is_known_to_have_changed(optim):
    p = torch.randn(8, device="cuda", requires_grad=True)
    loss = (p * p).sum()
    z = lambda: [torch.zeros(8, device="cuda")]  # noqa: E731
    optim.adamw_step([p], z(), z(), z(), torch.zeros(1, dtype=torch.int64, device="cuda"), lr=0.1)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


# ---------------------------------------------------------------- the class


def net(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(20, 33), torch.nn.GELU(), torch.nn.Linear(33, 7)).cuda().to(dtype)


def train(model, opt, steps, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    for _ in range(steps):
        x = torch.randn(16, 20, device="cuda", generator=g)
        opt.zero_grad(set_to_none=True)
        (model(x.to(model[0].weight.dtype)).float() ** 2).mean().backward()
        opt.step()


def test_the_class_does_what_torchs_does(optim):
    a, b = net(), net()
    kw = dict(lr=1e-2, betas=(0.8, 0.99), eps=1e-7, weight_decay=0.1)
    train(a, optim.AdamW(a.parameters(), **kw), 12)
    train(b, torch.optim.AdamW(b.parameters(), **kw), 12)
    for p, q in zip(a.parameters(), b.parameters()):
        # twelve steps of 0.01, whose direction is a quotient of sums that differ by their rounding
        assert float((p - q).abs().max()) <= 12 * 1e-2 * 2.0**-10


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict(optim, bits, dtype):
    a = net(dtype)
    oa = optim.AdamW(a.parameters(), lr=1e-2, state_bits=bits, seed=4)
    train(a, oa, 3)
    b = copy.deepcopy(a)
    ob_ = optim.AdamW(b.parameters(), lr=1e-2, state_bits=bits, seed=4)
    saved = copy.deepcopy(oa.state_dict())
    ob_.load_state_dict(saved)
    for p, q in zip(a.parameters(), b.parameters()):
        sa, sb = oa.state[p], ob_.state[q]
        assert sa.keys() == sb.keys()
        for k in sa:
            assert sa[k].dtype == sb[k].dtype and sa[k].data_ptr() != sb[k].data_ptr()
    train(a, oa, 2, 1)
    train(b, ob_, 2, 1)
    for p, q in zip(a.parameters(), b.parameters()):
        assert same(p, q)
    # what was saved is not what goes on
    assert all(int(s["step"]) == 3 for s in saved["state"].values())


def test_parameters_without_gradients_and_groups(optim):
    a = net()
    opt = optim.AdamW([dict(params=a[0].parameters(), lr=0.1), dict(params=a[2].parameters(), lr=0.0, weight_decay=0.0, state_bits=8)])
    before = [p.detach().clone() for p in a.parameters()]
    assert opt.step(lambda: 5) == 5  # no gradients: nothing
    assert all(same(p, q) for p, q in zip(a.parameters(), before)) and not opt.state
    a[0].weight.grad = torch.ones_like(a[0].weight)
    a[2].weight.grad = torch.ones_like(a[2].weight).t().contiguous().t()
    opt.step()
    assert not same(a[0].weight, before[0]) and same(a[0].bias, before[1]) and same(a[2].weight, before[2])
    assert set(opt.state) == {a[0].weight, a[2].weight}
    assert opt.state[a[2].weight]["exp_avg"].dtype == ob.E4M3 and int(opt.state[a[2].weight]["step"]) == 1


def test_a_first_step_cannot_be_captured(optim):
    p = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    p.grad = torch.ones(5, device="cuda")
    opt = optim.AdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert int(opt.state[p]["step"]) == 4


def test_refusals(optim):
    s = make([300, 20], torch.float32, 32)
    t = make([300, 20], torch.float32, 8)
    before = copied(s)
    one = torch.zeros((), dtype=torch.int64, device="cuda")
    base = dict(params=s["p"], grads=s["g"], exp_avgs=s["m"], exp_avg_sqs=s["v"], steps=s["steps"], lr=1e-3)
    for bad, error in [
        (dict(grads=s["g"][:1]), "each of 2"), (dict(steps=s["steps"][:1]), "step counts"), (dict(steps=[one]), "each of 2"),
        (dict(steps=[one, one.float()]), "step count"), (dict(steps=s["steps"].cpu()), "step counts"),
        (dict(params=[s["p"][0].cpu(), s["p"][1]]), "on the GPU"), (dict(params=[s["p"][0], s["p"][1].half()]), "parameter"),
        (dict(params=[s["p"][0].int(), s["p"][1].int()]), "float32"), (dict(grads=[s["g"][0].half(), s["g"][1]]), "gradient"),
        (dict(grads=[s["g"][0][:5], s["g"][1]]), "gradient"), (dict(exp_avgs=[s["m"][0], s["m"][1].half()]), "exp_avg"),
        (dict(exp_avg_sqs=[s["v"][0], s["v"][1][:3]]), "exp_avg_sq"), (dict(exp_avgs=t["m"]), "exp_avg"),
        (dict(exp_avg_scales=t["ms"]), "come together"), (dict(exp_avg_scales=t["ms"], exp_avg_sq_scales=t["vs"]), "exp_avg"),
        (dict(exp_avgs=t["m"], exp_avg_sqs=t["v"], exp_avg_scales=[t["ms"][0][:1], t["ms"][1]], exp_avg_sq_scales=t["vs"]), "exp_avg_scale"),
        (dict(params=[torch.zeros(20, 15, device="cuda").t()[:15], s["p"][1]]), "not contiguous|exp_avg|gradient"),
        (dict(lr=-1.0), "lr"), (dict(lr=float("nan")), "lr"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"),
        (dict(eps=-1e-8), "eps"), (dict(weight_decay=float("inf")), "weight_decay"), (dict(seed=-1), "seed"),
    ]:
        with pytest.raises(ValueError, match=error):
            optim.adamw_step(**{**base, **bad})
    for bad in (dict(params=[s["p"][0], s["p"][0]], grads=[s["g"][0]] * 2, exp_avgs=[s["m"][0]] * 2, exp_avg_sqs=[s["v"][0]] * 2),
                dict(steps=[one, one])):
        with pytest.raises(RuntimeError, match="share"):
            optim.adamw_step(**{**base, **bad})
    for k in s:
        for a, b in zip(s[k], before[k]):
            assert same(a, b), k
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))], state_bits=16)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="on the GPU"):
        optim.AdamW([p]).step()


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_written_shares_no_memory(optim, bits):
    s = make([200, 200], torch.float32, bits)
    before = copied(s)
    both = torch.zeros(300, device="cuda")
    twice = [dict(p=[both[:200], both[100:]]), dict(m=[s["m"][0]] * 2), dict(v=[s["v"][1]] * 2), dict(v=s["m"])]
    twice += [dict(ms=[s["ms"][0]] * 2), dict(vs=s["ms"])] if bits == 8 else []
    for bad in twice:
        with pytest.raises(RuntimeError, match="share"):
            call(optim, {**s, **bad})
    for k in s:
        for a, b in zip(s[k], before[k]):
            assert same(a, b), k
    call(optim, {**s, "p": [both[:150], both[150:]], **{k: [t[:150] for t in s[k]] for k in ("g", "m", "v")}})  # neighbours do not
    call(optim, {**s, "g": [s["g"][0]] * 2})  # nor what is read


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("step", [0, 3])
def test_roots_of_tiny_and_huge_numbers(optim, dtype, step):
    """Gradients from 1e-25, whose squares are nothing in 32 bits, to 1e18, side by side and in runs of
    neighbours; exact zeros between them. Their squares' roots are taken in two ways by their size."""
    n = 8192
    s = make([n], dtype, step=step)
    e = torch.linspace(-25, 18, n, device="cuda")
    mixed = torch.cat([e[: n // 2], e[n // 2:][torch.randperm(n // 2, device="cuda", generator=torch.Generator("cuda").manual_seed(1))]])
    s["g"][0].copy_((10.0 ** mixed.double() * torch.where(torch.arange(n, device="cuda") % 3 == 0, -1, 1)).to(dtype))
    s["g"][0][::7] = 0
    if step:
        s["v"][0].copy_((0.1 * s["g"][0].double() ** 2).float())
        s["m"][0].copy_((0.3 * s["g"][0].double()).float())
    old = copied(s)
    call(optim, s)
    want = ob.adamw(old["p"][0], old["g"][0], old["m"][0], old["v"][0], step + 1, 1e-3, 0.9, 0.999, 1e-8, 0.01)
    ob.check(s["p"][0], *want["p"], dtype, "p")
    ob.check(s["m"][0], *want["m"], torch.float32, "m")
    ob.check(s["v"][0], *want["v"], torch.float32, "v")
