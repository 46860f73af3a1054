"""diffrast.layers.dropout: its documented mask, drawn again here in Python's integers."""

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


def plain(x, p, seed, offset, res=None):
    """The formula in the type's own steps: one product and one sum in 32 bits, one rounding."""
    t = min(int(round(p * 65536)), 65535)
    keep = lb.philox_keep(x.numel(), t / 65536, seed, offset).reshape(x.shape).to(x.device)
    scale = torch.tensor(65536.0 / (65536 - t), dtype=torch.float32, device=x.device)
    y = torch.where(keep, x.float() * scale, torch.zeros((), device=x.device))
    return (y if res is None else y + res.float()).to(x.dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (257, 1003), (64, 2048), (2, 3, 4, 5), (100001,)])
def test_forward_and_gradients(layers, shape, dtype):
    g = torch.Generator("cuda").manual_seed(sum(shape))
    x, r, gy = (torch.randn(*shape, device="cuda", generator=g).to(dtype) for _ in range(3))
    x.requires_grad_(True)
    r.requires_grad_(True)
    for p, seed, offset in ((0.1, 5, 0), (0.5, (1 << 63) + 12345, 7), (0.937, 1 << 40, (1 << 64) - 1)):
        y = layers.dropout(x, p, seed=seed, offset=offset, residual=r)
        dx, dr = torch.autograd.grad(y, [x, r], gy)
        assert same(y, plain(x.detach(), p, seed, offset, r.detach()))
        assert same(dx, plain(gy, p, seed, offset)) and same(dr, gy)
        assert same(layers.dropout(x.detach(), p, seed=seed, offset=offset), plain(x.detach(), p, seed, offset))


def test_the_generators_published_outputs(layers):
    """Philox4x32-10's known answers (the counter and key all zero, and all ones), through the mask."""
    from struct import pack, unpack

    def halves(words):
        return list(unpack("<8H", pack("<4I", *words)))

    zero = halves((0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8))
    for p in (0.1, 0.25, 0.4, 0.5, 0.6, 0.75, 0.9):
        x = torch.ones(8, device="cuda")
        kept = layers.dropout(x, p, seed=0, offset=0) != 0
        assert kept.tolist() == [h >= round(p * 65536) for h in zero], p


def test_p_at_its_ends(layers):
    x = torch.randn(5000, device="cuda")
    assert same(layers.dropout(x, 0.0, seed=1), x)
    assert same(layers.dropout(x, 1e-6, seed=1), x)  # below the step of 2^-16
    y = layers.dropout(torch.ones(1 << 20, device="cuda"), 1 - 2.0**-30, seed=3)
    kept = int((y != 0).sum())
    assert 1 <= kept <= 60 and float(y.max()) == 65536.0  # 16 expected, one draw in 2^16 stays


def test_what_is_kept_and_how_offsets_differ(layers):
    n, p = 1 << 20, 0.3
    ones = torch.ones(n, device="cuda")
    a, b = (layers.dropout(ones, p, seed=9, offset=o) != 0 for o in (1, 2))
    q = 1 - round(p * 65536) / 65536
    six = 6 * (q * (1 - q) / n) ** 0.5
    assert abs(float(a.float().mean()) - q) < six and abs(float(b.float().mean()) - q) < six
    both = float((a & b).float().mean())
    assert abs(both - q * q) < 6 * (q * q * (1 - q * q) / n) ** 0.5
    # neighbours within one counter and across counters
    for d in (1, 2, 4, 8, 1024):
        pair = float((a[:-d] & a[d:]).float().mean())
        assert abs(pair - q * q) < 6 * (q * q * (1 - q * q) / (n - d)) ** 0.5 * 2


def test_infinities_and_nan(layers):
    """What is dropped is zero whatever it was; what is kept stays infinite or NaN."""
    n = 4096
    for v in (float("inf"), float("nan")):
        x = torch.full((n,), v, device="cuda")
        keep = lb.philox_keep(n, 0.4, 11, 3).cuda()
        y = layers.dropout(x, 0.4, seed=11, offset=3)
        assert not bool(y[~keep].any()) and not bool(torch.isfinite(y[keep]).any())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views(layers, dtype):
    """The mask goes by an element's place in the tensor, whatever its strides."""
    x = torch.randn(40, 72, device="cuda").to(dtype)
    want = layers.dropout(x, 0.3, seed=2)
    xt = x.t().contiguous().t()
    assert same(layers.dropout(xt, 0.3, seed=2, residual=xt), plain(x, 0.3, 2, 0, x))
    flat = torch.zeros(40 * 72 + 1, device="cuda", dtype=dtype)
    flat[1:] = x.reshape(-1)
    assert same(layers.dropout(flat[1:].view(40, 72), 0.3, seed=2), want)
    leaf = x.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(layers.dropout(leaf, 0.3, seed=2).sum(), leaf)
    assert same(d, plain(torch.ones_like(x), 0.3, 2, 0))
    assert layers.dropout(x[:0], 0.3, seed=2).shape == (0, 72)


def test_other_stream_and_cpu_tensors(layers):
    x = torch.randn(1000, 64, device="cuda")
    want = layers.dropout(x, 0.2, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layers.dropout(x, 0.2, seed=4)
    torch.cuda.current_stream().wait_stream(side)
    assert same(got, want)
    y = layers.dropout(x.cpu(), 0.2, seed=4)
    assert y.device.type == "cpu" and same(y, want.cpu())


@pytest.mark.parametrize("args,error", [
    (dict(p=1.0), "p must"), (dict(p=-0.1), "p must"), (dict(p=float("nan")), "p must"), (dict(seed=-1), "seed"),
    (dict(seed=1 << 64), "seed"), (dict(offset=1.5), "offset"), (dict(residual=torch.zeros(4)), "residual"),
    (dict(residual=torch.zeros(3, 4, dtype=torch.float16)), "residual"), (dict(x=torch.zeros(3, 4, dtype=torch.int64)), "float32"),
])
def test_refusals(layers, args, error):
    kw = dict(x=torch.zeros(3, 4), p=0.5, seed=0, offset=0, residual=None)
    kw.update(args)
    with pytest.raises(ValueError, match=error):
        layers.dropout(kw.pop("x"), kw.pop("p"), **kw)
