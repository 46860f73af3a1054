"""The norms, products and optimiser step of the C ABI that test_gpu_layers_abi.py does not hold:
nothing is written past the ends of outputs and workspaces, and what the header refuses is refused
before anything is launched."""

import ctypes

import pytest
import torch

from test_gpu_layers_abi import DT, Guarded, ctx, refused, size, stream  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f32", "bf16", "f16"])


@pytest.fixture(scope="module")
def L():
    from diffrast import _lib

    return _lib


def tight(t):
    """t's values at the end of an allocation's pages' worth of NaN, so that a read past them is seen."""
    room = torch.full((t.numel() + 4096,), float("nan"), device="cuda").to(t.dtype)
    room[2048:2048 + t.numel()] = t.reshape(-1)
    return room[2048:2048 + t.numel()].view(t.shape)


@TYPES
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 5), (5, 1000), (51, 2050), (7, 4099), (3, 8191), (2, 8193), (9, 1024), (17, 3), (2, 16385),
                                    (2, 32769)])
def test_rms_norm_keeps_within_its_outputs(L, ctx, rows, D, dtype):  # noqa: F811
    x, r, g, gs = (tight(torch.randn(rows, D, device="cuda").to(DT[dtype])) for _ in range(4))
    w = tight(torch.randn(D, device="cuda").to(DT[dtype]))
    y, s, rstd = Guarded(rows * D, DT[dtype]), Guarded(rows * D, DT[dtype]), Guarded(rows, torch.float32)
    q, scale, s2 = Guarded(rows * D, torch.uint8), Guarded(rows, torch.float32), Guarded(rows * D, DT[dtype])
    q3, scale3 = Guarded(rows * D, torch.uint8), Guarded(rows, torch.float32)
    f, h = L.lib(), ctx.handle
    L.check(f.drh_rms_norm(h, x.data_ptr(), r.data_ptr(), w.data_ptr(), rows, D, D, D, dtype, dtype, 1e-5, y.ptr, s.ptr, rstd.ptr,
                           stream(), 0))
    L.check(f.drh_rms_norm_8bit(h, x.data_ptr(), r.data_ptr(), w.data_ptr(), rows, D, D, D, dtype, dtype, 1e-5, q.ptr, scale.ptr, s2.ptr,
                                stream(), 0))
    L.check(f.drh_quantize_8bit(h, x.data_ptr(), rows, D, D, dtype, q3.ptr, scale3.ptr, stream(), 0))
    n = size(L, f.drh_rms_norm_backward_bytes, rows, D, dtype)
    dx, dw, ws = Guarded(rows * D, DT[dtype]), Guarded(D, DT[dtype]), Guarded(n, torch.uint8)
    L.check(f.drh_rms_norm_backward(h, s.ptr, w.data_ptr(), rstd.ptr, g.data_ptr(), gs.data_ptr(), rows, D, D, D, D, dtype, dtype, dx.ptr,
                                    dw.ptr, ws.ptr, n, stream(), L.SYNC))
    for name, b in dict(y=y, s=s, rstd=rstd, q=q, scale=scale, s2=s2, q3=q3, scale3=scale3, dx=dx, dw=dw, ws=ws).items():
        b.check(name)
        if name not in ("ws", "q", "q3"):
            kind = DT[dtype] if name in ("y", "s", "s2", "dx", "dw") else torch.float32
            assert bool(torch.isfinite(b.raw[4096:4096 + b.bytes].view(kind).float()).all()), name


PRODUCTS = [(1, 1, 1), (1, 17, 5), (64, 15, 130), (65, 1, 9), (129, 257, 33), (300, 130, 1000), (257, 513, 64), (2500, 1290, 72),
            (70, 20, 5000)]


@TYPES
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_gated_linear_keeps_within_its_outputs(L, ctx, M, N, K, dtype):  # noqa: F811
    x, w, g = (tight(torch.randn(*s, device="cuda").to(DT[dtype])) for s in ((M, K), (2 * N, K), (M, N)))
    b = tight(torch.randn(2 * N, device="cuda").to(DT[dtype]))
    f, h = L.lib(), ctx.handle
    n = size(L, f.drh_gated_linear_bytes, M, N, K, K, K, dtype)
    y, kept, ws = Guarded(M * N, DT[dtype]), Guarded(M * N * (8, 5, 6)[dtype], torch.uint8), Guarded(n, torch.uint8)
    L.check(f.drh_gated_linear(h, x.data_ptr(), w.data_ptr(), b.data_ptr(), M, N, K, K, K, dtype, 4, y.ptr, kept.ptr, ws.ptr, n, stream(), 0))
    m = size(L, f.drh_gated_linear_backward_bytes, M, N, K, K, K, dtype)
    dx, dw, db, ws2 = Guarded(M * K, DT[dtype]), Guarded(2 * N * K, DT[dtype]), Guarded(2 * N, DT[dtype]), Guarded(m, torch.uint8)
    L.check(f.drh_gated_linear_backward(h, x.data_ptr(), w.data_ptr(), kept.ptr, g.data_ptr(), M, N, K, K, K, dtype, dx.ptr, dw.ptr, db.ptr,
                                        ws2.ptr, m, stream(), L.SYNC))
    for name, buf in dict(y=y, kept=kept, ws=ws, dx=dx, dw=dw, db=db, ws2=ws2).items():
        buf.check(name)
        if name in ("y", "dx", "dw", "db"):
            assert bool(torch.isfinite(buf.raw[4096:4096 + buf.bytes].view(DT[dtype]).float()).all()), name


@TYPES
@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 17, 48), (64, 15, 144), (65, 1, 16), (129, 257, 32), (300, 130, 1008), (2500, 2570, 80),
                                   (70, 20, 8000)])
def test_linear_8bit_keeps_within_its_outputs(L, ctx, M, N, K, dtype):  # noqa: F811
    def codes(rows):
        room = torch.full((rows * K + 8192,), 0x7F, dtype=torch.uint8, device="cuda")  # NaN
        room[4096:4096 + rows * K] = torch.randint(0, 127, (rows * K,), device="cuda").to(torch.uint8)
        return room[4096:4096 + rows * K]

    x, w = codes(M), codes(N)
    xs, ws = (tight(torch.rand(k, device="cuda") * 2.0**-12) for k in (M, N))
    b, r = (tight(torch.randn(*s, device="cuda").to(DT[dtype])) for s in ((N,), (M, N)))
    f, h = L.lib(), ctx.handle
    n = size(L, f.drh_linear_8bit_bytes, M, N, K, K, K, dtype)
    y, space = Guarded(M * N, DT[dtype]), Guarded(n, torch.uint8)
    L.check(f.drh_linear_8bit(h, x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), b.data_ptr(), r.data_ptr(), M, N, K, K, K, dtype, 2,
                              y.ptr, space.ptr, n, stream(), L.SYNC))
    y.check("y"), space.check("workspace")
    assert bool(torch.isfinite(y.raw[4096:4096 + y.bytes].view(DT[dtype]).float()).all())


@TYPES
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_keeps_within_its_tensors(L, ctx, dtype, bits):  # noqa: F811
    sizes = [1, 3, 255, 256, 257, 2049, 5000, 0, 7]
    held, table = [], (L.AdamWTensor * len(sizes))()
    steps = Guarded(len(sizes), torch.int64)
    steps.raw[4096:4096 + steps.bytes] = 0
    for i, n in enumerate(sizes):
        blocks = -(-n // 256)
        p, m, v = Guarded(n, DT[dtype]), *(Guarded(n, torch.uint8 if bits == 8 else torch.float32) for _ in range(2))
        ms, vs = Guarded(blocks, torch.float32), Guarded(blocks, torch.float32)
        for b in (p, m, v, ms, vs):
            b.raw[4096:4096 + b.bytes] = 0
        g = tight(torch.randn(n, device="cuda").to(DT[dtype]))
        held.append((p, m, v, ms, vs, g))
        small = bits == 8
        table[i] = L.AdamWTensor(p.ptr, g.data_ptr(), m.ptr, v.ptr, ms.ptr if small else None, vs.ptr if small else None, steps.ptr + 8 * i, n)
    for _ in range(2):
        L.check(L.lib().drh_adamw(ctx.handle, table, len(sizes), dtype, bits, 1e-3, 0.9, 0.999, 1e-8, 0.01, 5, stream(), L.SYNC))
    for i, bufs in enumerate(held):
        for b in bufs[:5]:
            b.check(f"tensor {i}")
        p = bufs[0].raw[4096:4096 + bufs[0].bytes].view(DT[dtype]).float()
        assert bool(torch.isfinite(p).all()) and bool((p != 0).all())
    steps.check("steps")
    assert steps.raw[4096:4096 + steps.bytes].view(torch.int64).tolist() == [2] * len(sizes)


def test_refusals(L, ctx):  # noqa: F811
    f, t = L.lib(), torch.zeros(64, 64, device="cuda")
    p, h, s = t.data_ptr(), ctx.handle, stream()

    def caller(fn, **base):
        return lambda **k: fn(*{**base, **k}.values())

    rms = caller(f.drh_rms_norm, ctx=h, x=p, r=p, w=p, rows=4, cols=8, xs=8, rs=8, dt=0, wdt=0, eps=1e-5, y=p, sum=p, rstd=None, s=s, flags=0)
    shared = [dict(ctx=None), dict(x=None), dict(y=None), dict(rows=-1), dict(cols=0), dict(dt=3), dict(wdt=1), dict(eps=-1.0),
              dict(eps=float("nan")), dict(flags=L.HOST_PTRS), dict(xs=-8), dict(rs=-8), dict(r=None)]  # the last: a sum of nothing
    for bad in shared:
        refused(L, 6, lambda: rms(**bad))
    rms8 = caller(f.drh_rms_norm_8bit, ctx=h, x=p, r=p, w=p, rows=4, cols=8, xs=8, rs=8, dt=0, wdt=0, eps=1e-5, y=p, sc=p, sum=p, s=s, flags=0)
    for bad in [*shared, dict(sc=None)]:
        refused(L, 6, lambda: rms8(**bad))
    q8 = caller(f.drh_quantize_8bit, ctx=h, x=p, rows=4, cols=8, xs=8, dt=0, y=p, sc=p, s=s, flags=0)
    for bad in (dict(ctx=None), dict(x=None), dict(y=None), dict(sc=None), dict(rows=-1), dict(cols=0), dict(dt=3), dict(xs=-1), dict(flags=4)):
        refused(L, 6, lambda: q8(**bad))
    for call in (rms, rms8, q8):
        refused(L, 5, lambda: call(rows=1 << 31))
        refused(L, 5, lambda: call(cols=(1 << 30) + 1))
        refused(L, 5, lambda: call(xs=1 << 60))
    n = size(L, f.drh_rms_norm_backward_bytes, 4, 8, 0)
    back = caller(f.drh_rms_norm_backward, ctx=h, x=p, w=p, rstd=p, g=p, gs=p, rows=4, cols=8, xs=8, gst=8, gss=8, dt=0, wdt=0, dx=p, dw=p, ws=p,
                  n=n, s=s, flags=0)
    for bad in (dict(x=None), dict(rstd=None), dict(g=None), dict(ws=None), dict(n=n - 1), dict(ws=p + 4), dict(flags=4), dict(gss=-1),
                dict(gst=-8)):
        refused(L, 6, lambda: back(**bad))

    ga = caller(f.drh_gated_linear, ctx=h, x=p, w=p, b=None, rows=4, N=8, K=8, xs=8, ws=8, dt=0, act=4, y=p, kept=None, space=None, n=0, s=s,
                flags=0)
    for bad in (dict(ctx=None), dict(x=None), dict(w=None), dict(y=None), dict(N=0), dict(K=-1), dict(xs=7), dict(ws=4), dict(dt=-1),
                dict(act=5), dict(act=-1), dict(flags=L.HOST_PTRS), dict(kept=p + 4), dict(rows=1000, K=100, xs=101, ws=100)):
        refused(L, 6, lambda: ga(**bad))
    refused(L, 5, lambda: ga(N=(1 << 29) + 1))
    refused(L, 5, lambda: ga(K=1 << 31, xs=1 << 31, ws=1 << 31))
    m = size(L, f.drh_gated_linear_backward_bytes, 4, 8, 8, 8, 8, 0)
    gb = caller(f.drh_gated_linear_backward, ctx=h, x=p, w=p, kept=p, g=p, rows=4, N=8, K=8, xs=8, ws=8, dt=0, dx=p, dw=p, db=p, space=p, n=m,
                s=s, flags=0)
    for bad in (dict(x=None), dict(w=None), dict(kept=None), dict(kept=p + 8), dict(g=None), dict(space=None), dict(n=m - 1),
                dict(space=p + 8)):
        refused(L, 6, lambda: gb(**bad))

    li = caller(f.drh_linear_8bit, ctx=h, x=p, xsc=p, w=p, wsc=p, b=None, r=None, rows=4, N=8, K=16, xs=16, ws=16, dt=0, act=0, y=p, space=None,
                n=0, s=s, flags=0)
    for bad in (dict(ctx=None), dict(x=None), dict(w=None), dict(xsc=None), dict(wsc=None), dict(y=None), dict(N=0), dict(K=0), dict(K=8),
                dict(xs=24), dict(ws=40), dict(xs=0), dict(x=p + 8), dict(w=p + 1), dict(dt=3), dict(act=7), dict(flags=1)):
        refused(L, 6, lambda: li(**bad))
    refused(L, 5, lambda: li(xs=1 << 24))

    one = torch.zeros(4, dtype=torch.int64, device="cuda")
    tensor = lambda **k: L.AdamWTensor(*{**dict(p=p, g=p, m=p, v=p, ms=None, vs=None, step=one.data_ptr(), n=4), **k}.values())  # noqa: E731
    ad = lambda ts, **k: f.drh_adamw(*{**dict(ctx=h, t=(L.AdamWTensor * len(ts))(*ts), count=len(ts), dt=0, bits=32, lr=0.1, b1=0.9, b2=0.9,  # noqa: E731
                                              eps=0.0, wd=0.0, seed=0, s=s, flags=0), **k}.values())
    for bad in (dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(step=None), dict(n=-1), dict(ms=p, vs=p), dict(p=p + 2),
                dict(m=p + 1), dict(step=one.data_ptr() + 4)):
        refused(L, 6, lambda: ad([tensor(**bad)]))
    refused(L, 5, lambda: ad([tensor(n=(1 << 40) + 1)]))
    refused(L, 6, lambda: ad([tensor(), tensor(step=one.data_ptr() + 8)]))  # one parameter twice
    refused(L, 6, lambda: ad([tensor(), tensor(p=p + 256)]))  # one count twice
    refused(L, 6, lambda: ad([tensor(ms=p)], bits=8))
    for bad in (dict(ctx=None), dict(t=None), dict(count=-1), dict(dt=3), dict(bits=16), dict(lr=-1.0), dict(lr=float("nan")),
                dict(lr=float("inf")), dict(b1=1.0), dict(b2=-0.1), dict(eps=float("nan")), dict(wd=-1.0), dict(flags=4)):
        refused(L, 6, lambda: ad([tensor()], **bad))
    torch.cuda.synchronize()
    assert not bool(t.any()) and not bool(one.any())


def test_nothing_to_do(L, ctx):  # noqa: F811
    f, h, s = L.lib(), ctx.handle, stream()
    L.check(f.drh_rms_norm(h, None, None, None, 0, 8, 8, 8, 0, 0, 1e-5, None, None, None, s, 0))
    L.check(f.drh_rms_norm_8bit(h, None, None, None, 0, 8, 8, 8, 0, 0, 1e-5, None, None, None, s, 0))
    L.check(f.drh_quantize_8bit(h, None, 0, 8, 8, 0, None, None, s, 0))
    L.check(f.drh_gated_linear(h, None, None, None, 0, 8, 8, 8, 8, 0, 0, None, None, None, 0, s, 0))
    L.check(f.drh_linear_8bit(h, None, None, None, None, None, None, 0, 8, 16, 16, 16, 0, 0, None, None, 0, s, 0))
    L.check(f.drh_adamw(h, None, 0, 0, 32, 0.1, 0.9, 0.9, 0.0, 0.0, 0, s, 0))
