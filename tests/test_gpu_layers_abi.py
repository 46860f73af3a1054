"""The network layers at the C ABI: nothing is written past the ends of outputs and
workspaces, and what the header refuses is refused before anything is launched."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}
PAD = 4096  # bytes of sentinel on both sides


@pytest.fixture(scope="module")
def L():
    from diffrast import _lib

    return _lib


@pytest.fixture(scope="module")
def ctx(L):
    c = L.Context()
    yield c
    c.close()


class Guarded:
    """`n` elements between sentinels that check() wants untouched."""

    def __init__(self, n, dtype):
        self.bytes = n * torch.empty((), dtype=dtype).element_size()
        self.raw = torch.full((self.bytes + 2 * PAD,), 0xA5, dtype=torch.uint8, device="cuda")
        self.ptr = self.raw.data_ptr() + PAD

    def check(self, what):
        edge = torch.cat([self.raw[:PAD], self.raw[PAD + self.bytes:]])
        assert bool((edge == 0xA5).all()), f"{what}: written past an end"


def stream():
    return torch.cuda.current_stream().cuda_stream


def size(L, fn, *args):
    n = ctypes.c_uint64()
    L.check(fn(*args, ctypes.byref(n)))
    return n.value


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 5), (5, 1000), (51, 2050), (7, 4099), (3, 8191), (2, 8193), (9, 1024), (17, 3)])
def test_layer_norm_keeps_within_its_outputs(L, ctx, rows, D, dtype):
    x, g = (torch.randn(rows, D, device="cuda").to(DT[dtype]) for _ in range(2))
    w = torch.randn(D, device="cuda").to(DT[dtype])
    y, mean, rstd = Guarded(rows * D, DT[dtype]), Guarded(rows, torch.float32), Guarded(rows, torch.float32)
    L.check(L.lib().drh_layer_norm(ctx.handle, x.data_ptr(), w.data_ptr(), w.data_ptr(), rows, D, D, dtype, dtype, 1e-5,
                                   y.ptr, mean.ptr, rstd.ptr, stream(), 0))
    n = size(L, L.lib().drh_layer_norm_backward_bytes, rows, D, dtype)
    dx, dw, db, ws = Guarded(rows * D, DT[dtype]), Guarded(D, DT[dtype]), Guarded(D, DT[dtype]), Guarded(n, torch.uint8)
    L.check(L.lib().drh_layer_norm_backward(ctx.handle, x.data_ptr(), w.data_ptr(), mean.ptr, rstd.ptr, g.data_ptr(), rows, D,
                                            D, D, dtype, dtype, dx.ptr, dw.ptr, db.ptr, ws.ptr, n, stream(), L.SYNC))
    for name, b in dict(y=y, mean=mean, rstd=rstd, dx=dx, dw=dw, db=db, ws=ws).items():
        b.check(name)


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 17, 5), (64, 15, 130), (65, 1, 9), (129, 257, 33), (300, 130, 1000), (257, 513, 64),
                                   (2500, 2570, 72), (70, 20, 5000)])
def test_linear_keeps_within_its_outputs(L, ctx, M, N, K, dtype):
    x, w, g = (torch.randn(*s, device="cuda").to(DT[dtype]) for s in ((M, K), (N, K), (M, N)))
    b = torch.randn(N, device="cuda").to(DT[dtype])
    n = size(L, L.lib().drh_linear_bytes, M, N, K, K, K, dtype)
    y, kept, ws = Guarded(M * N, DT[dtype]), Guarded(M * N, torch.float32 if dtype == 0 else torch.float16), Guarded(n, torch.uint8)
    L.check(L.lib().drh_linear(ctx.handle, x.data_ptr(), w.data_ptr(), b.data_ptr(), g.data_ptr(), M, N, K, K, K, dtype, 2,
                               y.ptr, kept.ptr, ws.ptr, n, stream(), 0))
    m = size(L, L.lib().drh_linear_backward_bytes, M, N, K, K, K, dtype, 2)
    dx, dw, db, ws2 = Guarded(M * K, DT[dtype]), Guarded(N * K, DT[dtype]), Guarded(N, DT[dtype]), Guarded(m, torch.uint8)
    L.check(L.lib().drh_linear_backward(ctx.handle, x.data_ptr(), w.data_ptr(), kept.ptr, g.data_ptr(), M, N, K, K, K, dtype, 2,
                                        dx.ptr, dw.ptr, db.ptr, ws2.ptr, m, stream(), L.SYNC))
    for name, buf in dict(y=y, kept=kept, ws=ws, dx=dx, dw=dw, db=db, ws2=ws2).items():
        buf.check(name)


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2049, 100003])
def test_dropout_keeps_within_its_output(L, ctx, n, dtype):
    x, y = torch.randn(n, device="cuda").to(DT[dtype]), Guarded(n, DT[dtype])
    L.check(L.lib().drh_dropout(ctx.handle, x.data_ptr(), x.data_ptr(), n, dtype, 0.3, 1, 2, y.ptr, stream(), L.SYNC))
    y.check("y")


def refused(L, code, call):
    with pytest.raises(L.DiffrastError) as e:
        L.check(call())
    assert e.value.code == code, e.value


def test_refusals(L, ctx):
    f, t = L.lib(), torch.zeros(64, 64, device="cuda")
    p, h, s = t.data_ptr(), ctx.handle, stream()
    ln = lambda **k: f.drh_layer_norm(*{**dict(ctx=h, x=p, w=p, b=p, rows=4, cols=8, xs=8, dt=0, wdt=0, eps=1e-5, y=p, mean=None,  # noqa: E731
                                               rstd=None, s=s, flags=0), **k}.values())
    for bad in (dict(ctx=None), dict(x=None), dict(y=None), dict(rows=-1), dict(cols=0), dict(dt=3), dict(wdt=1), dict(eps=-1.0),
                dict(eps=float("nan")), dict(mean=p), dict(flags=L.HOST_PTRS), dict(xs=-8)):
        refused(L, 6, lambda: ln(**bad))
    refused(L, 5, lambda: ln(rows=1 << 31))
    n = size(L, f.drh_layer_norm_backward_bytes, 4, 8, 0)
    lb = lambda **k: f.drh_layer_norm_backward(*{**dict(ctx=h, x=p, w=p, mean=p, rstd=p, g=p, rows=4, cols=8, xs=8, gs=8, dt=0, wdt=0,  # noqa: E731
                                                        dx=p, dw=p, db=p, ws=p, n=n, s=s, flags=0), **k}.values())
    for bad in (dict(x=None), dict(mean=None), dict(g=None), dict(ws=None), dict(n=n - 1), dict(ws=p + 4), dict(flags=4)):
        refused(L, 6, lambda: lb(**bad))
    li = lambda **k: f.drh_linear(*{**dict(ctx=h, x=p, w=p, b=None, r=None, rows=4, N=8, K=8, xs=8, ws=8, dt=0, act=0, y=p, kept=None,  # noqa: E731
                                           space=None, n=0, s=s, flags=0), **k}.values())
    for bad in (dict(ctx=None), dict(x=None), dict(w=None), dict(y=None), dict(N=0), dict(K=-1), dict(xs=7), dict(ws=4), dict(dt=-1),
                dict(act=5), dict(act=-1), dict(flags=L.HOST_PTRS), dict(rows=1000, K=100, xs=101, ws=100)):  # the last: no workspace
        refused(L, 6, lambda: li(**bad))
    refused(L, 5, lambda: li(K=1 << 31, xs=1 << 31, ws=1 << 31))
    m = size(L, f.drh_linear_backward_bytes, 4, 8, 8, 8, 8, 0, 1)
    lib = lambda **k: f.drh_linear_backward(*{**dict(ctx=h, x=p, w=p, kept=p, g=p, rows=4, N=8, K=8, xs=8, ws=8, dt=0, act=1, dx=p, dw=p,  # noqa: E731
                                                     db=p, space=p, n=m, s=s, flags=0), **k}.values())
    for bad in (dict(x=None), dict(w=None), dict(kept=None), dict(g=None), dict(space=None), dict(n=m - 1), dict(space=p + 8)):
        refused(L, 6, lambda: lib(**bad))
    dr = lambda **k: f.drh_dropout(*{**dict(ctx=h, x=p, r=None, n=64, dt=0, p=0.5, seed=0, off=0, y=p, s=s, flags=0), **k}.values())  # noqa: E731
    for bad in (dict(x=None), dict(y=None), dict(n=-1), dict(p=1.0), dict(p=-0.5), dict(p=float("nan")), dict(dt=9), dict(flags=2 | 8)):
        refused(L, 6, lambda: dr(**bad))
    refused(L, 5, lambda: dr(n=(1 << 40) + 1))
    torch.cuda.synchronize()
    assert not bool(t.any())


def test_nothing_to_do(L, ctx):
    f, h, s = L.lib(), ctx.handle, stream()
    L.check(f.drh_layer_norm(h, None, None, None, 0, 8, 8, 0, 0, 1e-5, None, None, None, s, 0))
    L.check(f.drh_linear(h, None, None, None, None, 0, 8, 8, 8, 8, 0, 0, None, None, None, 0, s, 0))
    L.check(f.drh_dropout(h, None, None, 0, 0, 0.5, 0, 0, None, s, 0))
