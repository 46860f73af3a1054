"""drh_linear and drh_linear_backward with what only a caller of the C ABI gives them."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}


@pytest.fixture(scope="module")
def L():
    from diffrast import _lib

    return _lib


@pytest.fixture(scope="module")
def ctx(L):
    c = L.Context()
    yield c
    c.close()


def backward(L, ctx, x, w, g, xs, ws, dtype):
    (M, K), N = x.shape, w.shape[0]
    f, n = L.lib(), ctypes.c_uint64()
    L.check(f.drh_linear_backward_bytes(M, N, K, xs, ws, dtype, 0, ctypes.byref(n)))
    dx, dw, db = (torch.full(s, 7.0, device="cuda", dtype=DT[dtype]) for s in ((M, K), (N, K), (N,)))
    space = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    L.check(f.drh_linear_backward(ctx.handle, x.data_ptr(), w.data_ptr(), None, g.data_ptr(), M, N, K, xs, ws, dtype, 0,
                                  dx.data_ptr(), dw.data_ptr(), db.data_ptr(), space.data_ptr(), n.value,
                                  torch.cuda.current_stream().cuda_stream, L.SYNC))
    return dx, dw, db


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("stride", [0, 8, 96, 4096])
def test_the_stride_of_a_single_row_counts_for_nothing(L, ctx, stride, dtype):
    """An infinity in it stays in its own products, whose other factor is 1 or 2: all are exact."""
    K, many = 96, 200
    one = torch.ones(1, K, device="cuda", dtype=DT[dtype])
    one[0, 5] = float("inf")
    rest = torch.ones(many, K, device="cuda", dtype=DT[dtype])
    g = 1 + torch.arange(many, device="cuda").remainder(2).to(DT[dtype])  # 1, 2, 1, ...
    # one row of x: dW = g x
    _, dw, db = backward(L, ctx, one, rest, g.view(1, many), stride, K, dtype)
    assert bool(torch.equal(dw, g[:, None] * one)) and bool(torch.equal(db, g))
    # one output: dx = g w
    dx, _, db = backward(L, ctx, rest, one, g.view(many, 1), K, stride, dtype)
    assert bool(torch.equal(dx, g[:, None] * one)) and float(db) == 300


def test_strides_past_any_memory_are_refused(L, ctx):
    f, t = L.lib(), torch.zeros(64, 64, device="cuda")
    p, h, big = t.data_ptr(), ctx.handle, 1 << 46
    calls = (lambda: f.drh_linear(h, p, p, None, None, 100, 8, 8, big, 8, 0, 0, p, None, None, 0, None, 0),
             lambda: f.drh_linear(h, p, p, None, None, 4, 8, 8, 8, big, 0, 0, p, None, None, 0, None, 0),
             lambda: f.drh_linear_backward(h, p, p, None, p, 100, 8, 8, big, 8, 0, 0, p, p, None, p, 1 << 30, None, 0),
             lambda: f.drh_layer_norm(h, p, None, None, 100, 8, big, 0, 0, 1e-5, p, None, None, None, 0),
             lambda: f.drh_layer_norm_backward(h, p, None, p, p, p, 100, 8, 8, big, 0, 0, p, None, None, None, 0, None, 0))
    for call in calls:
        assert call() == 5, L.last_error()
    torch.cuda.synchronize()
    assert not bool(t.any())
