"""Arrays that need more threads than one launch has (2^32): the rows and elements about the
launches' borders and at the end are those of a small call on them alone."""

import ctypes

import pytest
import torch

import layer_bounds as lb

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def L():
    from diffrast import _lib

    return _lib


@pytest.fixture(scope="module")
def layers():
    from diffrast import layers

    return layers


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def same(a, b):
    return bool(torch.equal(a, b))


def need(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of free device memory")


def test_layer_norm_of_many_short_rows(layers):
    """A wave a row: 2^26 rows are 2^32 threads."""
    rows, D = (1 << 26) + 1003, 8
    need(8)
    x, g = (torch.randn(rows, D, device="cuda", generator=torch.Generator("cuda").manual_seed(s)).to(BF) for s in (1, 2))
    w, b = torch.randn(D, device="cuda").to(BF), torch.randn(D, device="cuda").to(BF)
    leaf = x.requires_grad_(True)
    y = layers.layer_norm(leaf, w, b)
    (dx,) = torch.autograd.grad(y, leaf, g)
    half = rows // 2
    for part in (slice(0, half), slice(half, rows)):
        small = x.detach()[part].clone().requires_grad_(True)
        ys = layers.layer_norm(small, w, b)
        (ds,) = torch.autograd.grad(ys, small, g[part])
        assert same(y.detach()[part], ys.detach()) and same(dx[part], ds)


def test_layer_norm_of_many_wide_rows(L):
    """A workgroup of 1024 a row: 2^22 rows are 2^32 threads. All rows are one and the same in memory."""
    rows, D = (1 << 22) + 5, 8193
    need(75)
    ctx, s = L.Context(), torch.cuda.current_stream().cuda_stream
    x, g, w = (torch.randn(D, device="cuda").to(BF) for _ in range(3))
    out = torch.zeros(rows, D, dtype=BF, device="cuda")
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")

    def check(label):
        for first in (0, rows // 2, (1 << 22) - 1002, rows - 1000):
            assert same(out[first:first + 1000], out[:1].expand(1000, D)), (label, first)
        assert bool((out[:, D - 1] == out[0, D - 1]).all()) and bool(out[0].any()), label

    L.check(L.lib().drh_layer_norm(ctx.handle, x.data_ptr(), w.data_ptr(), None, rows, D, 0, 1, 1, 1e-5, out.data_ptr(),
                                   mean.data_ptr(), rstd.data_ptr(), s, L.SYNC))
    check("y")
    want = lb.layer_norm(x[None], w, None, 1e-5, g[None])
    lb.check(out[:1], *want["y"], BF, "y")
    assert bool((mean == mean[0]).all()) and bool((rstd == rstd[0]).all())
    out.zero_()
    L.check(L.lib().drh_layer_norm_backward(ctx.handle, x.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                            g.data_ptr(), rows, D, 0, 0, 1, 1, out.data_ptr(), None, None, None, 0, s, L.SYNC))
    check("dx")
    lb.check(out[:1], *want["dx"], BF, "dx")
    ctx.close()


def test_dropout(layers):
    """Four 32-bit elements a thread."""
    n = (1 << 34) + 4099
    need(135)
    x = torch.ones(n, device="cuda")
    y = layers.dropout(x, 0.25, seed=8, offset=1)
    for first in (0, (1 << 34) - 2048, n - 1000):
        keep = lb.philox_keep(1000, 0.25, 8, 1, first=first // 8 * 8).cuda()
        assert same(y[first // 8 * 8:][:1000] != 0, keep[:n - first // 8 * 8]), first
    border = lb.philox_keep(6000, 0.25, 8, 1, first=(1 << 34) - 3000).cuda()
    assert same(y[(1 << 34) - 3000:][:6000] != 0, border)


def test_linear_of_one_row_and_many_outputs(layers):
    """Sixteen outputs a workgroup of 512 threads: 2^27 outputs are 2^32 threads."""
    N, K = (1 << 27) + 77, 8
    need(16)
    x = torch.randn(1, K, device="cuda").to(BF)
    w = torch.randn(N, K, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(BF)
    y = layers.linear(x, w)
    for first in (0, (1 << 27) - 500, N - 1000):
        part = w[first:first + 1000]
        lb.check(y[:, first:first + 1000], *lb.linear(x, part, None, None, None, None)["y"], BF, str(first))


def test_linear_of_many_rows_and_one_output(layers):
    """Tiles of 64 rows by 256 threads: 2^30 rows are 2^32 threads."""
    M, K = (1 << 30) + 77, 8
    need(60)
    g = torch.Generator("cuda").manual_seed(4)
    x = torch.empty(M, K, dtype=BF, device="cuda")
    for i in range(0, M, 1 << 27):
        x[i:i + (1 << 27)] = torch.randn(min(1 << 27, M - i), K, device="cuda", generator=g).to(BF)
    w = torch.randn(1, K, device="cuda", generator=g).to(BF)
    leaf = x.requires_grad_(True)
    y = layers.linear(leaf, w)
    (dx,) = torch.autograd.grad(y, leaf, torch.ones((), dtype=BF, device="cuda").expand_as(y))
    for first in (0, 1 << 29, (1 << 30) - 500, M - 1000):
        part = x.detach()[first:first + 1000]
        want = lb.linear(part, w, None, None, None, torch.ones(part.shape[0], 1, dtype=BF, device="cuda"))
        lb.check(y.detach()[first:first + 1000], *want["y"], BF, f"y {first}")
        lb.check(dx[first:first + 1000], *want["dx"], BF, f"dx {first}")


def test_what_no_launch_holds_is_refused(L):
    """2^38 outputs by the kernel that takes any alignment, which has a tile of 64 x 64 a workgroup."""
    f, ctx, t = L.lib(), L.Context(), torch.zeros(256, device="cuda", dtype=torch.uint8)
    p, n = t.data_ptr(), ctypes.c_uint64()
    M, N, K = 1 << 24, 1 << 14, 8
    L.check(f.drh_linear_bytes(M, N, K, K, K, 1, ctypes.byref(n)))
    assert n.value == 0
    for args in ((p + 2, p), (p, p + 2)):
        with pytest.raises(L.DiffrastError) as e:
            L.check(f.drh_linear(ctx.handle, *args, None, None, M, N, K, K, K, 1, 0, p, None, None, 0, None, 0))
        assert e.value.code == 5, e.value
    torch.cuda.synchronize()
    assert not bool(t.any())
    ctx.close()
