"""Plain forms of the network layers in 64 bits, and how far a right implementation in
32 bits may be from them, element by element.

u is half the relative spacing of the result's type, 2^-p for p significant bits; every
result is rounded once, to within u |y|, or half the smallest number below the normal ones. A sum of n terms in 32 bits, in any order, is
within n 2^-24 of the sum of magnitudes. Activations: float32's expf, erff and division
are within a few 2^-24 (16 are allowed for their composition); the 16-bit types' erf is
within 1.5e-7 and their exp and reciprocal within a few 2^-22 (2^-20 allowed).
"""

from __future__ import annotations

import math

import torch

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}
E = 2.0**-24
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def act(kind, z):
    if kind is None:
        return z
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z**3))


def slope(kind, z):
    z = z.detach().requires_grad_(True)
    with torch.enable_grad():
        (d,) = torch.autograd.grad(act(kind, z).sum(), z)
    return d


def act_error(kind, dtype):
    """Of an activation's value, over |z|, and of its slope, both beside z's own error."""
    if kind in (None, "relu"):
        return 0.0, 0.0
    return (16 * E, 64 * E) if dtype == torch.float32 else (2.0**-20, 2.0**-18)


def check(got, want, bound, dtype, label=""):
    """got (of type dtype) within bound of want before its one rounding."""
    assert got.dtype == dtype and got.shape == want.shape, (label, got.dtype, got.shape, want.shape)
    if want.numel() == 0:
        return
    d = (got.double() - want).abs()
    lim = bound + U[dtype] * (want.abs() + bound) + TINY[dtype]
    worst = float((d / lim).max())
    assert bool((d <= lim).all()), f"{label}: {worst:.3f} times its bound"


def linear(x, w, b, kind, res, g, check_fwd=None):
    """{name: (value, bound)} of y and the gradients, from tensors of the type under test."""
    dt, K, (N, _) = x.dtype, x.shape[-1], w.shape
    X, W, G = x.double().reshape(-1, K), w.double(), None if g is None else g.double().reshape(-1, N)
    M = X.shape[0]
    z = X @ W.t()
    ez = (K + 1) * E * (X.abs() @ W.abs().t())
    if b is not None:
        z = z + b.double()
        ez = ez + E * z.abs()
    a, (ea, es) = act(kind, z), act_error(kind, dt)
    y, ey = a, 1.13 * ez + ea * z.abs()
    if res is not None:
        y = y + res.double().reshape(-1, N)
        ey = ey + E * y.abs()
    out = {"y": (y, ey)}
    if g is None:
        return out
    if kind is None:
        dz, edz = G, torch.zeros_like(G)
    else:
        # no slope changes faster than 1.13 per unit of z; it is kept in 32 bits, or in float16
        d = slope(kind, z)
        ds = 1.13 * ez + es
        ds = ds + (E if dt == torch.float32 else 2.0**-11) * (d.abs() + ds) + 2.0**-25
        if kind == "relu":  # its slope turns at zero alone
            ds = torch.where(z.abs() <= ez, torch.ones_like(z), torch.zeros_like(z))
        dz = G * d
        edz = G.abs() * ds + E * dz.abs()
    # dz is rounded to its type for the products, not for the bias gradient
    er = edz + (U[dt] * (dz.abs() + edz) + TINY[dt] if kind is not None else 0.0)
    out["dx"] = (dz @ W, er @ W.abs() + (N + 1) * E * ((dz.abs() + er) @ W.abs()))
    out["dweight"] = (dz.t() @ X, er.t() @ X.abs() + (M + 1) * E * ((dz.abs() + er).t() @ X.abs()))
    out["dbias"] = (dz.sum(0), edz.sum(0) + (M + 1) * E * (dz.abs() + edz).sum(0))
    return out


def layer_norm(x, w, b, eps, g):
    """{name: (value, bound)}; a row's statistics are within D 2^-24 of its magnitudes."""
    D = x.shape[-1]
    X = x.double().reshape(-1, D)
    one = torch.ones(D, dtype=torch.float64, device=x.device)
    W, B = (one if w is None else w.double()), (0 * one if b is None else b.double())
    mu = X.mean(1, keepdim=True)
    var = ((X - mu) ** 2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (X - mu) * r
    emu = (D + 1) * E * X.abs().mean(1, keepdim=True)
    # the variance about a mean that is emu off is emu^2 more; r moves by half its relative error
    er = 0.5 * ((D + 4) * E + emu**2 * r**2) + 4 * E
    eh = emu * r + h.abs() * er + 2 * E * (h.abs() + 1)
    y = h * W + B
    out = {"y": (y, eh * W.abs() + 2 * E * (y.abs() + (h * W).abs()))}
    if g is None:
        return out
    G = g.double().reshape(-1, D)
    rows = X.shape[0]
    u = G * W
    m1, m2 = u.mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
    dx = r * (u - m1 - h * m2)
    em1 = (D + 2) * E * u.abs().mean(1, keepdim=True)
    em2 = (D + 3) * E * (u * h).abs().mean(1, keepdim=True) + (u.abs() * eh).mean(1, keepdim=True)
    edx = r * (4 * E * (u.abs() + m1.abs() + (h * m2).abs()) + em1 + eh * m2.abs() + h.abs() * em2) + dx.abs() * (er + 4 * E)
    out["dx"] = (dx, edx)
    out["dweight"] = ((G * h).sum(0), (G.abs() * eh).sum(0) + (rows + 2) * E * (G * h).abs().sum(0))
    out["dbias"] = (G.sum(0), (rows + 1) * E * G.abs().sum(0))
    return out


def philox_keep(n, p, seed, offset, first=0):
    """The mask that drh_dropout documents for n elements from `first` on, in Python's own
    integers and numpy."""
    import numpy as np

    m32, u = 0xFFFFFFFF, np.uint64
    blocks = np.arange(first // 8, (first + n + 7) // 8, dtype=u)
    c = [blocks & u(m32), blocks >> u(32), np.full_like(blocks, offset & m32), np.full_like(blocks, offset >> 32)]
    k = [seed & m32, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & u(m32), (a >> u(32)) ^ c[3] ^ u(k[1]), a & u(m32)]
        k = [(k[0] + 0x9E3779B9) & m32, (k[1] + 0xBB67AE85) & m32]
    words = np.stack(c, 1)
    bits = np.stack([words & u(0xFFFF), words >> u(16)], 2).reshape(-1)[first % 8:][:n].astype(np.int64)
    return torch.from_numpy(bits >= int(round(p * 65536)))
