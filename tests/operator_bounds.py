"""Plain forms in 64 bits of the norms, products and optimiser steps of layers.py and optim.py
that layer_bounds.py does not hold, and how far a right implementation in 32 bits may be from
them, element by element, with layer_bounds.py's constants.

e4m3 has 4 significant bits down to 2^-6 and steps of 2^-9 below: rounded to nearest it is within
2^-4 of the value or 2^-10.
"""

from __future__ import annotations

import torch

from layer_bounds import E, TINY, U, act, act_error, check, slope  # noqa: F401

E4M3 = torch.float8_e4m3fn
LEAST = 2.0**-126


def rms_norm(x, w, res, eps, g=None, gs=None):
    """{name: (value, bound)}: y, sum, and with g the gradients; from tensors of the type under test."""
    D, dt = x.shape[-1], x.dtype
    s = x.double().reshape(-1, D)
    if res is not None:
        s = s + res.double().reshape(-1, D)
    W = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    r = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    h = s * r
    y = h * W
    # a square is 3 E off (its s is one), a sum of D of them D E more; r moves by half its argument's error
    er = 0.5 * (D + 8) * E + 4 * E
    out = {"y": (y, y.abs() * (er + 4 * E)), "sum": (s, s.abs() * E)}
    if g is None:
        return out
    G = g.double().reshape(-1, D)
    # the backward pass reads the sum as it was stored
    stored = U[dt] if res is not None else 0.0
    eh = h.abs() * (er + 3 * E + stored) + (TINY[dt] * r if res is not None else 0.0)
    u = G * W
    m = (u * h).mean(1, keepdim=True)
    em = (D + 3) * E * (u * h).abs().mean(1, keepdim=True) + (u.abs() * eh).mean(1, keepdim=True)
    dn = r * (u - h * m)
    edx = r * (4 * E * (u.abs() + (h * m).abs()) + eh * m.abs() + h.abs() * em + eh * em) + dn.abs() * (er + 4 * E)
    dx = dn
    if gs is not None:
        dx = dn + gs.double().reshape(-1, D)
        edx = edx + 2 * E * (dn.abs() + dx.abs())
    out["dx"] = (dx, edx)
    rows = s.shape[0]
    out["dweight"] = ((G * h).sum(0), (G.abs() * eh).sum(0) + (rows + 2) * E * (G * h).abs().sum(0))
    return out


def check_8bit(q, scale, y, ey, label=""):
    """q and scale stand for y, whose value in 32 bits may be ey off."""
    assert q.dtype == E4M3 and scale.dtype == torch.float32 and q.shape[:-1] == scale.shape, label
    v, s = q.double().reshape(y.shape), scale.double().reshape(-1, 1)
    want = (y.abs().max(1, keepdim=True).values / 448).clamp(min=LEAST)
    lim = (ey.max(1, keepdim=True).values / 448) * (1 + 4 * E) + 4 * E * want
    assert bool(((s - want).abs() <= lim).all()), f"{label}: scale"
    lim = 2.0**-4 * (y.abs() + ey) + 2.0**-10 * s + ey + 4 * E * y.abs()
    d = (v * s - y).abs()
    assert bool((d <= lim).all()), f"{label}: {float((d / lim).max()):.3f} times its bound"


def _activated(kind, z, ez, dt):
    """act(z) and its slope with their bounds, where z is ez off."""
    a, (ea, es) = act(kind, z), act_error(kind, dt)
    eact = 1.13 * ez + ea * z.abs()
    if kind is None:
        return a, ez, torch.ones_like(z), torch.zeros_like(z)
    d = slope(kind, z)
    if kind == "relu":  # its slope turns at zero alone
        ed = torch.where(z.abs() <= ez, torch.ones_like(z), torch.zeros_like(z))
    else:
        ed = 1.13 * ez + es
    return a, eact, d, ed


# what the gated layer keeps its pairs in, cut off: 12 and 16 significant bits
KEPT = {torch.float32: 0.0, torch.bfloat16: 2.0**-11, torch.float16: 2.0**-15}


def gated_linear(x, w, b, kind, g=None):
    dt, K = x.dtype, x.shape[-1]
    N = w.shape[0] // 2
    X, W = x.double().flatten(0, -2) if x.dim() > 1 else x.double()[None], w.double()
    z = X @ W.t()
    ez = (K + 1) * E * (X.abs() @ W.abs().t())
    if b is not None:
        z = z + b.double()
        ez = ez + E * z.abs()
    if dt == torch.float32:  # what thirds drop of a term, and split sums' additions
        ez = ez + 2.0**-21 * (X.abs() @ W.abs().t())
    zg, zu, eg, eu = z[:, :N], z[:, N:], ez[:, :N], ez[:, N:]
    a, ea, d, ed = _activated(kind, zg, eg, dt)
    y = a * zu
    out = {"y": (y, a.abs() * eu + zu.abs() * ea + ea * eu + E * y.abs())}
    if g is None:
        return out
    G = g.double().reshape(-1, N)
    M = G.shape[0]
    b2 = d * zu
    eb = d.abs() * eu + zu.abs() * ed + ed * eu + E * b2.abs()
    k = KEPT[dt]
    ea, eb = ea + k * (a.abs() + ea), eb + k * (b2.abs() + eb)
    dz = torch.cat([G * b2, G * a], 1)
    edz = torch.cat([G.abs() * eb, G.abs() * ea], 1) + E * dz.abs()
    er = edz + U[dt] * (dz.abs() + edz) + TINY[dt]
    cut = 2.0**-21 if dt == torch.float32 else 0.0
    out["dx"] = (dz @ W, er @ W.abs() + ((2 * N + 1) * E + cut) * ((dz.abs() + er) @ W.abs()))
    out["dweight"] = (dz.t() @ X, er.t() @ X.abs() + ((M + 1) * E + cut) * ((dz.abs() + er).t() @ X.abs()))
    out["dbias"] = (dz.sum(0), edz.sum(0) + (M + 1) * E * (dz.abs() + edz).sum(0))
    return out


def linear_8bit(x, xs, w, ws, b, kind, res, dt):
    """(value, bound) of y."""
    K, N = x.shape[-1], w.shape[0]
    X = x.double().reshape(-1, K) * xs.double().reshape(-1, 1)
    W = w.double() * ws.double()[:, None]
    z, terms = X @ W.t(), X.abs() @ W.abs().t()
    # the 8-bit instructions lose up to 2^-10 of the terms' magnitudes; two scales and a bias follow
    ez = ((K + 1) * E + (0.0 if dt == torch.float32 else 2.0**-10)) * terms + 3 * E * z.abs()
    if b is not None:
        z = z + b.double()
        ez = ez + E * z.abs()
    y, ey, _, _ = _activated(kind, z, ez, dt)
    if res is not None:
        y = y + res.double().reshape(-1, N)
        ey = ey + E * y.abs()
    return y, ey


def adamw(p, g, m, v, t, lr, b1, b2, eps, wd):
    """{name: (value, bound)} of a parameter, m and v (m and v in 64 bits or 32)."""
    p, g, m, v = (a.double() for a in (p, g, m, v))
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    # the constants' rounding, a product each and the sum
    em = 4 * E * ((b1 * m).abs() + ((1 - b1) * g).abs())
    ev = 6 * E * v1 + 2.0**-148
    c1, c2 = 1 - b1**t, 1 - b2**t
    den = torch.sqrt(v1 / c2) + eps
    step = lr / c1 * m1 / den
    # the root moves by half of v's relative error, or by the root of what v lost below the normal numbers
    eden = torch.sqrt(v1 / c2) * 12 * E + 2.0**-74 / c2**0.5
    estep = lr / c1 * em / den + step.abs() * (eden / den + 12 * E)
    new = p - lr * wd * p - step
    ep = 4 * E * (p.abs() + step.abs()) + estep
    return {"p": (new, ep), "m": (m1, em), "v": (v1, ev)}
