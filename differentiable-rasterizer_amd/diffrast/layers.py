"""Layers of a network that answers with triangles, on MI355X through libdiffrast_hip.so.

    h = layer_norm(x, g1, b1)
    h = linear(h, w1, c1, activation="gelu")
    h = linear(h, w2, c2)
    x = dropout(h, 0.1, seed=seed, offset=step, residual=x)      # a residual block
    params = linear(x, w3, c3).float().view(B, T, 10)            # -> torch_layer.rasterize

The reference builds such a network from PyTorch's own layers (python/diffrast/model.py)
and has no counterpart of these. All of them are differentiable once, take float32,
bfloat16 and float16, compute in 32 bits and round each result once. As in `torch_layer`,
tensors on the GPU stay there and run on torch's current stream, CPU tensors are moved to
the current GPU and the results returned on the caller's device, wrong arguments raise
ValueError, and there is no CPU path. The calls may be captured into a HIP graph.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from . import _lib, torch_layer

DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _dtype(t: Tensor) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"expected float32, bfloat16 or float16, got {t.dtype}")
    return code


def _rows(x: Tensor) -> Tensor:
    """x as (rows, features) with contiguous features: a view where x's strides allow."""
    if x.dim() == 2:
        if x.is_contiguous():
            return x
        v = x
    else:
        D = x.shape[-1]
        v = x.reshape(x.numel() // D if D else math.prod(x.shape[:-1]), D)
    if v.stride(1) != 1 or (v.shape[0] > 1 and v.stride(0) < v.shape[1]):
        v = v.contiguous()
    return v


def _stride(v: Tensor) -> int:
    """Elements between the rows of _rows' view; one row has no stride of its own."""
    return v.stride(0) if v.shape[0] > 1 else v.shape[1]


def _flat(t: Tensor | None) -> Tensor | None:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _ptr(t: Tensor | None):
    return None if t is None else t.data_ptr()


def _enter(dev: torch.device):
    """(context handle, stream handle) of a call on `dev`. The stream is torch's current
    one, without the Stream object around it, which costs 2 us a call."""
    ctx = torch_layer._contexts.get(dev.index)
    if ctx is None:
        ctx = torch_layer._context(dev)
    torch_layer._note_gpu()
    return ctx.handle, torch._C._cuda_getCurrentRawStream(dev.index)


def _bytes(fn, *sizes) -> int:
    n = ctypes.c_uint64()
    _lib.check(fn(*sizes, ctypes.byref(n)))
    return n.value


def _workspace(n: int, dev: torch.device) -> Tensor | None:
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _elsewhere(x: Tensor, *others: Tensor | None) -> bool:
    """Whether a tensor is not on the GPU that x is on (or x on none)."""
    if not x.is_cuda:
        return True
    for t in others:
        if t is not None and t.device != x.device:
            return True
    return False


def _moved(x: Tensor, *others: Tensor | None):
    """The tensors on the GPU that x is on, or on the current one."""
    dev = x.device if x.is_cuda else torch_layer._gpu()
    return [t if t is None else t.to(dev) for t in (x, *others)]


def _once(backward):
    """`backward`, differentiable once. torch's own wrapper for that is entered only where a
    graph of the backward pass is asked for, since it costs 4 us a call."""
    wrapped = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return wrapped(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


# ---------------------------------------------------------------- layer norm


def _layer_norm_forward(x, weight, bias, eps, keep):
    dev = x.device
    xv = _rows(x)
    rows, cols = xv.shape
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    if keep:
        stats = torch.empty((2, rows), dtype=torch.float32, device=dev)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    else:
        stats = mean = rstd = None
    code = DTYPES[x.dtype]
    wcode = DTYPES[weight.dtype] if weight is not None else DTYPES[bias.dtype] if bias is not None else code
    handle, stream = _enter(dev)
    _lib.check(_lib.lib().drh_layer_norm(
        handle, xv.data_ptr(), _ptr(weight), _ptr(bias), rows, cols, _stride(xv), code, wcode, eps, y.data_ptr(),
        mean, rstd, stream, 0))
    return y, xv, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        weight, bias = _flat(weight), _flat(bias)
        y, xv, stats = _layer_norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(xv, weight, bias, stats)
        return y

    @staticmethod
    @_once
    def backward(ctx, g):
        xv, weight, bias, stats = ctx.saved_tensors
        dev = xv.device
        rows, cols = xv.shape
        gv = _rows(g)
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        dx = torch.empty_like(g, memory_format=torch.contiguous_format) if want_x else None
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        code = DTYPES[xv.dtype]
        wcode = DTYPES[weight.dtype] if weight is not None else DTYPES[bias.dtype] if bias is not None else code
        L = _lib.lib()
        n = _bytes(L.drh_layer_norm_backward_bytes, rows, cols) if want_w or want_b else 0
        ws = _workspace(n, dev)
        mean = stats.data_ptr()
        handle, stream = _enter(dev)
        _lib.check(L.drh_layer_norm_backward(
            handle, xv.data_ptr(), _ptr(weight), mean, mean + 4 * rows, gv.data_ptr(), rows, cols, _stride(xv),
            _stride(gv), code, wcode, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n, stream, 0))
        return dx, dw, db, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """Layer norm over the last dimension: (x - mean) / sqrt(var + eps) * weight + bias.

    Args:
        x: `(..., D)`.
        weight, bias: `(D,)` each or None, of x's type or both float32.
        eps: added to the variance, which is the mean of squares about the mean.
    """
    _dtype(x)
    D = x.shape[-1] if x.dim() else 0
    if D == 0:
        raise ValueError(f"expected x of shape (..., D), got {tuple(x.shape)}")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != D:
            raise ValueError(f"expected {name} of shape ({D},), got {tuple(t.shape)}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise ValueError(f"expected {name} in {x.dtype} or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight is {weight.dtype} but bias {bias.dtype}")
    if _elsewhere(x, weight, bias):
        return layer_norm(*_moved(x, weight, bias), eps=eps).to(x.device)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _layer_norm_forward(x, _flat(weight), _flat(bias), eps, False)[0]


# ---------------------------------------------------------------- linear


def _linear_forward(x, weight, bias, act, residual, keep):
    dev = x.device
    xv = _rows(x)
    rows, n_in = xv.shape
    n_out = weight.shape[0]
    y = x.new_empty((rows, n_out) if x.dim() == 2 else (*x.shape[:-1], n_out))
    kept = None
    if keep and act:
        kept = torch.empty((rows, n_out), dtype=torch.float32 if x.dtype == torch.float32 else torch.float16, device=dev)
    xs, wst, code = _stride(xv), _stride(weight), DTYPES[x.dtype]
    L = _lib.lib()
    n = _bytes(L.drh_linear_bytes, rows, n_out, n_in, xs, wst, code)
    ws = _workspace(n, dev)
    handle, stream = _enter(dev)
    _lib.check(L.drh_linear(
        handle, xv.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(residual), rows, n_out, n_in, xs, wst, code, act,
        y.data_ptr(), _ptr(kept), _ptr(ws), n, stream, 0))
    return y, xv, kept


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        weight = _rows(weight)
        y, xv, kept = _linear_forward(x, weight, _flat(bias), act, _flat(residual), True)
        ctx.save_for_backward(xv, weight, kept)
        ctx.act = act
        ctx.x_shape = x.shape
        return y

    @staticmethod
    @_once
    def backward(ctx, g):
        xv, weight, kept = ctx.saved_tensors
        dev, dt = xv.device, xv.dtype
        rows, n_in = xv.shape
        n_out = weight.shape[0]
        want_x, want_w, want_b, _, want_r = ctx.needs_input_grad
        dx = xv.new_empty(ctx.x_shape) if want_x else None
        dw = xv.new_empty((n_out, n_in)) if want_w else None
        db = xv.new_empty(n_out) if want_b else None
        if want_x or want_w or want_b:
            g = g.contiguous()
            L = _lib.lib()
            xs, wst, code = _stride(xv), _stride(weight), DTYPES[dt]
            n = _bytes(L.drh_linear_backward_bytes, rows, n_out, n_in, xs, wst, code, ctx.act)
            ws = _workspace(n, dev)
            handle, stream = _enter(dev)
            _lib.check(L.drh_linear_backward(
                handle, xv.data_ptr(), weight.data_ptr(), _ptr(kept), g.data_ptr(), rows, n_out, n_in, xs, wst, code,
                ctx.act, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n, stream, 0))
        return dx, dw, db, None, g if want_r else None


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = None,
           residual: Tensor | None = None) -> Tensor:
    """activation(x @ weight.T + bias) + residual, in one kernel.

    Args:
        x: `(..., K)`.
        weight: `(N, K)`, of x's type, as are bias and residual.
        bias: `(N,)` or None.
        activation: None, "relu", "gelu" (z Phi(z)), "gelu_tanh" or "silu".
        residual: `(..., N)` or None, added after the activation.

    The backward pass rounds dz = dy act'(z) to x's type for its two products, and keeps z
    for it in float16 beside 16-bit types (in float32 otherwise), where there is an activation.
    """
    _dtype(x)
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r} — expected one of {list(ACTIVATIONS)}")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] == 0:
        raise ValueError(f"expected x (..., K) and weight (N, K), got {tuple(x.shape)} and {tuple(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"expected bias of shape ({weight.shape[0]},), got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], weight.shape[0]):
        raise ValueError(f"expected residual of shape {(*x.shape[:-1], weight.shape[0])}, got {tuple(residual.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise ValueError(f"x is {x.dtype} but {name} {t.dtype}")
    if _elsewhere(x, weight, bias, residual):
        xd, wd, bd, rd = _moved(x, weight, bias, residual)
        return linear(xd, wd, bd, activation, rd).to(x.device)
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, act, residual)
    return _linear_forward(x, _rows(weight), _flat(bias), act, _flat(residual), False)[0]


# ---------------------------------------------------------------- dropout


def _dropout(x, residual, p, seed, offset):
    x = x.contiguous()
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    handle, stream = _enter(x.device)
    _lib.check(_lib.lib().drh_dropout(handle, x.data_ptr(), _ptr(residual), x.numel(), DTYPES[x.dtype], p, seed, offset,
                                      y.data_ptr(), stream, 0))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, residual):
        ctx.draw = (p, seed, offset)
        return _dropout(x, _flat(residual), p, seed, offset)

    @staticmethod
    @_once
    def backward(ctx, g):
        dx = _dropout(g, None, *ctx.draw) if ctx.needs_input_grad[0] else None
        return dx, None, None, None, g if ctx.needs_input_grad[4] else None


def dropout(x: Tensor, p: float, *, seed: int, offset: int = 0, residual: Tensor | None = None) -> Tensor:
    """x with elements zeroed with probability p and the others scaled up, plus residual.

    The mask is a function of (seed, offset) and the element's place alone
    (drh_dropout in include/diffrast_hip.h says which) and is never stored: the backward
    pass draws it again. Call with another offset for another mask, say the step's
    number times the layers plus the layer's. p is applied in steps of 2^-16, and the
    scale is the inverse of what is applied.

    Args:
        x: any shape; p: in [0, 1); seed, offset: integers in [0, 2^64).
        residual: x's shape and type, or None.
    """
    _dtype(x)
    if not 0.0 <= p < 1.0:
        raise ValueError("p must be in [0, 1)")
    for name, v in (("seed", seed), ("offset", offset)):
        if not (isinstance(v, int) and 0 <= v < 1 << 64):
            raise ValueError(f"{name} must be an integer in [0, 2^64)")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"expected a residual of shape {tuple(x.shape)} in {x.dtype}, got "
                         f"{tuple(residual.shape)} in {residual.dtype}")
    if _elsewhere(x, residual):
        xd, rd = _moved(x, residual)
        return dropout(xd, p, seed=seed, offset=offset, residual=rd).to(x.device)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, p, seed, offset, residual)
    return _dropout(x, _flat(residual), p, seed, offset)
