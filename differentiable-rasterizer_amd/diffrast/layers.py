"""Layers of a network that answers with triangles, on MI355X through libdiffrast_hip.so.

    h = layer_norm(x, g1, b1)
    h = linear(h, w1, c1, activation="gelu")
    h = linear(h, w2, c2)
    x = dropout(h, 0.1, seed=seed, offset=step, residual=x)      # a residual block
    params = linear(x, w3, c3).float().view(B, T, 10)            # -> torch_layer.rasterize

or, with gated blocks (and `optim.AdamW` to train them),

    y, x = rms_norm(h, g1, residual=x)                           # x: the stream with h added
    h = linear(gated_linear(y, w1), w2)

and, to answer in 8 bits,

    q, t, x = rms_norm_8bit(h, g1, residual=x)
    h = linear_8bit(q, t, *w1_in_8_bits, activation="gelu")      # weights: quantize_8bit(w1)

The reference builds such a network from PyTorch's own layers (python/diffrast/model.py)
and has no counterpart of these. All of them but those in 8 bits are differentiable once; they take
float32, bfloat16 and float16, compute in 32 bits and round each result once. As in `torch_layer`,
tensors on the GPU stay there and run on torch's current stream, CPU tensors are moved to
the current GPU and the results returned on the caller's device, wrong arguments raise
ValueError, and there is no CPU path. Differentiating a gradient again raises RuntimeError, and
forward-mode derivatives and tracers (torch.jit.trace, make_fx, fake tensors) NotImplementedError;
torch.compile runs the calls outside of its graphs. The calls may be captured into a HIP graph.
`torch_layer.shutdown_gpu` does not concern them: they keep no buffers between calls.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import _lib, torch_layer

_lib.lib()  # the native module links against it

from . import _torch_layers  # noqa: E402

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _act(activation: str | None) -> int:
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r} — expected one of {list(ACTIVATIONS)}")
    return act


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """Layer norm over the last dimension: (x - mean) / sqrt(var + eps) * weight + bias.

    Args:
        x: `(..., D)`.
        weight, bias: `(D,)` each or None, of x's type or both float32.
        eps: added to the variance, which is the mean of squares about the mean.
    """
    y = _torch_layers.layer_norm(x, weight, bias, eps)
    torch_layer._note_gpu()
    return y


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = None,
           residual: Tensor | None = None) -> Tensor:
    """activation(x @ weight.T + bias) + residual, in one kernel.

    Args:
        x: `(..., K)`.
        weight: `(N, K)`, of x's type, as are bias and residual.
        bias: `(N,)` or None.
        activation: None, "relu", "gelu" (z Phi(z)), "gelu_tanh" or "silu".
        residual: `(..., N)` or None, added after the activation.

    The backward pass rounds dz = dy act'(z) to x's type for its two products; act'(z) is kept
    for it in float16 beside 16-bit types (in float32 otherwise), where there is an activation.
    """
    y = _torch_layers.linear(x, weight, bias, _act(activation), residual)
    torch_layer._note_gpu()
    return y


def gated_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = "silu") -> Tensor:
    """activation(z[..., :N]) * z[..., N:] with z = x @ weight.T + bias, in one kernel.

    Args:
        x: `(..., K)`.
        weight: `(2 N, K)`, the gate's rows first, of x's type, as is bias.
        bias: `(2 N,)` or None.
        activation: of the gate: None, "relu", "gelu" (z Phi(z)), "gelu_tanh" or "silu".

    The backward pass rounds the gradient of z to x's type for its two products (in float16 it ends at
    65504, as y does). For it the forward pass keeps the gate's value, and its slope times the other half: 5 bytes an output beside bfloat16
    (20 bits each), 6 beside float16 (24 bits) and 8 beside float32.
    """
    y = _torch_layers.gated_linear(x, weight, bias, _act(activation))
    torch_layer._note_gpu()
    return y


def rms_norm(x: Tensor, weight: Tensor | None = None, residual: Tensor | None = None, eps: float = 1e-5):
    """s / sqrt(mean(s^2) + eps) * weight over the last dimension, with s = x + residual.

    Returns y, or with a residual (y, s): the norm and the stream that it was taken of, both
    differentiable (of s the weight's gradient is zero, where s alone is used too). y is made
    from s in 32 bits; s is rounded to its type where it is stored, and the backward pass starts from that. The mean of squares is held in float32, which ends at 3e38.

    Args:
        x: `(..., D)`.
        weight: `(D,)` or None, of x's type or float32.
        residual: x's shape and type, or None.
    """
    r = _torch_layers.rms_norm(x, weight, residual, eps)
    torch_layer._note_gpu()
    return r[0] if residual is None else (r[0], r[1])


def rms_norm_8bit(x: Tensor, weight: Tensor | None = None, residual: Tensor | None = None, eps: float = 1e-5):
    """`rms_norm` with y in 8 bits: (q, scale), or with a residual (q, scale, s); for `linear_8bit`
    where D is a multiple of 16.

    q is float8_e4m3fn, y / scale rounded to nearest even, and scale `(...)` in float32 has
    max(max |y| / 448, 2^-126) for each row. No gradients: raises RuntimeError where they are wanted.
    """
    r = _torch_layers.rms_norm_8bit(x, weight, residual, eps)
    torch_layer._note_gpu()
    return tuple(r)


def quantize_8bit(x: Tensor) -> tuple[Tensor, Tensor]:
    """x `(..., D)` as (q, scale) of `rms_norm_8bit`, without the norm: activations, or a `(N, K)` weight.

    D may be any width; `linear_8bit` takes multiples of 16.
    """
    r = _torch_layers.quantize_8bit(x)
    torch_layer._note_gpu()
    return r[0], r[1]


def linear_8bit(x: Tensor, x_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Tensor | None = None,
                activation: str | None = None, residual: Tensor | None = None,
                dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """activation((x * x_scale) @ (weight * weight_scale).T + bias) + residual, in one kernel.

    Args:
        x: `(..., K)` and weight: `(N, K)`, float8_e4m3fn, K a multiple of 16.
        x_scale: `(...)` and weight_scale: `(N,)`, float32: a factor for each row.
        bias: `(N,)` or None; residual: `(..., N)` or None; of type dtype.
        activation: as in `linear`.
        dtype: of the output: float32, bfloat16 or float16. Sums of products are held in 32 bits for
            float32, and for the others, at twice the speed, as the matrix cores' 8-bit instructions hold
            them: within 2^-10 of their terms' magnitudes. For normal numbers that is 8e-6 of the result; in rows
            with outliers it may pass float16's own rounding, and bfloat16's where large terms cancel.

    No gradients: raises RuntimeError where they are wanted.
    """
    y = _torch_layers.linear_8bit(x, x_scale, weight, weight_scale, bias, _act(activation), residual, dtype)
    torch_layer._note_gpu()
    return y


def dropout(x: Tensor, p: float, *, seed: int, offset: int = 0, residual: Tensor | None = None) -> Tensor:
    """x with elements zeroed with probability p and the others scaled up, plus residual.

    The mask is a function of (seed, offset) and the element's place alone
    (drh_dropout in include/diffrast_hip.h says which) and is never stored: the backward
    pass draws it again. Call with another offset for another mask, say the step's
    number times the layers plus the layer's. p is applied in steps of 2^-16, and the
    scale is the inverse of what is applied. In a captured HIP graph seed and offset are
    what they were at capture: every replay draws the same mask.

    Args:
        x: any shape; p: in [0, 1); seed, offset: integers in [0, 2^64).
        residual: x's shape and type, or None.
    """
    for name, v in (("seed", seed), ("offset", offset)):
        if not (isinstance(v, int) and 0 <= v < 1 << 64):
            raise ValueError(f"{name} must be an integer in [0, 2^64)")
    y = _torch_layers.dropout(x, p, seed, offset, residual)
    torch_layer._note_gpu()
    return y
