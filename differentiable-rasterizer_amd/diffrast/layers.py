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
ValueError, and there is no CPU path. Differentiating a gradient again raises RuntimeError, and
forward-mode derivatives and tracers (torch.jit.trace, make_fx, fake tensors) NotImplementedError;
torch.compile runs the calls outside of its graphs. The calls may be captured into a HIP graph.
`torch_layer.shutdown_gpu` does not concern them: they keep no buffers between calls.
"""

from __future__ import annotations

from torch import Tensor

from . import _lib, torch_layer

_lib.lib()  # the native module links against it

from . import _torch_layers  # noqa: E402

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


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
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r} — expected one of {list(ACTIVATIONS)}")
    y = _torch_layers.linear(x, weight, bias, act, residual)
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
