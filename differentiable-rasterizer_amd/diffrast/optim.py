"""The optimiser's step of a network that answers with triangles, on MI355X through
libdiffrast_hip.so: AdamW over all of its tensors in one kernel, with states in 32 or 8 bits.

    opt = optim.AdamW(net.parameters(), lr=1e-3, state_bits=8)
    ...
    loss.backward()
    opt.step()

The reference trains its networks with PyTorch's own optimisers (python/train.py) and has no
counterpart of these. (Its fits' Adam, which projects triangles, is `drh_fit`.)
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch
from torch import Tensor

from . import layers, torch_layer

_step = layers._torch_layers.adamw

BLOCK = 256  # elements of an 8-bit state that share a scale


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor],
               steps: Tensor | Sequence[Tensor], *, exp_avg_scales: Sequence[Tensor] | None = None,
               exp_avg_sq_scales: Sequence[Tensor] | None = None, lr: float, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, seed: int = 0) -> None:
    """One AdamW step over all parameters, in place, on torch's current stream.

    For each parameter, with t = step + 1 (which its step becomes) and in 32 bits:

        exp_avg = beta1 exp_avg + (1 - beta1) grad
        exp_avg_sq = beta2 exp_avg_sq + (1 - beta2) grad^2
        param = param (1 - lr weight_decay)
                - lr / (1 - beta1^t) exp_avg / (sqrt(exp_avg_sq / (1 - beta2^t)) + eps)

    Args:
        params, grads: of one type (float32, bfloat16 or float16), on one GPU. Parameters
            are contiguous; gradients that are not are copied. Of what is written no two share memory, nor
            does a gradient share any of it.
        exp_avgs, exp_avg_sqs: float32 of the parameters' shapes; or, with scales, float8_e4m3fn, the
            second of the root.
        steps: an int64 tensor with a count for each parameter, or one tensor of shape () each, on
            the GPU: steps done so far.
        exp_avg_scales, exp_avg_sq_scales: float32, one scale for 256 elements in order (drh_adamw in
            include/diffrast_hip.h says how states are rounded to them).
        seed: of the random rounding of 8-bit states, in [0, 2^64).

    The call may be captured into a HIP graph: steps count on when it is replayed, lr and the other
    numbers are those of the capture. Wrong arguments raise before anything is written.
    """
    if not (isinstance(seed, int) and 0 <= seed < 1 << 64):
        raise ValueError("seed must be an integer in [0, 2^64)")
    lr, eps, weight_decay, (beta1, beta2) = float(lr), float(eps), float(weight_decay), betas
    _check_numbers(lr, beta1, beta2, eps, weight_decay)
    one = isinstance(steps, Tensor)
    _step(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, steps if one else None,
          None if one else steps, lr, beta1, beta2, eps, weight_decay, seed)
    torch_layer._note_gpu()


def _check_numbers(lr: float, beta1: float, beta2: float, eps: float, weight_decay: float) -> None:
    for name, v in (("lr", lr), ("eps", eps), ("weight_decay", weight_decay)):
        if not 0.0 <= v < math.inf:
            raise ValueError(f"{name} must be finite and not negative, got {v}")
    for v in (beta1, beta2):
        if not 0.0 <= v < 1.0:
            raise ValueError(f"betas must be in [0, 1), got {v}")


def _check_group(g: dict) -> None:
    _check_numbers(float(g["lr"]), *g["betas"], g["eps"], g["weight_decay"])
    if g["state_bits"] not in (32, 8):
        raise ValueError(f"state_bits must be 32 or 8, got {g['state_bits']}")
    if not (isinstance(g["seed"], int) and 0 <= g["seed"] < 1 << 63):
        raise ValueError("seed must be an integer in [0, 2^63)")


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW by `adamw_step`: one call for all parameters of a group that are of one type
    and on one GPU, one kernel for 48 of them.

    Args:
        params, lr, betas, eps, weight_decay: as torch.optim.AdamW's.
        state_bits: 32, or 8: a byte for each state and a float for 256 of them, 2.03 bytes a
            parameter instead of 8, rounded at random. The root of exp_avg_sq keeps its mean so, its square does not:
            for normal gradients and beta2 0.999 exp_avg_sq is 3 to 5% above that of 32 bits and deviates by a
            third of itself, which is a sixth in a step's length. Elements whose root is below 2^-15 of the largest of
            their 256 are coarser, and below 2^-18 held at that: they take shorter steps than they should.
        seed: of that rounding; the i-th call of a step takes its group's seed + i. It stands in the groups,
            and so in copies and state dicts: a run that loads one goes on with the seed it was saved with.

    A step may be captured into a HIP graph once every parameter has had one outside of it.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, seed: int = 0):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed)
        _check_group(defaults)
        super().__init__(params, defaults)

    def add_param_group(self, param_group: dict) -> None:
        _check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        for group in self.param_groups:  # of a state dict without a seed
            group.setdefault("seed", self.defaults.get("seed", 0))

    @property
    def seed(self) -> int:
        return self.param_groups[0]["seed"]

    def _state_of(self, p: Tensor, bits: int) -> dict:
        state = self.state[p]
        if not state:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a parameter's first step cannot be captured: its states would start anew with every replay")
            if not (p.is_cuda and p.layout == torch.strided and p.is_contiguous()):
                raise ValueError("parameters must be contiguous and on the GPU")
            state["step"] = torch.zeros((), dtype=torch.int64, device=p.device)
            kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=kind, device=p.device)
                if bits == 8:
                    state[name + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        call = 0
        for group in self.param_groups:
            bits, calls = group["state_bits"], {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                s = self.state.get(p) or self._state_of(p, bits)
                calls.setdefault((p.device, p.dtype, "exp_avg_scale" in s), []).append((p, p.grad, s))
            for (_, _, small), of in calls.items():
                states = [s for _, _, s in of]
                adamw_step([p for p, _, _ in of], [g for _, g, _ in of], [s["exp_avg"] for s in states],
                           [s["exp_avg_sq"] for s in states], [s["step"] for s in states],
                           exp_avg_scales=[s["exp_avg_scale"] for s in states] if small else None,
                           exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states] if small else None, lr=group["lr"],
                           betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], seed=group["seed"] + call)
                call += 1
        return loss

    def load_state_dict(self, state_dict) -> None:
        loaded = []

        def keep(_, d):  # behind the caller's own hooks: the dictionary as they leave it
            loaded.append(d)

        def restore(_):  # before theirs; as they were saved: the base class gives states the parameters' type
            saved = [i for g in loaded[-1]["param_groups"] for i in g["params"]]
            for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
                if i in loaded[-1]["state"]:
                    self.state[p] = {k: v.to(device=p.device, copy=True) if isinstance(v, Tensor) else v
                                     for k, v in loaded[-1]["state"][i].items()}

        with self.register_load_state_dict_pre_hook(keep), self.register_load_state_dict_post_hook(restore, prepend=True):
            super().load_state_dict(state_dict)
