"""How far 8-bit states of noisy gradients are from 32-bit ones.

A root is rounded to one of two neighbours, `step` apart (1/16 to 1/8 of it), with its own value as the mean; its square then
gains the rounding's variance. From one step to the next a root moves on its grid by (1 - beta2) / 2 of |X - X'|, X the
chi-squared of its gradient and X' that of its block's largest, whose scale the grid has: 4 / pi of it in the mean. A root that
was on the grid and has moved by d is rounded with a variance below d step, so that v gains up to 0.0005 (4 / pi) / 8 of itself a step, where the
average forgets 0.001: a factor of 1 / (1 - 0.0796) = 1.087 at the most. And v's own variance gains 4 times as much, of which
1 - beta2^2 = 0.002 is forgotten: 0.159, a deviation of 0.40 of v's mean at the most, 0.43 of what it is in 32 bits."""

import pytest
import torch

import operator_bounds as ob
from test_gpu_adamw import values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spread", [0.0, 1.0])
def test_averages_of_noisy_gradients(spread):
    from diffrast import optim

    n, steps = 64 * 256, 6000
    gen = torch.Generator("cuda").manual_seed(11)
    size = torch.exp(spread * torch.randn(n, device="cuda", generator=gen))
    z = lambda **k: [torch.zeros(n, device="cuda", **k)]  # noqa: E731
    c = lambda: [torch.zeros(n // 256, device="cuda")]  # noqa: E731
    one = lambda: torch.zeros(1, dtype=torch.int64, device="cuda")  # noqa: E731
    small = dict(exp_avgs=z(dtype=ob.E4M3), exp_avg_sqs=z(dtype=ob.E4M3), exp_avg_scales=c(), exp_avg_sq_scales=c(), params=z(), steps=one())
    whole = dict(exp_avgs=z(), exp_avg_sqs=z(), params=z(), steps=one())
    sums = torch.zeros(3, dtype=torch.float64, device="cuda")
    for i in range(steps):
        g = [size * torch.randn(n, device="cuda", generator=gen)]
        optim.adamw_step(grads=g, seed=1, lr=1e-3, **small)
        optim.adamw_step(grads=g, lr=1e-3, **whole)
        if i >= steps // 2 and i % 50 == 0:
            x = values(small["exp_avg_sqs"][0], small["exp_avg_sq_scales"][0], True) / whole["exp_avg_sqs"][0].double()
            sums += torch.stack([x.mean(), (x * x).mean(), torch.ones((), dtype=torch.float64, device="cuda")])
    mean, square = float(sums[0] / sums[2]), float(sums[1] / sums[2])
    deviation = (square - mean * mean) ** 0.5
    # 16384 elements that deviate by 0.4: a hundredth is three of their mean's
    assert 0.99 <= mean <= 1.087 + 0.01 and deviation <= 0.43 + 0.01, (mean, deviation)
    assert mean > 1.0  # not the mean of v, but of its root
