"""diffrast.layers.quantize_8bit's codes are those of a division by the row's scale, to the bit: what lies
half way between two codes goes to the even one."""

import pytest
import torch

import operator_bounds as ob

pytestmark = pytest.mark.gpu
MOST = [49.0, 3.0625, 7.0, 448.0, 0.875, 35.0, 1.71875, 100.0, 55.75, 2.0**-9 * 49]  # scales that are exact, and not


def codes(x, scale):
    return (x.float().cpu() / scale.cpu()[:, None]).to(ob.E4M3).view(torch.uint8)


# rows in a wave's registers, in a workgroup's, and read again for each sum
@pytest.mark.parametrize("D", [255, 1500, 4096, 9000, 33001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_codes_are_a_divisions(dtype, D):
    from diffrast import layers

    g = torch.Generator().manual_seed(D)
    grid = torch.arange(126, dtype=torch.uint8).view(ob.E4M3).float()
    half = (grid + torch.arange(1, 127, dtype=torch.uint8).view(ob.E4M3).float()) / 2
    rows = []
    for most in MOST + ([49 * 2.0**-118, 49 * 2.0**-75, 49 * 2.0**100] if dtype != torch.float16 else []):
        at = half[torch.randint(len(half), (D,), generator=g)] * torch.where(torch.rand(D, generator=g) < 0.5, -1.0, 1.0)
        row = (at * (most / 448)).to(dtype)  # exact where the type holds them
        row[::3] = ((torch.rand(len(row[::3]), generator=g) * 2 - 1) * most).to(dtype)
        row[D // 2] = most
        rows.append(row)
    x = torch.stack(rows)
    q, s = layers.quantize_8bit(x.cuda())
    assert torch.equal(s.cpu(), x.float().abs().amax(1) / 448)
    ties = ((x.double() / s.cpu().double()[:, None]).abs()[..., None] == half.double()).any(-1).sum()
    assert int(ties) > D  # there are some
    assert torch.equal(q.cpu().view(torch.uint8), codes(x, s))


def test_two_numbers():
    """49 / 448 is 0.109375: 0.1708984375 and 0.341796875 are 1.5625 and 3.125 of it, half way."""
    from diffrast import layers

    q, s = layers.quantize_8bit(torch.tensor([[49.0, 0.1708984375, 0.341796875]], dtype=torch.bfloat16, device="cuda"))
    assert float(s[0]) == 0.109375 and q[0].float().tolist() == [448.0, 1.5, 3.0]


def test_any_numbers():
    from diffrast import layers

    x = torch.randn(20000, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    x *= torch.exp2(torch.linspace(-130, 110, 20000, device="cuda"))[:, None]
    q, s = layers.quantize_8bit(x)
    assert torch.equal(q.view(torch.uint8), (x / s[:, None]).to(ob.E4M3).view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_zeros_keep_their_signs(dtype):
    from diffrast import layers

    for D in (300, 40000):
        x = torch.zeros(3, D, dtype=dtype, device="cuda")
        x[:, ::3] = -0.0
        x[1, 1], x[2, 1] = 3.0, -1e-4
        q, s = layers.quantize_8bit(x)
        assert torch.equal(q.view(torch.uint8), (x.float() / s[:, None]).to(ob.E4M3).view(torch.uint8))
