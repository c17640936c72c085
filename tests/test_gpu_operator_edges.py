"""Values at which the FP8 operators and the balance loss are hard to get
right, on the GPU against 64-bit definitions."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from dsv4_plugin import ops
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def e4m3_grid(v):
    """Nearest E4M3 value of float64 v, ties to even, saturating."""
    v = v.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


@pytest.mark.parametrize("cols", [128, 127])
@pytest.mark.parametrize("steps", [0, 1, -1])
def test_act_quant_fp32_ties(ops, cols, steps):
    """fp32 x whose 448 x / amax is a tie of E4M3, or one step of x beside it.
    With amax = 448 m and x = t m for an integer m of 19 bits and a tie t of 5,
    both are fp32 numbers and the quotient is t.  The float64 quotient has an
    error of 2^-53 and a step of x moves it by 2^-24, so the reference's code
    is the nearest one: no tolerance."""
    rows, g = 4000, gen(cols + steps)
    m = torch.randint(1 << 18, 1 << 19, (rows, 1), generator=g, device="cuda").double() * 2.0 ** -19
    odd = 2 * torch.randint(8, 16, (rows, cols), generator=g, device="cuda").double() + 1
    t = odd * torch.exp2(torch.randint(-10, 4, (rows, cols), generator=g, device="cuda").double())
    t = t * (1 - 2 * torch.randint(0, 2, (rows, cols), generator=g, device="cuda").double())
    x = (t * m).float()
    assert torch.equal(x.double(), t * m)
    if steps:
        x = torch.nextafter(x, torch.full_like(x, steps * float("inf")))
    x[:, 5] = (448 * m[:, 0]).float()
    q, s = ops.act_quant(x, 128, None)
    amax = x.double().abs().amax(1, keepdim=True)
    assert torch.equal(amax, 448 * m)
    assert torch.equal(q.double(), e4m3_grid(x.double() * 448.0 / amax))
