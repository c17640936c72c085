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


def balance64(l, fn):
    if fn == "softmax":
        return torch.exp(l - l.max(1, keepdim=True).values)
    return torch.sigmoid(l) if fn == "sigmoid" else torch.sqrt(torch.nn.functional.softplus(l, threshold=1000.0))


def balance_grad(ops, lg, idx, fn, alpha, up):
    """(loss, gradient) and the same in float64."""
    t, e = lg.shape
    x = lg.clone().requires_grad_(True)
    loss, counts = ops.balance_loss(x, idx, fn, alpha)
    grad, = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"))
    l64 = lg.double().requires_grad_(True)
    s = balance64(l64, fn)
    want = alpha * (counts.double() * e / counts.sum() * (s / s.sum(1, keepdim=True))).sum() / t
    gw, = torch.autograd.grad(want * up, l64)
    return loss.detach(), grad, want.detach(), gw


@pytest.mark.parametrize("fn,lo,top,budget", [("softmax", -86, 0, 24), ("sigmoid", -86, 40, 28),
                                              ("sqrtsoftplus", -170, 16, 48)])
@pytest.mark.parametrize("t", [200, 3000])
def test_balance_gradient_far_below_the_maximum(ops, fn, lo, top, budget, t):
    """Two experts, every pick on the first, whose logit is `top`; the second's
    is far below.  Then sum score = the first's score, p of it is 1, g of the
    second is 0, and its gradient is -alpha up p r g0 / t: a product of few
    factors.  Logits are multiples of 1/8, so differences are exact.  Steps of
    2^-24: the exponential 6; softmax adds p, 1 / sum, d, its scaling and two
    products, 2 each (16 in all); sigmoid a quotient of a square, 8 (24);
    sqrtsoftplus the series 4, quotients 8, two roots 6 and the first score's
    6 twice, 44."""
    l = torch.randint(lo * 8, -20 * 8, (t,), generator=gen(t), device="cuda").float() / 8
    lg = torch.stack([torch.full_like(l, float(top)), l], 1)
    idx = torch.zeros(t, 1, dtype=torch.int32, device="cuda")
    _, grad, _, gw = balance_grad(ops, lg, idx, fn, float(t), 1.0)
    assert ((grad[:, 1].double() - gw[:, 1]).abs() <= budget * 2.0 ** -24 * gw[:, 1].abs()).all()


@pytest.mark.parametrize("fn,l", [("sigmoid", -84.0), ("sqrtsoftplus", -100.0), ("sqrtsoftplus", -160.0)])
@pytest.mark.parametrize("t", [40, 1000])
def test_balance_rows_of_small_scores(ops, fn, l, t):
    """Rows whose scores are all small, and a large upstream gradient (a loss
    scale): p is what it is for large scores, and nothing overflows.  Steps of
    2^-24: 96 as for any row of the balance loss."""
    lg = l + torch.randint(0, 16, (t, 8), generator=gen(t), device="cuda").float() / 8
    idx = torch.topk(lg + torch.arange(8, device="cuda"), 2, dim=1).indices.int()
    loss, grad, want, gw = balance_grad(ops, lg, idx, fn, 1.0, 65536.0)
    tol = 96 * 2.0 ** -24
    assert abs(float(loss) - float(want)) <= tol * float(want)
    # |g| + |d| bounds what cancels: at most twice E / t for one expert with every pick
    s = balance64(lg.double(), fn)
    p = s / s.sum(1, keepdim=True)
    assert ((grad.double() - gw).abs() <= tol * 65536.0 * p * 16 / t).all()
