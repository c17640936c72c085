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


@pytest.mark.parametrize("n", [2304, 2432, 4480, 4608, 4736])
@pytest.mark.parametrize("m", [16, 32, 64])
@pytest.mark.parametrize("k", [512, 2048, 4096])
def test_fp8_linear_is_its_parts_where_clusters_fill_the_gpu(ops, m, n, k):
    """As many clusters as the SMs take, and one more: a cluster size that
    does not fit is made smaller, in one launch as in two."""
    g = gen(m + n + k)
    w = (torch.randn((n, k), generator=g, device="cuda") * 100).clamp(-448, 448).to(F8)
    ws = torch.exp2(torch.randint(-15, -8, (-(-n // 128), -(-k // 128)), generator=g, device="cuda").float()).to(E8)
    x = torch.randn((m, k), generator=g, device="cuda").bfloat16()
    want = ops.fp8_matmul(*ops.act_quant(x, 128, "ue8m0", E8), w, ws)
    assert torch.equal(ops.fp8_linear(x, w, ws), want)
    ops.fp8_status()


def test_fp8_operators_beside_the_routed_layer(ops):
    """Clusters that split K, CTA pairs, the routed layer and the prompt's
    router on four streams together: the bits of a serial run."""
    from dsv4_plugin import synthetic as S
    from helpers import SyntheticLayer, bf16_tensor
    cfg = S.CFG0
    layer = SyntheticLayer(cfg)
    xt = bf16_tensor(S.make_tokens(cfg, 3, 512))
    gate = torch.from_numpy(layer.gate_w).cuda()
    plan = ops.MoEPlan(cfg.hidden, cfg.inter, cfg.n_experts, cfg.topk, 512, cfg.swiglu_limit, layer.arena)
    w, idx = ops.route_topk(xt, gate, None, cfg.topk, cfg.score_func, cfg.renormalize)
    g = gen(1)
    f8 = lambda n, k: ((torch.randn((n, k), generator=g, device="cuda") * 100).clamp(-448, 448).to(F8),  # noqa: E731
                       torch.full((-(-n // 128), -(-k // 128)), 2.0 ** -10, device="cuda"))
    big, small = f8(2304, 2048), f8(1024, 4096)
    xb = torch.randn((1500, 2048), generator=g, device="cuda").bfloat16()
    xs = torch.randn((100, 4096), generator=g, device="cuda").bfloat16()
    calls = [lambda: ops.fp8_linear(xb, *big), lambda: ops.fp8_linear(xs, *small),
             lambda: plan.forward(xt, w, idx, layer.slot_of).clone(),
             lambda: ops.route_topk(xt, gate, None, cfg.topk, cfg.score_func, cfg.renormalize)[0]]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    ops.fp8_status()
    plan.status()
    for i, w0 in enumerate(want):
        assert all(torch.equal(y, w0) for y in got[i])
