"""balance_loss on the GPU against a plain 64-bit implementation (autograd in
float64) and against differences.

Tolerances.  A score takes at most an exponential (2 + 1.2 |l| steps of
2^-24), a logarithm or a reciprocal and a root (2 to 4 each); a row's sums
over E experts are trees over 32 lanes after E / 32 terms per lane, and the
gradient adds about ten more operations:
    U = (96 + E / 32 + 2 max |l|) * 2^-24
bounds the relative error of p, r and of the loss (a sum of positive terms),
and U * c p r (|g| + |d|) that of a gradient, whose difference g - d is what
cancels.  A bf16 gradient adds half a step, 2^-8.  The loss is rounded once
more, 2^-24."""

import numpy as np
import pytest
import torch

from dsv4_plugin import synthetic as S
from helpers import bf16_tensor

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from dsv4_plugin import ops
    return ops


def make(seed, t, e, k, dtype=torch.float32, pad=0.1, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lg = (torch.randn((t, e), generator=g, device="cuda") * spread).to(dtype)
    bias = torch.randn(e, generator=g, device="cuda")
    idx = torch.topk(lg.float() + bias, k, dim=-1).indices.int()
    idx[torch.rand(t, generator=g, device="cuda") < pad] = -1
    return lg, idx


def score64(l, fn):
    if fn == "softmax":
        return torch.exp(l - l.max(1, keepdim=True).values)
    if fn == "sigmoid":
        return torch.sigmoid(l)
    return torch.sqrt(torch.nn.functional.softplus(l, threshold=500.0))


def loss64(l, idx, off, fn, alpha):
    """(loss, counts [S, E], p, g / alpha-free per row pieces) in float64."""
    t, e = l.shape
    off = [0, t] if off is None else off
    s = score64(l, fn)
    p = s / s.sum(1, keepdim=True)
    idx = idx.cpu()
    counts, losses, g = torch.zeros(len(off) - 1, e, dtype=torch.int64), [], torch.zeros(t, e, dtype=torch.float64)
    for i, (a, b) in enumerate(zip(off[:-1], off[1:])):
        part = idx[a:b]
        ok = (part >= 0) & (part < e)
        counts[i] = torch.bincount(part[ok].long(), minlength=e)
        rows = a + ok.any(1).nonzero()[:, 0]
        if len(rows):
            f = counts[i].double() * e / counts[i].sum()
            losses.append((f.to(l.device) * p[rows.to(l.device)].mean(0)).sum())
            g[rows] = f / len(rows)
    loss = alpha * torch.stack(losses).mean() if losses else l.sum() * 0.0
    return loss, counts, p.detach(), (alpha * g / max(len(losses), 1)).to(l.device)


def check(ops, lg, idx, off, fn, alpha=0.01, up=1.7):
    t, e = lg.shape
    offs = None if off is None else torch.tensor(off, dtype=torch.int32, device="cuda")
    x = lg.clone().requires_grad_(True)
    loss, counts = ops.balance_loss(x, idx, fn, alpha, offs)
    grad, = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"))
    l64 = lg.double().requires_grad_(True)
    want, c64, p, g = loss64(l64, idx, off, fn, alpha)
    gw, = torch.autograd.grad(want * float(np.float32(up)), l64)
    assert counts.dtype == torch.int32
    assert torch.equal(counts.cpu().long(), c64 if off is not None else c64[0])
    size = lg.float().abs()
    U = (96 + e / 32 + 2 * float(size[size < 1e30].max())) * 2.0 ** -24      # a masked logit's score is exactly 0
    assert abs(float(loss) - float(want)) <= (U + 2.0 ** -24) * abs(float(want))
    d = (g * p).sum(1, keepdim=True)
    tol = U * up * p * (g.abs() + d) + (2.0 ** -8 * gw.abs() if lg.dtype == torch.bfloat16 else 0)
    assert grad.dtype == lg.dtype
    bad = (grad.double() - gw).abs() > tol + 1e-45
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())
    return loss, counts, grad


@pytest.mark.parametrize("fn", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,e,k", [(1, 8, 1), (7, 16, 4), (64, 256, 8), (256, 60, 3), (257, 256, 8), (1000, 257, 8),
                                   (33, 1, 1), (130, 384, 6), (300, 1024, 2), (2048, 64, 8), (5, 130, 40)])
def test_one_sequence(ops, fn, dtype, t, e, k):
    check(ops, *make(t + e, t, e, min(k, e), dtype, pad=0.1 if t > 1 else 0.0), None, fn)


@pytest.mark.parametrize("fn", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("t,off", [
    (100, [0, 100]), (100, [0, 0, 40, 40, 90, 90]), (100, [10, 11, 12, 13]), (600, [0, 1, 2, 300, 599]),
    (600, [0] * 20 + [600] * 3), (3000, list(range(0, 2900, 100))), (700, [700, 700]), (40, [0] + list(range(41)))])
def test_packed_sequences(ops, fn, t, off):
    lg, idx = make(t + len(off), t, 64, 4)
    _, _, grad = check(ops, lg, idx, off, fn)
    assert (grad[off[-1]:] == 0).all() and (grad[:off[0]] == 0).all()
    assert (grad[(idx < 0).all(1)] == 0).all()


@pytest.mark.parametrize("t,s", [(20000, 20000), (5000, 1500), (70000, 3)])
def test_many_sequences(ops, t, s):
    """A sequence per token; sequences around the piece that is counted in
    shared memory; more rows per warp than a batch."""
    g = np.random.RandomState(t)
    cuts = np.sort(g.randint(0, t + 1, s - 1)).tolist() if s != t else list(range(1, t))
    lg, idx = make(t, t, 16, 2, spread=1.0)
    off = [0, *cuts, t]
    offs = torch.tensor(off, device="cuda")
    x = lg.clone().requires_grad_(True)
    loss, counts = ops.balance_loss(x, idx, "sigmoid", 1.0, offs)
    grad, = torch.autograd.grad(loss, x)
    # the definition over all rows at once (a loop over sequences would be slow)
    l64 = lg.double().requires_grad_(True)
    p = torch.sigmoid(l64)
    p = p / p.sum(1, keepdim=True)
    seq = torch.bucketize(torch.arange(t, device="cuda"), offs, right=True) - 1
    live = (idx >= 0).any(1)
    c = torch.zeros(s * 16, dtype=torch.int64, device="cuda")
    c = c.index_add_(0, (seq[:, None] * 16 + idx)[live].reshape(-1), torch.ones(int(live.sum()) * 2, dtype=torch.int64,
                                                                               device="cuda")).view(s, 16)
    n = torch.zeros(s, dtype=torch.int64, device="cuda").index_add_(0, seq[live], torch.ones_like(seq[live]))
    f = c.double() * 16 / c.sum(1, keepdim=True).clamp(min=1) / n.clamp(min=1)[:, None]
    want = (f[seq] * p)[live].sum() / (n > 0).sum()
    gw, = torch.autograd.grad(want, l64)
    assert torch.equal(counts.long(), c)
    U = (96 + 2 * float(lg.abs().max())) * 2.0 ** -24
    assert abs(float(loss.detach()) - float(want.detach())) <= (U + 2.0 ** -24) * float(want.detach())
    gg = f[seq] / (n > 0).sum()
    tol = U * p.detach() * (gg + (gg * p.detach()).sum(1, keepdim=True))
    assert ((grad.double() - gw).abs() <= tol + 1e-45).all()


def test_offsets_beyond_32_bits(ops):
    """Logits of more than 2^32 bytes: the last sequence as computed alone."""
    t, e, tail = 8_500_000, 256, 1000
    lg = torch.zeros((t, e), dtype=torch.bfloat16, device="cuda")
    last, idx_last = make(1, tail, e, 8, torch.bfloat16, pad=0.0)
    lg[-tail:] = last
    idx = torch.full((t, 8), -1, dtype=torch.int32, device="cuda")
    idx[-tail:] = idx_last
    x = lg.requires_grad_(True)
    loss, counts = ops.balance_loss(x, idx, "sigmoid")
    grad, = torch.autograd.grad(loss, x)
    y = last.clone().requires_grad_(True)
    l2, c2 = ops.balance_loss(y, idx_last, "sigmoid")
    g2, = torch.autograd.grad(l2, y)
    assert torch.equal(counts, c2) and abs(float(loss.detach()) - float(l2.detach())) <= 2.0 ** -20 * float(l2.detach())
    assert torch.equal(grad[-tail:], g2)
    assert not grad[:-tail].any()


@pytest.mark.parametrize("t", [40, 900])
def test_nothing_counts(ops, t):
    """Only padding; and no rows at all."""
    lg, idx = make(1, t, 32, 4)
    idx[:] = -1
    lg[3] = float("nan")
    x = lg.requires_grad_(True)
    loss, counts = ops.balance_loss(x, idx, "sigmoid")
    loss.backward()
    assert float(loss) == 0.0 and int(counts.abs().sum()) == 0 and (x.grad == 0).all()
    x = torch.zeros(0, 32, device="cuda", requires_grad=True)
    loss, counts = ops.balance_loss(x, torch.zeros(0, 4, dtype=torch.int32, device="cuda"))
    loss.backward()
    assert float(loss) == 0.0 and int(counts.sum()) == 0 and x.grad.shape == (0, 32)
    off = torch.zeros(3000, dtype=torch.int32, device="cuda")
    loss, counts = ops.balance_loss(x, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), seq_offsets=off)
    assert float(loss) == 0.0 and counts.shape == (2999, 32) and int(counts.sum()) == 0


@pytest.mark.parametrize("fn", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("t", [50, 500])
def test_masked_experts_and_empty_rows(ops, fn, t):
    """Experts masked with -inf or the type's lowest value have p = 0 and no
    gradient; a row that is masked whole has no probabilities and no gradient."""
    lg, idx = make(9, t, 64, 4, pad=0.0)
    lg[:, 5] = float("-inf")
    lg[:, 9] = torch.finfo(torch.float32).min
    idx[(idx == 5) | (idx == 9)] = 20
    gone = lg.clone()
    loss0, c0, g0 = check(ops, lg, idx, None, fn) if fn == "softmax" else (None, None, None)
    gone[7] = float("-inf")
    x = gone.requires_grad_(True)
    loss, counts = ops.balance_loss(x, idx, fn, 0.01)
    grad, = torch.autograd.grad(loss, x)
    assert torch.isfinite(loss) and torch.isfinite(grad).all()
    assert (grad[7] == 0).all() and (grad[:, 5] == 0).all() and (grad[:, 9] == 0).all()
    # the same with the masked columns taken out: p of the others is unchanged
    keep = [i for i in range(64) if i not in (5, 9)]
    l64 = gone.detach().double()
    s = torch.where(torch.isinf(l64), 0.0, score64(l64.clamp(min=-1e30), fn)) if fn != "softmax" else \
        torch.exp(l64 - l64.max(1, keepdim=True).values.clamp(min=-1e300))
    p = torch.nan_to_num(s / s.sum(1, keepdim=True))
    f = counts.double() * 64 / counts.sum()
    want = 0.01 * (f * p).sum() / t
    assert abs(float(loss) - float(want)) <= 128 * 2.0 ** -24 * float(want)
    assert counts[keep].sum() == counts.sum()


def test_nan_and_infinity_stay_in_their_row(ops):
    for t in (60, 600):
        lg, idx = make(4, t, 32, 2, pad=0.0)
        idx[1] = -1
        lg[0, 3], lg[1, 3], lg[2, 3] = float("nan"), float("nan"), float("inf")
        x = lg.requires_grad_(True)
        loss, _ = ops.balance_loss(x, idx, "sqrtsoftplus")
        grad, = torch.autograd.grad(loss, x)
        assert torch.isnan(loss) and torch.isnan(grad[0]).any()
        assert (grad[1] == 0).all() and torch.isfinite(grad[3:]).all()


@pytest.mark.parametrize("t", [30, 3000])
def test_bad_picks_and_offsets_are_reported(ops, t):
    lg, idx = make(2, t, 16, 3, pad=0.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.balance_loss(lg, idx, status=status)
    assert int(status) == 0
    bad = idx.clone()
    bad[4, 1], bad[5, 2], bad[6] = 16, -2, 99
    loss, counts = ops.balance_loss(lg, bad, status=status)
    assert int(status) == -1
    skipped = bad.clone()
    skipped[(bad < 0) | (bad >= 16)] = -1
    l2, c2 = ops.balance_loss(lg, skipped)
    assert torch.equal(loss, l2) and torch.equal(counts, c2)
    l3, c3 = ops.balance_loss(lg, bad.long() + torch.where(bad == 99, 1 << 32, 0))   # no wrap to a valid id
    assert torch.equal(l3, l2) and torch.equal(c3, c2)
    for off in ([0, 20, 10, t], [-1, t], [0, t + 1]):
        status.zero_()
        ops.balance_loss(lg, idx, seq_offsets=torch.tensor(off, device="cuda"), status=status)
        assert int(status) == -1


def test_duplicate_picks_count_each(ops):
    lg = torch.randn(10, 8, device="cuda")
    idx = torch.full((10, 4), 3, dtype=torch.int32, device="cuda")
    _, counts = ops.balance_loss(lg, idx)
    assert int(counts[3]) == 40 and int(counts.sum()) == 40


@pytest.mark.parametrize("fn", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_gradient_against_differences(ops, fn):
    """The slope of the 64-bit loss along random directions.  Central
    differences with h: h^2 / 6 of the third derivative (scores and their
    derivatives are within a factor of ten of 1 for these logits) and 2^-52
    of the loss over h."""
    lg, idx = make(11, 300, 40, 4, spread=1.0)
    off = [0, 100, 290]
    _, _, grad = check(ops, lg, idx, off, fn, alpha=1.0, up=1.0)
    h = 2.0 ** -13
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(4):
        v = torch.randn(lg.shape, generator=g, device="cuda", dtype=torch.float64)
        up = float(loss64(lg.double() + h * v, idx, off, fn, 1.0)[0])
        dn = float(loss64(lg.double() - h * v, idx, off, fn, 1.0)[0])
        slope = float((grad.double() * v).sum())
        scale = float((grad.double() * v).abs().sum())
        assert abs((up - dn) / (2 * h) - slope) <= 1e-4 * scale + 2.0 ** -50 / h * abs(up)


def test_strided_logits_streams_and_repeat(ops):
    lg, idx = make(3, 5000, 256, 8)
    off = torch.tensor([0, 2000, 4800], dtype=torch.int32, device="cuda")
    x = lg.clone().requires_grad_(True)
    loss, counts = ops.balance_loss(x, idx, "sigmoid", 1.0, off)
    grad, = torch.autograd.grad(loss, x)
    for _ in range(3):                                        # the same bits each time
        l2, c2 = ops.balance_loss(x, idx, "sigmoid", 1.0, off)
        g2, = torch.autograd.grad(l2, x)
        assert torch.equal(l2, loss) and torch.equal(c2, counts) and torch.equal(g2, grad)
    wide = torch.zeros(5000, 300, device="cuda")
    wide[:, 7:263] = lg
    v = wide[:, 7:263].requires_grad_(True)
    l3, _ = ops.balance_loss(v, idx.t().contiguous().t(), "sigmoid", 1.0, off)
    g3, = torch.autograd.grad(l3, v)
    assert torch.equal(l3, loss) and torch.equal(g3, grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        l4, c4 = ops.balance_loss(x, idx, "sigmoid", 1.0, off)
        g4, = torch.autograd.grad(l4, x)
    side.synchronize()
    assert torch.equal(l4, loss) and torch.equal(c4, counts) and torch.equal(g4, grad)
    # the counts are the caller's: changing them does not change the gradient
    l5, c5 = ops.balance_loss(x, idx, "sigmoid", 1.0, off)
    c5.zero_()
    assert torch.equal(torch.autograd.grad(l5, x)[0], grad)


@pytest.mark.parametrize("t", [100, 4000])
def test_captured(ops, t):
    """Forward and backward in a graph, two graphs replayed in turn."""
    sets = [make(s, t, 64, 4) for s in range(3)]
    want = []
    for lg, idx in sets:
        x = lg.clone().requires_grad_(True)
        loss, counts = ops.balance_loss(x, idx, "softmax", 1.0)
        want.append((loss.detach().clone(), counts.clone(), torch.autograd.grad(loss, x)[0]))
    del loss, x
    graphs = []
    for _ in range(2):
        bl, bi = sets[0][0].clone().requires_grad_(True), sets[0][1].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, counts = ops.balance_loss(bl, bi, "softmax", 1.0)
            grad, = torch.autograd.grad(loss, bl)
        graphs.append((g, bl, bi, loss.detach(), counts, grad))
        del loss
    for i in range(3):
        for j, (g, bl, bi, *_) in enumerate(graphs):
            with torch.no_grad():
                bl.copy_(sets[(i + j) % 3][0])
            bi.copy_(sets[(i + j) % 3][1])
            g.replay()
        torch.cuda.synchronize()
        for j, (_, _, _, *got) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(got, want[(i + j) % 3]))


def test_after_the_router(ops):
    """Router, its counts and its loss together: the counts are the align's,
    and they make a placement."""
    from dsv4_plugin.parallel_ep import balanced_placement
    cfg = S.CFG0
    gw, _ = S.make_gate(cfg, 0)
    x = S.make_tokens(cfg, 0, 500)
    xt, gt = bf16_tensor(x), torch.from_numpy(gw).cuda()
    _, idx = ops.route_topk(xt, gt, None, cfg.topk, cfg.score_func, cfg.renormalize)
    w = gt.clone().requires_grad_(True)
    loss, counts = ops.balance_loss(xt.float() @ w.t(), idx, cfg.score_func, 0.01)
    loss.backward()
    assert torch.equal(counts, ops.moe_align(idx, cfg.n_experts)["counts"])
    assert sorted(set(balanced_placement(counts.tolist(), 4))) == [0, 1, 2, 3]
    l64 = (xt.double() @ gt.double().t()).requires_grad_(True)
    want, *_ = loss64(l64, idx, None, cfg.score_func, 0.01)
    gl, = torch.autograd.grad(want, l64)
    ref = gl.t() @ xt.double()
    # 500 rows summed in fp32 by the two products around the loss
    mag = gl.abs().t() @ xt.double().abs()
    assert ((w.grad.double() - ref).abs() <= 1e-4 * mag).all()
