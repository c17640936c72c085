"""Cases of the FP8 block-scaled operators and of the expert balance loss.

Four operators, each with its plain form (elementary torch operations in 32
bits, 64 for long sums and values next to a border), the framework's call, and
its value in 64 bits:

* ``act_quant``    x -> E4M3 codes and one scale per row and 128 columns: the
                   power of two that brings the block within 448, or amax / 448;
* ``fp8_matmul``   product of E4M3 matrices, a scale for each row and 128 of K
                   on the left, for each 128 x 128 block on the right;
* ``fp8_linear``   the two together on a frozen FP8 weight, with the gradient
                   of its input;
* ``balance_loss`` the router's load balance loss and per-expert counts, with
                   the gradient of the logits.

``own`` selects the side: False computes the plain form, True calls
``dsv4_plugin.ops``.
"""

import os
import sys

import numpy as np
import torch

own = False

BLOCK = 128
F8 = torch.float8_e4m3fn
E8 = torch.float8_e8m0fnu
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ops():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v4-flash-offload_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from dsv4_plugin import ops
    return ops


# -- cases ---------------------------------------------------------------------

def listed():
    return [
        # tokens of a decode batch (the default benchmark's 64) before the shared expert's first product
        {"name": "quant_decode", "op": "act_quant", "rows": 64, "cols": 4096, "dtype": "bf16", "scale": "e8m0"},
        # a whole 8192-token step
        {"name": "quant_prefill", "op": "act_quant", "rows": 8192, "cols": 4096, "dtype": "bf16", "scale": "e8m0"},
        # 32-bit values whose row does not end on a block, with 32-bit scales
        {"name": "quant_ragged", "op": "act_quant", "rows": 4095, "cols": 2008, "dtype": "f32", "scale": "f32"},
        # one token through a gate or up projection
        {"name": "mm_token", "op": "fp8_matmul", "m": 1, "n": 2048, "k": 4096, "scale": "e8m0", "out": "bf16", "trans_b": True},
        # ragged in every size, 32-bit scales and output
        {"name": "mm_ragged", "op": "fp8_matmul", "m": 300, "n": 1001, "k": 2000, "scale": "f32", "out": "f32", "trans_b": True},
        # the prefill benchmark's 2048 tokens
        {"name": "mm_prefill", "op": "fp8_matmul", "m": 2048, "n": 4096, "k": 4096, "scale": "e8m0", "out": "bf16", "trans_b": True},
        # the input gradient of an up projection: the weight is read along its rows
        {"name": "mm_dx", "op": "fp8_matmul", "m": 2048, "n": 4096, "k": 2048, "scale": "e8m0", "out": "bf16", "trans_b": False},
        # the largest step, with the 32-bit block scales that other checkpoints carry
        {"name": "mm_large", "op": "fp8_matmul", "m": 8192, "n": 8192, "k": 4096, "scale": "f32", "out": "bf16", "trans_b": True},
        # a decode batch through the down projection: quantisation and product in one call
        {"name": "linear_decode", "op": "fp8_linear", "m": 64, "n": 4096, "k": 2048, "scale": "e8m0", "train": False},
        # forward and input gradient of a projection while something before it is tuned
        {"name": "linear_train", "op": "fp8_linear", "m": 4096, "n": 2048, "k": 4096, "scale": "e8m0", "train": True},
        # a small batch with padding tokens, the router's own score function
        {"name": "balance_small", "op": "balance_loss", "tokens": 64, "experts": 256, "topk": 8, "seqs": 0, "score": "sqrtsoftplus", "dtype": "f32"},
        # a packed training batch: ragged sequences, rows behind the last one
        {"name": "balance_packed", "op": "balance_loss", "tokens": 65536, "experts": 256, "topk": 8, "seqs": 24, "score": "sigmoid", "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(2.0 ** rng.uniform(np.log2(lo), np.log2(hi))))


def draw(rng):
    op = rng.choice(["act_quant", "fp8_matmul", "fp8_linear", "balance_loss"])
    if op == "act_quant":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 96, 4096), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "scale": rng.choice(["e8m0", "f32"])}
    if op == "balance_loss":
        e = rng.choice([8, 16, 60, 64, 128, 160, 256, 256, 257, 384])
        return {"op": op, "tokens": _log(rng, 1, 65536 * 256 // max(e, 256)), "experts": e, "topk": rng.randint(1, 8),
                "seqs": rng.choice([0, 0, 1, 3, 17, 64]), "score": rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]),
                "dtype": rng.choice(["f32", "f32", "bf16"])}
    m, k = _log(rng, 1, 8192), 16 * _log(rng, 4, 256)
    if op == "fp8_linear":
        train = rng.random() < 0.5
        return {"op": op, "m": min(m, 4096), "n": _log(rng, 64, 4096), "k": k, "scale": rng.choice(["e8m0", "f32"]), "train": train}
    trans = rng.random() < 0.7
    n = _log(rng, 64, 8192)
    return {"op": op, "m": m, "n": n if trans else (n + 15) // 16 * 16, "k": k, "scale": rng.choice(["e8m0", "f32"]),
            "out": rng.choice(["bf16", "bf16", "f32"]), "trans_b": trans}


# -- inputs --------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _activations(gen, rows, cols):
    """Hidden states: normal, every 61st channel an outlier, rows of unlike size."""
    x = _normal(gen, rows, cols)
    x *= torch.exp(0.5 * _normal(gen, rows, 1))
    x[:, 7::61] *= 20.0
    return x


def _weight(gen, n, k, fmt):
    """An FP8 checkpoint matrix: codes over the type's range, one scale per 128 x 128 block."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    q = (_normal(gen, n, k) * 100.0).clamp_(-448.0, 448.0).to(F8)
    e = torch.randint(-15, -10, (nb, kb), generator=gen, device="cuda").float()
    s = torch.exp2(e)
    if fmt == "f32":
        s = s * (1.0 + torch.rand((nb, kb), generator=gen, device="cuda"))
    return q, s.to(E8) if fmt == "e8m0" else s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, st = case["op"], {"case": case}
    if op == "act_quant":
        st["x"] = _activations(gen, case["rows"], case["cols"]).to(DTYPES[case["dtype"]])
    elif op == "fp8_matmul":
        m, n, k, fmt = case["m"], case["n"], case["k"], case["scale"]
        st["a"], st["as"] = _quantise(_activations(gen, m, k), fmt)
        st["b"], st["bs"] = _weight(gen, n, k, fmt) if case["trans_b"] else _weight(gen, k, n, fmt)
    elif op == "fp8_linear":
        m, n, k = case["m"], case["n"], case["k"]
        st["x"] = _activations(gen, m, k).to(torch.bfloat16)
        st["w"], st["ws"] = _weight(gen, n, k, case["scale"])
        if case["train"]:
            st["x"].requires_grad_(True)
            st["dy"] = (_activations(gen, m, n) * 1e-3).to(torch.bfloat16)
    else:
        t, e, k, s = case["tokens"], case["experts"], case["topk"], case["seqs"]
        logits = _normal(gen, t, e).to(DTYPES[case["dtype"]])
        # skewed picks, as a selection bias over experts leaves them
        bias = -0.3 * torch.log(torch.randperm(e, generator=gen, device="cuda") + 1.0)
        st["idx"] = torch.topk(logits.float() + bias, k, dim=-1).indices.to(torch.int32)
        st["logits"] = logits.requires_grad_(True)
        st["up"] = 0.5 + torch.rand((), generator=gen, device="cuda")
        st["off"] = None
        if s:
            # ragged sequences in a packed batch, its last rows belong to none
            used = t - t // 17
            cuts = np.sort(np.random.RandomState(int(seed) % (1 << 31)).randint(0, used + 1, s - 1))
            st["off"] = torch.tensor([0, *cuts.tolist(), used], dtype=torch.int32, device="cuda")
        else:
            st["idx"][torch.rand(t, generator=gen, device="cuda") < 0.03] = -1   # padding tokens have no pick
    return st


# -- the plain forms -----------------------------------------------------------

def _wide(s, size):
    """One value per 128 columns -> one per column."""
    return s.float().repeat_interleave(BLOCK, dim=-1)[..., :size]


def _quantise(x, fmt):
    x = x.float()
    rows, cols = x.shape
    nb = -(-cols // BLOCK)
    amax = torch.nn.functional.pad(x.abs(), (0, nb * BLOCK - cols)).view(rows, nb, BLOCK).amax(-1).clamp(min=1e-4)
    if fmt == "e8m0":
        # the smallest power of two that brings the block within 448, decided in 64 bits
        mant, expo = torch.frexp(amax.double() / 448.0)
        s = torch.exp2((expo - (mant == 0.5).to(expo.dtype)).float())
        return (x / _wide(s, cols)).clamp(-448.0, 448.0).to(F8), s.to(E8)
    # the code nearest to 448 x / amax, in 64 bits: two 16-bit values often put it on a tie
    q = x.double() * 448.0 / amax.double().repeat_interleave(BLOCK, dim=-1)[:, :cols]
    return q.clamp(-448.0, 448.0).float().to(F8), amax / 448.0


def _product(a, a_s, b, b_s, trans_b, out):
    af = a.float() * _wide(a_s, a.shape[1])
    bf = b.float() * _wide(b_s.float().repeat_interleave(BLOCK, dim=0)[: b.shape[0]], b.shape[1])
    return (af @ (bf.t() if trans_b else bf)).to(out)


def _balance(st):
    case, idx, off = st["case"], st["idx"].long(), st["off"]
    t, e = st["logits"].shape
    l = st["logits"].detach().float()
    if case["score"] == "softmax":
        s = torch.exp(l - l.amax(-1, keepdim=True))
        r = torch.ones_like(l)
    elif case["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
        r = 1.0 - s
    else:
        sp = torch.log1p(torch.exp(-l.abs())) + l.clamp(min=0.0)
        s = torch.sqrt(sp)
        r = 0.5 / ((1.0 + torch.exp(-l)) * sp)
    p = s / s.sum(-1, keepdim=True)
    rows = torch.arange(t, device=l.device)
    n_seq = 1 if off is None else off.numel() - 1
    seq = torch.zeros_like(rows) if off is None else torch.bucketize(rows, off.long(), right=True) - 1
    live = (idx >= 0).any(-1) & (seq >= 0) & (seq < n_seq)
    seq = torch.where(live, seq, n_seq)                          # one row more, for what does not count
    flat = (seq[:, None] * e + idx)[idx >= 0]
    c = torch.zeros((n_seq + 1) * e, dtype=torch.int64, device=l.device).index_add_(0, flat, torch.ones_like(flat))
    c = c.view(n_seq + 1, e)[:n_seq]
    n = torch.zeros(n_seq + 1, dtype=torch.int64, device=l.device).index_add_(0, seq, torch.ones_like(seq))[:n_seq]
    total = torch.zeros((n_seq + 1, e), dtype=torch.float64, device=l.device).index_add_(0, seq, p.double())[:n_seq]
    f = c.double() * e / c.sum(-1, keepdim=True).clamp(min=1)
    each = n.clamp(min=1).double()
    loss = 0.01 * ((f * total).sum(-1) / each).sum() / (n > 0).sum().clamp(min=1)
    g = 0.01 * f / (each * (n > 0).sum().clamp(min=1))[:, None]
    g = torch.cat([g, torch.zeros_like(g[:1])]).float()[seq]
    d = p * r * (g - (g * p).sum(-1, keepdim=True)) * st["up"]
    d = torch.where(live[:, None], d, 0.0).to(st["logits"].dtype)
    return loss.float(), (c[0] if off is None else c).to(torch.int32), d


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        ops = _ops()
        if op == "act_quant":
            fmt = "ue8m0" if case["scale"] == "e8m0" else None
            return ops.act_quant(state["x"], 128, fmt, E8 if fmt else torch.float32)
        if op == "fp8_matmul":
            return ops.fp8_matmul(state["a"], state["as"], state["b"], state["bs"], trans_b=case["trans_b"], out_dtype=DTYPES[case["out"]])
        if op == "fp8_linear":
            y = ops.fp8_linear(state["x"], state["w"], state["ws"])
            return (y.detach(), *torch.autograd.grad(y, state["x"], state["dy"])) if case["train"] else y
        loss, counts = ops.balance_loss(state["logits"], state["idx"], score_func=case["score"], alpha=0.01, seq_offsets=state["off"])
        return loss.detach(), counts, *torch.autograd.grad(loss, state["logits"], state["up"])
    if op == "act_quant":
        return _quantise(state["x"], case["scale"])
    if op == "fp8_matmul":
        return _product(state["a"], state["as"], state["b"], state["bs"], case["trans_b"], DTYPES[case["out"]])
    if op == "fp8_linear":
        fmt = case["scale"]
        y = _product(*_quantise(state["x"].detach(), fmt), state["w"], state["ws"], True, torch.bfloat16)
        return (y, _product(*_quantise(state["dy"], fmt), state["w"], state["ws"], False, torch.bfloat16)) if case["train"] else y
    return _balance(state)


def work(case):
    op = case["op"]
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if op == "act_quant":
        r, c = case["rows"], case["cols"]
        blocks = r * -(-c // BLOCK)
        return {"bytes": r * c * (size[case["dtype"]] + 1) + blocks * (1 if case["scale"] == "e8m0" else 4), "flops": 3 * r * c}
    if op == "balance_loss":
        t, e = case["tokens"], case["experts"]
        # the logits, the picks, the gradient, the counts
        return {"bytes": 2 * t * e * size[case["dtype"]] + 4 * t * case["topk"] + 4 * max(case["seqs"], 1) * e, "flops": 16 * t * e}
    m, n, k = case["m"], case["n"], case["k"]
    sb = 1 if case["scale"] == "e8m0" else 4
    blocks = -(-n // BLOCK) * -(-k // BLOCK)
    if op == "fp8_matmul":
        return {"bytes": m * k + n * k + sb * (m * -(-k // BLOCK) + blocks) + m * n * size[case["out"]], "flops": 2 * m * n * k}
    twice = 2 if case["train"] else 1
    return {"bytes": n * k + sb * blocks + twice * 2 * m * (n + k), "flops": twice * 2 * m * n * k}


# -- in 64 bits, from the definitions ------------------------------------------

def _e4m3_64(v):
    """The E4M3 value nearest to v (even mantissa on a tie), at most 448."""
    v = v.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def _quantise_64(x, fmt):
    x = x.double()
    out, scales = torch.empty_like(x), []
    for c in range(0, x.shape[1], BLOCK):
        b = x[:, c:c + BLOCK]
        amax = b.abs().max(dim=1, keepdim=True).values.clamp(min=float(np.float32(1e-4)))
        ratio = amax / 448.0
        if fmt == "e8m0":
            # log2 in 64 bits is too coarse next to a power of two: correct it by comparison
            s = torch.exp2(torch.ceil(torch.log2(ratio)))
            s = torch.where(s / 2 >= ratio, s / 2, torch.where(s < ratio, s * 2, s))
        out[:, c:c + BLOCK] = _e4m3_64(b / s if fmt == "e8m0" else b * 448.0 / amax)
        scales.append(s if fmt == "e8m0" else ratio)
    return out, torch.cat(scales, dim=1)


def _product_64(a, a_s, b, b_s, trans_b):
    col = torch.arange(max(a.shape[1], *b.shape), device=a.device) // BLOCK
    a = a.double() * a_s.double()[:, col[:a.shape[1]]]
    b = b.double() * b_s.double()[col[:b.shape[0]]][:, col[:b.shape[1]]]
    return torch.einsum("mk,nk->mn" if trans_b else "mk,kn->mn", a, b)


def _balance_64(st):
    case, t, e = st["case"], *st["logits"].shape
    x, idx = st["logits"].detach().double(), st["idx"].cpu().numpy()
    off = [0, t] if st["off"] is None else st["off"].tolist()
    if case["score"] == "softmax":
        fn = torch.exp
    elif case["score"] == "sigmoid":
        fn = torch.sigmoid
    else:
        fn = lambda v: torch.sqrt(torch.nn.functional.softplus(v, threshold=1000.0))  # noqa: E731
    x.requires_grad_(True)
    score = fn(x)
    prob = score / score.sum(dim=1, keepdim=True)
    rows, losses = np.zeros((len(off) - 1, e), dtype=np.int64), []
    for i, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        mine = idx[lo:hi]
        keep = np.nonzero((mine >= 0).any(axis=1))[0]
        rows[i] = np.bincount(mine[mine >= 0], minlength=e)
        if keep.size:
            f = torch.from_numpy(rows[i] * (e / rows[i].sum())).to(x.device)
            losses.append((f * prob[lo + torch.from_numpy(keep).to(x.device)].mean(dim=0)).sum())
    loss = 0.01 * torch.stack(losses).mean() if losses else 0.0 * x.sum()
    grad, = torch.autograd.grad(loss * st["up"].double(), x)
    return loss.detach(), torch.from_numpy(rows[0] if st["off"] is None else rows).to(torch.int32), grad


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "act_quant":
        return _quantise_64(st["x"], case["scale"])
    if op == "fp8_matmul":
        return _product_64(st["a"], st["as"], st["b"], st["bs"], case["trans_b"])
    if op == "balance_loss":
        return _balance_64(st)
    y = _product_64(*_quantise_64(st["x"].detach(), case["scale"]), st["w"], st["ws"], True)
    return (y, _product_64(*_quantise_64(st["dy"], case["scale"]), st["w"], st["ws"], False)) if case["train"] else y
