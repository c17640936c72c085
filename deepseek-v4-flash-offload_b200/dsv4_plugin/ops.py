"""torch-facing wrappers of the CUDA library, named after the reference ops.

| here                    | reference                                           |
|-------------------------|-----------------------------------------------------|
| ``dequant_fp4_weight``  | npu_ops.dequant_fp4_weight (npu_ops.py:142-158)     |
| ``act_quant``           | npu_ops.act_quant (npu_ops.py:73-104)               |
| ``fp8_matmul``,         | a dense layer on a checkpoint's FP8 weight          |
| ``fp8_linear``          | (npu_ops.dequant_fp8_weight, npu_ops.py:161-167)    |
| ``dynamic_mx_quant``    | torch_npu.npu_dynamic_mx_quant (deepseek_v4.py:212) |
| ``route_topk``          | OffloadDeepseekV4MoE._route (deepseek_v4.py:118-148)|
| ``moe_align``           | the align block of _routed (deepseek_v4.py:154-164) |
| ``MoEPlan.forward``     | _routed / _routed_mxfp4 (deepseek_v4.py:150-245)    |
| ``balance_loss``        | none (the reference's router only serves)           |

All tensors must live on a CUDA device; work runs on the current torch
stream.  There is no CPU path.
"""

from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad

from ._lib import (DT_BF16, DT_FP16, DT_FP32, PROFILES, ROWS_BF16, ROWS_FP8, ROWS_MXFP4,  # noqa: F401
                   SCALE_E8M0, SCALE_FP32, SCALE_FP32_POW2, SCORE_FUNCS, check, lib)

_E8M0 = getattr(torch, "float8_e8m0fnu", None)
_E4M3 = torch.float8_e4m3fn
_DT = {torch.bfloat16: DT_BF16, torch.float16: DT_FP16, torch.float32: DT_FP32}


# the handle alone, where torch gives it: a Stream object costs 2 us a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev: torch.device) -> int:
    if _raw_stream is not None and dev.index is not None:
        return _raw_stream(dev.index)
    return torch.cuda.current_stream(dev).cuda_stream


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("dsv4 ops need CUDA tensors (there is no CPU path)")


def _u8(t: torch.Tensor) -> torch.Tensor:
    if t.dtype in (torch.uint8, torch.int8) or (_E8M0 is not None and t.dtype == _E8M0):
        return t.contiguous().view(torch.uint8)
    raise TypeError(f"expected a uint8/int8/e8m0 tensor, got {t.dtype}")


def dequant_fp4_weight(w_packed: torch.Tensor, scale: torch.Tensor, out_dtype=torch.bfloat16) -> torch.Tensor:
    """[N, K//2] packed E2M1 + [N, K//32] E8M0 -> [N, K] bf16 (bit-exact)."""
    if out_dtype != torch.bfloat16:
        raise NotImplementedError("the CUDA dequant produces bf16")
    _need_cuda(w_packed, scale)
    w, s = _u8(w_packed), _u8(scale)
    n, kh = w.shape
    out = torch.empty((n, kh * 2), dtype=torch.bfloat16, device=w.device)
    check(lib().dsv4_dequant_mxfp4(w.data_ptr(), s.data_ptr(), out.data_ptr(), n, kh * 2, _stream(w.device)))
    return out


def act_quant(x: torch.Tensor, block_size: int = 128, scale_fmt: str | None = "ue8m0", scale_dtype=None,
              inplace: bool = False):
    """FP8-E4M3 quantisation per row and 128 columns.

    ``inplace=True``: the round trip of a contiguous bf16 ``x`` with
    power-of-two scales, in place; returns ``x``.

    ``inplace=False``: (q, s) with q E4M3 of ``x``'s shape and s [..,
    ceil(C / 128)].  ``x`` is bf16, fp16 or fp32, with any number of columns.
    ``scale_fmt="ue8m0"``: the smallest power of two that brings the block
    within 448, as ``scale_dtype`` float32 (also None) or float8_e8m0fnu;
    ``scale_fmt=None``: amax / 448 in float32.  amax is at least 1e-4.  A NaN
    stays NaN and leaves its block's scale alone; an infinity saturates.  The
    result carries no gradient (``fp8_linear`` does)."""
    if block_size != 128 or scale_fmt not in ("ue8m0", None):
        raise NotImplementedError("act_quant provides block_size 128 and scale_fmt 'ue8m0' or None")
    if inplace:
        if scale_fmt != "ue8m0":
            raise NotImplementedError("only act_quant(x, 128, 'ue8m0', _, inplace=True) is provided in place")
        _need_cuda(x)
        if x.dtype != torch.bfloat16 or not x.is_contiguous():
            raise TypeError("act_quant expects a contiguous bf16 tensor")
        check(lib().dsv4_act_quant_fp8_rt(x.data_ptr(), x.numel() // x.shape[-1], x.shape[-1], _stream(x.device)))
        return x
    if x.dtype not in _DT:
        raise TypeError(f"act_quant expects bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("act_quant needs at least one column")
    if scale_dtype not in (None, torch.float32) and (_E8M0 is None or scale_dtype != _E8M0 or scale_fmt is None):
        raise TypeError("scale_dtype must be float32, or float8_e8m0fnu with scale_fmt 'ue8m0'")
    _need_cuda(x)
    if not x.is_contiguous():
        x = x.detach().contiguous()
    cols = x.shape[-1]
    rows = x.numel() // cols
    kind = SCALE_FP32 if scale_fmt is None else (SCALE_E8M0 if scale_dtype == _E8M0 else SCALE_FP32_POW2)
    q = x.new_empty(x.shape, dtype=_E4M3)
    s = x.new_empty((*x.shape[:-1], (cols + 127) // 128), dtype=_E8M0 if kind == SCALE_E8M0 else torch.float32)
    check(lib().dsv4_act_quant_fp8(x.data_ptr(), _DT[x.dtype], rows, cols, cols, q.data_ptr(), cols, s.data_ptr(), kind,
                                   _stream(x.device)))
    return q, s


def _fp8_rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(FP8 matrix the kernels can read, its row stride in bytes): rows that
    start on 16 bytes, columns next to each other; copied when it is not."""
    r, c = t.shape
    if c % 16 == 0 and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, c
    ld = t.stride(0) if r > 1 else (c + 15) // 16 * 16
    if (t.stride(1) == 1 or c == 1) and ld % 16 == 0 and ld >= c and t.data_ptr() % 16 == 0:
        return t, ld
    ld = (c + 15) // 16 * 16
    p = torch.empty((r, ld), dtype=torch.uint8, device=t.device)
    p[:, :c].copy_(t.contiguous().view(torch.uint8))
    return p, ld


def _fp8_scale(s: torch.Tensor) -> torch.Tensor:
    """Scales as the kernels read them: contiguous E8M0 bytes or float32."""
    return s.contiguous() if s.dtype == torch.float32 else _u8(s)


def _is_e8m0(s: torch.Tensor) -> bool:
    dt = s.dtype
    if dt == torch.float32:
        return False
    if dt == torch.uint8 or (_E8M0 is not None and dt == _E8M0):
        return True
    raise TypeError(f"FP8 scales are float32 or E8M0 (float8_e8m0fnu or uint8), got {dt}")


def _e8m0_float(s: torch.Tensor) -> torch.Tensor:
    return (s.view(_E8M0) if s.dtype == torch.uint8 else s).float()


def _same_device(*ts):
    _need_cuda(*ts)
    first = ts[0].device
    for t in ts[1:]:
        if t is not None and t.device != first:
            raise ValueError("the tensors live on different devices")


def _check_fp8_weight(b: torch.Tensor, b_scale: torch.Tensor):
    if b.dtype != _E4M3:
        raise TypeError(f"expected a float8_e4m3fn matrix, got {b.dtype}")
    if b.dim() != 2 or b_scale.shape != ((b.shape[0] + 127) // 128, (b.shape[1] + 127) // 128):
        raise ValueError(f"a matrix of shape {tuple(b.shape)} needs one scale per 128 x 128 block, "
                         f"got {tuple(b_scale.shape)}")


def fp8_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, trans_b: bool = True,
               out_dtype=torch.bfloat16) -> torch.Tensor:
    """Product of E4M3 matrices with a scale for each row and 128 of K of ``a``
    ([.., K], a_scale [.., ceil(K / 128)]) and each 128 x 128 block of ``b``
    ([N, K]; with ``trans_b=False`` [K, N]; b_scale one per block):
    dequant(a) @ dequant(b).T (or @ dequant(b)) with fp32 sums, in bf16 or
    fp32.  Scales: float32 or E8M0 (float8_e8m0fnu or uint8); where the two
    differ, both are taken as float32.  No gradient: see ``fp8_linear``.

    Rows of ``a`` and ``b`` may be strided.  Where they do not start on 16
    bytes the matrix is copied first."""
    if a.dtype != _E4M3:
        raise TypeError(f"expected a float8_e4m3fn matrix, got {a.dtype}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("out_dtype must be bfloat16 or float32")
    _check_fp8_weight(b, b_scale)
    if a.dim() < 1 or a.shape[-1] == 0:
        raise ValueError("fp8_matmul needs K > 0")
    k = a.shape[-1]
    n, kb = b.shape if trans_b else b.shape[::-1]
    if kb != k:
        raise ValueError(f"a has K = {k}, b has K = {kb}")
    if a_scale.shape != (*a.shape[:-1], (k + 127) // 128):
        raise ValueError(f"a_scale must be {(*a.shape[:-1], (k + 127) // 128)}, got {tuple(a_scale.shape)}")
    e8 = _is_e8m0(a_scale)
    if e8 != _is_e8m0(b_scale):
        a_scale, b_scale = (_e8m0_float(a_scale), b_scale) if e8 else (a_scale, _e8m0_float(b_scale))
        e8 = False
    _same_device(a, a_scale, b, b_scale)
    y = a.new_empty((*a.shape[:-1], n), dtype=out_dtype)
    m = y.numel() // n if n else 0
    if m == 0:
        return y
    a2, lda = _fp8_rows(a if a.dim() == 2 else a.reshape(m, k))
    b2, ldb = _fp8_rows(b)
    sa, sb = _fp8_scale(a_scale), _fp8_scale(b_scale)
    check(lib().dsv4_fp8_matmul(a2.data_ptr(), lda, sa.data_ptr(), b2.data_ptr(), ldb, sb.data_ptr(),
                                SCALE_E8M0 if e8 else SCALE_FP32, int(bool(trans_b)), m, n, k, y.data_ptr(), n,
                                _DT[out_dtype], _stream(a.device)))
    return y


def fp8_status(device=None) -> None:
    """Synchronise the current stream of ``device`` and raise if a wait of an
    ``fp8_matmul`` / ``fp8_linear`` kernel ran out since the last call (its
    outputs are then undefined)."""
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise ValueError("fp8_status needs a CUDA device")
    index = torch.cuda.current_device() if dev.index is None else dev.index
    check(lib().dsv4_fp8_status(index, _stream(dev)))


def _fp8_linear_call(x: torch.Tensor, w: torch.Tensor, ws: torch.Tensor, trans: bool) -> torch.Tensor:
    """act_quant(x) times w (trans: w.T) -> x's type; scales of ws's type."""
    k = x.shape[-1]
    n = w.shape[0 if trans else 1]
    if k == 0:      # the gradient of a layer without outputs
        return x.new_zeros((*x.shape[:-1], n))
    y = x.new_empty((*x.shape[:-1], n))
    m = y.numel() // n if n else 0
    if m == 0:
        return y
    if not x.is_contiguous():
        x = x.detach().contiguous()
    w2, ldw = _fp8_rows(w)
    sw = _fp8_scale(ws)
    kind = SCALE_FP32 if sw.dtype == torch.float32 else SCALE_E8M0
    # the codes (rows padded to 16 bytes) and the scales: dsv4_fp8_linear_workspace_bytes
    nb = m * ((k + 15) // 16 * 16 + (k + 127) // 128 * (4 if kind == SCALE_FP32 else 1))
    buf = x.new_empty((nb + 1) // 2)       # x's type: at least two bytes an element
    check(lib().dsv4_fp8_linear(x.data_ptr(), _DT[x.dtype], k, w2.data_ptr(), ldw, sw.data_ptr(), kind, int(trans), m, n,
                                k, y.data_ptr(), n, buf.data_ptr(), nb, _stream(x.device)))
    return y


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, ws):
        ctx.save_for_backward(w, ws)
        return _fp8_linear_call(x, w, ws, True)

    @staticmethod
    def backward(ctx, dy):
        if dy.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("fp8_linear is differentiable once")
        w, ws = ctx.saved_tensors
        return _fp8_linear_call(dy, w, ws, False), None, None


def _has_tangent(*ts) -> bool:
    """A tensor is a forward-mode dual one (outside a dual level none is)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and \
        any(forward_ad.unpack_dual(t).tangent is not None for t in ts)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    """Linear layer on a frozen FP8 weight [N, K] with one scale per 128 x 128
    block: ``act_quant(x)`` (power-of-two scales for an E8M0 ``weight_scale``,
    amax / 448 for a float32 one), then ``fp8_matmul``.  ``x`` [.., K] is bf16
    or fp32, and so is the result [.., N].

    Differentiable in ``x``: the gradient dy is quantised the same way, along
    N, and multiplied with the same stored weight (the rounding of x is passed
    through).  The weight is a checkpoint's and gets no gradient.  Forward-mode
    tangents are refused.  As with
    torch's own operators, a backward pass is captured into a CUDA graph only
    while no eager graph of the same leaves is alive."""
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"fp8_linear expects bf16 or fp32, got {x.dtype}")
    _check_fp8_weight(weight, weight_scale)
    if weight.requires_grad or weight_scale.requires_grad:
        raise ValueError("fp8_linear has no gradient for the weight or its scales")
    if x.dim() == 0 or x.shape[-1] != weight.shape[1] or x.shape[-1] == 0:
        raise ValueError(f"x {tuple(x.shape)} does not match the weight {tuple(weight.shape)}")
    _is_e8m0(weight_scale)
    _same_device(x, weight, weight_scale)
    if (x.requires_grad and torch.is_grad_enabled()) or _has_tangent(x, weight, weight_scale):
        return _Fp8Linear.apply(x, weight, weight_scale)      # which refuses a tangent
    return _fp8_linear_call(x, weight, weight_scale, True)


def dynamic_mx_quant(x: torch.Tensor):
    """bf16 [.., C] -> (packed E2M1 uint8 [.., C//2], E8M0 uint8 [.., C//32])."""
    _need_cuda(x)
    if x.dtype != torch.bfloat16:
        raise TypeError("dynamic_mx_quant expects bf16")
    x = x.contiguous()
    cols = x.shape[-1]
    rows = x.numel() // cols
    q = torch.empty((*x.shape[:-1], cols // 2), dtype=torch.uint8, device=x.device)
    s = torch.empty((*x.shape[:-1], cols // 32), dtype=torch.uint8, device=x.device)
    check(lib().dsv4_act_quant_mxfp4(x.data_ptr(), rows, cols, q.data_ptr(), s.data_ptr(), _stream(x.device)))
    return q, s


def route_topk(x: torch.Tensor, gate_weight: torch.Tensor, bias: torch.Tensor | None, topk: int,
               score_func: str = "sqrtsoftplus", renormalize: bool = True, route_scale: float = 1.5,
               tid2eid: torch.Tensor | None = None, input_ids: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None, out=None):
    """Router of the MoE layer.  Returns (weights fp32 [T,k], indices int32 [T,k]),
    written into ``out`` = (weights, indices) when given."""
    _need_cuda(x, gate_weight, bias, tid2eid, input_ids)
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    x = x.contiguous()
    w = gate_weight.contiguous().float()
    t, h = x.shape
    e = w.shape[0]
    if tid2eid is not None:
        if input_ids is None:
            raise RuntimeError("hash routing needs input_ids (forward_context.input_ids is missing)")
        tid2eid = tid2eid.to(torch.int32).contiguous()
        input_ids = input_ids.to(torch.int64).reshape(-1).contiguous()
        if input_ids.numel() != t:
            raise ValueError("input_ids must have one id per token")
    b = None if bias is None else bias.float().contiguous()
    need = lib().dsv4_route_workspace_bytes(t, h, e)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 4), dtype=torch.uint8, device=x.device)
    if out is not None:
        wo, io = out
        if (wo.shape != (t, topk) or io.shape != (t, topk) or wo.dtype != torch.float32 or io.dtype != torch.int32
                or not (wo.is_contiguous() and io.is_contiguous())):
            raise ValueError("out must be contiguous (float32 [T, k], int32 [T, k]) tensors")
    else:
        wo = torch.empty((t, topk), dtype=torch.float32, device=x.device)
        io = torch.empty((t, topk), dtype=torch.int32, device=x.device)
    check(lib().dsv4_route_topk(
        x.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(),
        None if tid2eid is None else tid2eid.data_ptr(), None if input_ids is None else input_ids.data_ptr(),
        0 if tid2eid is None else tid2eid.shape[0], t, h, e, topk, SCORE_FUNCS[score_func], int(bool(renormalize)), float(route_scale),
        wo.data_ptr(), io.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        _stream(x.device)))
    return wo, io


def route_workspace_bytes(n_tokens: int, hidden: int, n_experts: int) -> int:
    n = lib().dsv4_route_workspace_bytes(n_tokens, hidden, n_experts)
    if n < 0:
        check(int(n))
    return int(n)


def moe_align(indices: torch.Tensor, n_experts: int) -> dict:
    """Stable counting sort of the [T,k] expert indices (int32) on the GPU."""
    _need_cuda(indices)
    idx = indices.to(torch.int32).contiguous()
    t, k = idx.shape
    p = t * k
    dev = idx.device
    out = {
        "counts": torch.empty(n_experts, dtype=torch.int32, device=dev),
        "offsets": torch.empty(n_experts + 1, dtype=torch.int32, device=dev),
        "sorted_flat": torch.empty(max(p, 1), dtype=torch.int32, device=dev),
        "inv": torch.empty(max(p, 1), dtype=torch.int32, device=dev),
        "active": torch.full((n_experts,), -1, dtype=torch.int32, device=dev),
        "n_active": torch.zeros(1, dtype=torch.int32, device=dev),
        "status": torch.zeros(1, dtype=torch.int32, device=dev),
    }
    o = out
    check(lib().dsv4_moe_align(idx.data_ptr(), t, k, n_experts, o["counts"].data_ptr(), o["offsets"].data_ptr(),
                               o["sorted_flat"].data_ptr(), o["inv"].data_ptr(), o["active"].data_ptr(),
                               o["n_active"].data_ptr(), o["status"].data_ptr(), _stream(dev)))
    out["sorted_flat"] = out["sorted_flat"][:p]
    out["inv"] = out["inv"][:p]
    return out


class _DifferentiatedOnce(torch.autograd.Function):
    """A gradient computed from ``inputs`` outside autograd: differentiating
    it raises (an untracked result would only leave the term out)."""

    @staticmethod
    def forward(ctx, what, grad, *inputs):
        ctx.what = what
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} is differentiable once")


class _BalanceLoss(torch.autograd.Function):
    # logits: contiguous
    @staticmethod
    def forward(ctx, logits, indices, offsets, n_seqs, score, alpha, status):
        t, e = logits.shape
        nb = lib().dsv4_balance_workspace_bytes(t, e, n_seqs)
        ws = logits.new_empty(nb, dtype=torch.uint8)
        loss = logits.new_empty((), dtype=torch.float32)
        counts = logits.new_empty(e if offsets is None else (n_seqs, e), dtype=torch.int32)
        check(lib().dsv4_balance_forward(logits.data_ptr(), _DT[logits.dtype], t, e, indices.data_ptr(),
                                         indices.shape[1], None if offsets is None else offsets.data_ptr(), n_seqs,
                                         score, alpha, loss.data_ptr(), counts.data_ptr(), ws.data_ptr(), nb,
                                         None if status is None else status.data_ptr(), _stream(logits.device)))
        ctx.save_for_backward(logits, ws)
        ctx.args = (n_seqs, score, alpha)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)      # no zeros for the counts
        return loss, counts

    @staticmethod
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None, None, None
        logits, ws = ctx.saved_tensors
        n_seqs, score, alpha = ctx.args
        t, e = logits.shape
        up = grad_loss if grad_loss.dtype == torch.float32 else grad_loss.float()
        out = torch.empty_like(logits)
        check(lib().dsv4_balance_backward(logits.data_ptr(), _DT[logits.dtype], t, e, n_seqs, score, alpha,
                                          up.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(),
                                          _stream(logits.device)))
        if torch.is_grad_enabled():           # create_graph
            out = _DifferentiatedOnce.apply("balance_loss", out, logits, up)
        return out, None, None, None, None, None, None


def balance_loss(logits: torch.Tensor, indices: torch.Tensor, score_func: str = "sqrtsoftplus", alpha: float = 1.0,
                 seq_offsets: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """Load balance loss of a router (float32 scalar, differentiable once in
    ``logits``: a second derivative raises) and the picks per expert (int32 [E], or [S, E] with
    ``seq_offsets``, which ``parallel_ep.balanced_placement`` takes as loads).

    ``logits`` [T, E] fp32 or bf16 (E <= 1024), ``indices`` [T, k] the
    router's picks (``route_topk``; -1 = empty; T k < 2^31).  ``seq_offsets`` [S + 1]
    (integer, ascending, on the device) packs S sequences: rows o[s] ..
    o[s+1]-1 are sequence s.  A row without a pick and a row outside the
    sequences are padding: they do not count and their gradient is 0.  With p
    = score / sum score, the picks c and the tokens n of a sequence:
        alpha * mean_s sum_e (c[e] E / sum c) * (sum_t p[t, e] / n)
    over the sequences that have tokens; the counts are constants of the
    gradient.  A pick outside [-1, E) is skipped; it and offsets that descend
    or leave [0, T] set DSV4_EINVAL (-1) in ``status`` (int32 [1], zeroed by
    the caller) when it is given."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("logits must be fp32 or bf16 [T, E]")
    t, e = logits.shape
    if not 1 <= e <= 1024:
        raise ValueError("balance_loss handles 1 to 1024 experts")
    if indices.dim() != 2 or indices.shape[0] != t or indices.shape[1] < 1:
        raise ValueError("indices must be [T, k], one row per row of logits")
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError("indices must be int32 or int64")
    if score_func not in SCORE_FUNCS:
        raise ValueError(f"score_func must be one of {sorted(SCORE_FUNCS)}")
    n_seqs = 1
    if seq_offsets is not None:
        if seq_offsets.dim() != 1 or seq_offsets.numel() < 2 or seq_offsets.dtype not in (torch.int32, torch.int64):
            raise ValueError("seq_offsets must be int32 or int64 [S + 1] with S >= 1")
        n_seqs = seq_offsets.numel() - 1
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise TypeError("status must be an int32 tensor")
    _same_device(logits, indices, seq_offsets, status)
    if indices.dtype == torch.int64:
        indices = indices.clamp(-2, e).to(torch.int32)     # what is out of range stays out of range
    if seq_offsets is not None:
        if seq_offsets.dtype == torch.int64:
            seq_offsets = seq_offsets.clamp(-1, 0x7fffffff).to(torch.int32)
        seq_offsets = seq_offsets.contiguous()
    loss, counts = _BalanceLoss.apply(logits.contiguous(), indices.contiguous(), seq_offsets, n_seqs,
                                      SCORE_FUNCS[score_func], float(alpha), status)
    return loss, counts


def combine_ordered(rows: torch.Tensor, order: torch.Tensor) -> torch.Tensor:
    """y[t] = bf16(sum_j rows[order[t, j]]) in float32, j ascending; -1 skips."""
    _need_cuda(rows, order)
    rows = rows.contiguous()
    o = order.to(torch.int32).contiguous()
    t, k = o.shape
    y = torch.empty((t, rows.shape[1]), dtype=torch.bfloat16, device=rows.device)
    check(lib().dsv4_moe_combine_ordered(rows.data_ptr(), o.data_ptr(), t, k, rows.shape[1], y.data_ptr(),
                                         _stream(rows.device)))
    return y


def expert_slot_bytes(hidden: int, inter: int) -> int:
    n = lib().dsv4_expert_slot_bytes(hidden, inter)
    if n < 0:
        check(int(n))
    return int(n)


def pack_expert(w1p, w1s, w2p, w2s, w3p, w3s, hidden: int, inter: int, out=None) -> torch.Tensor:
    """Pack the six checkpoint tensors of one expert (CPU) into one slot
    (CPU uint8 tensor, optionally written into ``out``)."""
    ts = [t.detach().contiguous().view(torch.uint8) if t.dtype != torch.uint8 else t.detach().contiguous()
          for t in (w1p, w1s, w2p, w2s, w3p, w3s)]
    for t in ts:
        if t.is_cuda:
            raise ValueError("pack_expert packs host tensors")
    nb = expert_slot_bytes(hidden, inter)
    if out is None:
        out = torch.empty(nb, dtype=torch.uint8)
    if out.is_cuda or out.numel() < nb or not out.is_contiguous():
        raise ValueError("out must be a contiguous host uint8 buffer of at least the slot size")
    check(lib().dsv4_pack_expert_host(*[t.data_ptr() for t in ts], hidden, inter, out.data_ptr()))
    return out


def shared_slot_bytes(hidden: int, inter: int) -> int:
    n = lib().dsv4_shared_slot_bytes(hidden, inter)
    if n < 0:
        check(int(n))
    return int(n)


def pack_shared_expert(w1, s1, w2, s2, w3, s3, hidden: int, inter: int, out=None) -> torch.Tensor:
    """Pack the shared expert's FP8 checkpoint tensors (w1 / w3 [I, H], w2
    [H, I] E4M3 bytes; s* [ceil(N/128), ceil(K/128)] E8M0 bytes; host) into
    its FP8 slot (host uint8 tensor)."""
    ts = [t.detach().contiguous().view(torch.uint8) if t.dtype != torch.uint8 else t.detach().contiguous()
          for t in (w1, s1, w2, s2, w3, s3)]
    for t in ts:
        if t.is_cuda:
            raise ValueError("pack_shared_expert packs host tensors")
    nb = shared_slot_bytes(hidden, inter)
    if out is None:
        out = torch.empty(nb, dtype=torch.uint8)
    if out.is_cuda or out.numel() < nb or not out.is_contiguous():
        raise ValueError("out must be a contiguous host uint8 buffer of at least the slot size")
    check(lib().dsv4_pack_shared_host(*[t.data_ptr() for t in ts], hidden, inter, out.data_ptr()))
    return out


def unpack_expert(slot: torch.Tensor, hidden: int, inter: int) -> dict:
    """Inverse of ``pack_expert`` (host tensors) -> six checkpoint tensors."""
    s = slot.detach().cpu().contiguous()
    h, i = hidden, inter
    out = {"w1p": torch.empty((i, h // 2), dtype=torch.uint8), "w1s": torch.empty((i, h // 32), dtype=torch.uint8),
           "w2p": torch.empty((h, i // 2), dtype=torch.uint8), "w2s": torch.empty((h, i // 32), dtype=torch.uint8),
           "w3p": torch.empty((i, h // 2), dtype=torch.uint8), "w3s": torch.empty((i, h // 32), dtype=torch.uint8)}
    check(lib().dsv4_unpack_expert_host(s.data_ptr(), h, i, *[out[k].data_ptr() for k in
                                                            ("w1p", "w1s", "w2p", "w2s", "w3p", "w3s")]))
    return out


def slot_dequant(slot: torch.Tensor, hidden: int, inter: int) -> dict:
    """bf16 w1/w2/w3 of one device-resident slot (ExpertBank.get semantics)."""
    _need_cuda(slot)
    dev = slot.device
    w1 = torch.empty((inter, hidden), dtype=torch.bfloat16, device=dev)
    w3 = torch.empty((inter, hidden), dtype=torch.bfloat16, device=dev)
    w2 = torch.empty((hidden, inter), dtype=torch.bfloat16, device=dev)
    check(lib().dsv4_slot_dequant(slot.data_ptr(), hidden, inter, w1.data_ptr(), w2.data_ptr(), w3.data_ptr(),
                                  _stream(dev)))
    return {"w1": w1, "w2": w2, "w3": w3}


class MoEPlan:
    """Binds a slot arena (uint8 CUDA tensor [n_slots, slot_bytes]) and a
    workspace to the layer dims; ``forward`` runs the fused routed-expert
    layer on the current stream."""

    def __init__(self, hidden: int, inter: int, n_experts: int, topk: int, max_tokens: int,
                 swiglu_limit: float, arena: torch.Tensor, with_shared: bool = False):
        _need_cuda(arena)
        if arena.dtype != torch.uint8 or not arena.is_contiguous() or arena.dim() != 2:
            raise TypeError("arena must be a contiguous uint8 CUDA tensor [n_slots, slot_bytes]")
        if arena.shape[1] != expert_slot_bytes(hidden, inter):
            raise ValueError("arena row size must equal the expert slot size")
        self.hidden, self.inter, self.n_experts, self.topk = hidden, inter, n_experts, topk
        self.with_shared = bool(with_shared)
        self.max_tokens = int(max_tokens)
        self.arena = arena
        self.device = arena.device
        sh = int(self.with_shared)
        nb = lib().dsv4_moe_workspace_bytes_ex(hidden, inter, n_experts, topk, self.max_tokens, sh)
        if nb < 0:
            check(int(nb))
        self.workspace = torch.empty(int(nb), dtype=torch.uint8, device=self.device)
        h = C.c_void_p()
        check(lib().dsv4_moe_plan_create_ex(C.byref(h), hidden, inter, n_experts, topk, self.max_tokens,
                                            float(swiglu_limit), arena.data_ptr(), arena.shape[0],
                                            self.workspace.data_ptr(), int(nb), sh))
        self._h = h

    def forward(self, x: torch.Tensor, weights: torch.Tensor, indices: torch.Tensor, slot_of: torch.Tensor,
                profile: str = "bf16", out: torch.Tensor | None = None,
                shared_slot: torch.Tensor | None = None) -> torch.Tensor:
        """Routed experts (plus the shared expert, whose FP8 slot a plan made
        ``with_shared`` takes) of the [T, H] bf16 tokens -> [T, H] bf16."""
        _need_cuda(x, weights, indices, slot_of)
        x = x.contiguous()
        if x.dtype != torch.bfloat16:
            raise TypeError("x must be bf16")
        t = x.shape[0]
        if t > self.max_tokens:
            raise ValueError(f"{t} tokens exceed the plan's max_tokens={self.max_tokens}")
        w = weights.contiguous().float()
        idx = indices.contiguous().to(torch.int32)
        so = slot_of.contiguous().to(torch.int32)
        if so.numel() < self.n_experts:
            raise ValueError("slot_of needs one entry per expert")
        if out is None:
            out = torch.empty((t, self.hidden), dtype=torch.bfloat16, device=x.device)
        if self.with_shared:
            if shared_slot is None or not shared_slot.is_cuda or shared_slot.dtype != torch.uint8:
                raise ValueError("this plan runs the shared expert: pass its FP8 slot (uint8 CUDA tensor)")
            check(lib().dsv4_moe_forward_shared(self._h, PROFILES[profile], x.data_ptr(), t, w.data_ptr(),
                                                idx.data_ptr(), so.data_ptr(), shared_slot.data_ptr(), out.data_ptr(),
                                                _stream(x.device)))
            return out
        check(lib().dsv4_moe_forward(self._h, PROFILES[profile], x.data_ptr(), t, w.data_ptr(), idx.data_ptr(),
                                     so.data_ptr(), out.data_ptr(), _stream(x.device)))
        return out

    def route(self, x: torch.Tensor, gate_weight: torch.Tensor, bias: torch.Tensor | None, topk: int,
              score_func: str = "sqrtsoftplus", renormalize: bool = True, route_scale: float = 1.5,
              tid2eid: torch.Tensor | None = None, input_ids: torch.Tensor | None = None):
        """``route_topk`` for a decode batch (< 256 tokens) in this plan's
        workspace: one launch (partial logits, grid barrier, top-k) when the
        grid fits on the GPU.  Returns (weights fp32 [T,k], indices int32 [T,k])."""
        _need_cuda(x, gate_weight, bias, tid2eid, input_ids)
        if x.dtype != torch.bfloat16:
            x = x.to(torch.bfloat16)
        x = x.contiguous()
        w = gate_weight.contiguous().float()
        t = x.shape[0]
        if tid2eid is not None:
            if input_ids is None:
                raise RuntimeError("hash routing needs input_ids (forward_context.input_ids is missing)")
            tid2eid = tid2eid.to(torch.int32).contiguous()
            input_ids = input_ids.to(torch.int64).reshape(-1).contiguous()
            if input_ids.numel() != t:
                raise ValueError("input_ids must have one id per token")
        b = None if bias is None else bias.float().contiguous()
        wo = torch.empty((t, topk), dtype=torch.float32, device=x.device)
        io = torch.empty((t, topk), dtype=torch.int32, device=x.device)
        check(lib().dsv4_moe_route(
            self._h, x.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(),
            None if tid2eid is None else tid2eid.data_ptr(), None if input_ids is None else input_ids.data_ptr(),
            0 if tid2eid is None else tid2eid.shape[0], t, topk, SCORE_FUNCS[score_func], int(bool(renormalize)),
            float(route_scale), wo.data_ptr(), io.data_ptr(), _stream(x.device)))
        return wo, io

    def forward_rows(self, x: torch.Tensor, weights: torch.Tensor, indices: torch.Tensor, slot_of: torch.Tensor,
                     profile: str = "bf16", n_tokens_dev: torch.Tensor | None = None):
        """The layer without its combine, for a token count that may be known
        only on the device (``n_tokens_dev``: int32 [1]; the first n rows of
        ``x`` / ``weights`` / ``indices`` are used, at most ``x.shape[0]``).
        Returns (rows bf16 [row capacity, H], inv int32 [T * k]): the output of
        assignment a is ``rows[inv[a]]``; both live in the plan's workspace
        until its next forward."""
        _need_cuda(x, weights, indices, slot_of)
        if x.dtype != torch.bfloat16 or not x.is_contiguous():
            raise TypeError("x must be contiguous bf16")
        t = x.shape[0]
        if t > self.max_tokens:
            raise ValueError(f"{t} tokens exceed the plan's max_tokens={self.max_tokens}")
        w = weights if weights.dtype == torch.float32 and weights.is_contiguous() else weights.contiguous().float()
        idx = indices if indices.dtype == torch.int32 and indices.is_contiguous() else \
            indices.contiguous().to(torch.int32)
        so = slot_of.contiguous().to(torch.int32)
        check(lib().dsv4_moe_forward_rows(self._h, PROFILES[profile], x.data_ptr(), t,
                                          None if n_tokens_dev is None else n_tokens_dev.data_ptr(), w.data_ptr(),
                                          idx.data_ptr(), so.data_ptr(), None, _stream(x.device)))
        return self.output_rows(t * self.topk)

    def forward_scatter(self, x: torch.Tensor, weights: torch.Tensor, indices: torch.Tensor, slot_of: torch.Tensor,
                        assign_dst_ptr: int, profile: str = "bf16", n_tokens_dev: torch.Tensor | None = None,
                        x_format: int = ROWS_BF16) -> None:
        """The layer whose down GEMM stores the output row of assignment a
        straight to the device address table ``assign_dst_ptr`` [T * k]
        (another GPU's memory included; null entries are dropped).  With
        ``x_format`` ROWS_FP8 (bf16 profile) or ROWS_MXFP4 (a4w4), x is uint8
        [T, row_bytes] rows quantised at their source."""
        _need_cuda(x, weights, indices, slot_of)
        if x_format == ROWS_BF16 and (x.dtype != torch.bfloat16 or not x.is_contiguous()):
            raise TypeError("x must be contiguous bf16")
        if x_format != ROWS_BF16 and (x.dtype != torch.uint8 or not x.is_contiguous()):
            raise TypeError("quantised rows must be a contiguous uint8 tensor")
        t = x.shape[0]
        if t > self.max_tokens:
            raise ValueError(f"{t} tokens exceed the plan's max_tokens={self.max_tokens}")
        w = weights if weights.dtype == torch.float32 and weights.is_contiguous() else weights.contiguous().float()
        idx = indices if indices.dtype == torch.int32 and indices.is_contiguous() else \
            indices.contiguous().to(torch.int32)
        so = slot_of.contiguous().to(torch.int32)
        check(lib().dsv4_moe_forward_scatter_q(self._h, PROFILES[profile], x.data_ptr(), int(x_format), t,
                                               None if n_tokens_dev is None else n_tokens_dev.data_ptr(),
                                               w.data_ptr(), idx.data_ptr(), so.data_ptr(), assign_dst_ptr,
                                               _stream(x.device)))

    def output_rows(self, n_assign: int):
        rp, ip = C.c_void_p(), C.c_void_p()
        check(lib().dsv4_moe_output_rows(self._h, C.byref(rp), C.byref(ip)))
        rows = torch.as_tensor(_DevArray(rp.value, (self._rows_cap(), self.hidden), "<i2"), device=self.device)
        inv = torch.as_tensor(_DevArray(ip.value, (max(n_assign, 1),), "<i4"), device=self.device)
        return rows.view(torch.bfloat16), inv[:n_assign]

    def _rows_cap(self) -> int:
        # padded row capacity of the plan (same rule as the library's workspace layout)
        p = self.max_tokens * self.topk
        bn = 128
        return (p + (bn - 1) * min(self.n_experts, p) + bn - 1) // bn * bn + bn

    STAGES = ("align", "quant_gather", "gate_up_gemm", "down_gemm", "combine")

    def set_gemm_tile(self, tokens_per_tile: int = 0) -> None:
        """Tokens per GEMM tile: 64, 112, or 0 for the library default."""
        check(lib().dsv4_moe_set_gemm_tile(self._h, int(tokens_per_tile)))

    def set_ffn_fusion(self, enable=None) -> None:
        """Gate/up and down GEMMs in one launch (True), two (False), or the
        library's choice (None: one launch with the decode tile)."""
        check(lib().dsv4_moe_set_ffn_fusion(self._h, -1 if enable is None else int(bool(enable))))

    def enable_timing(self, enable: bool = True) -> None:
        check(lib().dsv4_moe_enable_timing(self._h, int(bool(enable))))

    def stage_times(self) -> dict:
        """ms per stage of the last forward (waits for it)."""
        buf = (C.c_float * 5)()
        check(lib().dsv4_moe_stage_times(self._h, buf, 5))
        return dict(zip(self.STAGES, [float(v) for v in buf]))

    def n_active(self) -> int:
        """Active experts of the last forward (synchronises)."""
        ptrs = [C.c_void_p() for _ in range(6)]
        check(lib().dsv4_moe_debug_align(self._h, *[C.byref(p) for p in ptrs]))
        buf = (C.c_int32 * 1)()
        torch.cuda.synchronize(self.device)
        _memcpy_d2h(buf, ptrs[5].value, 4)
        return int(buf[0])

    def status(self) -> None:
        """Synchronise and raise if a kernel recorded an error."""
        check(lib().dsv4_moe_status(self._h, _stream(self.device)))

    def debug_align(self, n_tokens: int) -> dict:
        ptrs = [C.c_void_p() for _ in range(6)]
        check(lib().dsv4_moe_debug_align(self._h, *[C.byref(p) for p in ptrs]))
        p = n_tokens * self.topk
        e = self.n_experts
        names = ("counts", "offsets", "sorted_flat", "inv", "active", "n_active")
        sizes = (e, e + 1, p, p, e, 1)
        out = {}
        for name, ptr, n in zip(names, ptrs, sizes):
            if n == 0:
                out[name] = torch.zeros(0, dtype=torch.int32)
                continue
            buf = (C.c_int32 * n)()
            torch.cuda.synchronize(self.device)
            _memcpy_d2h(buf, ptr.value, 4 * n)
            out[name] = torch.tensor(list(buf), dtype=torch.int32)
        return out

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                lib().dsv4_moe_plan_destroy(h)
            except Exception:
                pass
            self._h = None


class _DevArray:
    def __init__(self, ptr: int, shape, typestr: str):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False),
                                         "version": 3}


def _memcpy_d2h(dst, src_ptr: int, nbytes: int):
    """Copy device memory at a raw address into a ctypes buffer via torch."""
    import numpy as np
    arr = np.frombuffer(dst, dtype=np.uint8)
    # wrap the device address as a torch tensor through __cuda_array_interface__
    class _View:
        __cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (src_ptr, False), "version": 3}
    t = torch.as_tensor(_View(), device="cuda")
    arr[:] = t.cpu().numpy()
