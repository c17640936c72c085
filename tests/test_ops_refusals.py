"""Arguments that the FP8 operators and the balance loss refuse: the Python
wrappers raise before they touch a device, the C entry points return
DSV4_EINVAL with a message.  Needs no GPU."""

import ctypes as C

import pytest
import torch

from dsv4_plugin import _lib, ops

F8 = torch.float8_e4m3fn


def f8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(F8)


def test_act_quant_refuses():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        ops.act_quant(x, 64)
    with pytest.raises(NotImplementedError):
        ops.act_quant(x, 128, "e5m3")
    with pytest.raises(NotImplementedError):
        ops.act_quant(x, 128, None, None, inplace=True)
    with pytest.raises(TypeError):
        ops.act_quant(x.double())
    with pytest.raises(TypeError):
        ops.act_quant(x, 128, None, torch.float8_e8m0fnu)
    with pytest.raises(TypeError):
        ops.act_quant(x, 128, "ue8m0", torch.float16)
    with pytest.raises(ValueError):
        ops.act_quant(x[:, :0])
    with pytest.raises(ValueError, match="CUDA"):
        ops.act_quant(x)


def test_fp8_matmul_refuses():
    a, sa = f8(4, 256), torch.ones(4, 2)
    b, sb = f8(130, 256), torch.ones(2, 2)
    with pytest.raises(TypeError):
        ops.fp8_matmul(a.view(torch.uint8), sa, b, sb)
    with pytest.raises(TypeError):
        ops.fp8_matmul(a, sa, b.float(), sb)
    with pytest.raises(TypeError):
        ops.fp8_matmul(a, sa.double(), b, sb)
    with pytest.raises(TypeError):
        ops.fp8_matmul(a, sa, b, sb, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.fp8_matmul(a, sa, b, torch.ones(1, 2))             # 130 rows are two blocks
    with pytest.raises(ValueError):
        ops.fp8_matmul(a, torch.ones(4, 1), b, sb)
    with pytest.raises(ValueError):
        ops.fp8_matmul(a, sa, b, sb, trans_b=False)            # K = 256 against 130
    with pytest.raises(ValueError):
        ops.fp8_matmul(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0])
    with pytest.raises(ValueError):
        ops.fp8_matmul(a, sa, b[0], sb)
    with pytest.raises(ValueError, match="CUDA"):
        ops.fp8_matmul(a, sa, b, sb)


def test_fp8_linear_refuses():
    w, s = f8(130, 256), torch.ones(2, 2)
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        ops.fp8_linear(x.half(), w, s)
    with pytest.raises(ValueError):
        ops.fp8_linear(x[:, :128], w, s)
    with pytest.raises(ValueError):
        ops.fp8_linear(x, w, s.clone().requires_grad_())
    with pytest.raises(TypeError):
        ops.fp8_linear(x, w, s.half())
    with pytest.raises(ValueError, match="CUDA"):
        ops.fp8_linear(x, w, s)
    with pytest.raises(ValueError):
        ops.fp8_status("cpu")


def test_balance_loss_refuses():
    lg, idx = torch.zeros(6, 8), torch.zeros(6, 2, dtype=torch.int32)
    off = torch.tensor([0, 6], dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.balance_loss(lg.half(), idx)
    with pytest.raises(TypeError):
        ops.balance_loss(lg, idx.float())
    with pytest.raises(ValueError):
        ops.balance_loss(torch.zeros(6, 1025), idx)
    with pytest.raises(ValueError):
        ops.balance_loss(lg, idx[:5])
    with pytest.raises(ValueError):
        ops.balance_loss(lg, idx[:, :0])
    with pytest.raises(ValueError):
        ops.balance_loss(lg, idx, score_func="tanh")
    with pytest.raises(ValueError):
        ops.balance_loss(lg, idx, seq_offsets=off[:1])
    with pytest.raises(ValueError):
        ops.balance_loss(lg, idx, seq_offsets=off.float())
    with pytest.raises(TypeError):
        ops.balance_loss(lg, idx, status=torch.zeros(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.balance_loss(lg, idx, seq_offsets=off)


P = 4096   # an address that is never read: every call below is refused first


def refused(name, *args):
    L = _lib.lib()
    assert getattr(L, name)(*args) == _lib.DSV4_EINVAL
    return L.dsv4_last_error_string().decode()


def test_act_quant_entry_refuses():
    def call(x=P, dt=0, rows=4, cols=256, ldx=256, q=P, ldq=256, s=P, kind=0):
        return refused("dsv4_act_quant_fp8", x, dt, rows, cols, ldx, q, ldq, s, kind, None)

    assert "null" in call(x=None) and "null" in call(q=None) and "null" in call(s=None)
    assert "bf16" in call(dt=3)
    assert "scale type" in call(kind=3)
    assert "cols" in call(cols=0) and "rows" in call(rows=-1)
    assert "stride" in call(ldx=255) and "stride" in call(ldq=255)
    assert "misaligned" in call(x=P + 1) and "misaligned" in call(s=P + 2, kind=1)
    assert "too many" in call(rows=1 << 40)
    assert _lib.lib().dsv4_act_quant_fp8(None, 0, 0, 256, 256, None, 256, None, 0, None) == 0


def test_fp8_matmul_entry_refuses():
    def call(a=P, lda=256, sa=P, b=P, ldb=256, sb=P, kind=0, tb=1, m=4, n=16, k=256, y=P, ldy=16, out=0):
        return refused("dsv4_fp8_matmul", a, lda, sa, b, ldb, sb, kind, tb, m, n, k, y, ldy, out, None)

    for name in ("a", "sa", "b", "sb", "y"):
        assert "null" in call(**{name: None})
    assert "E8M0" in call(kind=2)
    assert "bf16" in call(out=1)
    assert "k > 0" in call(k=0) and "k > 0" in call(m=-1)
    assert "stride" in call(lda=240) and "stride" in call(ldb=240) and "stride" in call(ldy=15)
    assert "stride" in call(tb=0, n=272, ldy=272)
    assert "16 bytes" in call(a=P + 8) and "16 bytes" in call(lda=264) and "16 bytes" in call(b=P + 1)
    assert "misaligned" in call(y=P + 1) and "misaligned" in call(sa=P + 2, kind=1)
    assert "too large" in call(m=1 << 40)
    L = _lib.lib()
    assert L.dsv4_fp8_matmul(None, 256, None, None, 256, None, 0, 1, 0, 16, 256, None, 16, 0, None) == 0


def test_fp8_linear_entry_refuses():
    L = _lib.lib()
    assert L.dsv4_fp8_linear_workspace_bytes(100, 250, 0) == 100 * (256 + 2)
    assert L.dsv4_fp8_linear_workspace_bytes(100, 256, 1) == 100 * (256 + 8)
    for bad in ((-1, 256, 0), (4, 0, 0), (4, 256, 2), (1 << 40, 256, 0)):
        assert L.dsv4_fp8_linear_workspace_bytes(*bad) == _lib.DSV4_EINVAL

    def call(x=P, dt=0, ldx=256, w=P, ldw=256, sw=P, kind=0, tw=1, m=100, n=16, k=256, y=P, ldy=16, ws=P, nb=1 << 20):
        return refused("dsv4_fp8_linear", x, dt, ldx, w, ldw, sw, kind, tw, m, n, k, y, ldy, ws, nb, None)

    for name in ("x", "w", "sw", "y", "ws"):
        assert "null" in call(**{name: None})
    assert "bf16" in call(dt=1) and "E8M0" in call(kind=2) and "k > 0" in call(k=0)
    assert "stride" in call(ldx=255) and "stride" in call(ldw=240) and "stride" in call(ldy=15)
    assert "stride" in call(tw=0, n=272, ldy=272)
    assert "16 bytes" in call(w=P + 8) and "16 bytes" in call(ldw=264)
    assert "misaligned" in call(x=P + 1) and "misaligned" in call(y=P + 1) and "misaligned" in call(sw=P + 2, kind=1)
    assert "workspace" in call(nb=100) and "workspace" in call(ws=P + 8)
    assert "too large" in call(m=1 << 40)


def test_balance_entries_refuse():
    L = _lib.lib()
    big = L.dsv4_balance_workspace_bytes(100, 8, 2)
    assert big > 0
    for bad in ((-1, 8, 1), (1 << 31, 8, 1), (4, 0, 1), (4, 1025, 1), (4, 8, 0), (4, 1024, 1 << 22)):
        assert L.dsv4_balance_workspace_bytes(*bad) == _lib.DSV4_EINVAL

    def fwd(lg=P, dt=2, t=100, e=8, idx=P, k=2, off=P, s=2, score=0, loss=P, counts=P, ws=P, nb=big):
        return refused("dsv4_balance_forward", lg, dt, t, e, idx, k, off, s, score, C.c_float(1.0), loss, counts, ws,
                       nb, None, None)

    for name in ("lg", "idx", "loss", "counts", "ws"):
        assert "null" in fwd(**{name: None})
    assert "fp32" in fwd(dt=1)
    assert "topk" in fwd(k=0)
    assert "score" in fwd(score=3)
    assert "offsets" in fwd(off=None)
    assert "workspace" in fwd(nb=big - 1) and "aligned" in fwd(ws=P + 8)
    assert "n_experts" in fwd(e=2000)

    def bwd(lg=P, dt=2, t=100, e=8, s=2, score=0, up=P, out=P, ws=P, nb=big):
        return refused("dsv4_balance_backward", lg, dt, t, e, s, score, C.c_float(1.0), up, out, ws, nb, None)

    for name in ("lg", "up", "out", "ws"):
        assert "null" in bwd(**{name: None})
    assert "fp32" in bwd(dt=1) and "score" in bwd(score=-1) and "workspace" in bwd(nb=16)


@pytest.mark.parametrize("t,k", [(1 << 30, 2), (1 << 28, 8), ((1 << 31) - 1, 2)])
def test_balance_refuses_more_picks_than_it_can_count(t, k):
    """The picks of a sequence are counted in 32 bits."""
    nb = _lib.lib().dsv4_balance_workspace_bytes(t, 8, 1)
    assert "picks" in refused("dsv4_balance_forward", P, _lib.DT_FP32, t, 8, P, k, None, 1, 0, C.c_float(1.0), P, P, P,
                              nb, None, None)
