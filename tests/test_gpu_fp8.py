"""act_quant with separate outputs, fp8_matmul and fp8_linear on the GPU,
against plain 64-bit implementations of their definitions.

Tolerances.  Quantisation: scales and codes are exact for 16-bit input (the
quotient of two short significands is a tie of E4M3 or at least 2^-20 away
from one); for fp32 input a code may be the neighbour when 448 x / amax lies
within 2^-21 of a tie.  Products: every product of two E4M3 values is exact
in fp32; an MMA adds 32 of K at a time to an fp32 accumulator, so at most K /
32 + 32 roundings (or truncations, 2^-23 each) of a running sum that is never
above the sum of the magnitudes, plus three roundings of scales (2^-24 each):
    |err| <= (K / 32 + 34) * 2^-23 * sum_k |terms|,
plus half a step (2^-8) of the value for a bf16 result."""

import numpy as np
import pytest
import torch

from oracle import moe_oracle as O
from dsv4_plugin import synthetic as S
from helpers import SyntheticLayer, bf16_tensor, bf16_to_np

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


def blocks(x):
    """[R, C] -> [R, nb, 128] zero padded."""
    r, c = x.shape
    nb = -(-c // 128)
    return torch.nn.functional.pad(x, (0, nb * 128 - c)).view(r, nb, 128)


def e4m3_grid(v):
    """Nearest E4M3 value of float64 v, ties to even, saturating."""
    v = v.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def quant64(x, pow2):
    """(codes' values, scales, exact quotients) in float64."""
    x = x.double()
    c = x.shape[1]
    amax = blocks(x).abs().amax(-1).clamp(min=float(np.float32(1e-4)))
    if pow2:
        m, e = torch.frexp(amax / 448.0)
        s = torch.exp2((e - (m == 0.5).int()).double())
        v = x / s.repeat_interleave(128, 1)[:, :c]
    else:
        s = amax / 448.0
        v = x * 448.0 / amax.repeat_interleave(128, 1)[:, :c]
    return e4m3_grid(v), s, v


def activations(seed, m, k):
    g = gen(seed)
    x = torch.randn((m, k), generator=g, device="cuda") * torch.exp(torch.randn((m, 1), generator=g, device="cuda"))
    x[:, 3::29] *= 30.0
    return x


def weight(seed, n, k, e8):
    g = gen(seed)
    q = (torch.randn((n, k), generator=g, device="cuda") * 100).clamp(-448, 448).to(F8)
    s = torch.exp2(torch.randint(-15, -8, (-(-n // 128), -(-k // 128)), generator=g, device="cuda").float())
    return q, s.to(E8) if e8 else s * (1 + torch.rand(s.shape, generator=g, device="cuda"))


def deq64(q, s, rows128):
    s = s.double()
    if rows128:
        s = s.repeat_interleave(128, 0)[: q.shape[0]]
    return q.double() * s.repeat_interleave(128, 1)[:, : q.shape[1]]


def check_product(y, a64, b64, k, what=""):
    """y against a64 @ b64 ([M, K] and [K, N], float64) within the bound above."""
    ref, mag = a64 @ b64, a64.abs() @ b64.abs()
    tol = (k / 32 + 34) * 2.0 ** -23 * mag + (2.0 ** -8 * ref.abs() if y.dtype == torch.bfloat16 else 0)
    bad = (y.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (1, 128), (5, 129), (64, 4096), (33, 1000), (2, 1032),
                                       (257, 2008), (7, 136)])
def test_act_quant(ops, dtype, rows, cols):
    x = (activations(rows * 7 + cols, rows, cols)).to(dtype)
    x[0, 0] = 0
    for fmt, sd in (("ue8m0", E8), ("ue8m0", torch.float32), ("ue8m0", None), (None, None)):
        q, s = ops.act_quant(x, 128, fmt, sd)
        ref, s64, v = quant64(x, fmt is not None)
        assert q.dtype == F8 and q.shape == x.shape and s.shape == (rows, -(-cols // 128))
        assert s.dtype == (E8 if sd is E8 else torch.float32)
        assert torch.equal(s.float(), s64.float())
        if fmt is None and dtype == torch.float32:
            off = (q.double() - v).abs() - (ref - v).abs()   # how much further than the nearest code
            assert (off <= v.abs() * 2.0 ** -20).all()
        else:
            assert torch.equal(q.double(), ref)


def test_act_quant_edges(ops):
    """Zero rows, a block at its limit, tiny and huge values, NaN and infinity."""
    x = torch.zeros(8, 384, device="cuda")
    x[1, :128] = 448.0
    x[1, 128] = 448.0 * (1 + 2.0 ** -23)     # one step above: the next power of two
    x[2, 0] = 3e38
    x[3, 5] = 1e-30
    x[4, 200] = float("inf")
    x[4, 201] = 1.0
    x[5, 300] = float("nan")
    x[5, 301] = 2.0
    x[6] = -0.0
    x[7, 383] = -57.0
    q, s = ops.act_quant(x, 128, "ue8m0", torch.float32)
    ref, s64, _ = quant64(torch.nan_to_num(x, nan=0.0, posinf=3.4028234663852886e38), True)
    assert torch.equal(s, s64.float())
    assert s[0, 0] == 2.0 ** -22 and s[1, 0] == 1.0 and s[1, 1] == 2.0
    assert torch.isnan(q.float()[5, 300]) and q.float()[4, 200] == 448.0 and q.float()[4, 201] == 0.0
    q2 = q.double()
    q2[5, 300] = 0.0
    ref[4, 200] = 448.0
    assert torch.equal(q2, ref)
    q, s = ops.act_quant(x, 128, None)
    assert s[1, 0] == 1.0 and torch.isnan(q.float()[5, 300]) and q.float()[4, 200] == 448.0
    assert (q.float()[0] == 0).all() and q.float()[2, 0] == 448.0 and q.float()[7, 383] == -448.0


def test_act_quant_round_trip_equals_in_place_form(ops):
    x = activations(1, 40, 1024).bfloat16()
    q, s = ops.act_quant(x, 128, "ue8m0")
    back = (q.float() * s.repeat_interleave(128, 1)).bfloat16()
    assert torch.equal(back, ops.act_quant(x.clone(), 128, "ue8m0", None, True))


def test_act_quant_shapes_and_strides(ops):
    x = activations(2, 24, 512).bfloat16()
    q, s = ops.act_quant(x.view(2, 3, 4, 512))
    q0, s0 = ops.act_quant(x)
    assert q.shape == (2, 3, 4, 512) and s.shape == (2, 3, 4, 4)
    assert torch.equal(q.view(24, 512).view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s.view(24, 4), s0)
    wide = torch.cat([x, x], 1)
    q1, _ = ops.act_quant(wide[:, 1:257])          # unaligned, strided rows
    q2, _ = ops.act_quant(wide[:, 1:257].contiguous())
    assert torch.equal(q1.view(torch.uint8), q2.view(torch.uint8))
    q3, s3 = ops.act_quant(x[:0])
    assert q3.shape == (0, 512) and s3.shape == (0, 4)


SIZES = [(1, 128, 128), (1, 16, 16), (2, 1000, 144), (16, 130, 512), (17, 256, 640), (33, 127, 1040), (64, 384, 4096),
         (65, 144, 256), (127, 512, 2000), (129, 128, 1024), (300, 1001, 2000), (257, 272, 528)]


@pytest.mark.parametrize("e8", [True, False])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_fp8_matmul(ops, m, n, k, e8):
    q, s = ops.act_quant(activations(m + n, m, k), 128, "ue8m0" if e8 else None, E8 if e8 else None)
    w, ws = weight(k, n, k, e8)
    y = ops.fp8_matmul(q, s, w, ws, out_dtype=torch.float32)
    check_product(y, deq64(q, s, False), deq64(w, ws, True).t(), k, "fp32")
    yb = ops.fp8_matmul(q, s, w, ws)
    assert yb.dtype == torch.bfloat16 and torch.equal(yb, y.bfloat16())      # one rounding of the same sums
    n16 = (n + 15) // 16 * 16
    w, ws = weight(k + 1, k, n16, e8)
    y = ops.fp8_matmul(q, s, w, ws, trans_b=False, out_dtype=torch.float32)
    check_product(y, deq64(q, s, False), deq64(w, ws, True), k, "trans_b=False")
    ops.fp8_status()


@pytest.mark.parametrize("e8", [True, False])
@pytest.mark.parametrize("m,n,k", [(512, 768, 4096), (1000, 1100, 1040), (2049, 520, 2048), (260, 4096, 256)])
def test_fp8_matmul_larger(ops, m, n, k, e8):
    q, s = ops.act_quant(activations(m + n, m, k).bfloat16(), 128, "ue8m0" if e8 else None, E8 if e8 else None)
    for trans in (True, False):
        nn = n if trans else (n + 15) // 16 * 16
        w, ws = weight(k, *((nn, k) if trans else (k, nn)), e8)
        y = ops.fp8_matmul(q, s, w, ws, trans_b=trans)
        b = deq64(w, ws, True)
        check_product(y, deq64(q, s, False), b.t() if trans else b, k)
    ops.fp8_status()


@pytest.mark.parametrize("e8", [True, False])
def test_fp8_matmul_unaligned_is_copied(ops, e8):
    """K that is no multiple of 16, column slices, expanded rows, uint8 E8M0 scales, 3-D a."""
    q, s = ops.act_quant(activations(5, 12, 333), 128, "ue8m0" if e8 else None, E8 if e8 else None)
    w, ws = weight(6, 50, 333, e8)
    y = ops.fp8_matmul(q, s, w, ws, out_dtype=torch.float32)
    check_product(y, deq64(q, s, False), deq64(w, ws, True).t(), 333)
    big, bs = weight(7, 256, 512, e8)
    q, s = ops.act_quant(activations(8, 6, 256), 128, "ue8m0" if e8 else None, E8 if e8 else None)
    y = ops.fp8_matmul(q, s, big[:, 128:384], bs[:, 1:3], out_dtype=torch.float32)      # strided rows, as they are
    check_product(y, deq64(q, s, False), deq64(big[:, 128:384], bs[:, 1:3], True).t(), 256)
    y1 = ops.fp8_matmul(q[:1].expand(5, 256), s[:1].expand(5, 2), big[:, :256], bs[:, :2], out_dtype=torch.float32)
    y2 = ops.fp8_matmul(q[:1], s[:1], big[:, :256], bs[:, :2], out_dtype=torch.float32)
    assert torch.equal(y1, y2.expand(5, 256))
    y3 = ops.fp8_matmul(q.view(2, 3, 256), s.view(2, 3, 2), big[:, :256], bs[:, :2], out_dtype=torch.float32)
    assert torch.equal(y3.view(6, 256), ops.fp8_matmul(q, s, big[:, :256], bs[:, :2], out_dtype=torch.float32))
    wt = big[:, :256].t()                                        # columns not next to each other
    y4 = ops.fp8_matmul(q, s, wt, bs[:, :2].t(), trans_b=False, out_dtype=torch.float32)
    check_product(y4, deq64(q, s, False), deq64(wt, bs[:, :2].t(), True), 256)
    if e8:
        assert torch.equal(y4, ops.fp8_matmul(q, s.view(torch.uint8), wt, bs[:, :2].t(), trans_b=False,
                                              out_dtype=torch.float32))
        y5 = ops.fp8_matmul(q, s.float(), wt, bs[:, :2].t(), trans_b=False, out_dtype=torch.float32)   # mixed
        check_product(y5, deq64(q, s, False), deq64(wt, bs[:, :2].t(), True), 256)


@pytest.mark.parametrize("e8", [True, False])
@pytest.mark.parametrize("k", [128, 1024, 1536, 2048, 2560, 3000, 3584, 4096, 4104, 12288])
def test_fp8_matmul_every_cluster_size(ops, k, e8):
    """K split over 1 to 8 CTAs, with shares that end inside a group of scales."""
    for m in (1, 40, 128):
        q, s = ops.act_quant(activations(k + m, m, k), 128, "ue8m0" if e8 else None, E8 if e8 else None)
        w, ws = weight(k, 200, k, e8)
        y = ops.fp8_matmul(q, s, w, ws, out_dtype=torch.float32)
        check_product(y, deq64(q, s, False), deq64(w, ws, True).t(), k, f"m {m}")


@pytest.mark.parametrize("e8", [True, False])
@pytest.mark.parametrize("n,k", [(4096, 1536), (4100, 1040), (2304, 4096), (8192, 100)])
def test_fp8_matmul_pairs(ops, n, k, e8):
    """More 128 x 128 tiles than SMs: the CTA pairs, ragged in every size."""
    m = 148 * 128 * 128 // n // 128 * 128 + 300
    q, s = ops.act_quant(activations(n, m, k).bfloat16(), 128, "ue8m0" if e8 else None, E8 if e8 else None)
    for trans in (True, False):
        nn = n if trans else (n + 15) // 16 * 16
        w, ws = weight(k, *((nn, k) if trans else (k, nn)), e8)
        b = deq64(w, ws, True)
        for out in (torch.bfloat16, torch.float32):
            y = ops.fp8_matmul(q, s, w, ws, trans_b=trans, out_dtype=out)
            check_product(y, deq64(q, s, False), b.t() if trans else b, k)
    ops.fp8_status()


def test_offsets_beyond_32_bits(ops):
    """x, a and y of more than 2^32 bytes: the last rows as computed alone."""
    rows, k = 1_060_000, 4096
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    x[-200:] = activations(1, 200, k).bfloat16()
    q, s = ops.act_quant(x, 128, "ue8m0", E8)
    q1, s1 = ops.act_quant(x[-200:].clone(), 128, "ue8m0", E8)
    del x
    assert torch.equal(q[-200:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-200:].float(), s1.float())
    for n in (64, 2304):                                        # one CTA per tile; pairs
        w, ws = weight(2, n, k, True)
        y = ops.fp8_matmul(q, s, w, ws)
        check_product(y[-200:], deq64(q1, s1, False), deq64(w, ws, True).t(), k)
        assert (y[:-200] == 0).all()
        del y
    ops.fp8_status()


def test_large_and_small_products_at_once(ops):
    """CTA pairs, clusters that split K and the routed layer's kernels on three
    streams together: clusters whose CTAs wait for one another must all get
    their tensor memory."""
    big, bs = weight(1, 2304, 2048, False)
    w, ws = weight(2, 1024, 4096, True)
    w2, ws2 = weight(3, 1024, 4096, False)
    xb, xs = activations(4, 1500, 2048).bfloat16(), activations(5, 100, 4096).bfloat16()
    want = [ops.fp8_linear(xb, big, bs), ops.fp8_linear(xs, w, ws), ops.fp8_linear(xs, w2, ws2), ops.fp8_linear(xs[:9], w, ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [[] for _ in range(4)]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                a, b = ((xb, (big, bs)), (xs, (w, ws)), (xs, (w2, ws2)), (xs[:9], (w, ws)))[i]
                got[i].append(ops.fp8_linear(a, *b))
    torch.cuda.synchronize()
    ops.fp8_status()
    for i in range(4):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_first_call_of_a_thread(ops):
    """A thread without a CUDA context of its own yet, as autograd's are."""
    import threading
    w, ws = weight(1, 256, 512, True)
    q, s = ops.act_quant(activations(1, 8, 512), 128, "ue8m0", E8)
    x = activations(2, 8, 512).bfloat16()
    want = [ops.fp8_matmul(q, s, w, ws), ops.fp8_linear(x, w, ws)]
    got = [None, None]

    def run(i):
        got[i] = ops.fp8_matmul(q, s, w, ws) if i == 0 else ops.fp8_linear(x, w, ws)
        torch.cuda.current_stream().synchronize()

    for i in range(2):
        t = threading.Thread(target=run, args=(i,))
        t.start()
        t.join()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_first_call_of_a_process_in_a_capture(ops):
    """Nothing has to run before a capture: kernels load and set up inside it."""
    import os
    import subprocess
    import sys
    import textwrap
    code = textwrap.dedent("""
        import torch
        from dsv4_plugin import ops
        x = torch.randn(20, 512, device="cuda").bfloat16()
        w = torch.ones(256, 512, device="cuda").to(torch.float8_e4m3fn)
        ws = torch.ones(2, 4, device="cuda")
        lg = torch.randn(20, 16, device="cuda")
        idx = torch.zeros(20, 2, dtype=torch.int32, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.fp8_linear(x, w, ws)
            loss, counts = ops.balance_loss(lg, idx, "softmax")
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.fp8_linear(x, w, ws)) and int(counts[0]) == 40
        assert torch.equal(loss, ops.balance_loss(lg, idx, "softmax")[0])
        print("captured")
    """)
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_fp8_matmul_empty(ops):
    w, ws = weight(1, 64, 128, True)
    q, s = ops.act_quant(activations(1, 4, 128), 128, "ue8m0", E8)
    assert ops.fp8_matmul(q[:0], s[:0], w, ws).shape == (0, 64)
    assert ops.fp8_matmul(q, s, w[:0], ws[:0]).shape == (4, 0)


@pytest.mark.parametrize("m", [3, 200])
def test_fp8_matmul_extreme_scales_and_nan(ops, m):
    """E8M0 from 2^-100 to 2^100 that cancel, a NaN code spoils its row alone,
    a NaN scale (byte 255) its row alone."""
    q, s = ops.act_quant(activations(3, m, 512), 128, "ue8m0", E8)
    w, _ = weight(4, 256, 512, True)
    sa = torch.full((m, 4), 27, dtype=torch.uint8, device="cuda")
    sb = torch.full((2, 4), 227, dtype=torch.uint8, device="cuda")
    y = ops.fp8_matmul(q, sa, w, sb, out_dtype=torch.float32)
    check_product(y, q.double(), w.double().t(), 512)
    q.view(torch.uint8)[1, 300] = 0x7f
    sa[2, 1] = 255
    y2 = ops.fp8_matmul(q, sa, w, sb, out_dtype=torch.float32)
    assert torch.isnan(y2[1:3]).all() and torch.equal(y2[0], y[0]) and torch.equal(y2[3:], y[3:])


@pytest.mark.parametrize("e8", [True, False])
def test_fp8_matmul_leaves_neighbours(ops, e8):
    """Nothing outside the result is written (odd n, one row past the last)."""
    from dsv4_plugin import _lib
    m, n, k = 19, 141, 256
    q, s = ops.act_quant(activations(3, m, k), 128, "ue8m0" if e8 else None, E8 if e8 else None)
    w, ws = weight(4, n, k, e8)
    out = torch.full((m + 2, 160), 7.0, dtype=torch.bfloat16, device="cuda")
    _lib.check(_lib.lib().dsv4_fp8_matmul(q.data_ptr(), k, s.data_ptr(), w.data_ptr(), k, ws.data_ptr(), 0 if e8 else 1, 1,
                                          m, n, k, out[1].data_ptr(), 160, 0, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[1:-1, :n], ops.fp8_matmul(q, s, w, ws))
    out[1:-1, :n] = 7.0
    assert (out == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("e8", [True, False])
@pytest.mark.parametrize("m,n,k", [(1, 256, 128), (16, 130, 1024), (70, 1000, 528), (300, 384, 1000)])
def test_fp8_linear_and_its_gradient(ops, m, n, k, e8, dtype):
    """y and dx against their definitions in 64 bits.  fp32 input takes bf16
    values, so that both sides choose the same codes."""
    w, ws = weight(n, n, k, e8)
    w64 = deq64(w, ws, True)
    x = activations(k, m, k).bfloat16().to(dtype).requires_grad_(True)
    dy = (activations(n + 1, m, n) * 1e-3).bfloat16().to(dtype)
    y = ops.fp8_linear(x, w, ws)
    assert y.dtype == dtype and y.requires_grad
    dx, = torch.autograd.grad(y, x, dy)
    qx, sx, _ = quant64(x.detach(), e8)
    qy, sy, _ = quant64(dy, e8)
    check_product(y.detach(), deq64(qx, sx, False), w64.t(), k, "y")
    check_product(dx, deq64(qy, sy, False), w64, n, "dx")
    with torch.no_grad():
        assert torch.equal(ops.fp8_linear(x, w, ws), y)
    # differences: y is linear in the dequantised rows, dx its slope along any direction
    v = torch.randn(k, device="cuda", dtype=torch.float64)
    h = 2.0 ** -10
    d64 = deq64(qy, sy, False)
    up = (d64 * ((deq64(qx, sx, False) + h * v) @ w64.t())).sum(1)
    dn = (d64 * ((deq64(qx, sx, False) - h * v) @ w64.t())).sum(1)
    slope = (dx.double() * v).sum(1)
    mag = (d64.abs() @ w64.abs()) @ v.abs()
    # dx is within its own bound; the difference loses 2^-52 of the two values over 2 h
    lost = 2.0 ** -50 / h * ((d64.abs() * ((deq64(qx, sx, False).abs() + h * v.abs()) @ w64.abs().t())).sum(1))
    tol = ((n / 32 + 34) * 2.0 ** -23 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * mag + lost
    assert ((up - dn) / (2 * h) - slope).abs().le(tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("e8", [True, False])
@pytest.mark.parametrize("m,n,k", [(1, 2048, 4096), (2, 130, 1), (5, 100, 333), (16, 256, 1000), (17, 4096, 2048),
                                   (33, 127, 3584), (64, 1001, 4104), (64, 20000, 512), (65, 300, 1024), (400, 256, 520)])
def test_fp8_linear_is_its_parts(ops, m, n, k, e8, dtype):
    """Quantisation and product in one launch (up to 64 rows) or two: the bits
    of act_quant and fp8_matmul called one after the other, forward and for
    the gradient; values with a NaN, an infinity and a row of zeros."""
    w, ws = weight(n + k, n, k, e8)
    x = activations(m + k, m, k).to(dtype)
    x[m // 2] = 0
    if k > 10:
        x[0, 3], x[-1, 10] = float("nan"), float("inf")
    dy = activations(m + n, m, n).to(dtype)
    fmt, sd = ("ue8m0", E8) if e8 else (None, None)
    xr = x.clone().requires_grad_(True)
    y = ops.fp8_linear(xr, w, ws)
    dx, = torch.autograd.grad(y, xr, dy)
    same = lambda a, b: torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))  # noqa: E731
    assert same(y.detach(), ops.fp8_matmul(*ops.act_quant(x, 128, fmt, sd), w, ws, out_dtype=dtype))
    assert same(dx, ops.fp8_matmul(*ops.act_quant(dy, 128, fmt, sd), w, ws, trans_b=False, out_dtype=dtype))
    ops.fp8_status()


def test_fp8_linear_shapes(ops):
    w, ws = weight(1, 96, 256, True)
    x = activations(2, 12, 256).bfloat16()
    y = ops.fp8_linear(x, w, ws)
    assert torch.equal(ops.fp8_linear(x.view(3, 4, 256), w, ws).view(12, 96), y)
    assert torch.equal(ops.fp8_linear(x.t().contiguous().t(), w, ws), y)
    assert ops.fp8_linear(x[:0], w, ws).shape == (0, 96)
    x3 = x.view(3, 4, 256).clone().requires_grad_(True)
    ops.fp8_linear(x3, w, ws).sum().backward()                 # an expanded gradient
    g, = torch.autograd.grad(ops.fp8_linear(x3, w, ws), x3, torch.ones(3, 4, 96, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(x3.grad, g)


def test_a_row_does_not_depend_on_its_neighbours(ops):
    """The same rows in a batch of the same size give the same bits; a second
    run too."""
    w, ws = weight(1, 640, 2048, True)
    for m in (8, 100, 600):
        x = activations(m, m, 2048).bfloat16()
        y = ops.fp8_linear(x, w, ws)
        z = x.clone()
        z[1:] = activations(m + 1, m - 1, 2048).bfloat16()
        assert torch.equal(ops.fp8_linear(z, w, ws)[0], y[0])
        assert torch.equal(ops.fp8_linear(x, w, ws), y)


def test_side_stream_and_graph(ops):
    """On a side stream, and captured: two graphs of one call replay with new
    inputs, in turn and one after the other."""
    w, ws = weight(1, 512, 1024, True)
    xs = [activations(i, 48, 1024).bfloat16() for i in range(4)]
    want = [ops.fp8_linear(x, w, ws) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.fp8_linear(xs[1], w, ws)
    side.synchronize()
    assert torch.equal(y, want[1])
    graphs = []
    for _ in range(2):
        buf = xs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.fp8_linear(buf, w, ws)
        graphs.append((g, buf, out))
    for i in (1, 2, 3):
        for j, (g, buf, out) in enumerate(graphs):
            buf.copy_(xs[(i + j) % 4])
            g.replay()
        torch.cuda.synchronize()
        for j, (_, _, out) in enumerate(graphs):
            assert torch.equal(out, want[(i + j) % 4])
    ops.fp8_status()


def test_gradient_in_a_graph(ops):
    w, ws = weight(2, 256, 512, False)
    x = activations(1, 40, 512).bfloat16()
    dy = activations(2, 40, 256).bfloat16()
    xr = x.clone().requires_grad_(True)
    want, = torch.autograd.grad(ops.fp8_linear(xr, w, ws), xr, dy)
    bx, bd = torch.zeros_like(x).requires_grad_(True), torch.zeros_like(dy)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dx, = torch.autograd.grad(ops.fp8_linear(bx, w, ws), bx, bd)
    with torch.no_grad():
        bx.copy_(x)
    bd.copy_(dy)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(dx, want)


def test_shared_expert_from_fp8_linear(ops):
    """The shared expert as a user would write it from the operators, beside
    the routed layer: gate and up, SwiGLU, down; against the oracle, and
    added to the routed output against the plan that fuses it."""
    cfg = S.CFG0
    layer = SyntheticLayer(cfg)
    sh = S.make_shared_expert(cfg, 0)
    dev = {}
    for n in ("w1", "w2", "w3"):
        dev[n] = (torch.from_numpy(sh[n]).cuda().view(F8), torch.from_numpy(sh[n + "s"]).cuda().view(E8))
    x = S.make_tokens(cfg, 3, 24)
    xt = bf16_tensor(x)
    gate, up = ops.fp8_linear(xt, *dev["w1"]).float(), ops.fp8_linear(xt, *dev["w3"]).float()
    h = torch.nn.functional.silu(gate.clamp(max=cfg.swiglu_limit)) * up.clamp(-cfg.swiglu_limit, cfg.swiglu_limit)
    y = ops.fp8_linear(h.bfloat16(), *dev["w2"])
    ref = O.shared_expert(x, O.shared_weights_f32(sh), cfg.swiglu_limit)
    # the layer's own bound against the oracle: 1e-2 of the largest value
    assert np.abs(bf16_to_np(y) - ref).max() <= 1e-2 * np.abs(ref).max()
    w, idx = ops.route_topk(xt, torch.from_numpy(layer.gate_w).cuda(), None, cfg.topk, cfg.score_func, cfg.renormalize)
    nb = ops.shared_slot_bytes(cfg.hidden, cfg.inter)
    slot = ops.pack_shared_expert(*[torch.from_numpy(sh[k]) for k in ("w1", "w1s", "w2", "w2s", "w3", "w3s")], cfg.hidden,
                                  cfg.inter).cuda()
    assert slot.numel() == nb
    args = (cfg.hidden, cfg.inter, cfg.n_experts, cfg.topk, 24, cfg.swiglu_limit, layer.arena)
    plain, fused = ops.MoEPlan(*args), ops.MoEPlan(*args, with_shared=True)
    routed = plain.forward(xt, w, idx, layer.slot_of)
    both = fused.forward(xt, w, idx, layer.slot_of, shared_slot=slot)
    plain.status(), fused.status(), ops.fp8_status()
    got, want = routed.float() + y.float(), both.float()
    assert (got - want).abs().max() <= 1e-2 * want.abs().max()
