"""What the operators' autograd functions answer beyond a first derivative,
on the CPU: a stand-in for the library accepts every call, so only the Python
side runs.  Needs no GPU."""

import pytest
import torch

from dsv4_plugin import ops


class FakeLibrary:
    """Every entry point returns DSV4_OK; sizes are generous."""

    def __getattr__(self, name):
        return (lambda *a: 4096) if name.endswith("_bytes") else (lambda *a: 0)


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    fake = FakeLibrary()
    monkeypatch.setattr(ops, "lib", lambda: fake)
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)


def router_batch(strided=False):
    logits = torch.zeros(6, 16)[:, :8] if strided else torch.zeros(6, 8)
    return logits.requires_grad_(True), torch.zeros(6, 2, dtype=torch.int32)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("constant", [True, False])
def test_balance_loss_refuses_a_second_derivative(strided, constant):
    """The gradient depends on the logits, also where the upstream gradient is
    a constant: differentiating it raises instead of leaving the term out."""
    logits, idx = router_batch(strided)
    loss, _ = ops.balance_loss(logits, idx)
    scale = 1.0 if constant else torch.ones((), requires_grad=True)
    with pytest.raises(RuntimeError, match="once"):
        g, = torch.autograd.grad((logits ** 2).sum() + scale * loss, logits, create_graph=True)
        g.pow(2).sum().backward()


@pytest.mark.parametrize("strided", [False, True])
def test_balance_loss_first_derivative_under_create_graph(strided):
    """A graph of the first derivative that nobody differentiates is no error."""
    logits, idx = router_batch(strided)
    loss, _ = ops.balance_loss(logits, idx)
    g, = torch.autograd.grad((logits ** 2).sum() + loss, logits, create_graph=True)
    assert g.shape == logits.shape and g.requires_grad
    loss, _ = ops.balance_loss(logits, idx)
    loss.backward()
    assert logits.grad.shape == logits.shape and not logits.grad.requires_grad


def fp8_layer(n=16, k=128):
    w = torch.zeros(n, k, dtype=torch.uint8).view(torch.float8_e4m3fn)
    return w, torch.ones((n + 127) // 128, 1)


@pytest.mark.parametrize("grad", [True, False])
def test_fp8_linear_refuses_forward_mode(grad):
    """A tangent is refused, not dropped, whether or not x requires a gradient."""
    from torch.autograd import forward_ad
    w, s = fp8_layer()
    x = torch.zeros(3, 128, requires_grad=grad)
    with forward_ad.dual_level():
        assert ops.fp8_linear(x, w, s).shape == (3, 16)        # no tangent: as outside
        with pytest.raises(RuntimeError, match="forward"):
            ops.fp8_linear(forward_ad.make_dual(x, torch.ones(3, 128)), w, s)
        with pytest.raises(RuntimeError, match="forward"):
            ops.fp8_linear(x, w, forward_ad.make_dual(s, torch.ones_like(s)))


@pytest.mark.parametrize("shape", [(3, 128), (2, 3, 128), (0, 128)])
def test_fp8_linear_with_an_empty_weight(shape):
    """No output columns: the gradient of x is a sum over nothing."""
    w, s = fp8_layer(0)
    x = torch.ones(shape, requires_grad=True)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(ops, "lib", lambda: pytest.fail("an empty product calls no kernel"))
        y = ops.fp8_linear(x, w, s)
        assert y.shape == (*shape[:-1], 0)
        dx, = torch.autograd.grad(y, x, torch.zeros_like(y))
    assert dx.shape == x.shape and dx.dtype == x.dtype and not dx.any()
