"""What follows a tensor besides reverse-mode autograd: forward-mode derivatives and traces must not go past the operators."""

import pytest
import torch
from torch.autograd import forward_ad

from forge_b200 import FusedLinear, native
from forge_b200.fp8 import Fp8Weight, fp8_linear, fp8_matmul, quantize_fp8
from forge_b200.loss import token_logprobs

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.fixture(params=["direct", "python"])
def path(request, monkeypatch):
    monkeypatch.setenv("FORGE_NATIVE_AUTOGRAD", "1" if request.param == "direct" else "0")
    native.reset()
    yield request.param
    monkeypatch.undo()
    native.reset()


def test_forward_mode_is_refused(path):
    """(instead of results whose derivative reads as zero)"""
    x = torch.randn(4, 256, device=DEV)
    t = torch.randint(0, 256, (4,), device=DEV)
    w = Fp8Weight.from_weight(torch.randn(128, 256, device=DEV).bfloat16())
    b = torch.randn(128, device=DEV).bfloat16()
    with forward_ad.dual_level():
        for grad in (False, True):
            d = forward_ad.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x))
            db = forward_ad.make_dual(x.bfloat16().requires_grad_(grad), torch.ones_like(x).bfloat16())
            for call in (lambda: token_logprobs(d, t), lambda: token_logprobs(d, None, top_k=2), lambda: fp8_linear(db, w),
                         lambda: fp8_linear(x.bfloat16(), w, forward_ad.make_dual(b, torch.ones_like(b)))):
                with pytest.raises(RuntimeError):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError):
                    call()
        token_logprobs(x, t), fp8_linear(x.bfloat16(), w)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("shape", [(4,), (2, 3)])
def test_a_trace_holds_the_log_probabilities(path, shape):
    """A traced function computes its results from its inputs (they are not constants of the trace)."""
    x, y = (torch.randn(*shape, 256, device=DEV) for _ in range(2))
    t = torch.randint(0, 256, shape, device=DEV)
    f = torch.jit.trace(lambda v: tuple(token_logprobs(v, t, top_k=3)), (x,), check_trace=False)
    for a, b in zip(f(y), token_logprobs(y, t, top_k=3)):
        assert torch.equal(a, b)


@pytest.mark.filterwarnings("ignore")
def test_8_bit_products_cannot_be_traced(path):
    x = torch.randn(4, 256, device=DEV).bfloat16()
    weight = torch.randn(128, 256, device=DEV).bfloat16()
    w = Fp8Weight.from_weight(weight)
    lin = FusedLinear(256, 128, bias=False).to(DEV).to(torch.bfloat16).train().use_fp8_products()
    for f in (lambda v: fp8_linear(v, w), lambda v: quantize_fp8(v)[1], lambda v: quantize_fp8(v, 128, True)[3], lin,
              lambda v: fp8_matmul(w.codes, w.scales[:, :1].expand(1, 2), w.codes, w.scales) + v[:, :128]):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,), check_trace=False)
    fp8_linear(x, w)


def _strided(t):
    """The same values in memory of another order."""
    return t.detach().t().contiguous().t() if t.dim() == 2 else t.detach()


@pytest.mark.parametrize("hooks", [torch.autograd.graph.save_on_cpu, lambda: torch.autograd.graph.saved_tensors_hooks(_strided, lambda t: t),
                                   lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), _strided)])
def test_saved_tensors_that_come_back_otherwise(path, hooks):
    """Layouts that hooks on saved tensors change: rows become columns, pitches are lost."""
    x = torch.randn(12, 264, device=DEV)
    t = torch.randint(0, 200, (12,), device=DEV)
    w = Fp8Weight.from_weight((torch.randn(392, 264, device=DEV)).bfloat16())       # codes_t: 264 rows of 392, pitch 400
    dy = torch.randn(12, 392, device=DEV).bfloat16()

    def results():
        out = []
        for view in (lambda v: v, lambda v: v[:, 3:250], lambda v: v.view(3, 4, 264)):
            xr = x.clone().requires_grad_(True)
            v = view(xr)
            tt = t.view(v.shape[:-1])
            o = token_logprobs(v, tt, top_k=2)
            out += torch.autograd.grad(o.logprobs.sum() + o.entropy.sum(), xr)
        xr = x.bfloat16().requires_grad_(True)
        return out + list(torch.autograd.grad(fp8_linear(xr, w), xr, dy))

    want = results()
    with hooks():
        got = results()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("wrong", [lambda t: t.cpu(), lambda t: t.to(torch.float64) if t.is_floating_point() else t,
                                   lambda t: t.reshape(-1)[:-1] if t.numel() > 1 else t])
def test_saved_tensors_that_are_something_else_are_refused(path, wrong):
    x = torch.randn(12, 256, device=DEV).requires_grad_(True)
    t = torch.randint(0, 256, (12,), device=DEV)
    w = Fp8Weight.from_weight(torch.randn(128, 256, device=DEV).bfloat16())
    xb = x.detach().bfloat16().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.detach(), wrong):
        out = token_logprobs(x, t)
        y = fp8_linear(xb, w)
        with pytest.raises((RuntimeError, ValueError, IndexError)):
            out.logprobs.sum().backward()
        with pytest.raises((RuntimeError, ValueError, IndexError)):
            y.sum().backward()
