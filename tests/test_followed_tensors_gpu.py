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
