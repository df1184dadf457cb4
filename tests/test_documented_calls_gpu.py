"""Calls of the loss, multi-tensor and 8-bit entry points that their documentation allows and that no other test makes:
argument forms, modes of autograd, the optimizer's surroundings, sizes beyond 32 bits."""

import copy
import io
import math

import pytest
import torch
import torch.distributed as dist
from torch.utils.checkpoint import checkpoint

from forge_b200 import FusedLinear, FusedOptimizerManager, native
from forge_b200.fp8 import Fp8Weight, fp8_linear, fp8_matmul, quantize_fp8
from forge_b200.loss import token_logprobs
from forge_b200.multi_tensor import MultiTensorAdamW, multi_tensor_adamw, multi_tensor_grad_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["direct", "python"])
def path(request, monkeypatch):
    monkeypatch.setenv("FORGE_NATIVE_AUTOGRAD", "1" if request.param == "direct" else "0")
    native.reset()
    yield request.param
    monkeypatch.undo()
    native.reset()


def rows(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g) * 2


def grad_of(x, t, **kw):
    xr = x.detach().requires_grad_(True)
    out = token_logprobs(xr, t, **kw)
    (dx,) = torch.autograd.grad((out.logprobs + 0.5 * out.entropy).sum(), xr)
    return (*(o if o is None else o.detach() for o in out), dx)


def same(a, b):
    assert len(a) == len(b)
    for p, q in zip(a, b):
        assert (p is None and q is None) or torch.equal(p, q)


# ----- loss ------------------------------------------------------------------------------------------
def test_log_probabilities_of_any_shape(path):
    x = rows(24, 777)
    t = torch.randint(0, 777, (24,), device=DEV)
    want = grad_of(x, t, top_k=3)
    for lead in ((2, 12), (2, 3, 4), (24, 1), (1, 1, 24)):
        got = grad_of(x.view(*lead, 777), t.view(lead), top_k=3)
        assert got[0].shape == lead and got[2].shape == (*lead, 3)
        same([g.reshape(w.shape) for g, w in zip(got, want)], want)
    one = grad_of(x[5], t[5], top_k=3)
    assert one[0].shape == () and one[3].shape == (3,)
    same(one, [w[5] for w in want])
    for dt in (torch.int32, torch.int16):
        same(grad_of(x, t.to(dt), top_k=3), want)
    same(grad_of(x, torch.stack([t, t], 1)[:, 0], top_k=3), want)            # strided targets
    none = grad_of(x.view(2, 12, 777)[:, :0], t.view(2, 12)[:, :0], top_k=2)
    assert none[0].shape == (2, 0) and none[2].shape == (2, 0, 2) and none[4].shape == (2, 0, 777)


def test_log_probabilities_in_every_mode(path):
    x, t = rows(9, 1001), torch.randint(0, 1001, (9,), device=DEV)
    want = [o.detach() for o in token_logprobs(x, t, top_k=2)]
    with torch.inference_mode():
        same(token_logprobs(x, t, top_k=2), want)
        same(token_logprobs(x.clone(), t.clone(), top_k=2), want)
    with torch.no_grad():
        same(token_logprobs(x.clone().requires_grad_(True), t, top_k=2), want)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        same(token_logprobs(x, t, top_k=2), want)
    dx = grad_of(x, t)[-1]
    for reentrant in (False, True):
        xr = x.clone().requires_grad_(True)
        out = checkpoint(lambda v: tuple(token_logprobs(v, t)[:2]), xr, use_reentrant=reentrant)
        (out[0] + 0.5 * out[1]).sum().backward()
        assert torch.equal(xr.grad, dx)
    xr = x.clone().requires_grad_(True)
    out = token_logprobs(xr, t)
    loss = (out.logprobs + 0.5 * out.entropy).sum()
    loss.backward(retain_graph=True)
    loss.backward()
    assert torch.equal(xr.grad, 2 * dx)
    x16 = x.bfloat16().requires_grad_(True)                                   # gradients of another type than the results
    (a,) = torch.autograd.grad(token_logprobs(x16, t).logprobs.to(torch.float64).sum(), x16)
    (b,) = torch.autograd.grad(token_logprobs(x16, t).logprobs.sum(), x16)
    assert torch.equal(a, b)


def test_log_probabilities_of_a_group_of_one(path):
    dist.init_process_group("nccl", rank=0, world_size=1, store=dist.HashStore(), device_id=torch.device(DEV, 0))
    try:
        x, t = rows(3, 5, 1000), torch.randint(0, 1000, (3, 5), device=DEV)
        t[1, 2] = -100
        kw = dict(vocab_total=1000, group=dist.group.WORLD)
        for targets, top in ((t, 0), (t, 4), (None, 2), (t.int(), 0)):
            got, want = grad_of(x, targets, top_k=top, temperature=0.7, **kw), grad_of(x, targets, top_k=top, temperature=0.7)
            for a, b in zip(got, want):                                       # (the join is formed in another order)
                assert (a is None and b is None) or (a.shape == b.shape and a.dtype == b.dtype and (a - b).abs().max() < 1e-5)
        empty = grad_of(x[:0], t[:0], top_k=1, **kw)
        assert empty[0].shape == (0, 5) and empty[-1].shape == (0, 5, 1000)
        with pytest.raises(ValueError, match="vocab_total"):
            token_logprobs(x, t, group=dist.group.WORLD)
    finally:
        dist.destroy_process_group()


def test_log_probabilities_beyond_32_bits():
    """More than 2^31 logits, and rows whose pitch takes them there: some of them against the same rows by themselves."""
    vocab, n = 100003, 21504
    x = torch.empty(n, vocab, dtype=torch.bfloat16, device=DEV)
    for i in range(0, n, 4096):
        x[i:i + 4096] = rows(min(4096, n - i), vocab, seed=i).bfloat16()
    t = torch.randint(0, vocab, (n,), device=DEV)
    some = torch.tensor([0, 1, 5000, n - 2, n - 1], device=DEV)
    want = grad_of(x[some], t[some])
    got = grad_of(x, t)
    for a, b in zip(got, want):
        if a is not None:
            # (fewer rows are cut over clusters: sums in another order, 4e-5 of a value; a step of bf16 in the gradient)
            assert ((a[some].double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 8e-5).all()
    del got
    pitch = x.view(-1)[: (n // 4096) * 4096 * vocab].view(-1, 4096 * vocab)[:, :vocab]          # 5 rows, 8e8 elements apart
    near = torch.empty(len(pitch), 100008, dtype=x.dtype, device=DEV)[:, :vocab].copy_(pitch)     # rows on 16-byte boundaries, too
    same(grad_of(pitch, t[:len(pitch)]), grad_of(near, t[:len(pitch)]))


# ----- many tensors -----------------------------------------------------------------------------------
def _lists(seed=0, dtype=torch.float32):
    shapes = [(), (5, 7), (0,), (4096,), (3, 1, 65)]
    g = torch.Generator(device=DEV).manual_seed(seed)
    p = [torch.randn(s, device=DEV, generator=g).to(dtype) for s in shapes]
    gr = [torch.randn(s, device=DEV, generator=g).to(dtype) for s in shapes]
    return p, gr, [torch.zeros_like(v, dtype=torch.float32) for v in p], [torch.zeros_like(v, dtype=torch.float32) for v in p]


def test_lists_of_any_kind(path):
    want = _lists()
    norm = multi_tensor_adamw(*want, max_norm=1.0)
    for kind in (tuple, iter, lambda v: (u for u in v)):
        got = _lists()
        n = multi_tensor_adamw(*(kind(v) for v in got), max_norm=1.0)
        assert torch.equal(n, norm)
        for a, b in zip(got, want):
            same(a, b)
    grads = _lists()[1]
    for kind in (tuple, iter):
        same(multi_tensor_grad_norm(kind(grads), 2.0), multi_tensor_grad_norm(grads, 2.0))
    got = _lists()                                                            # the clip factor by hand
    multi_tensor_adamw(*got, grad_coef=multi_tensor_grad_norm(got[1], 1.0)[1])
    for a, b in zip(got, want):
        same(a, b)
    got = _lists()                                                            # one gradient for two parameters, an expanded one
    got[1][1] = torch.ones((), device=DEV).expand(5, 7)
    multi_tensor_adamw(*got)
    twice = _lists()
    twice[1][1] = torch.ones(5, 7, device=DEV)
    multi_tensor_adamw(*twice)
    for a, b in zip(got, twice):
        same(a, b)


def test_the_optimizer_among_what_torch_puts_around_it(path):
    def make():
        g = torch.Generator().manual_seed(3)
        return [torch.nn.Parameter(torch.randn(n, generator=g).to(DEV)) for n in [(9, 64), (33,)]]

    a, b = make(), make()
    mine, ref = MultiTensorAdamW(a, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(b, lr=1e-2, weight_decay=0.1)
    schedules = [torch.optim.lr_scheduler.LambdaLR(o, lambda s: 1.0 / (1 + s)) for o in (mine, ref)]
    calls = []
    mine.register_step_post_hook(lambda *_: calls.append(1))
    for step in range(3):
        def closure(ps):
            for i, p in enumerate(ps):
                p.grad = torch.full_like(p, 0.1 * (i + 1 + step))
            return torch.tensor(float(step))
        assert float(mine.step(lambda: closure(a))) == step == float(ref.step(lambda: closure(b)))
        for s in schedules:
            s.step()
        mine.zero_grad(set_to_none=step % 2 == 0)
    assert calls == [1, 1, 1]
    for p, q in zip(a, b):
        assert (p - q).abs().max() < 1e-6
    # through a file, to the host and back
    f = io.BytesIO()
    torch.save(mine.state_dict(), f)
    f.seek(0)
    c = make()
    other = MultiTensorAdamW(c, lr=7.0)
    other.load_state_dict(torch.load(f, map_location="cpu", weights_only=True))
    for p, q in zip(a, c):
        for k, v in mine.state[p].items():
            u = other.state[q][k]
            assert (u == v) if k == "step" else (torch.equal(u, v) and u.device == v.device)
    scaler = torch.amp.GradScaler("cuda")                                     # a step with infinite gradients is left out
    before = [p.detach().clone() for p in a]
    for p in a:
        p.grad = torch.full_like(p, math.inf)
    scaler.scale(torch.zeros((), device=DEV))
    scaler.step(mine)
    scaler.update()
    for p, q in zip(a, before):
        assert torch.equal(p, q)


# ----- 8-bit products ---------------------------------------------------------------------------------
def test_8_bit_linears_of_any_shape(path):
    w = rows(200, 272, seed=1).bfloat16()
    w8 = Fp8Weight.from_weight(w)
    x = rows(24, 272, seed=2).bfloat16()
    dy = rows(24, 200, seed=3).bfloat16()

    def both(v, g, bias=None):
        v = v.detach().requires_grad_(True)
        y = fp8_linear(v, w8, bias)
        (dx,) = torch.autograd.grad(y, v, g)
        return y.detach(), dx

    want = both(x, dy)
    for lead in ((2, 12), (2, 3, 4), (24, 1)):
        y, dx = both(x.view(*lead, 272), dy.view(*lead, 200))
        assert y.shape == (*lead, 200) and dx.shape == (*lead, 272)
        same((y.view(24, 200), dx.view(24, 272)), want)
    same(both(x[3], dy[3]), [fp8_linear(x[3:4], w8)[0], both(x[3:4], dy[3:4])[1][0]])
    same(both(torch.cat([x, x], 1)[:, :272], torch.cat([dy, dy], 1)[:, 200:]), want)         # rows of a wider pitch
    same(both(x.t().contiguous().t(), dy.t().contiguous().t()), want)
    y, dx = both(x[:0], dy[:0])
    assert y.shape == (0, 200) and dx.shape == (0, 272)
    y, dx = both(x.view(2, 12, 272)[:, :0], dy.view(2, 12, 200)[:, :0])
    assert y.shape == (2, 0, 200) and dx.shape == (2, 0, 272)
    (dx,) = torch.autograd.grad(fp8_linear(v := x.clone().requires_grad_(True), w8).sum(), v)    # an expanded gradient
    same((dx,), both(x, torch.ones_like(dy))[1:])
    b = torch.ones(200, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    y = fp8_linear(x, w8, b)                                                   # only the bias has a gradient
    y.backward(dy)
    assert torch.equal(y.detach(), want[0] + 1) and torch.equal(b.grad, dy.sum(0))
    with torch.inference_mode():
        assert torch.equal(fp8_linear(x, w8), want[0])
        fresh = Fp8Weight.from_weight(w).update_(w)
        assert torch.equal(fp8_linear(x.clone(), fresh), want[0])
    for reentrant in (False, True):
        v = x.clone().requires_grad_(True)
        checkpoint(lambda u: fp8_linear(u, w8), v, use_reentrant=reentrant).backward(dy)
        assert torch.equal(v.grad, want[1])


def test_8_bit_weights_of_any_form(path):
    w = rows(130, 200, seed=4)
    for weight in (w, torch.nn.Parameter(w), w.t().contiguous().t(), torch.cat([w, w], 1)[:, :200]):
        w8 = Fp8Weight.from_weight(weight)
        for a, b in zip((w8.codes, w8.scales, w8.codes_t, w8.scales_t), quantize_fp8(w, 128, True)):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        assert tuple(w8.shape) == (130, 200)
    plain = Fp8Weight.from_weight(w, transposed=False)
    assert plain.codes_t is None
    x = rows(5, 200).bfloat16()
    assert torch.equal(fp8_linear(x, plain), fp8_linear(x, w8))
    with pytest.raises(ValueError, match="transposed"):
        fp8_linear(x.requires_grad_(True), plain)
    with torch.no_grad():
        fp8_linear(x, plain)
    for bad in (w[:129], w[:, :199], w.cpu()):
        with pytest.raises((ValueError, RuntimeError)):
            w8.update_(bad)
    for bad in (x[:, :199], x.float(), x.detach()[:, :0]):
        with pytest.raises(ValueError):
            fp8_linear(bad, w8)
    with pytest.raises((ValueError, RuntimeError)):
        fp8_linear(x.detach().cpu(), w8)
    same((fp8_matmul(*quantize_fp8(x.detach()), w8.codes, w8.scales),), (fp8_linear(x.detach(), w8),))


@pytest.mark.parametrize("optimizer,mode", [("adamw", "bf16"), ("adamw", "int8"), ("adamw", "fp8_block"), ("sgd", None), ("lion", None)])
def test_8_bit_products_under_every_optimizer_and_accumulation(optimizer, mode):
    """Two micro-steps a step, grouped and not: the same weights."""
    results = []
    for grouped in (False, True):
        torch.manual_seed(6)
        kw = {} if mode is None else dict(state_mode=mode)
        net = torch.nn.Sequential(FusedLinear(128, 256, optimizer_type=optimizer, **kw), torch.nn.SiLU(),
                                  FusedLinear(256, 64, optimizer_type=optimizer, **kw)).to(DEV).to(torch.bfloat16).train()
        manager = FusedOptimizerManager(net, gradient_accumulation_steps=2).use_fp8_products()
        if grouped:
            manager.group_updates("layer")
        start = copy.deepcopy([p.detach() for p in net.parameters()])
        for micro in range(4):
            manager.pre_step(lr=1e-2)
            net(rows(40, 128, seed=micro).bfloat16()).float().square().mean().backward()
        manager.flush_updates()
        for p, q in zip(net.parameters(), start):
            assert p.isfinite().all() and not torch.equal(p, q) and p.grad is None
        results.append([p.detach() for p in net.parameters()])
    same(*results)


def test_a_tensor_beyond_32_bits_is_updated_to_its_end():
    n = 2 ** 31 + 2 ** 20 + 64 * 5 + 3
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEV)
    m, v = (torch.zeros(n, dtype=torch.int8, device=DEV) for _ in range(2))
    ms, vs = (torch.ones(-(-n // 64), device=DEV) for _ in range(2))
    cuts = [(0, 6400), (2 ** 31 - 640, 2 ** 31 + 640), (n - 64 * 4 - n % 64, n)]
    for i, (a, b) in enumerate(cuts):
        p[a:b], g[a:b] = rows(b - a, seed=i).bfloat16(), rows(b - a, seed=i + 7).bfloat16()
    parts = [[t[a:b].clone() for t in (p, g, m, v)] + [s[a // 64:-(-b // 64)].clone() for s in (ms, vs)] for a, b in cuts]
    norm, coef = multi_tensor_grad_norm([g], 1.0)
    exact = math.sqrt(sum(float(g[i:i + 2 ** 28].double().square().sum()) for i in range(0, n, 2 ** 28)))
    assert abs(float(norm) - exact) <= 2.0 ** -21 * exact
    multi_tensor_adamw([p], [g], [m], [v], [ms], [vs], grad_coef=coef, lr=1e-2)
    multi_tensor_adamw(*([q[i] for q in parts] for i in range(6)), grad_coef=coef, lr=1e-2)
    for (a, b), q in zip(cuts, parts):
        same([t[a:b] for t in (p, g, m, v)] + [s[a // 64:-(-b // 64)] for s in (ms, vs)], q)
    inner = p[10 ** 9:10 ** 9 + 64]
    assert (inner == inner[0]).all() and inner[0] != 0


def test_8_bit_products_beyond_32_bits():
    """More than 2^31 codes of activations."""
    tokens, n, k = 2 ** 20 + 2 ** 17 + 77, 136, 2048
    x = torch.zeros(tokens, k, dtype=torch.bfloat16, device=DEV)
    some = torch.tensor([0, 5, 2 ** 20 - 1, 2 ** 20, tokens - 200, tokens - 1], device=DEV)
    x[some] = rows(6, k, seed=8).bfloat16()
    w8 = Fp8Weight.from_weight(rows(n, k, seed=9).bfloat16())
    y = fp8_linear(x, w8)
    want = fp8_linear(x[some], w8)
    # sums of the same terms in another order: 2^-24 of their absolute values each, and one rounding to bf16 each
    xq, xs = quantize_fp8(x[some])
    value = lambda q, s, r: q.double() * s.double().repeat_interleave(r, 0)[:q.shape[0]].repeat_interleave(128, 1)      # noqa: E731
    size = value(xq, xs, 1).abs() @ value(w8.codes, w8.scales, 128).abs().t()
    assert ((y[some].double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -23 * (131 + 16) * size).all()
    y[some] = 0
    assert (y == 0).all()
