"""The loss, the rest optimizer and the 8-bit products together with the fused linears, as a training step uses them."""

import copy

import pytest
import torch
import torch.distributed as dist
import torch.nn as nn
import torch.nn.functional as F

from forge_b200 import FusedLinear, FusedOptimizerManager, OptimizerConfig
from forge_b200 import kernel as K
from forge_b200.fp8 import Fp8Weight, fp8_linear
from forge_b200.loss import token_logprobs
from forge_b200.multi_tensor import MultiTensorAdamW, multi_tensor_adamw

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB, HID, TOKENS = 1000, 256, 130


class Block(nn.Module):
    def __init__(self, linear):
        super().__init__()
        self.gamma = nn.Parameter(torch.ones(HID, dtype=torch.bfloat16))
        self.up, self.down = linear(HID, 2 * HID), linear(2 * HID, HID)

    def forward(self, h):
        x = F.rms_norm(h.float(), (HID,)).to(h.dtype) * self.gamma
        return h + self.down(F.silu(self.up(x)))


class Net(nn.Module):
    def __init__(self, linear):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, HID, dtype=torch.bfloat16)
        self.blocks = nn.ModuleList([Block(linear) for _ in range(2)])
        self.head = linear(HID, VOCAB)

    def forward(self, ids):
        h = self.embed(ids)
        for b in self.blocks:
            h = b(h)
        return self.head(h)


def fused(i, o):
    return FusedLinear(i, o, optimizer_type="adamw", state_mode="int8", weight_decay=0.01).to(torch.bfloat16)


def plain(i, o):
    return nn.Linear(i, o, bias=False, dtype=torch.bfloat16)


def make(seed=0):
    torch.manual_seed(seed)
    a = Net(fused).to(DEV).train()
    with torch.no_grad():
        for p in a.parameters():
            if p.dim() == 2:
                p.normal_(0.0, 0.05)
    b = Net(plain).to(DEV)
    b.load_state_dict(a.state_dict())
    return a, b


def batch(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, VOCAB, (2, TOKENS), device=DEV, generator=g)


def loss_of(model, ids):
    out = token_logprobs(model(ids)[:, :-1], ids[:, 1:])
    return -out.logprobs.mean() - 0.01 * out.entropy.mean()


@pytest.mark.parametrize("fp8", [False, True])
def test_gradients_of_the_rest(fp8):
    """Against the same network on torch's own linears and loss.  bf16: some ten tensors on the way are rounded to half a
    step, 2^-8 relative at most: 3 %.  fp8: twelve operands of six products are rounded to e4m3 besides, 2^-4 at most and a
    quarter of that in the mean square, independently: sqrt(12) / 64 + 3 % = 9 %, and twice that for the tail."""
    a, b = make()
    m = FusedOptimizerManager(a).group_updates("layer")
    if fp8:
        m.use_fp8_products()
    ids = batch(1)
    m.pre_step(lr=1e-3)
    loss_of(a, ids).backward()
    logits = b(ids)[:, :-1].float().reshape(-1, VOCAB)
    lp = torch.log_softmax(logits, -1)
    ref = F.nll_loss(lp, ids[:, 1:].reshape(-1)) + 0.01 * (lp.exp() * lp).sum(-1).mean()
    ref.backward()
    for (n, p), q in zip(a.named_parameters(), b.parameters()):
        if isinstance(dict(a.named_modules())[n.rsplit(".", 1)[0]], FusedLinear):
            assert p.grad is None and not torch.equal(p, q), n            # updated on the way
            continue
        rel = (p.grad.double() - q.grad.double()).norm() / q.grad.double().norm()
        assert rel < (0.18 if fp8 else 0.03), (n, float(rel))


@pytest.mark.parametrize("fp8", [False, True])
def test_eager_steps_equal_graph_replays(fp8):
    nets = [make(2)[0] for _ in range(2)]
    managers = [FusedOptimizerManager(n).group_updates("layer") for n in nets]
    opts = [MultiTensorAdamW(m.get_non_fused_params(), lr=1e-3, state_mode="int8", max_grad_norm=0.5) for m in managers]
    if fp8:
        for m in managers:
            m.use_fp8_products()
    for m in managers:
        m.enable_device_hyper()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = torch.zeros(2, TOKENS, dtype=torch.long, device=DEV)

    def step(i):
        loss = loss_of(nets[i], static)
        loss.backward()
        opts[i].step()
        opts[i].zero_grad(set_to_none=True)
        return loss.detach()

    with torch.cuda.stream(side):
        for i in range(2):                              # one eager step allocates the states
            static.copy_(batch(10))
            managers[i].pre_step(lr=1e-3)
            step(i)
        for o in opts:
            o.enable_device_hyper()
        graph = torch.cuda.CUDAGraph()
        managers[1].pre_step(lr=1e-3)
        opts[1].pre_step()
        static.copy_(batch(11))
        with torch.cuda.graph(graph, stream=side):
            captured = step(1)
        for k in range(3):
            static.copy_(batch(11 + k))
            lr = 1e-3 * (k + 1)
            for o in opts:
                o.param_groups[0]["lr"] = lr
            if k:
                managers[1].pre_step(lr=lr)
                opts[1].pre_step()
            graph.replay()
            managers[0].pre_step(lr=lr)
            opts[0].pre_step()
            eager = step(0)
            assert torch.equal(eager, captured)
    torch.cuda.current_stream().wait_stream(side)
    for (n, p), q in zip(nets[0].named_parameters(), nets[1].parameters()):
        assert torch.equal(p, q), n


def test_first_replay_uses_the_captured_steps_rate():
    """(the graph above is first replayed with the hyper-parameters that pre_step wrote before the capture)"""
    p = torch.nn.Parameter(torch.ones(100, device=DEV))
    q = torch.nn.Parameter(torch.ones(100, device=DEV))
    p.grad, q.grad = torch.ones(100, device=DEV), torch.ones(100, device=DEV)
    a, b = MultiTensorAdamW([p], lr=1e-2).enable_device_hyper(), MultiTensorAdamW([q], lr=1e-2)
    a.pre_step()
    a.step()
    b.step()
    assert torch.equal(p, q) and a.state[p]["step"] == 1
    sd = copy.deepcopy(a.state_dict())
    c = MultiTensorAdamW([torch.nn.Parameter(p.detach().clone())], lr=1.0)
    c.load_state_dict(sd)
    assert c.state[c.param_groups[0]["params"][0]]["step"] == 1


@pytest.mark.parametrize("bias", [False, True])
def test_fp8_products_of_a_fused_linear(bias):
    torch.manual_seed(4)
    lin = FusedLinear(272, 392, bias=bias).to(DEV).to(torch.bfloat16).train()
    x = torch.randn(3, 37, 272, device=DEV).bfloat16().requires_grad_(True)
    dy = (torch.randn(3, 37, 392, device=DEV) * 0.1).bfloat16()
    w0 = lin.weight.detach().clone()
    lin.use_fp8_products()
    xr = x.detach().clone().requires_grad_(True)
    want = fp8_linear(xr, Fp8Weight.from_weight(w0), lin.bias)
    (dx,) = torch.autograd.grad(want, xr, dy)
    y = lin(x)                                        # no config yet: a plain linear's gradients
    y.backward(dy)
    assert torch.equal(y, want) and torch.equal(x.grad, dx)
    dw = dy.reshape(-1, 392).t() @ x.detach().reshape(-1, 272)
    assert torch.equal(lin.weight.grad, dw)
    lin.weight.grad = None
    # with one: the weight is updated from the bf16 operands, the input gradient is that of the weight before
    x.grad = None
    lin.update_optimizer_config(OptimizerConfig(lr=1e-2))
    lin(x).backward(dy)
    w1, m, v = w0.clone(), torch.zeros_like(w0), torch.zeros_like(w0)
    K.fused_grad_adamw(dy.reshape(-1, 392), x.detach().reshape(-1, 272), w1, m, v, lr=1e-2, step=1)
    assert torch.equal(lin.weight, w1) and torch.equal(x.grad, dx)
    # the next forward quantises the new weight
    assert torch.equal(lin(x), fp8_linear(x.detach(), Fp8Weight.from_weight(w1), lin.bias))
    assert torch.equal(lin.eval()(x), F.linear(x, lin.weight, lin.bias))
    lin.train()
    with pytest.raises(ValueError):
        lin(x.float())
    with pytest.raises(ValueError):
        FusedLinear(64, 64).half().use_fp8_products()


def test_fp8_products_of_a_row_sharded_linear_take_the_plain_path():
    """The forms that fuse a collective into the GEMM multiply the weight as it is: a linear with 8-bit products has none."""
    from forge_b200.tensor_parallel import RowShardedFusedLinear, RowShardedLinearSet
    x = torch.zeros(2, 32, device=DEV, dtype=torch.bfloat16)
    lin = RowShardedFusedLinear(64, 64, rank=0, world=2, dtype=torch.bfloat16, device=DEV, bias=False).train()
    part = RowShardedFusedLinear(64, 64, rank=0, world=2, gather_input=False, dtype=torch.bfloat16, device=DEV, bias=False).train()
    both = RowShardedLinearSet([part])
    both.attach_fused_scatter(object(), 0)            # only asked for by what runs fused
    lin.attach_fused_gather(object(), 0)
    for m in (lin, part):
        m.local.update_optimizer_config(OptimizerConfig(lr=1e-3))
    assert lin.returns_full_output(x) and both.fused(x)
    for m in (lin, part):
        m.local.use_fp8_products()
    assert not lin.returns_full_output(x) and not both.fused(x)


def test_calls_from_several_threads_and_streams():
    import threading
    torch.manual_seed(9)
    x = torch.randn(70, 33000, device=DEV).bfloat16()
    t = torch.randint(0, 33000, (70,), device=DEV)
    w = torch.randn(1000, 512, device=DEV).bfloat16()
    a = [torch.randn(n, 512, device=DEV).bfloat16() for n in (1, 40, 700)]
    g = [torch.randn(n, device=DEV) for n in (5, 4096, 100000)]

    def work():
        out = []
        for _ in range(6):
            xr = x.detach().requires_grad_(True)
            o = token_logprobs(xr, t, top_k=5)
            out += [*o, torch.autograd.grad(o.logprobs.sum() + o.entropy.sum(), xr)[0]]
            w8 = Fp8Weight.from_weight(w)
            out += [fp8_linear(v, w8) for v in a]
            p, m, v = ([torch.zeros_like(u) for u in g] for _ in range(3))
            out.append(multi_tensor_adamw(p, g, m, v, max_norm=1.0))
            out += p
        return [o.detach() for o in out]

    want = work()
    torch.cuda.synchronize()
    results = {}

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            results[i] = work()
        s.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert len(results) == 4
    for got in results.values():
        assert len(got) == len(want) and all(torch.equal(p, q) for p, q in zip(got, want))


def test_sharded_loss_of_one_rank_equals_the_torch_ops():
    from examples.tp_model import _VocabParallelCrossEntropy, library_cross_entropy
    dist.init_process_group("nccl", rank=0, world_size=1, store=dist.HashStore(), device_id=torch.device(DEV, 0))
    try:
        x = (torch.randn(77, 2048, device=DEV) * 3).bfloat16().requires_grad_(True)
        t = torch.randint(0, 2048, (77,), device=DEV)
        a = _VocabParallelCrossEntropy.apply(x, t, 0, dist.group.WORLD)
        (ga,) = torch.autograd.grad(a, x)
        b = library_cross_entropy(x, t, 0, 2048, None)
        (gb,) = torch.autograd.grad(b, x)
        assert abs(float(a.detach()) - float(b.detach())) < 1e-5 * abs(float(a.detach()))
        # the torch form rounds once to bf16 as the kernel does, from another fp32 value: one step at most
        assert ((ga.double() - gb.double()).abs() <= 2.0 ** -7 * ga.double().abs() + 1e-9).all()
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("bias", [False, True])
def test_fp8_products_of_an_fp32_linear(bias):
    """fp32 weight and bias, bf16 activations: the output is bf16 as the activations are (the bias added in fp32, one
    rounding), the weight's gradient and update come from the bf16 operands."""
    torch.manual_seed(5)
    lin = FusedLinear(272, 392, bias=bias).to(DEV).train().use_fp8_products()
    x = torch.randn(37, 272, device=DEV).bfloat16().requires_grad_(True)
    dy = (torch.randn(37, 392, device=DEV) * 0.1).bfloat16()
    w0 = lin.weight.detach().clone()
    y = lin(x)
    assert y.dtype == torch.bfloat16
    product = fp8_linear(x.detach(), Fp8Weight.from_weight(w0))
    assert torch.equal(y, product if not bias else (product.float() + lin.bias).bfloat16())
    y.backward(dy)
    xr = x.detach().clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(fp8_linear(xr, Fp8Weight.from_weight(w0)), xr, dy)
    assert torch.equal(x.grad, dx)
    want = dy.double().t() @ x.detach().double()
    # a sum of 37 exact products in fp32, rounded to bf16 at most
    assert lin.weight.grad.dtype == torch.float32
    bound = 2.0 ** -8 * want.abs() + 37 * 2.0 ** -24 * (dy.double().abs().t() @ x.detach().double().abs())
    assert ((lin.weight.grad.double() - want).abs() <= bound).all()
    if bias:
        want = dy.double().sum(0)
        assert lin.bias.grad.dtype == torch.float32
        assert ((lin.bias.grad.double() - want).abs() <= 37 * 2.0 ** -24 * dy.double().abs().sum(0)).all()
    # the update, fused and with the gradient accumulated before it
    lin.weight.grad = x.grad = None
    lin.update_optimizer_config(OptimizerConfig(lr=1e-2))
    lin(x).backward(dy)
    w1, m, v = w0.clone(), torch.zeros_like(w0), torch.zeros_like(w0)
    st = lin._state
    K.fused_grad_adamw(dy, x.detach(), w1, m.to(st.m.dtype), v.to(st.v.dtype), lr=1e-2, step=1)
    assert torch.equal(lin.weight, w1) and not torch.equal(w1, w0) and torch.equal(x.grad, dx)
    lin.set_accumulating(True)
    lin(x).backward(dy)
    lin.set_accumulating(False)
    lin(x).backward(dy)
    assert lin.weight.isfinite().all() and not torch.equal(lin.weight, w1)
