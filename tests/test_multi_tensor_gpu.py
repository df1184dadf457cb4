"""AdamW over lists of tensors: moments, codes and scales bit for bit against the oracle (fp32 and bf16 moments) or fp32
operations in the definition's order (8-bit moments), weights within the oracle's bar; the common
norm against 64 bits; the optimizer class against the function, torch.optim and itself after a checkpoint."""

import copy
import math

import numpy as np
import pytest
import torch

import oracle
from forge_b200 import _lib
from forge_b200 import kernel as K
from forge_b200.multi_tensor import MultiTensorAdamW, multi_tensor_adamw, multi_tensor_grad_norm

from tests.util import assert_bits_equal, assert_w_close, np32

pytestmark = pytest.mark.gpu
DEV = "cuda"
HP = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3)
CODE = {"int8": torch.int8, "fp8_block": torch.float8_e4m3fn}


def make(sizes, mode, pdt, gdt, seed=0, offset=0):
    """CPU tensors of the given sizes and their CUDA copies; `offset` elements of misalignment for param and grad."""
    g = torch.Generator().manual_seed(seed)

    def dev(t):
        if not offset:
            return t.to(DEV)
        big = torch.zeros(t.numel() + offset, dtype=t.dtype, device=DEV)
        big[offset:] = t.reshape(-1).to(DEV)
        return big[offset:].view(t.shape)

    out = []
    for n in sizes:
        p = (torch.randn(n, generator=g) * 0.02).to(pdt)
        gr = (torch.randn(n, generator=g) * 1e-2).to(gdt)
        num = math.prod(n)
        d = dict(p=p, g=gr)
        if mode in CODE:
            b = -(-num // 64)
            if mode == "int8":
                d["m"] = torch.randint(-127, 128, n, generator=g).to(torch.int8)
                d["v"] = torch.randint(0, 128, n, generator=g).to(torch.int8)
            else:
                d["m"] = (torch.randn(n, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
                d["v"] = (torch.randn(n, generator=g).abs() * 100).clamp(0, 448).to(torch.float8_e4m3fn)
            d["ms"] = torch.rand(b, generator=g) * 1e-4 + 1e-6
            d["vs"] = torch.rand(b, generator=g) * 1e-6 + 1e-8
        else:
            sdt = torch.float32 if mode == "f32" else torch.bfloat16
            d["m"] = (torch.randn(n, generator=g) * 1e-3).to(sdt)
            d["v"] = (torch.randn(n, generator=g).square() * 1e-5).to(sdt)
        out.append((d, {k: dev(t) if k in "pgmv" else t.to(DEV) for k, t in d.items()}))
    return out


def call(items, mode, **kw):
    quant = mode in CODE
    return multi_tensor_adamw([d["p"] for d in items], [d["g"] for d in items], [d["m"] for d in items], [d["v"] for d in items],
                              [d["ms"] for d in items] if quant else None, [d["vs"] for d in items] if quant else None,
                              **{**HP, **kw})


def expect(d, mode, coef=1.0):
    """The oracle's step on one tensor, the last block filled up with zeros."""
    h = oracle.Hyper(**HP)
    n = d["p"].numel()
    g = (d["g"].float() * coef).reshape(-1)
    wb = d["p"].dtype == torch.bfloat16
    if mode not in CODE:
        w, m, v = np32(d["p"]).reshape(-1).copy(), np32(d["m"]).reshape(-1).copy(), np32(d["v"]).reshape(-1).copy()
        oracle.adamw(w, m, v, np32(g), h, w_bf16=wb, s_bf16=mode == "bf16")
        return dict(p=w, m=m, v=v)
    # 8-bit moments: fp32 operations, each rounded once, over blocks of 64 elements in memory order
    f = np.float32
    b = -(-n // 64)

    def pad(t):
        out = np.zeros(b * 64, dtype=f)
        out[:n] = t.float().reshape(-1).numpy()
        return out.reshape(b, 64)

    live = (np.arange(b * 64) < n).reshape(b, 64)
    gr, ms, vs = pad(g), d["ms"].numpy()[:, None], d["vs"].numpy()[:, None]
    m, v = pad(d["m"]) * ms, np.maximum(pad(d["v"]) * vs, f(1e-8))
    m = f(h.c.beta1) * m + f(h.c.one_m_beta1) * gr
    v = f(h.c.beta2) * v + (f(h.c.one_m_beta2) * gr) * gr
    top = 127 if mode == "int8" else 448
    out = {}
    for k, x in (("m", m * live), ("v", v * live)):
        scale = np.abs(x).max(1, keepdims=True) * f(1 / top) + f(1e-12)
        q = torch.from_numpy(x / scale)
        q = q.round().clamp(-127, 127).to(torch.int8) if mode == "int8" else q.clamp(-448, 448).to(torch.float8_e4m3fn)
        out[k], out[k + "s"] = q.view(torch.uint8).reshape(-1)[:n].numpy(), scale.reshape(-1)
    w = pad(d["p"]).astype(np.float64)
    up = (m.astype(np.float64) / h.c.bc1) / (np.sqrt(v.astype(np.float64) / h.c.bc2) + h.c.eps)
    w = w * h.c.decay - h.c.lr * up
    out["p"] = w.astype(f).reshape(-1)[:n]
    return out


def verify(pairs, mode, coef=1.0):
    for i, (cpu, dev) in enumerate(pairs):
        e = expect(cpu, mode, coef)
        for k in ("m", "v"):
            got = dev[k].reshape(-1)
            assert_bits_equal(e[k], got.view(torch.uint8) if mode in CODE else got, f"tensor {i}: {k}")
        if mode in CODE:
            assert_bits_equal(e["ms"], dev["ms"], f"tensor {i}: m scale")
            assert_bits_equal(e["vs"], dev["vs"], f"tensor {i}: v scale")
        assert_w_close(e["p"], dev["p"].reshape(-1), cpu["p"].reshape(-1))


SIZES = [(1,), (7,), (64,), (65, 3), (4096,), (130, 64), (5, 5, 5), (2049,), (40, 1025)]


@pytest.mark.parametrize("mode", ["f32", "bf16", "int8", "fp8_block"])
@pytest.mark.parametrize("pdt,gdt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                     (torch.float32, torch.bfloat16), (torch.float32, torch.float32)])
def test_against_the_oracle(mode, pdt, gdt):
    pairs = make(SIZES, mode, pdt, gdt, seed=1)
    call([d for _, d in pairs], mode)
    verify(pairs, mode)


@pytest.mark.parametrize("mode", ["f32", "int8"])
@pytest.mark.parametrize("offset", [1, 3])
def test_tensors_that_start_anywhere(mode, offset):
    pairs = make(SIZES, mode, torch.bfloat16, torch.bfloat16, seed=2, offset=offset)
    guard = [(d["p"]._base[:offset].clone(), d["p"]._base) for _, d in pairs]
    call([d for _, d in pairs], mode)
    verify(pairs, mode)
    for before, base in guard:
        assert torch.equal(before, base[:offset])


def test_more_tensors_than_a_launch_holds_and_mixed_types():
    sizes = [((i * 37) % 300 + 1,) for i in range(1000)]
    pairs = make(sizes[:500], "f32", torch.bfloat16, torch.bfloat16, seed=3) + make(sizes[500:], "f32", torch.float32, torch.float32, seed=4)
    order = torch.randperm(1000, generator=torch.Generator().manual_seed(5)).tolist()
    pairs = [pairs[i] for i in order]
    call([d for _, d in pairs], "f32")
    verify(pairs, "f32")


@pytest.mark.parametrize("mode", ["bf16", "int8", "fp8_block"])
def test_against_the_single_tensor_operator(mode):
    """bf16 moments: the same bits.  8-bit moments: a scale is at most one ulp (2^-23) apart, which moves a quotient of up to
    127 (or a code's place among the 16 steps of its binade) by 1.5e-5 (2e-6): that share of the codes, with a wide margin,
    may round to the neighbouring one."""
    (a, dev), = make([(2000, 512)], mode, torch.bfloat16, torch.bfloat16, seed=6)
    one = {k: t.to(DEV) for k, t in a.items()}
    call([dev], mode)
    if mode == "bf16":
        K.optimizer_only_adamw(one["g"], one["p"], one["m"], one["v"], **HP)
        assert all(torch.equal(dev[k], one[k]) for k in dev)
        return
    fn = K.optimizer_only_adamw_int8state if mode == "int8" else K.optimizer_only_adamw_fp8block
    fn(one["g"], one["p"], one["m"], one["v"], one["ms"].view(2000, 8), one["vs"].view(2000, 8), **HP)
    assert torch.equal(dev["p"], one["p"])
    for k in ("ms", "vs"):
        assert ((dev[k] - one[k]).abs() <= one[k] * 2.0 ** -23).all()
    for k in ("m", "v"):
        x, y = dev[k].view(torch.int8).int(), one[k].view(torch.int8).int()
        assert (x - y).abs().max() <= 1 and (x != y).float().mean() < 1e-3


def test_large_tensor_several_passes_per_chunk():
    (cpu, dev), = make([(4001, 33000)], "int8", torch.bfloat16, torch.bfloat16, seed=7)
    call([dev], "int8")
    b = 64 * 1000
    for lo in (0, 4001 * 33000 // 2 // 64 * 64, 4001 * 33000 // 64 * 64 - b):        # slices on block boundaries
        hi = min(lo + b, 4001 * 33000)
        cut = {k: (t.reshape(-1)[lo:hi] if k in "pgmv" else t[lo // 64:-(-hi // 64)]) for k, t in cpu.items()}
        got = {k: (t.reshape(-1)[lo:hi] if k in "pgmv" else t[lo // 64:-(-hi // 64)]) for k, t in dev.items()}
        verify([(cut, got)], "int8")


@pytest.mark.parametrize("gdt", [torch.bfloat16, torch.float32])
def test_norm_and_clipping(gdt):
    pairs = make(SIZES + [(300000,)], "f32", torch.float32, gdt, seed=8)
    grads = [d["g"] for _, d in pairs]
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    norm, none = multi_tensor_grad_norm(grads)
    # eight squares in fp32 (8 * 2^-24 of the sum), fp64 from there on, one rounding of the root
    assert none is None and abs(float(norm) - exact) <= 1e-6 * exact
    again, coef = multi_tensor_grad_norm(grads, 0.5 * exact)
    assert torch.equal(norm, again) and abs(float(coef) - 0.5 * exact / (exact + 1e-6)) < 1e-6
    assert float(multi_tensor_grad_norm(grads, 2 * exact)[1]) == 1.0
    total = call([d for _, d in pairs], "f32", max_norm=0.5 * exact)
    assert torch.equal(total, norm)
    verify(pairs, "f32", coef.cpu())
    assert float(multi_tensor_grad_norm([torch.zeros(5, device=DEV), torch.zeros(0, device=DEV)])[0]) == 0.0
    assert float(multi_tensor_grad_norm([torch.zeros(0, device=DEV)])[0]) == 0.0
    bad = torch.ones(100, device=DEV)
    bad[3] = math.nan
    n, c = multi_tensor_grad_norm([bad], 1.0)
    assert n.isnan() and c.isnan()
    bad[3] = math.inf
    n, c = multi_tensor_grad_norm([bad], 1.0)
    assert n.isinf() and c == 0


def test_empty_and_expanded():
    assert multi_tensor_adamw([], [], [], []) is None
    pairs = make([(0,), (6, 4)], "f32", torch.float32, torch.float32, seed=9)
    cpu, dev = pairs[1]
    cpu["g"] = torch.full((1, 1), 0.25).expand(6, 4)
    dev["g"] = torch.full((1, 1), 0.25, device=DEV).expand(6, 4)
    call([d for _, d in pairs], "f32")
    verify(pairs[1:], "f32")


def test_device_hyper_stream_and_graph():
    pairs = make(SIZES, "int8", torch.bfloat16, torch.bfloat16, seed=10)
    devs = [d for _, d in pairs]
    start = copy.deepcopy(devs)
    hd = K.DeviceHyper(torch.device(DEV, 0))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm = call(devs, "int8", hyper_device=hd, max_norm=1e9)
        for step in (1, 2):
            hd.update(**{**HP, "step": step})
            graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    for step in (1, 2):
        want = call(start, "int8", step=step, max_norm=1e9)
    assert torch.equal(norm, want)
    for a, b in zip(devs, start):
        for k in a:
            assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)), k


def _params(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(n, generator=g) * 0.1).to(dtype).to(DEV)) for n in [(33, 64), (100,), (7,)]]


def _give_grads(params, seed, skip=()):
    g = torch.Generator().manual_seed(seed)
    for i, p in enumerate(params):
        gr = torch.randn(p.shape, generator=g).to(p.dtype).to(DEV)
        p.grad = None if i in skip else gr


def test_optimizer_class_follows_torch():
    a, b = _params(1), _params(1)
    mine = MultiTensorAdamW([{"params": a[:1]}, {"params": a[1:], "weight_decay": 0.0, "lr": 3e-3}], lr=1e-2, weight_decay=0.1,
                            max_grad_norm=2.0)
    ref = torch.optim.AdamW([{"params": b[:1]}, {"params": b[1:], "weight_decay": 0.0, "lr": 3e-3}], lr=1e-2, weight_decay=0.1)
    for step in range(4):
        skip = (1,) if step == 1 else ()             # one parameter sits a step out and counts its own steps
        _give_grads(a, step, skip)
        _give_grads(b, step, skip)
        total = torch.nn.utils.clip_grad_norm_(b, 2.0)
        mine.step()
        ref.step()
        assert abs(float(mine.last_grad_norm) - float(total)) < 1e-5 * float(total)
    assert mine.state[a[1]]["step"] == 3 and mine.state[a[0]]["step"] == 4
    for p, q in zip(a, b):
        # a step moves a weight by about lr; the two evaluate it in fp32 with a few roundings each
        assert (p - q).abs().max() < 4 * 1e-2 * 1e-5 + 1e-6


@pytest.mark.parametrize("mode", ["f32", "bf16", "int8", "fp8_block"])
def test_optimizer_checkpoint_continues_bit_for_bit(mode):
    a, b = _params(2, torch.bfloat16), _params(2, torch.bfloat16)
    opt = MultiTensorAdamW(a, lr=1e-2, state_mode=mode)
    for step in range(2):
        _give_grads(a, step)
        opt.step()
    for p, q in zip(b, a):
        p.data.copy_(q.data)
    other = MultiTensorAdamW(b, lr=5.0, state_mode=mode)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert other.param_groups[0]["lr"] == 1e-2
    for p, q in zip(a, b):
        for k, t in opt.state[p].items():
            u = other.state[q][k]
            assert (t == u) if k == "step" else (t.dtype == u.dtype and t.data_ptr() != u.data_ptr())
    for o, ps in ((opt, a), (other, b)):
        _give_grads(ps, 9)
        o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k, t in opt.state[p].items():
            u = other.state[q][k]
            assert t == u if k == "step" else torch.equal(t.view(torch.uint8), u.view(torch.uint8))


def test_optimizer_in_a_graph():
    a, b = _params(3, torch.bfloat16), _params(3, torch.bfloat16)
    opt, ref = MultiTensorAdamW(a, lr=1e-2, state_mode="int8"), MultiTensorAdamW(b, lr=1e-2, state_mode="int8")
    _give_grads(a, 0)
    _give_grads(b, 0)
    opt.step()                                        # allocates the state
    ref.step()
    opt.enable_device_hyper()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.pre_step()
        with torch.cuda.graph(graph, stream=side):
            opt.step()
        graph.replay()
        opt.param_groups[0]["lr"] = 2e-2
        opt.pre_step()
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    ref.step()
    ref.param_groups[0]["lr"] = 2e-2
    ref.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)


@pytest.mark.parametrize("strided", [False, True])
def test_autograd_sees_the_update(strided):
    """A graph that has saved a parameter refuses to go on once the step has changed it (both ways into the library)."""
    w = torch.nn.Parameter(torch.ones(8, 8, device=DEV))
    x = torch.ones(3, 8, device=DEV, requires_grad=True)
    y = (x @ w).sum()
    g = torch.ones(8, 16, device=DEV)[:, ::2] if strided else torch.ones(8, 8, device=DEV)
    multi_tensor_adamw([w.detach()], [g], [torch.zeros(8, 8, device=DEV)], [torch.zeros(8, 8, device=DEV)])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_replayed_steps_are_counted_in_checkpoints():
    p = torch.nn.Parameter(torch.ones(8, device=DEV))
    p.grad = torch.ones(8, device=DEV)
    opt = MultiTensorAdamW([p]).enable_device_hyper()
    opt.pre_step()
    opt.step()
    for _ in range(3):
        opt.pre_step()                                # (replays of a captured step() in between)
    assert opt.state_dict()["state"][0]["step"] == 4


def test_a_captured_step_goes_on_with_a_loaded_checkpoint():
    a, b = _params(6, torch.bfloat16), _params(6, torch.bfloat16)
    opt, ref = MultiTensorAdamW(a, lr=1e-2, state_mode="int8"), MultiTensorAdamW(b, lr=1e-2, state_mode="int8")
    for ps in (a, b):
        _give_grads(ps, 0)
    opt.step()
    ref.step()
    saved = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in a]
    opt.enable_device_hyper()
    graph = torch.cuda.CUDAGraph()
    opt.pre_step()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
        opt.pre_step()
    opt.load_state_dict(saved[0])
    opt.enable_device_hyper()                         # (again: what the graph reads stays where it is)
    with torch.no_grad():
        for p, q in zip(a, saved[1]):
            p.copy_(q)
    for _ in range(2):
        opt.pre_step()
        graph.replay()
        ref.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "step"):
            u, v = opt.state[p][k], ref.state[q][k]
            assert torch.equal(u, v) if isinstance(u, torch.Tensor) else u == v


def test_capture_without_a_state_is_refused():
    """A state created during a capture would be zeroed by every replay."""
    (p, *_), opt = _params(5), None
    opt = MultiTensorAdamW([p])
    p.grad = torch.ones_like(p)
    before = p.detach().clone()
    for hyper in (False, True):
        if hyper:
            opt.enable_device_hyper().pre_step()
        with pytest.raises(RuntimeError, match="before it is captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                opt.step()
    assert not opt.state and torch.equal(p, before)
    opt.step()
    assert not torch.equal(p, before)


def test_refusals():
    p, g = torch.zeros(8, 8, device=DEV), torch.zeros(8, 8, device=DEV)
    m, v = torch.zeros(8, 8, device=DEV), torch.zeros(8, 8, device=DEV)
    ok = [p], [g], [m], [v]
    q = torch.zeros(64, dtype=torch.int8, device=DEV)
    s = torch.ones(1, device=DEV)
    for args, kw in [(([p], [], [m], [v]), {}), (([p], [g[:4]], [m], [v]), {}), (([p], [g], [m[:4]], [v]), {}),
                     (([p.half()], [g], [m], [v]), {}), (([p], [g.half()], [m], [v]), {}), (([p], [g], [m.half()], [v.half()]), {}),
                     (([p], [g], [m], [v.bfloat16()]), {}), (([p.t()[:4]], [g[:4]], [m[:4]], [v[:4]]), {}),
                     (([p], [g], [q], [q.clone()]), {}), (([p], [g], [q], [q.clone()], [s], [torch.ones(2, device=DEV)]), {}),
                     (([p], [g], [q], [q.clone()], [s], [s.double()]), {}), (([p], [g], [m], [v], [s], [s]), {}),
                     (([p, p], [g, g], [m, m.clone()], [v, v.clone()]), {}), (([p, p.clone()], [g, g], [m, m], [v, v.clone()]), {}),
                     (([p], [g], [m], [m]), {}), (([p], [g], [q], [q.clone()], [s], [s]), {}),
                     (ok, dict(hyper_device=K.DeviceHyper(torch.device("cpu")))), (ok, dict(step=0)), (ok, dict(max_norm=0.0)), (ok, dict(max_norm=1.0, grad_coef=s)),
                     (ok, dict(grad_coef=torch.ones(2, device=DEV)))]:
        with pytest.raises(ValueError):
            multi_tensor_adamw(*args, **kw)
    with pytest.raises(_lib.ForgeLibraryError):
        multi_tensor_adamw([p.cpu()], [g], [m], [v])
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(p)], state_mode="fp4")
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(p)], max_grad_norm=-1.0)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(lr=math.nan)):
        with pytest.raises(ValueError):
            MultiTensorAdamW([torch.nn.Parameter(p)], **kw)
    with pytest.raises(ValueError):
        MultiTensorAdamW([torch.nn.Parameter(p)]).pre_step()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [1e20, 3e38, 1e-20, 1e-30, 1e-38])
def test_norm_of_gradients_whose_squares_leave_fp32(dtype, scale):
    """Against 64 bits; the norm itself is rounded to fp32 (and is infinite where it exceeds its range).  Eight squares in fp32 are
    off by 8 2^-24 of their sum at most, the root by half of that."""
    g = torch.Generator(device=DEV).manual_seed(3)
    big = torch.rand(70001, device=DEV, generator=g) * scale                 # up to `scale`, the type's normal range and a bit below
    grads = [big.to(dtype), (torch.rand(13, device=DEV, generator=g) * min(scale, 1.0)).to(dtype), torch.zeros(4096, device=DEV, dtype=dtype)]
    exact = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
    norm, coef = multi_tensor_grad_norm(grads, 0.5)
    if exact > torch.finfo(torch.float32).max:
        assert norm.isinf() and abs(float(coef) - 0.5 / exact) <= 2.0 ** -149        # (a subnormal number)
    else:
        assert abs(float(norm) - exact) <= 2.0 ** -21 * exact + 2.0 ** -149
        assert abs(float(coef) - min(1.0, 0.5 / (exact + 1e-6))) <= 1e-6 * min(1.0, 0.5 / (exact + 1e-6)) + 2.0 ** -149
    one = torch.zeros(9, device=DEV, dtype=dtype)
    one[4] = scale
    want = float(one.double().norm())
    norm, coef = multi_tensor_grad_norm([one], 1.0)
    assert abs(float(norm) - want) <= 2e-7 * want
    # a step clipped by it moves the parameters
    p, m, v = torch.zeros(9, device=DEV), torch.zeros(9, device=DEV), torch.zeros(9, device=DEV)
    if scale > 1:
        multi_tensor_adamw([p], [one], [m], [v], max_norm=1.0, weight_decay=0.0)
        assert abs(float(m[4]) - 0.1) < 1e-6 and p[4] < 0


def test_a_captured_step_goes_on_where_a_checkpoint_lacks_a_parameter():
    a = _params(7, torch.bfloat16)
    opt = MultiTensorAdamW(a, lr=1e-2, state_mode="int8")
    _give_grads(a, 0)
    opt.step()
    opt.enable_device_hyper()
    graph = torch.cuda.CUDAGraph()
    opt.pre_step()
    with torch.cuda.graph(graph):
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    del saved["state"][1]
    saved["state"][0]["step"] = saved["state"][2]["step"] = 4
    opt.load_state_dict(saved)
    b = [p.detach().clone() for p in a]
    states = [{k: v.clone() for k, v in opt.state[p].items() if k != "step"} for p in a]
    assert (states[1]["exp_avg"] == 0).all() and (states[1]["exp_avg_sq_scale"] == 1).all()
    opt.pre_step()
    graph.replay()
    for p, q, st in zip(a, b, states):
        multi_tensor_adamw([q], [p.grad], [st["exp_avg"]], [st["exp_avg_sq"]], [st["exp_avg_scale"]], [st["exp_avg_sq_scale"]],
                           lr=1e-2, step=5)
        assert torch.equal(p, q)
        for k, v in st.items():
            assert torch.equal(opt.state[p][k], v)


@pytest.mark.parametrize("direct", [True, False])
def test_errors_are_the_same_on_both_paths(direct, monkeypatch):
    """A code of the library is the same exception from the extension and from Python."""
    from forge_b200 import native
    monkeypatch.setenv("FORGE_NATIVE_AUTOGRAD", "1" if direct else "0")
    native.reset()

    class Hyper:                                         # off its boundary: refused by the host code, never read
        dev = torch.zeros(16, device=DEV)

        def data_ptr(self):
            return self.dev.data_ptr() + 4

    try:
        assert (native.module() is not None) == direct
        p, g, m, v = (torch.zeros(8, device=DEV) for _ in range(4))
        with pytest.raises(_lib.ForgeLibraryError, match="hyper_device is not aligned"):
            multi_tensor_adamw([p], [g], [m], [v], hyper_device=Hyper())
        with pytest.raises(ValueError, match="step must be"):
            multi_tensor_adamw([p], [g], [m], [v], step=0)
    finally:
        monkeypatch.undo()
        native.reset()
