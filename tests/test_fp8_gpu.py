"""e4m3 block quantisation against its definition, bit for bit, and products of codes against 64 bits.

Tolerance of a product: the 128 terms of a block are exact products of two e4m3 values added by the tensor cores with at least
24 bits relative to the largest partial sum, then scaled and added in fp32 (3 roundings per block and KB additions, 2^-24 each,
of at most the sum A of the terms' absolute values); 2^-24 (128 + 3 + KB) A covers both.  The result is rounded to bf16 once
(eps / 2 of the value)."""

import math

import pytest
import torch

from forge_b200 import _lib
from forge_b200.fp8 import Fp8Weight, fp8_linear, fp8_matmul, quantize_fp8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def quantize_reference(x, block_rows):
    """fp32 operations on the CPU, each rounded once as the definition has it."""
    x = x.cpu().float()
    r, c = x.shape
    f = torch.zeros(-(-r // block_rows) * block_rows, -(-c // 128) * 128)
    f[:r, :c] = x
    b = f.view(f.shape[0] // block_rows, block_rows, f.shape[1] // 128, 128)
    scale = b.abs().amax((1, 3)) * torch.tensor(1 / 448.0) + 1e-12
    q = (b / scale[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(f.shape)[:r, :c], scale


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 7), (2, 129), (130, 300), (128, 256), (257, 1000), (5, 4096), (1000, 130)])
def test_quantize_bit_for_bit(dtype, block, shape):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[0], 1, generator=g) * 3)
    x[0, 0] = 0.0
    x = x.to(dtype)
    got = quantize_fp8(x.to(DEV), block, transposed=block == 128)
    q, s = quantize_reference(x, block)
    assert torch.equal(got[1].cpu(), s)
    assert torch.equal(bits(got[0]), bits(q))
    assert got[0].data_ptr() % 16 == 0 and (got[0].stride(0) % 16 == 0 or shape[0] == 1)
    if block == 128:
        assert torch.equal(bits(got[2]), bits(q.t())) and torch.equal(got[3].cpu(), s.t())


def test_quantize_layouts_zeros_and_non_finite():
    x = torch.randn(70, 515, device=DEV).bfloat16()
    want = quantize_fp8(x)
    big = torch.zeros(70, 520, device=DEV, dtype=torch.bfloat16)
    big[:, 3:518] = x
    for view in (big[:, 3:518], x.t().contiguous().t()):
        got = quantize_fp8(view)
        assert torch.equal(bits(got[0]), bits(want[0])) and torch.equal(got[1], want[1])
    assert quantize_fp8(x[::2])[1].equal(want[1][::2])
    out = tuple(torch.zeros_like(t) for t in quantize_fp8(x, 128, True))
    back = quantize_fp8(x, 128, True, out=out)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(out, back))
    q, s = quantize_fp8(torch.zeros(4, 256, device=DEV))
    assert (q.float() == 0).all() and (s == 1e-12).all()
    y = torch.ones(3, 256, device=DEV)
    y[0, 5], y[1, 130] = math.inf, math.nan
    q, s = quantize_fp8(y)
    v = q.float() * s.repeat_interleave(128, 1)
    assert v[0, :128].isnan().all() and v[0, 128:].isfinite().all() and v[2].isfinite().all()
    assert v[1].isnan().sum() == 1 and v[1, 130].isnan()
    assert quantize_fp8(torch.zeros(0, 256, device=DEV))[0].shape == (0, 256)
    assert quantize_fp8(torch.zeros(3, 0, device=DEV))[1].shape == (3, 0)


def values(q, s, block_rows):
    r, c = q.shape
    return q.double() * s.double().repeat_interleave(block_rows, 0)[:r].repeat_interleave(128, 1)[:, :c]


def check_product(xq, xs, wq, ws, y):
    x, w = values(xq, xs, 1), values(wq, ws, 128)
    want = x @ w.t()
    a = x.abs() @ w.abs().t()
    kb = -(-xq.shape[1] // 128)
    tol = torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 2.0 ** -24 * (131 + kb) * a
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((y.double() - want).abs() / tol.clamp(min=1e-300)).max():.2f}x"


@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (1, 1, 1), (1, 1030, 4096), (1, 20000, 700), (2, 5000, 1040), (2, 130, 300), (3, 777, 5000), (4, 6000, 514), (4, 129, 16), (5, 20001, 1168), (8, 4100, 2064), (7, 33, 130), (16, 256, 512), (17, 129, 1000), (33, 640, 144),
                                   (64, 1024, 2048), (65, 257, 384), (128, 128, 128), (129, 300, 520), (200, 1024, 7168), (500, 2000, 640),
                                   (512, 4096, 1024), (700, 515, 260), (1100, 3000, 900), (5, 14336, 4096), (2048, 1024, 256),
                                   (300, 4090, 1000), (390, 4072, 640), (1500, 1000, 300)])
def test_product_against_64_bits(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    x = torch.randn(m, k, device=DEV, generator=g)
    x[:, ::37] *= 50
    w = torch.randn(n, k, device=DEV, generator=g) * torch.exp(torch.randn(n, 1, device=DEV, generator=g))
    xq, xs = quantize_fp8(x)
    wq, ws = quantize_fp8(w, 128)
    y = fp8_matmul(xq, xs, wq, ws)
    assert y.shape == (m, n) and y.dtype == torch.bfloat16
    check_product(xq, xs, wq, ws, y)
    assert torch.equal(y, fp8_matmul(xq, xs, wq, ws))


def test_rows_and_scales_of_other_layouts():
    x, w = torch.randn(70, 512, device=DEV), torch.randn(200, 512, device=DEV)
    xq, xs = quantize_fp8(x)
    wq, ws = quantize_fp8(w, 128)
    want = fp8_matmul(xq, xs, wq, ws)
    assert torch.equal(fp8_matmul(xq, xs.t().contiguous().t(), wq, ws.t().contiguous().t()), want)
    big = torch.zeros(70, 1024, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
    big[:, 512:].view(torch.uint8).copy_(xq.view(torch.uint8))
    assert torch.equal(fp8_matmul(big[:, 512:], xs, wq, ws), want)
    assert torch.equal(fp8_matmul(xq[::2], xs[::2], wq, ws), want[::2])
    assert torch.equal(fp8_matmul(xq[:1], xs[:1], wq, ws).isfinite(), torch.ones(1, 200, device=DEV, dtype=torch.bool))
    empty = fp8_matmul(xq[:0], xs[:0], wq, ws)
    assert empty.shape == (0, 200)
    nothing = fp8_matmul(xq[:, :0], xs[:, :0], wq[:, :0], ws[:, :0])
    assert nothing.shape == (70, 200) and (nothing == 0).all()


def test_non_finite_stays_in_its_row():
    x, w = torch.randn(40, 300, device=DEV), torch.randn(129, 300, device=DEV)
    x[3, 299] = math.nan
    x[7, 0] = math.inf
    y = fp8_matmul(*quantize_fp8(x), *quantize_fp8(w, 128))
    rows = torch.zeros(40, dtype=torch.bool, device=DEV)
    rows[3] = rows[7] = True
    assert torch.equal(y.isnan().all(1), rows) and y[~rows].isfinite().all()


def test_linear_and_its_gradients():
    g = torch.Generator(device=DEV).manual_seed(3)
    w = (torch.randn(384, 272, device=DEV, generator=g) * 0.1).bfloat16()
    x = torch.randn(3, 50, 272, device=DEV, generator=g).bfloat16().requires_grad_(True)
    b = torch.randn(384, device=DEV, generator=g).bfloat16().requires_grad_(True)
    dy = torch.randn(3, 50, 384, device=DEV, generator=g).bfloat16()
    fw = Fp8Weight.from_weight(w)
    y = fp8_linear(x, fw)
    check_product(*quantize_fp8(x.detach().view(150, 272)), fw.codes, fw.scales, y.detach().view(150, 384))
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx.shape == x.shape
    check_product(*quantize_fp8(dy.view(150, 384)), fw.codes_t, fw.scales_t, dx.view(150, 272))
    yb = fp8_linear(x, fw, b)
    dxb, db = torch.autograd.grad(yb, (x, b), dy)
    assert torch.equal(yb, (y + b)) and torch.equal(dxb, dx) and torch.equal(db, dy.view(150, 384).sum(0))
    # against differences: the map is linear once x is a multiple of its codes, so a step of one code changes y by w's values
    xq, xs = quantize_fp8(x.detach().view(150, 272))
    col = torch.zeros(1, 272, device=DEV)
    col[0, 9] = 2.0
    step = fp8_matmul(*quantize_fp8(col), fw.codes, fw.scales)
    want = 2.0 * values(fw.codes, fw.scales, 128)[:, 9]
    assert ((step[0].double() - want).abs() <= want.abs() * (2.0 ** -8 + 1e-6)).all()
    with torch.no_grad():
        assert torch.equal(fp8_linear(x, fw), y)
    w2 = w * 1.5
    fw.update_(w2)
    fresh = Fp8Weight.from_weight(w2)
    assert all(torch.equal(bits(getattr(fw, k)), bits(getattr(fresh, k))) for k in fw.__slots__)
    assert torch.equal(fp8_linear(x[0, 0].detach(), fw), fp8_linear(x[:1, :1].detach(), fw)[0, 0])


def test_streams_and_graph():
    w = Fp8Weight.from_weight(torch.randn(512, 256, device=DEV))
    x = torch.randn(100, 256, device=DEV).bfloat16().requires_grad_(True)
    dy = torch.randn(100, 512, device=DEV).bfloat16()

    def step():
        y = fp8_linear(x, w)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    a = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c = step()
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, r)


@pytest.mark.parametrize("bias", [False, True])
def test_codes_rewritten_before_the_backward_are_noticed(bias):
    w = torch.randn(256, 128, device=DEV)
    fw = Fp8Weight.from_weight(w)
    x = torch.randn(10, 128, device=DEV).bfloat16().requires_grad_(True)
    b = torch.zeros(256, device=DEV, dtype=torch.bfloat16) if bias else None
    y = fp8_linear(x, fw, b)
    fw.update_(w * 2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    fp8_linear(x, fw, b).sum().backward()
    with torch.inference_mode():
        Fp8Weight.from_weight(w).update_(w)


def test_refusals():
    x, w = torch.randn(8, 256, device=DEV), torch.randn(130, 256, device=DEV)
    xq, xs = quantize_fp8(x)
    wq, ws = quantize_fp8(w, 128)
    for args in [(xq[:, :128], xs, wq, ws), (xq, xs[:, :1], wq, ws), (xq, xs, wq, ws[:1]), (xq, xs.double(), wq, ws), (x, xs, wq, ws),
                 (xq[0], xs, wq, ws), (xq.t(), xs, wq, ws), (wq[:8].t().contiguous().t(), xs, wq, ws)]:
        with pytest.raises(ValueError):
            fp8_matmul(*args)
    with pytest.raises(_lib.ForgeLibraryError):                    # rows that start off a 16-byte boundary
        odd = torch.zeros(8, 264, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
        fp8_matmul(odd[:, :256], xs, wq, ws)
    with pytest.raises(_lib.ForgeLibraryError):
        odd = torch.zeros(8, 272, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
        fp8_matmul(odd[:, 8:264], xs, wq, ws)
    for a, kw in [((x[0],), {}), ((x, 64), {}), ((x, 1, True), {}), ((x.half(),), {}), ((x,), dict(out=(xq, ws)))]:
        with pytest.raises(ValueError):
            quantize_fp8(*a, **kw)
    fw = Fp8Weight(wq, ws)
    for bad in (x, x[:, :128].bfloat16()):
        with pytest.raises(ValueError):
            fp8_linear(bad, fw)
    with pytest.raises(ValueError):
        fp8_linear(x.bfloat16().requires_grad_(True), fw)
    with pytest.raises(ValueError):
        Fp8Weight(wq, ws, wq)
    with pytest.raises(_lib.ForgeLibraryError):
        quantize_fp8(x.cpu())
