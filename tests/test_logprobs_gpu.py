"""Token log probabilities, entropies, alternatives and their gradients against the definition in 64 bits.

Tolerances.  One exponential is off by the rounding of its argument (2 roundings of |z - m| 2^-24 each, weighted with the
probability: at most a few units of the entropy) and of the instruction (2^-22); a thread adds at most V / 512 + 8 terms in
a row before the joins.  For V <= 160000 that is 320 * 2^-24 = 1.9e-5 of S in the worst case: 4e-5 absolute for a logarithm,
twice that for the entropy, whose T has the same sums; z itself is rounded twice (2^-23 of |z|).  A gradient entry inherits
the error of log p relatively, and is rounded to its type by at most half a step (eps / 2 relative)."""

import math

import pytest
import torch

from forge_b200 import _lib
from forge_b200.loss import join_logprob_parts, logprob_parts, token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x, t, temperature, ignore):
    z = x.double() / temperature
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    kept = t != ignore
    chosen = torch.where(kept, lp.gather(-1, torch.where(kept, t, 0)[..., None])[..., 0], 0.0)
    return lp, p, ent, chosen, kept


def check(x, t, top_k=0, temperature=1.0, ignore=-100, grads=True):
    x = x.detach().requires_grad_(grads)
    out = token_logprobs(x, t, top_k=top_k, temperature=temperature, ignore_index=ignore)
    xd = x.detach()
    lp, p, ent, chosen, kept = reference(xd, t, temperature, ignore)
    finite = torch.where(torch.isfinite(xd), xd.abs(), 0)
    zmax = finite.float().amax(-1).double() / temperature
    tol = 4e-5 + 2.0 ** -22 * zmax
    neg = chosen == -math.inf
    assert torch.equal(neg, out.logprobs == -math.inf)
    assert (((out.logprobs.double() - chosen).abs() <= tol) | neg).all()
    assert ((out.entropy.double() - ent).abs() <= 2 * tol).all()
    if top_k:
        v, ids = torch.sort(xd, dim=-1, descending=True, stable=True)
        assert out.top_ids.dtype == torch.int64 and torch.equal(out.top_ids, ids[..., :top_k])
        want = lp.gather(-1, ids[..., :top_k])
        inf = want == -math.inf
        assert torch.equal(inf, out.top_logprobs == -math.inf)
        assert (((out.top_logprobs.double() - want).abs() <= tol[..., None]) | inf).all()
    if grads:
        g = torch.Generator(device=DEV).manual_seed(1)
        gl = torch.randn(t.shape, device=DEV, generator=g)
        gh = torch.randn(t.shape, device=DEV, generator=g)
        (dx,) = torch.autograd.grad((out.logprobs, out.entropy), (x,), (gl, gh))
        glk, ghd = torch.where(kept, gl.double(), 0.0)[..., None], gh.double()[..., None]
        lpc = torch.where(p > 0, lp, torch.zeros_like(lp))
        want = -glk * p - ghd * p * (lpc + ent[..., None])
        want.scatter_add_(-1, torch.where(kept, t, 0)[..., None], glk)
        want /= temperature
        terms = (glk.abs() * p + ghd.abs() * p * (lpc.abs() + ent[..., None])) / temperature
        terms.scatter_add_(-1, torch.where(kept, t, 0)[..., None], glk.abs() / temperature)
        assert dx.dtype == x.dtype and dx.shape == x.shape
        bound = torch.finfo(x.dtype).eps / 2 * want.abs() + (3 * tol[..., None] + 1e-6) * terms + 1e-30
        bad = (dx.double() - want).abs() > bound
        assert not bad.any(), f"{int(bad.sum())} gradient entries off, worst {((dx.double() - want).abs() / bound).max():.2f}x"
    return out


def make(rows, vocab, dtype, seed=0, masked=0.0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, vocab, device=DEV, generator=g) * spread
    if masked:
        hit = torch.rand(rows, vocab, device=DEV, generator=g) < masked
        hit[:, 0] = False
        x = x.masked_fill(hit, -math.inf)
    t = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    return x.to(dtype), t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 33, 32), (1, 1000, 5), (17, 4099, 20),
                                            (1, 128256, 5), (9, 65537, 32), (200, 32003, 0), (700, 1001, 1)])
def test_against_64_bits(dtype, rows, vocab, top):
    x, t = make(rows, vocab, dtype, seed=rows + vocab)
    if rows > 2:
        t[1] = -100
    check(x, t, top_k=top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("masked", [0.5, 0.999])
def test_masked_logits(dtype, masked):
    x, t = make(6, 9001, dtype, masked=masked, seed=4)
    check(x, t, top_k=4, temperature=0.7)
    low = torch.where(x == -math.inf, torch.finfo(dtype).min, x.float()).to(dtype)     # the type's lowest value as a mask
    check(low, t, top_k=4)


@pytest.mark.parametrize("temperature", [0.05, 0.7, 3.0])
def test_temperature_and_peaked_rows(temperature):
    x, t = make(8, 5003, torch.float32, seed=6)
    x[0, 17] = 60.0                                     # nearly all of the probability
    x[1] = 2.5                                          # a uniform row: every logit ties
    x[2, ::2] = -0.0
    x[2, 1::2] = 0.0                                    # zeros of both signs tie
    x[3] = torch.arange(5003, device=DEV) * 1e-3        # ascending: every element is a new best
    t[0] = 17
    check(x, t, top_k=32, temperature=temperature)


def test_layouts():
    x, t = make(12, 1003, torch.bfloat16, seed=8)
    check(x.view(3, 4, 1003), t.view(3, 4), top_k=2)
    check(x[::2], t[::2], top_k=2)                                        # a pitch of two rows
    wide, tw = make(12, 1010, torch.bfloat16, seed=9)
    check(wide[:, 3:1006], tw.clamp(max=1002), top_k=2)                    # rows that start anywhere
    check(x.view(3, 4, 1003)[:, :-1], t.view(3, 4)[:, :-1])               # no rows of one pitch: copied
    check(x.t().contiguous().t(), t, top_k=2)                             # columns first: copied
    check(x[0], t[0], top_k=3)                                            # one row
    assert token_logprobs(x, t.int(), top_k=1).logprobs.equal(token_logprobs(x, t).logprobs)
    e = x[:1].expand(4, -1)
    assert torch.equal(token_logprobs(e, t[:1].expand(4)).logprobs, token_logprobs(x[:1], t[:1]).logprobs.expand(4))


def test_rows_without_a_distribution():
    x, t = make(6, 3001, torch.float32, seed=10)
    x[1] = -math.inf
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x = x.requires_grad_(True)
    out = token_logprobs(x, t, top_k=3)
    lp = torch.log_softmax(x.detach(), -1)
    bad = torch.tensor([False, True, True, True, False, False], device=DEV)
    assert torch.equal(out.logprobs.isnan(), bad) and torch.equal(out.entropy.isnan(), bad)
    assert torch.equal(lp.isnan().any(-1), bad)
    assert (out.top_ids >= 0).all() and (out.top_ids < 3001).all()
    (dx,) = torch.autograd.grad(out.logprobs[~bad].sum(), x)
    assert dx[~bad].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(3, 70001), (400, 70001)])
def test_alternatives_of_hard_rows(dtype, rows, vocab):
    """Rows in which nearly every element passes for a candidate, for one CTA per row and for many."""
    x, t = make(rows, vocab, dtype, seed=21)
    x[0] = 1.0                                                              # all tie
    x[1] = torch.linspace(-9, 9, vocab, device=DEV).to(dtype)               # ascending, with ties in bf16
    x[2] = -math.inf
    x[2, vocab - 3:] = torch.tensor([1.0, 2.0, 2.0], device=DEV).to(dtype)  # three columns left
    for k in (1, 5, 32):
        check(x, t, top_k=k, grads=False)
    x[0] = math.nan
    out = token_logprobs(x, t, top_k=32)
    assert out.logprobs[0].isnan() and out.top_logprobs[0].isnan().all()
    assert (out.top_ids >= 0).all() and (out.top_ids < vocab).all()


def test_targets_outside_the_vocabulary():
    x, t = make(4, 515, torch.bfloat16, seed=11)
    x = x.requires_grad_(True)
    t[0], t[1], t[2] = 515, -7, -100
    out = token_logprobs(x, t)
    assert out.logprobs[:2].isnan().all() and out.logprobs[2] == 0 and out.logprobs[3].isfinite()
    assert out.entropy.isfinite().all()
    (dx,) = torch.autograd.grad(out.logprobs.sum(), x)
    assert dx[:2].isnan().all() and (dx[2] == 0).all() and dx[3].isfinite().all()
    none = token_logprobs(x.detach(), None, top_k=2)
    assert (none.logprobs == 0).all() and none.entropy.equal(out.entropy)
    check(x.detach()[3:], t[3:], ignore=int(t[3]))          # the ignored index may be a column


def test_one_gradient_only_and_empty():
    x, t = make(5, 700, torch.float32, seed=12)
    x = x.requires_grad_(True)
    out = token_logprobs(x, t)
    (a,) = torch.autograd.grad(out.logprobs.sum(), x, retain_graph=True)         # an expanded gradient arrives
    (b,) = torch.autograd.grad(out.entropy.sum(), x, retain_graph=True)
    (c,) = torch.autograd.grad((out.logprobs + out.entropy).sum(), x)
    assert (a + b - c).abs().max() < 1e-5
    y = torch.zeros(0, 700, device=DEV, requires_grad=True)
    out = token_logprobs(y, t[:0], top_k=2)
    assert out.logprobs.shape == (0,) and out.top_ids.shape == (0, 2)
    out.logprobs.sum().backward()
    assert y.grad.shape == (0, 700)


@pytest.mark.parametrize("mask", ["inf", "lowest"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_entropy_gradient_at_masked_logits(dtype, mask):
    """p log p is 0 at a masked logit, whatever its factor."""
    x, t = make(5, 2003, dtype, masked=0.4, seed=41)
    low = x if mask == "inf" else torch.where(x == -math.inf, torch.finfo(dtype).min, x.float()).to(dtype)
    low = low.detach().requires_grad_(True)
    out = token_logprobs(low, t, temperature=0.5)
    gh = torch.tensor([-50.0, 3.0, 1e6, -1e30, 0.0], device=DEV)
    (dx,) = torch.autograd.grad(out.entropy, low, gh)
    hidden = x == -math.inf
    assert (dx[hidden] == 0).all()
    # the other columns: the gradient for -1, which test_masked_logits holds against the definition, times -gh
    (unit,) = torch.autograd.grad(token_logprobs(low, t, temperature=0.5).entropy.sum(), low)
    want = unit.double() * gh.double()[:, None]
    # both are rounded to their type, from fp32 products of the same three factors (2^-22 each way)
    tol = (torch.finfo(dtype).eps + 2.0 ** -20) * want.abs() + 2.0 ** -20 * gh.double().abs()[:, None] * 30
    assert ((dx.double() - want).abs() <= tol)[~hidden].all()


def test_rows_without_a_gradient_of_their_own():
    """What a row holds is nobody's concern where neither of its results has a gradient: a padded row may be anything."""
    for dtype in (torch.bfloat16, torch.float32):
        for start in (0, 1):                              # rows that start off a 16-byte boundary, too
            x, t = make(7, 3001, dtype, seed=42)
            x[0], x[1], x[2, 7] = -math.inf, math.nan, math.inf
            t[:4] = -100
            view = x[:, start:].detach().requires_grad_(True)
            out = token_logprobs(view, t.clamp(max=2999))
            (dx,) = torch.autograd.grad(out.logprobs.sum(), view)
            assert (dx[:4] == 0).all() and dx[4:].isfinite().all() and (dx[4:] != 0).any()
            (dx,) = torch.autograd.grad(token_logprobs(view, t.clamp(max=2999)).logprobs[5:].sum(), view)
            assert (dx[:5] == 0).all() and (dx[5:] != 0).any()


def test_results_may_be_changed_in_place():
    x, t = make(3, 50, torch.float32, seed=43)
    x = x.requires_grad_(True)
    for view in (x, x[:, 1:]):                         # the direct call; rows of a wider pitch
        (want,) = torch.autograd.grad(token_logprobs(view, t.clamp(max=48)).logprobs.sum(), x)
        out = token_logprobs(view, t.clamp(max=48), top_k=2)
        out.logprobs.neg_()
        out.top_logprobs.exp_()
        (dx,) = torch.autograd.grad(out.logprobs.sum(), x)
        assert torch.equal(dx, -want)


def test_gradient_against_differences():
    # exact in fp32: logits of a few bits, differences of the 64-bit function
    x, t = make(2, 37, torch.float32, seed=13, spread=1.0)
    x = x.requires_grad_(True)
    out = token_logprobs(x, t, temperature=0.8)
    (dx,) = torch.autograd.grad(out.logprobs.sum() + 0.3 * out.entropy.sum(), x)

    def f(v):
        _, _, ent, chosen, _ = reference(v, t, 0.8, -100)
        return chosen.sum() + 0.3 * ent.sum()

    h = 1e-5
    base = x.detach().double()
    for r in range(2):
        for j in range(37):
            d = torch.zeros_like(base)
            d[r, j] = h
            assert abs(float((f(base + d) - f(base - d)) / (2 * h)) - float(dx[r, j])) < 1e-5


def test_second_derivatives_are_refused_and_changed_logits_noticed():
    x, t = make(3, 50, torch.float32, seed=31)
    x = x.requires_grad_(True)
    for view in (x, x[:, 1:]):                         # the direct call; rows of a wider pitch
        out = token_logprobs(view, t.clamp(max=48))
        (dx,) = torch.autograd.grad(out.logprobs.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(dx.sum(), x)
    y = x.detach().clone().requires_grad_(True)
    z = y * 1.0
    out = token_logprobs(z, t)
    z.data.add_(0)
    z.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()


def test_reproducible_streams_and_graph():
    x, t = make(33, 50001, torch.bfloat16, seed=14)
    x = x.requires_grad_(True)

    def step():
        out = token_logprobs(x, t, top_k=4)
        (dx,) = torch.autograd.grad(out.logprobs.sum() * 0.5 + out.entropy.sum(), x)
        return (*[o.detach() for o in out], dx)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            third = step()
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cuts", [[0, 5000, 10007], [0, 3, 4096, 10007], [0, 10007]])
def test_slices_of_the_vocabulary(dtype, cuts):
    x, t = make(11, 10007, dtype, seed=15, masked=0.2)
    t[2] = -100
    t[3] = 10007
    x[4, :4096] = -math.inf                            # a slice without a finite logit
    t[4] = 10006
    whole = token_logprobs(x, t, top_k=7, temperature=0.9)
    parts = [logprob_parts(x[:, a:b], t, a, 10007, top_k=7, temperature=0.9) for a, b in zip(cuts, cuts[1:])]
    lp, ent, lse, top, ids = join_logprob_parts(torch.stack([s for s, _ in parts]), torch.stack([k for _, k in parts]), t, 10007,
                                                temperature=0.9)
    assert torch.equal(ids, whole.top_ids)
    for a, b in ((lp, whole.logprobs), (ent, whole.entropy), (top, whole.top_logprobs)):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
        ok = a.isfinite()
        assert ((a - b)[ok].abs() <= 8e-5 + 2.0 ** -21 * 20).all()
    # each slice's columns of the gradient
    import ctypes
    xr = x.detach().requires_grad_(True)
    out = token_logprobs(xr, t, temperature=0.9)
    gl, gh = torch.randn(11, device=DEV), torch.randn(11, device=DEV)
    (dx,) = torch.autograd.grad((out.logprobs, out.entropy), (xr,), (gl, gh))
    from forge_b200.loss import _args, _call
    for a, b in zip(cuts, cuts[1:]):
        sl = x[:, a:b]
        args = _args(sl, t, 0, 0.9, -100, a, 10007)
        args.lse, args.entropy = lse.data_ptr(), ent.data_ptr()
        got = torch.empty(11, b - a, dtype=dtype, device=DEV)
        _call("forge_logprobs_backward", x.device, ctypes.byref(args), gl.data_ptr(), gh.data_ptr(), got.data_ptr(), b - a)
        want = dx[:, a:b]
        assert torch.equal(got.isnan(), want.isnan())
        ok = ~got.isnan()
        err = (got.double() - want.double()).abs()[ok]
        assert (err <= torch.finfo(dtype).eps * want.double().abs()[ok] + 1e-3 * want.double().abs()[ok] + 1e-6).all()


def test_refusals():
    x, t = make(4, 100, torch.float32, seed=16)
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan),
                dict(top_k=33), dict(top_k=-1), dict(vocab_start=4), dict(vocab_total=200)):
        with pytest.raises(ValueError):
            token_logprobs(x, t, **bad)
    for xx, tt in ((x.half(), t), (x, t.float()), (x, t[:3]), (x[:, :0], t), (x[:, :3], t)):
        with pytest.raises(ValueError):
            token_logprobs(xx, tt, top_k=4)
    with pytest.raises(_lib.ForgeLibraryError):
        token_logprobs(x, t.cpu())
    stats, keys = logprob_parts(x, t, 0, 100, top_k=4)
    stats, keys = stats[None], keys[None]
    for args in ((stats, keys, t.float(), 100), (stats, keys, t[:3], 100), (stats, keys, t.cpu(), 100), (stats.double(), keys, t, 100),
                 (stats, keys[:, :, 0], t, 100), (stats[:, :3], keys, t, 100)):
        with pytest.raises((ValueError, _lib.ForgeLibraryError)):
            join_logprob_parts(*args)
    with pytest.raises(ValueError):
        join_logprob_parts(stats, keys, t, 3)
