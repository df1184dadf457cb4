"""Token log probabilities where fp32 is short of room: masks of the type's lowest value at low temperatures, rows that are
nearly certain."""

import math

import pytest
import torch

from forge_b200.loss import join_logprob_parts, logprob_parts, token_logprobs

from tests.test_logprobs_gpu import DEV, make, reference

pytestmark = pytest.mark.gpu


def close(got, want, tol):
    """Equal where `want`, rounded to fp32, is infinite or NaN; elsewhere within `tol` and the roundings of a number that is a
    masked logit over the temperature (difference, reciprocal, product: 3 2^-24 of it)."""
    w, got = want.float(), got.detach()
    assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got == -math.inf, w == -math.inf)
    ok = w.isfinite()
    assert ((got.double() - want).abs() <= tol + 2.0 ** -22 * want.abs())[ok].all()


def lowest(x, dtype):
    return torch.where(x == -math.inf, torch.finfo(dtype).min, x.float()).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 1.6])
@pytest.mark.parametrize("rows,vocab", [(5, 128256), (700, 9001)])
def test_masks_of_the_lowest_value(dtype, temperature, rows, vocab):
    """Nearly everything masked, so that whole threads, warps and CTAs of a row hold nothing else: the definition in 64 bits,
    where such a logit has probability 0 too.  Tolerances as in test_logprobs_gpu.py."""
    x, t = make(rows, vocab, dtype, masked=0.999, seed=51)
    x[1, 1:] = -math.inf                                  # one column left
    x[2] = -math.inf                                      # none: a uniform row
    x[3, :vocab // 2] = -math.inf
    x[3, -1] = 2.0
    t[0], t[1] = 0, 0
    low = lowest(x, dtype).requires_grad_(True)
    out = token_logprobs(low, t, top_k=4, temperature=temperature)
    lp, p, ent, chosen, _ = reference(low.detach(), t, temperature, -100)
    tol = 4e-5 + 2.0 ** -22 * torch.where(x == -math.inf, 0.0, x.float()).abs().amax(-1).double() / temperature
    close(out.logprobs, chosen, tol)
    close(out.entropy, ent, 2 * tol)
    ids = torch.sort(low.detach(), dim=-1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(out.top_ids, ids)
    close(out.top_logprobs, lp.gather(-1, ids), tol[:, None].expand(-1, 4))
    g = torch.Generator(device=DEV).manual_seed(1)
    gl, gh = (torch.randn(rows, device=DEV, generator=g) for _ in range(2))
    (dx,) = torch.autograd.grad((out.logprobs, out.entropy), (low,), (gl, gh))
    gl, gh, at = gl.double()[:, None], gh.double()[:, None], t[:, None]
    lpc = torch.where(p > 0, lp, 0.0)
    want = (-gl * p - gh * p * (lpc + ent[:, None])).scatter_add_(-1, at, gl) / temperature
    # d(p (log p + H)) = p (log p + H + 1) dlog p + p dH: where log p + H is next to nothing, as in a row with one column left, the
    # errors of log p (tol) and H (2 tol) still come times p
    terms = (gl.abs() * p + gh.abs() * p * (lpc.abs() + ent[:, None] + 1)).scatter_add_(-1, at, gl.abs()) / temperature
    bound = torch.finfo(dtype).eps / 2 * want.abs() + (3 * tol[:, None] + 1e-6) * terms + 1e-30
    some = torch.arange(rows, device=DEV) != 2
    assert ((dx.double() - want).abs() <= bound)[some].all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.3, 0.9])
def test_slices_masked_with_the_lowest_value(dtype, temperature):
    vocab, cuts = 10007, [0, 3, 4096, 10007]
    x, t = make(11, vocab, dtype, seed=52, masked=0.99)
    x[4, :4096] = -math.inf                               # slices with nothing else
    x[5, 1:] = -math.inf
    x[6] = -math.inf
    t[4], t[5], t[7] = 10006, 0, -100
    x[4, 10006] = 1.0
    low = lowest(x, dtype)
    parts = [logprob_parts(low[:, a:b], t, a, vocab, top_k=3, temperature=temperature) for a, b in zip(cuts, cuts[1:])]
    lp, ent, lse, top, ids = join_logprob_parts(torch.stack([s for s, _ in parts]), torch.stack([k for _, k in parts]), t, vocab,
                                                temperature=temperature)
    want, _, want_ent, chosen, _ = reference(low, t, temperature, -100)
    tol = 4e-5 + 2.0 ** -22 * torch.where(x == -math.inf, 0.0, x.float()).abs().amax(-1).double() / temperature
    close(lp, chosen, tol)
    close(ent, want_ent, 2 * tol)
    close(lse, torch.logsumexp(low.double() / temperature, -1), 2 * tol)
    assert torch.equal(ids, torch.sort(low, dim=-1, descending=True, stable=True).indices[:, :3])
    close(top, want.gather(-1, ids), tol[:, None].expand(-1, 3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [1.0, 0.5])
def test_entropy_of_nearly_certain_rows(dtype, temperature):
    """Two logits a row, the smaller one first, in columns that one thread reads one after the other; the rest masked.  With
    g = gap / temperature, e = e^-g: S = 1 + e, H = log S + g e / S.  S is below 2 and rounded once: 2^-24.  e is off by
    g 2^-23 (two roundings of its argument) and 2^-22 (the instruction) of itself, which H feels times g e S < H S: 2^-20 H up to
    g = 8, and less than a hundredth of 2^-24 beyond.  The logarithm and the last sum are off by 2^-24 of H each.
    Together: 2^-23 + 2^-20 H."""
    rows, vocab = 700, 20008                              # one CTA per row, which reads 8192 or 4096 columns at a time
    gaps = torch.linspace(0.25, 16.0, rows, device=DEV).to(dtype)
    x = torch.full((rows, vocab), -math.inf, device=DEV, dtype=dtype)
    r = torch.arange(rows, device=DEV)
    t = r % 1024 + 8192
    x[r, t - 8192], x[r, t] = -gaps, 0.0
    out = token_logprobs(x, t, temperature=temperature)
    _, _, ent, chosen, _ = reference(x, t, temperature, -100)
    assert ((out.entropy.double() - ent).abs() <= 2.0 ** -23 + 2.0 ** -20 * ent).all()
    assert ((out.logprobs.double() - chosen).abs() <= 2.0 ** -23 + 2.0 ** -20 * chosen.abs()).all()


@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("offset", [50.0, -200.0, 1000.0])
@pytest.mark.parametrize("rows", [3, 700])
def test_a_constant_added_to_a_row_changes_nothing(rows, offset, temperature):
    """Logits on a grid of 2^-10, so that adding the constant is exact, and so is every difference of two: the same bits, by
    the direct call and, for rows of a wider pitch, by the Python one."""
    vocab = 32003
    g = torch.Generator(device=DEV).manual_seed(53)
    x = ((torch.randn(rows, vocab, device=DEV, generator=g) * 2.5).clamp(-16, 16) * 1024).round() / 1024
    t = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    x[torch.arange(rows, device=DEV), t] = 14.0
    gl, gh = (torch.randn(rows, device=DEV, generator=g) for _ in range(2))

    def results(x, three_dimensional):
        x = x.requires_grad_(True)
        if three_dimensional:
            v, tt = torch.cat([x, x.detach()], 1)[:, :vocab][None], t[None]
        else:
            v, tt = x, t
        out = token_logprobs(v, tt, top_k=3, temperature=temperature)
        (one,) = torch.autograd.grad(out.logprobs, x, gl.view_as(tt), retain_graph=True)
        (both,) = torch.autograd.grad((out.logprobs, out.entropy), x, (gl.view_as(tt), gh.view_as(tt)))
        return [r.reshape(rows, -1) for r in (*out, one, both)]

    for nd in (False, True):
        first, shifted = results(x.clone(), nd), results(x + offset, nd)
        for a, b in zip(first, shifted):
            assert torch.equal(a, b)


def test_a_constant_added_to_sliced_rows_changes_nothing():
    """As above for slices of the vocabulary: the joined base and sum give each slice its gradient."""
    import ctypes

    from forge_b200.loss import _SAVED, _args, _call, _join
    vocab, cuts, rows, temperature = 5000, [0, 3, 2048, 5000], 9, 0.7
    g = torch.Generator(device=DEV).manual_seed(54)
    x = (torch.randn(rows, vocab, device=DEV, generator=g) * 2.5 * 1024).round() / 1024
    t = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    gl, gh = (torch.randn(rows, device=DEV, generator=g) for _ in range(2))

    def results(x):
        parts = [logprob_parts(x[:, a:b], t, a, vocab, temperature=temperature) for a, b in zip(cuts, cuts[1:])]
        lp, ent, _, _, top, total = _join(torch.stack([s for s, _ in parts]), torch.stack([k for _, k in parts]), t, vocab, temperature,
                                          -100, (rows,), _SAVED)
        assert torch.equal(top, x.amax(1))
        grads = []
        for a, b in zip(cuts, cuts[1:]):
            args = _args(x[:, a:b], t, 0, temperature, -100, a, vocab)
            args.entropy, args.row_max, args.log_sum = ent.data_ptr(), top.data_ptr(), total.data_ptr()
            grads.append(torch.empty(rows, b - a, device=DEV))
            _call("forge_logprobs_backward", x.device, ctypes.byref(args), gl.data_ptr(), gh.data_ptr(), grads[-1].data_ptr(), b - a)
        return lp, ent, total, torch.cat(grads, 1)

    first, shifted = results(x), results(x + 1000.0)
    for a, b in zip(first, shifted):
        assert torch.equal(a, b)
    xr = x.clone().requires_grad_(True)
    out = token_logprobs(xr, t, temperature=temperature)
    (want,) = torch.autograd.grad((out.logprobs, out.entropy), (xr,), (gl, gh))
    # other orders of the same fp32 sums: 4e-5 of p, as in test_logprobs_gpu.py, and 2^-20 for what is formed of it
    p = torch.softmax(x.double() / temperature, 1)
    terms = (gl.abs()[:, None] + gh.abs()[:, None] * ((-p.clamp(min=1e-300).log()) + out.entropy.detach()[:, None] + 1)) * p / temperature
    terms.scatter_add_(1, t[:, None], gl.abs().double()[:, None] / temperature)
    assert ((first[3] - want).abs() <= (4 * 4e-5 + 2.0 ** -20) * terms).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0])
def test_gradient_of_a_row_of_the_lowest_value(dtype, temperature):
    """All logits equal: a uniform row, whatever their value.  Powers of two, so p = 1 / V is exact; log p and the entropy are off
    by 2^-22 of themselves at most, and cancel in the entropy's gradient."""
    vocab = 4096
    x = torch.full((2, vocab), torch.finfo(dtype).min, device=DEV, dtype=dtype, requires_grad=True)
    t = torch.tensor([5, 4000], device=DEV)
    out = token_logprobs(x, t, temperature=temperature)
    log_v = math.log(vocab)
    assert ((out.logprobs.double() + log_v).abs() <= 2.0 ** -22 * log_v).all()
    assert ((out.entropy.double() - log_v).abs() <= 2.0 ** -22 * log_v).all()
    (dx,) = torch.autograd.grad(out.logprobs.sum(), x, retain_graph=True)
    want = torch.full((2, vocab), -1.0 / vocab, device=DEV, dtype=torch.float64).scatter_add_(1, t[:, None], torch.ones(2, 1, device=DEV).double())
    want /= temperature
    # 2^-21: of the exponent -12, of its power, of the temperature's reciprocal
    assert ((dx.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 12 * 2.0 ** -22 + 2.0 ** -22) * want.abs() + 2.0 ** -23 / temperature / vocab).all()
    (dx,) = torch.autograd.grad(out.entropy.sum(), x)
    assert (dx.double().abs() <= 2 * 2.0 ** -21 * log_v / vocab / temperature).all()


@pytest.mark.parametrize("mask", ["inf", "lowest"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_extreme_temperatures(dtype, mask):
    """At 1e36 every logit that is not masked is as likely as the next, at 1e-36 the largest has all of the probability."""
    x, t = make(5, 3001, dtype, seed=55, masked=0.4)
    hidden = x == -math.inf
    if mask == "lowest":
        x = lowest(x, dtype)
    x[:, 7] = 20.0
    hidden[:, 7] = False
    t[0], t[1] = 7, 0
    x = x.requires_grad_(True)
    left = (~hidden).sum(1).double()
    out = token_logprobs(x, t, temperature=1e36)
    at = hidden.gather(1, t[:, None])[:, 0]
    assert ((out.logprobs.double() + left.log()).abs() <= 2.0 ** -20 * left.log())[~at].all() and (out.logprobs[at] < -100).all()
    assert ((out.entropy.double() - left.log()).abs() <= 2.0 ** -20 * left.log()).all()
    cold = token_logprobs(x, t, temperature=1e-36, top_k=1)
    close(cold.logprobs, (x.detach().double().gather(1, t[:, None])[:, 0] - 20.0) / 1e-36, torch.zeros(5, device=DEV))
    assert (cold.entropy == 0).all() and (cold.top_ids == 7).all() and (cold.top_logprobs == 0).all()
    (dx,) = torch.autograd.grad(cold.entropy.sum(), x)
    assert (dx == 0).all()


@pytest.mark.parametrize("wide", [False, True])
def test_entropy_gradient_without_targets(wide):
    """No targets: the same as targets that are all ignored, in the direct call and the Python one."""
    x, _ = make(6, 5000, torch.float32, seed=56)
    x = torch.cat([x, x], 1)[:, :5000] if wide else x
    t = torch.full((2, 3), -100, device=DEV)
    grads = []
    for targets in (None, t):
        xr = x.detach().requires_grad_(True)
        out = token_logprobs(xr.view(2, 3, 5000), targets, temperature=0.8)
        assert (out.logprobs == 0).all()
        grads += torch.autograd.grad((out.logprobs + out.entropy).sum(), xr)
    assert torch.equal(*grads) and (grads[0] != 0).any()


@pytest.mark.parametrize("temperature,factor", [(1e-36, 100.0), (1e-30, 1e8), (0.5, 1e37)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_entropy_gradients_of_improbable_columns(dtype, temperature, factor):
    """p log p is 0 where p is, also where factor / temperature times the logarithm leaves fp32."""
    x = torch.zeros(3, 2000, device=DEV, dtype=dtype)
    x[:, 1::2] = -200.0
    x[:, 0] = 200.0
    x = x.requires_grad_(True)
    out = token_logprobs(x, None, temperature=temperature)
    assert (out.entropy == 0).all()
    (dx,) = torch.autograd.grad(out.entropy, x, torch.full((3,), factor, device=DEV))
    assert (dx == 0).all()
