"""Log probabilities of given tokens at the logits, with the rows' entropies and most likely alternatives.

    out = token_logprobs(logits, targets)                  # logits (..., V) bf16 or fp32, targets (...) integers
    loss = -out.logprobs.sum() / (targets != -100).sum()   # next-token cross entropy
    (loss - 0.01 * out.entropy.mean()).backward()

    out = token_logprobs(logits, tokens, top_k=5, temperature=0.7)     # serving: out.top_logprobs, out.top_ids

One pass over the logits forward, one read and one write backward (``forge_logprobs_forward`` /
``forge_logprobs_backward``), nothing of the logits' size in between.  A row-sharded lm_head
(``forge_b200.tensor_parallel``) passes its slice of the columns and its process group: each rank reduces its
slice to a few numbers per row, those are gathered and joined, and each rank forms its own columns of the
gradient.  No reference counterpart (it leaves the loss to the model's own torch code).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from forge_b200 import _lib, native
from forge_b200.kernel import _require_cuda

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    """``logprobs``, ``entropy``: fp32, the targets' shape; ``top_logprobs`` (fp32), ``top_ids`` (int64): with a last
    dimension of top_k, or None.  Gradients flow through the first two."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _rows(logits):
    """The logits as rows of a pitch; copies only what has no such form."""
    x = logits.reshape(-1, logits.shape[-1])
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _args(x, targets, top_k, temperature, ignore_index, vocab_start, vocab_total):
    a = _lib.ForgeLogprobsArgs()
    a.logits, a.targets = x.data_ptr(), targets.data_ptr() if targets is not None else None
    a.rows, a.vocab = x.shape
    a.ld = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    a.vocab_start, a.vocab_total = vocab_start, vocab_total
    a.ignore_index, a.temperature = ignore_index, temperature
    a.dtype, a.top_k = _lib.dtype_id(x.dtype), top_k
    return a


def _check_targets(targets, device):
    if targets is not None:
        if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
            raise ValueError(f"targets must be integers (got {targets.dtype})")
        if targets.device != device:
            raise ValueError("targets and logits must be on the same device")


def _check(logits, targets, top_k, vocab_start, vocab_total):
    _require_cuda(logits, targets)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have a last dimension of at least one column (got {tuple(logits.shape)})")
    _lib.dtype_id(logits.dtype)
    _check_targets(targets, logits.device)
    if targets is not None and targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not match logits {tuple(logits.shape)}")
    if not 0 <= top_k <= MAX_TOP_K:
        raise ValueError(f"top_k must be 0 .. {MAX_TOP_K} (got {top_k})")
    if top_k > vocab_total:
        raise ValueError(f"top_k ({top_k}) exceeds the vocabulary ({vocab_total})")
    if vocab_start < 0 or vocab_start + logits.shape[-1] > vocab_total:
        raise ValueError(f"columns [{vocab_start}, {vocab_start + logits.shape[-1]}) of a vocabulary of {vocab_total}")


def _targets(targets):
    return None if targets is None else targets.reshape(-1).to(torch.int64).contiguous()


def _call(fn, device, *args):
    with torch.cuda.device(device):
        rc = getattr(_lib.load(), fn)(*args, _lib.current_stream_ptr(device))
    if rc:
        _lib.check(rc, fn)


_SAVED = ("row_max", "log_sum")      # what backward needs besides the entropy


def _outputs(a, lead, top_k, device, more):
    """``(logprobs, entropy, top_logprobs, top_ids, *more)``, `more` naming other outputs of a value per row."""
    # (tensors of their own and no views: what a user does in place to one result is not done to the saved ones)
    out = [torch.empty(lead, dtype=torch.float32, device=device) for _ in range(2 + len(more))]
    for name, t in zip(("logprobs", "entropy", *more), out):
        setattr(a, name, t.data_ptr())
    top = ids = None
    if top_k:
        top = torch.empty(*lead, top_k, dtype=torch.float32, device=device)
        ids = torch.empty(*lead, top_k, dtype=torch.int64, device=device)
        a.top_logprobs, a.top_ids = top.data_ptr(), ids.data_ptr()
    return out[0], out[1], top, ids, *out[2:]


def logprob_parts(logits, targets, vocab_start: int, vocab_total: int, top_k: int = 0, temperature: float = 1.0,
                  ignore_index: int = -100):
    """What one slice of the vocabulary, columns ``[vocab_start, vocab_start + V)`` of ``vocab_total``, contributes
    to its rows: ``(stats (rows, 5) fp32, keys (rows, top_k) int64)`` for ``join_logprob_parts``."""
    _check(logits, targets, top_k, vocab_start, vocab_total)
    x, t = _rows(logits), _targets(targets)
    a = _args(x, t, top_k, temperature, ignore_index, vocab_start, vocab_total)
    stats = torch.empty(x.shape[0], 5, dtype=torch.float32, device=x.device)
    keys = torch.empty(x.shape[0], top_k, dtype=torch.int64, device=x.device)
    a.stats, a.keys = stats.data_ptr(), keys.data_ptr()
    _call("forge_logprobs_forward", x.device, ctypes.byref(a))
    return stats, keys


def join_logprob_parts(stats, keys, targets, vocab_total: int, temperature: float = 1.0, ignore_index: int = -100):
    """The rows' results from the parts of all slices, ``stats`` (parts, rows, 5) and ``keys`` (parts, rows, top_k):
    ``(logprobs, entropy, lse, top_logprobs, top_ids)``, each with the rows as its first dimension.  ``temperature`` and
    ``ignore_index`` are those of the parts."""
    _require_cuda(stats, keys, targets)
    if keys.dim() != 3:
        raise ValueError(f"keys must be (parts, rows, top_k) (got {tuple(keys.shape)})")
    _check_targets(targets, stats.device)
    if keys.device != stats.device:
        raise ValueError("stats and keys must be on the same device")
    stats, keys, t = stats.contiguous(), keys.contiguous(), _targets(targets)
    parts, rows, top_k = keys.shape
    if stats.dtype != torch.float32 or keys.dtype != torch.int64 or tuple(stats.shape) != (parts, rows, 5):
        raise ValueError(f"stats must be (parts, rows, 5) fp32 and keys (parts, rows, top_k) int64 (got {tuple(stats.shape)}, "
                         f"{tuple(keys.shape)})")
    if t is not None and t.numel() != rows:
        raise ValueError(f"{t.numel()} targets for {rows} rows")
    lp, ent, top, ids, lse = _join(stats, keys, t, vocab_total, temperature, ignore_index, (rows,), ("lse",))
    return lp, ent, lse, top, ids


def _join(stats, keys, t, vocab_total, temperature, ignore_index, lead, more):
    parts, rows, top_k = keys.shape
    a = _lib.ForgeLogprobsArgs()
    a.targets = t.data_ptr() if t is not None else None
    a.rows, a.vocab_total, a.vocab, a.ld = rows, vocab_total, vocab_total, vocab_total
    a.ignore_index, a.temperature, a.top_k = ignore_index, temperature, top_k
    res = _outputs(a, lead, top_k, stats.device, more)
    _call("forge_logprobs_join", stats.device, ctypes.byref(a), stats.data_ptr(), keys.data_ptr(), parts)
    return res


def _gather_parts(stats, keys, group):
    """Every rank's parts, (world, rows, ...) in rank order."""
    import torch.distributed as dist
    world = dist.get_world_size(group)
    out = []
    for t in (stats, keys):
        parts = t.new_empty(world, *t.shape)
        if t.numel():
            dist.all_gather_into_tensor(parts.view(-1), t.reshape(-1), group=group)
        out.append(parts)
    return out


class _TokenLogprobs(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature, ignore_index, vocab_start, vocab_total, group):
        x, t = _rows(logits), _targets(targets)
        lead = logits.shape[:-1]
        if group is None:
            a = _args(x, t, top_k, temperature, ignore_index, vocab_start, vocab_total)
            lp, ent, top, ids, *saved = _outputs(a, lead, top_k, x.device, _SAVED)
            _call("forge_logprobs_forward", x.device, ctypes.byref(a))
        else:
            stats, keys = logprob_parts(x, t, vocab_start, vocab_total, top_k, temperature, ignore_index)
            lp, ent, top, ids, *saved = _join(*_gather_parts(stats, keys, group), t, vocab_total, temperature, ignore_index, lead,
                                              _SAVED)
        if top_k:
            ctx.mark_non_differentiable(top, ids)
        ctx.set_materialize_grads(False)
        # the logits themselves where they are rows already, so that autograd notices if they are changed
        ctx.save_for_backward(logits if x.data_ptr() == logits.data_ptr() else x, t, ent, *saved)
        ctx.shape = logits.shape
        ctx.settings = (temperature, ignore_index, vocab_start, vocab_total)
        return lp, ent, top, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_lp, g_ent, _g_top, _g_ids):
        x, t, *saved = ctx.saved_tensors
        _require_cuda(x, t, *saved)
        x = _rows(x)
        # (hooks on saved tensors may have brought them back in another layout, or as something else)
        t, saved = _targets(t), [s.contiguous() for s in saved]
        if any(s.shape.numel() != x.shape[0] or s.dtype != torch.float32 or s.device != x.device for s in saved) or (
                t is not None and (t.numel() != x.shape[0] or t.device != x.device)):
            raise RuntimeError("token_logprobs: what was saved for the backward pass came back as something else")
        none = (None,) * 7
        if g_lp is None and g_ent is None:
            return (None, *none)
        a = _args(x, t, 0, *ctx.settings)
        for name, s in zip(("entropy", *_SAVED), saved):
            setattr(a, name, s.data_ptr())
        g = [None if q is None else q.reshape(-1).to(torch.float32).contiguous() for q in (g_lp, g_ent)]
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _call("forge_logprobs_backward", x.device, ctypes.byref(a), *(None if q is None else q.data_ptr() for q in g),
              grad.data_ptr(), grad.shape[1])
        return (grad.view(ctx.shape), *none)


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor], *, top_k: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100, vocab_start: int = 0, vocab_total: Optional[int] = None,
                   group=None) -> TokenLogprobs:
    """Log probability of ``targets`` under ``softmax(logits / temperature)``, the rows' entropies and, with ``top_k``
    (at most 32), the most likely columns in descending order, equal logits by ascending column.

    ``logits`` (..., V) bf16 or fp32 on CUDA (rows of any pitch; what is not made of rows is copied, ``x[:, :-1]`` of a
    batch for one: give all positions and ``ignore_index`` as the last one's target instead), ``targets`` (...) integers
    or None.  A target equal to ``ignore_index`` gives 0 and no gradient of its own; one outside the vocabulary gives NaN,
    in the gradient too.  Logits of -inf have probability zero; rows of nothing else, or with NaN or +inf, give NaN as
    ``log_softmax`` does; logits of the type's lowest value have probability zero beside any other, and are uniform among
    themselves.  ``temperature``: 1e-36 .. 1e36.  Sums are fp32; the gradient comes in the logits' type, and a row neither of
    whose results has one (an ignored target without an entropy gradient) gets zeros, whatever it holds.

    ``group``: the logits are this rank's columns ``[vocab_start, vocab_start + V)`` of ``vocab_total``, every rank of the
    process group calls with its own slice of the same rows (collective: two small all-gathers), and the results are the
    same on every rank.  The gradient is that of this rank's columns for the gradients that reach this rank's results."""
    temperature = float(temperature)
    if not 1e-36 <= temperature <= 1e36:
        raise ValueError(f"temperature must be a positive number, 1e-36 .. 1e36 (got {temperature})")
    if group is None and (vocab_start != 0 or vocab_total is not None and vocab_total != logits.shape[-1]):
        raise ValueError("a slice of the vocabulary needs the process group of the other slices")
    if group is not None and vocab_total is None:
        raise ValueError("a slice of the vocabulary needs vocab_total")
    if group is None:
        nat = native.module()
        if nat is not None:
            out = nat.token_logprobs(logits, targets, top_k, temperature, ignore_index)
            if out is not None:
                return TokenLogprobs(*out)
    total = logits.shape[-1] if vocab_total is None else vocab_total
    _check(logits, targets, top_k, vocab_start, total)
    return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top_k, temperature, int(ignore_index), vocab_start, total,
                                               group))
