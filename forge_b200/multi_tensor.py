"""AdamW over many tensors at once: the step of the parameters that are not fused linears (embeddings, norms, biases).

    manager = FusedOptimizerManager(model)
    rest = MultiTensorAdamW(manager.get_non_fused_params(), lr=1e-4, weight_decay=0.01, state_mode="int8")
    ...
    loss.backward()                 # fused layers update their weights here
    rest.step(); rest.zero_grad()

One launch per combination of types and 448 tensors (``forge_multi_adamw``), with the arithmetic and the moment layouts of
the fused path: fp32, bf16, int8 or e4m3 moments, the last two with one fp32 scale for each 64 consecutive elements and,
as there, with a second moment of at least 1e-8 (where the gradients' rms is below 1e-4 the first moment is divided by
1e-4, and the steps are smaller than AdamW's).
``max_grad_norm`` scales the gradients by their common norm without a host synchronisation (``forge_multi_norm``).  The
reference leaves these parameters to ``torch.optim`` (``src/fused_grad_optimizer/module.py:218-222``).
"""

from __future__ import annotations

import copy
import ctypes

import torch

from forge_b200 import _lib, native
from forge_b200.kernel import DeviceHyper, _hyper, _require_cuda

STATE_MODES = ("f32", "bf16", "int8", "fp8_block")
QBLOCK = 64
_MODE_OF = {torch.float32: _lib.ST_F32, torch.bfloat16: _lib.ST_BF16, torch.int8: _lib.ST_INT8,
            torch.float8_e4m3fn: _lib.ST_FP8_BLOCK}
_DTYPE_OF = {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8, "fp8_block": torch.float8_e4m3fn}
_QUANTIZED = (torch.int8, torch.float8_e4m3fn)


def _dense(t, what):
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous (got shape {tuple(t.shape)}, strides {tuple(t.stride())})")


def _grads(grads):
    """Contiguous CUDA gradients; one that is not contiguous (an expanded one, say) is copied."""
    out = []
    for g in grads:
        _require_cuda(g)
        if g.is_sparse:
            raise ValueError("sparse gradients are not supported")
        _lib.dtype_id(g.dtype)
        out.append(g if g.is_contiguous() else g.contiguous())
    return out


def _one_device(tensors):
    dev = tensors[0].device
    if any(t.device != dev for t in tensors):
        raise ValueError("all tensors must be on the same device")
    return dev


def multi_tensor_grad_norm(grads, max_norm: float | None = None):
    """``(norm, coef)`` of a list of CUDA gradients, fp32 scalars on their device: the 2-norm of all elements and, with
    ``max_norm``, ``min(1, max_norm / (norm + 1e-6))`` (None without).  A norm above fp32's range reads as inf, its ``coef`` is
    right; an infinite gradient gives 0.  Bit-reproducible; no host synchronisation."""
    nat = native.module()
    if nat is not None and (max_norm is None or max_norm > 0):
        out = nat.multi_norm(grads, max_norm or 0.0)
        if out is not None:
            return out
    grads = _grads(grads)
    if max_norm is not None and not max_norm > 0:
        raise ValueError(f"max_norm must be positive (got {max_norm})")
    if not grads:
        raise ValueError("no gradients")
    dev = _one_device(grads)
    items = (_lib.ForgeNormItem * len(grads))()
    for it, g in zip(items, grads):
        it.grad, it.numel, it.dtype = g.data_ptr(), g.numel(), _lib.dtype_id(g.dtype)
    lib = _lib.load()
    nbytes = lib.forge_multi_norm_scratch_bytes(items, len(grads))
    with torch.cuda.device(dev):
        out = torch.empty(2, dtype=torch.float32, device=dev)
        scratch = torch.empty(max(nbytes, 8), dtype=torch.uint8, device=dev)
        rc = lib.forge_multi_norm(items, len(grads), float(max_norm or 0.0), out.data_ptr(),
                                  out[1:].data_ptr() if max_norm is not None else None, scratch.data_ptr(), nbytes,
                                  _lib.current_stream_ptr(dev))
    _lib.check(rc, "forge_multi_norm")
    return out[0], (out[1] if max_norm is not None else None)


def multi_tensor_adamw(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales=None, exp_avg_sq_scales=None, *,
                       lr: float = 1e-4, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
                       weight_decay: float = 0.01, step: int = 1, max_norm: float | None = None, grad_coef=None,
                       hyper_device: DeviceHyper | None = None):
    """One AdamW step of every tensor of ``params`` (bf16 or fp32, contiguous, any sizes), in place.

    ``exp_avgs`` / ``exp_avg_sqs``: the moments, all of one dtype, of the parameters' sizes: fp32, bf16, int8 or
    float8_e4m3fn; the 8-bit ones with ``exp_avg_scales`` / ``exp_avg_sq_scales``, fp32, ceil(numel / 64) values each.
    No two of the tensors that are written may overlap (one that is given twice is refused).
    ``max_norm``: multiply the gradients by ``min(1, max_norm / (norm + 1e-6))`` of their common norm, which is returned
    (an fp32 device scalar; None without ``max_norm``); ``grad_coef``: multiply them by a device scalar instead.
    ``hyper_device``: read lr, betas, eps, decay and step from a ``DeviceHyper`` block (for captured graphs)."""
    if not isinstance(params, (list, tuple)):
        params = list(params)
    if hyper_device is not None and params and hyper_device.dev.device != params[0].device:
        raise ValueError(f"hyper_device is on {hyper_device.dev.device}, the parameters are on {params[0].device}")
    nat = native.module()
    if nat is not None and (max_norm is None or max_norm > 0):
        out = nat.multi_adamw(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, lr, beta1, beta2, eps,
                              weight_decay, step, max_norm or 0.0, hyper_device.data_ptr() if hyper_device is not None else 0,
                              grad_coef)
        if out is not None:
            return out[1]
    params, exp_avgs, exp_avg_sqs = list(params), list(exp_avgs), list(exp_avg_sqs)
    grads = _grads(grads)
    n = len(params)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n):
        raise ValueError(f"lists of different lengths: {n} params, {len(grads)} grads, {len(exp_avgs)}, {len(exp_avg_sqs)} moments")
    if max_norm is not None and grad_coef is not None:
        raise ValueError("give max_norm or grad_coef, not both")
    if n == 0:
        return None
    _require_cuda(*params, *exp_avgs, *exp_avg_sqs)
    sdt = exp_avgs[0].dtype
    if sdt not in _MODE_OF or any(t.dtype != sdt for t in exp_avgs) or any(t.dtype != sdt for t in exp_avg_sqs):
        raise ValueError("the moments must share one dtype: float32, bfloat16, int8 or float8_e4m3fn")
    quant = sdt in _QUANTIZED
    if quant:
        if exp_avg_scales is None or exp_avg_sq_scales is None:
            raise ValueError("8-bit moments need exp_avg_scales and exp_avg_sq_scales")
        ms, vs = list(exp_avg_scales), list(exp_avg_sq_scales)
        if len(ms) != n or len(vs) != n:
            raise ValueError("one scale tensor per moment is needed")
        _require_cuda(*ms, *vs)
    elif exp_avg_scales is not None or exp_avg_sq_scales is not None:
        raise ValueError("scales belong to 8-bit moments only")
    dev = _one_device([*params, *grads, *exp_avgs, *exp_avg_sqs, *((*ms, *vs) if quant else ())])
    items = (_lib.ForgeMultiItem * n)()
    seen = set()
    for i in range(n):
        p, g, m, v, it = params[i], grads[i], exp_avgs[i], exp_avg_sqs[i], items[i]
        num = p.numel()
        if g.shape != p.shape or m.numel() != num or v.numel() != num:
            raise ValueError(f"tensor {i}: param {tuple(p.shape)}, grad {tuple(g.shape)}, moments {tuple(m.shape)}, {tuple(v.shape)}")
        for t, what in ((p, "param"), (m, "exp_avg"), (v, "exp_avg_sq")):
            _dense(t, f"tensor {i}: {what}")
        it.param, it.grad, it.m, it.v, it.numel = p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), num
        it.param_dtype, it.grad_dtype = _lib.dtype_id(p.dtype), _lib.dtype_id(g.dtype)
        if quant:
            blocks = -(-num // QBLOCK)
            for t, what in ((ms[i], "exp_avg_scale"), (vs[i], "exp_avg_sq_scale")):
                _dense(t, f"tensor {i}: {what}")
                if t.dtype != torch.float32 or t.numel() != blocks:
                    raise ValueError(f"tensor {i}: {what} must hold {blocks} fp32 values (got {t.numel()} of {t.dtype})")
            it.m_scale, it.v_scale = ms[i].data_ptr(), vs[i].data_ptr()
        if num:
            for q in (it.param, it.m, it.v, *((it.m_scale, it.v_scale) if quant else ())):
                if q in seen:
                    raise ValueError(f"tensor {i}: a parameter, moment or scale tensor appears twice")
                seen.add(q)
    norm = None
    if max_norm is not None:
        norm, grad_coef = multi_tensor_grad_norm(grads, max_norm)
    if grad_coef is not None and (grad_coef.dtype != torch.float32 or grad_coef.numel() != 1 or grad_coef.device != dev):
        raise ValueError("grad_coef must be one fp32 value on the parameters' device")
    a = _lib.ForgeMultiArgs()
    a.items, a.count, a.state_mode = items, n, _MODE_OF[sdt]
    a.hyper = _hyper(lr, beta1, beta2, eps, weight_decay, step)
    a.hyper_device = hyper_device.data_ptr() if hyper_device is not None else None
    a.grad_coef = grad_coef.data_ptr() if grad_coef is not None else None
    with torch.cuda.device(dev):
        rc = _lib.load().forge_multi_adamw(ctypes.byref(a), _lib.current_stream_ptr(dev))
    _lib.check(rc, "forge_multi_adamw")
    # (for autograd: a graph that has saved one of these tensors must not go on with other values)
    torch.autograd.graph.increment_version([t for t in (*params, *exp_avgs, *exp_avg_sqs) if not t.is_inference()])
    return norm


class MultiTensorAdamW(torch.optim.Optimizer):
    """``torch.optim`` interface over ``multi_tensor_adamw``.  ``state_mode``: "f32", "bf16", "int8" or "fp8_block"
    (per parameter group); ``max_grad_norm``: clip by the common norm of all gradients (``last_grad_norm`` then holds it,
    on the device).

    For CUDA graphs run one eager step, which creates the moments, call ``enable_device_hyper()`` and, before each captured
    or replayed ``step()``, ``pre_step()``: it counts the step and writes the groups' hyper-parameters to device memory, where
    ``step()`` reads them; every parameter with a gradient is then taken to be updated in every step."""

    def __init__(self, params, lr: float = 1e-4, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_mode: str = "f32", max_grad_norm: float | None = None):
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"max_grad_norm must be positive (got {max_grad_norm})")
        if not lr >= 0 or not eps >= 0 or not weight_decay >= 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError(f"lr={lr}, betas={betas}, eps={eps}, weight_decay={weight_decay}: out of range")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_mode=state_mode))
        self.max_grad_norm = max_grad_norm
        self.last_grad_norm = None
        self._device_hyper: dict[tuple, DeviceHyper] | None = None
        self._device_step = 0

    @staticmethod
    def _check_group(group):
        if group["state_mode"] not in STATE_MODES:
            raise ValueError(f"Unknown state_mode: {group['state_mode']}. Use one of {STATE_MODES}.")

    def add_param_group(self, group):
        self._check_group({**self.defaults, **group})
        super().add_param_group(group)

    def _state_of(self, p, mode):
        st = self.state[p]
        if not st:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                del self.state[p]
                raise RuntimeError("the moments are created (zeroed) in the first step: run one step before it is captured")
            dt, dev = _DTYPE_OF[mode], p.device
            new = {k: torch.empty(p.shape, dtype=dt, device=dev) for k in ("exp_avg", "exp_avg_sq")}
            if dt in _QUANTIZED:
                for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                    new[k] = torch.empty(-(-p.numel() // QBLOCK), dtype=torch.float32, device=dev)
            self._start(new)
            st.update(new)
        return st

    @staticmethod
    def _start(st):
        """What the first step begins with, written to the tensors of a parameter's state."""
        st["step"] = 0
        for k, t in st.items():
            if k != "step":
                t.fill_(1.0) if k.endswith("_scale") else t.zero_()

    def enable_device_hyper(self):
        if self._device_hyper is None:             # (captured steps read the blocks that are there)
            self._device_hyper = {}
        self._device_step = max((st["step"] for st in self.state.values() if st), default=0)
        return self

    @property
    def reads_device_hyper(self) -> bool:
        return self._device_hyper is not None

    def _hyper_block(self, index, device):
        hd = self._device_hyper.get((index, device))
        if hd is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call pre_step() before a step and before it is captured")
            hd = self._device_hyper[(index, device)] = DeviceHyper(device)
            self._write_hyper(hd, self.param_groups[index])
        return hd

    def _write_hyper(self, hd, group):
        b1, b2 = group["betas"]
        hd.update(lr=group["lr"], beta1=b1, beta2=b2, eps=group["eps"], weight_decay=group["weight_decay"],
                  step=max(self._device_step, 1))

    def pre_step(self):
        """Count the coming step and write the groups' hyper-parameters to the device (see ``enable_device_hyper``)."""
        if self._device_hyper is None:
            raise ValueError("pre_step() belongs to enable_device_hyper()")
        self._device_step += 1
        for index, group in enumerate(self.param_groups):
            for p in group["params"]:              # (a replayed step() does not come by here)
                if self.state.get(p):
                    self.state[p]["step"] = self._device_step
            for dev in {p.device for p in group["params"]}:
                hd = self._device_hyper.get((index, dev))
                if hd is None:
                    self._hyper_block(index, dev)
                else:
                    self._write_hyper(hd, group)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        coefs = {}
        if self.max_grad_norm is not None:
            every = [p.grad for g in self.param_groups for p in g["params"] if p.grad is not None]
            if every:
                if len({g.device for g in every}) > 1:
                    raise ValueError("max_grad_norm needs all parameters on one device")
                self.last_grad_norm, coef = multi_tensor_grad_norm(every, self.max_grad_norm)
                coefs[every[0].device] = coef
        for index, group in enumerate(self.param_groups):
            self._check_group(group)
            # one call per device and step count (a parameter without a gradient in some step counts its own steps)
            calls: dict[tuple, tuple] = {}
            mode = group["state_mode"]
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                st = self.state[p] or self._state_of(p, mode)
                count = st["step"] = st["step"] + 1 if self._device_hyper is None else self._device_step
                m = st["exp_avg"]
                key = p.device, count, m.dtype
                lists = calls.get(key)
                if lists is None:
                    lists = calls[key] = [], [], [], [], [], []
                lists[0].append(p)
                lists[1].append(grad)
                lists[2].append(m)
                lists[3].append(st["exp_avg_sq"])
                if m.dtype in _QUANTIZED:
                    lists[4].append(st["exp_avg_scale"])
                    lists[5].append(st["exp_avg_sq_scale"])
            b1, b2 = group["betas"]
            for (dev, count, sdt), lists in calls.items():
                multi_tensor_adamw(*lists[:4 if sdt not in _QUANTIZED else 6], lr=group["lr"], beta1=b1, beta2=b2,
                                   eps=group["eps"], weight_decay=group["weight_decay"], step=max(count, 1),
                                   grad_coef=coefs.get(dev),
                                   hyper_device=self._hyper_block(index, dev) if self._device_hyper is not None else None)
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As in ``torch.optim``, but the moments keep the types they were saved in (the base class would cast them to the
        parameters' type), and are loaded into the tensors that are there where those fit: a captured ``step()`` goes on
        with them.  Moments of a parameter that the checkpoint lacks stay as well and start again from zero.  After
        ``enable_device_hyper()`` a checkpoint that does not fit the moments (another ``state_mode``) is refused."""
        there = dict(self.state)
        pairs = [(p, state_dict["state"].get(index)) for group, saved in zip(self.param_groups, state_dict["param_groups"])
                 for p, index in zip(group["params"], saved["params"])]
        if self._device_hyper is not None:
            for p, st in pairs:
                old = there.get(p)
                for k in {*old, *st} if old and st else ():
                    if k != "step" and not self._fits(old.get(k), st.get(k), p.device):
                        raise ValueError(f"{k} of the checkpoint does not fit the moments that a captured step may be using; load it "
                                         f"before enable_device_hyper(), or into another optimizer")
        super().load_state_dict(state_dict)
        for p, st in pairs:
            old = there.get(p, {})
            if st:
                self.state[p] = {k: self._load(old.get(k), v, p.device) for k, v in st.items()}
            elif old:
                self._start(old)
                self.state[p] = old
        self._device_step = max((st["step"] for st in self.state.values() if st), default=0)

    @staticmethod
    def _fits(old, new, device):
        return (isinstance(old, torch.Tensor) and isinstance(new, torch.Tensor) and old.shape == new.shape and old.dtype == new.dtype
                and old.device == device)

    @classmethod
    def _load(cls, old, new, device):
        if not isinstance(new, torch.Tensor):
            return copy.deepcopy(new)
        return old.copy_(new) if cls._fits(old, new, device) else new.to(device, copy=True)
