"""Linear products in 8-bit floating point (e4m3) with one fp32 scale for each block of 128.

    w = Fp8Weight.from_weight(linear.weight)       # codes and scales of 128 x 128 blocks, both ways round
    y = fp8_linear(x, w)                           # x (..., K) bf16 is quantised by rows (1 x 128 blocks) in the call
    y.backward(dy)                                 # dX = dY W through the transposed codes
    w.update_(linear.weight)                       # after the weight has changed

``quantize_fp8`` and ``fp8_matmul`` are the two steps by themselves (``forge_fp8_quantize``, ``forge_fp8_product``).  The
weight gets no gradient here: in training the fused update forms it from the bf16 activations
(``FusedLinear.use_fp8_products``).  No reference counterpart.
"""

from __future__ import annotations

import ctypes

import torch

from forge_b200 import _lib, native
from forge_b200.kernel import _require_cuda

BLOCK = 128
_CODE = torch.float8_e4m3fn
_registered: set = set()      # devices whose status word the extension knows


def _empty_codes(rows, cols, device):
    """(rows, cols) codes whose rows start on 16-byte boundaries, as the product wants them."""
    return torch.empty(rows, -(-cols // 16) * 16, dtype=_CODE, device=device)[:, :cols]


def _blocks(n):
    return -(-n // BLOCK)


def _matrix(t, what):
    if t.dim() != 2:
        raise ValueError(f"{what} must be 2-D (got {tuple(t.shape)})")


def _pitch(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), -(-t.shape[1] // 16) * 16)


def _no_trace(what):
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} cannot be traced: its result would be a constant of the trace")


def quantize_fp8(x: torch.Tensor, block_rows: int = 1, transposed: bool = False, out=None):
    """e4m3 codes and fp32 scales of a bf16 or fp32 matrix ``x`` (R, C) in blocks of ``block_rows`` x 128 (1 or 128):
    ``scale = absmax * (1 / 448) + 1e-12``, ``code = e4m3(x / scale)`` in fp32.  Returns ``(codes (R, C), scales (ceil(R / block_rows),
    ceil(C / 128)))``; with ``transposed`` (128 x 128 blocks) also the codes (C, R) and scales of the transpose.  Code rows
    start on 16-byte boundaries.  An infinity makes its block NaN, a NaN only itself.  Codes carry no gradient.  ``out``: tensors
    of an earlier call to write to."""
    nat = native.module() if out is None else None
    if nat is not None:
        res = nat.fp8_quantize(x, block_rows, transposed)
        if res is not None:
            return res
    _no_trace("quantize_fp8")
    _require_cuda(x)
    _matrix(x, "x")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK} (got {block_rows})")
    if transposed and block_rows != BLOCK:
        raise ValueError("transposed codes need 128 x 128 blocks")
    dt = _lib.dtype_id(x.dtype)
    R, C = x.shape
    if C > 1 and x.stride(1) != 1 or R > 1 and x.stride(0) < C:
        x = x.contiguous()
    dev = x.device
    sr = R if block_rows == 1 else _blocks(R)
    if out is None:
        out = (_empty_codes(R, C, dev), torch.empty(sr, _blocks(C), dtype=torch.float32, device=dev))
        if transposed:
            out += (_empty_codes(C, R, dev), torch.empty(_blocks(C), sr, dtype=torch.float32, device=dev))
    else:
        shapes = ((R, C), (sr, _blocks(C)), (C, R), (_blocks(C), sr))[:4 if transposed else 2]
        if (len(out) != len(shapes) or any(tuple(t.shape) != s or t.device != dev for t, s in zip(out, shapes))
                or any(t.dtype != (torch.float32 if i % 2 else _CODE) for i, t in enumerate(out))
                or any(t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1] for t in out[::2])
                or any(not t.is_contiguous() for t in out[1::2])):
            raise ValueError("out does not fit x: pass the tensors that an earlier call returned")
    a = _lib.ForgeFp8QuantizeArgs()
    a.x, a.rows, a.cols, a.ld_x = x.data_ptr(), R, C, x.stride(0) if R > 1 else C
    a.dtype, a.block_rows = dt, block_rows
    a.codes, a.ld_codes, a.scales = out[0].data_ptr(), _pitch(out[0]), out[1].data_ptr()
    if transposed:
        a.codes_t, a.ld_codes_t, a.scales_t = out[2].data_ptr(), _pitch(out[2]), out[3].data_ptr()
    with torch.cuda.device(dev):
        rc = _lib.load().forge_fp8_quantize(ctypes.byref(a), _lib.current_stream_ptr(dev))
    if rc:
        _lib.check(rc, "forge_fp8_quantize")
    # (for autograd: a graph that has saved these codes must not go on with other values)
    torch.autograd.graph.increment_version([t for t in out if not t.is_inference()])
    return tuple(out)


def fp8_matmul(x_codes, x_scales, w_codes, w_scales) -> torch.Tensor:
    """``Y = X W^T`` (M, N) bf16 of codes with scales: X (M, K) with scales (M, ceil(K / 128)), W (N, K) with scales
    (ceil(N / 128), ceil(K / 128)).  Code rows start on 16-byte boundaries (those of ``quantize_fp8`` do)."""
    _no_trace("fp8_matmul")
    _require_cuda(x_codes, x_scales, w_codes, w_scales)
    for t, what in ((x_codes, "x_codes"), (w_codes, "w_codes"), (x_scales, "x_scales"), (w_scales, "w_scales")):
        _matrix(t, what)
    (M, K), (N, K2) = x_codes.shape, w_codes.shape
    if x_codes.dtype != _CODE or w_codes.dtype != _CODE or x_scales.dtype != torch.float32 or w_scales.dtype != torch.float32:
        raise ValueError("codes must be float8_e4m3fn and scales float32")
    if K != K2 or tuple(x_scales.shape) != (M, _blocks(K)) or tuple(w_scales.shape) != (_blocks(N), _blocks(K)):
        raise ValueError(f"shape mismatch: x {tuple(x_codes.shape)} with scales {tuple(x_scales.shape)}, w {tuple(w_codes.shape)} "
                         f"with scales {tuple(w_scales.shape)}")
    for t, what in ((x_codes, "x_codes"), (w_codes, "w_codes")):
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{what} must have a contiguous last dimension (got strides {tuple(t.stride())})")
    dev = x_codes.device
    if any(t.device != dev for t in (x_scales, w_codes, w_scales)):
        raise ValueError("all tensors must be on the same device")
    y = torch.empty(M, N, dtype=torch.bfloat16, device=dev)
    if K == 0:
        return y.zero_()
    a = _lib.ForgeFp8ProductArgs()
    a.x_codes, a.x_scales, a.w_codes, a.w_scales, a.y = (t.data_ptr() for t in (x_codes, x_scales, w_codes, w_scales, y))
    a.M, a.N, a.K = M, N, K
    a.ld_x, a.ld_w, a.ld_y = _pitch(x_codes), _pitch(w_codes), N
    a.x_scale_row, a.x_scale_col = x_scales.stride()
    a.w_scale_row, a.w_scale_col = w_scales.stride()
    a.status = _lib.status_word(dev).data_ptr()
    with torch.cuda.device(dev):
        rc = _lib.load().forge_fp8_product(ctypes.byref(a), _lib.current_stream_ptr(dev))
    if rc:
        _lib.check(rc, "forge_fp8_product")
    return y


class Fp8Weight:
    """Codes and scales of a weight (N, K) in 128 x 128 blocks and, for input gradients, of its transpose, which a backward
    pass reads: call ``update_`` after it (autograd refuses to go on with codes that have been rewritten)."""

    __slots__ = ("codes", "scales", "codes_t", "scales_t")

    def __init__(self, codes, scales, codes_t=None, scales_t=None):
        if (codes_t is None) != (scales_t is None):
            raise ValueError("codes_t and scales_t belong together")
        self.codes, self.scales, self.codes_t, self.scales_t = codes, scales, codes_t, scales_t

    @classmethod
    def from_weight(cls, weight: torch.Tensor, transposed: bool = True):
        return cls(*quantize_fp8(weight.detach(), BLOCK, transposed))

    def update_(self, weight: torch.Tensor):
        """Quantise ``weight`` into the tensors held here (same shape and device)."""
        t = self.codes_t is not None
        quantize_fp8(weight.detach(), BLOCK, t, out=(self.codes, self.scales) + ((self.codes_t, self.scales_t) if t else ()))
        return self

    @property
    def shape(self):
        return self.codes.shape


def _product(x2d, codes, scales):
    return fp8_matmul(*quantize_fp8(x2d), codes, scales)


class _Fp8Linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, bias, w):
        ctx.save_for_backward(w.codes_t, w.scales_t)
        ctx.shape = x.shape
        ctx.bias_dtype = None if bias is None else bias.dtype
        return _forward(x, bias, w)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dy2d = dy.reshape(-1, dy.shape[-1])
        dx = None
        if ctx.needs_input_grad[0]:
            codes, scales = ctx.saved_tensors
            if codes.dim() != 2 or codes.dtype != _CODE:
                raise RuntimeError("fp8_linear: what was saved for the backward pass came back as something else")
            if _pitch(codes) % 16 or codes.data_ptr() % 16:     # (save_on_cpu brings them back without their pitch)
                codes = _empty_codes(*codes.shape, codes.device).copy_(codes)
            dx = _product(dy2d, codes, scales).view(ctx.shape)
        db = dy2d.sum(0).to(ctx.bias_dtype) if ctx.needs_input_grad[1] else None
        return dx, db, None


def _forward(x, bias, w):
    y = _product(x.reshape(-1, x.shape[-1]), w.codes, w.scales).view(*x.shape[:-1], w.shape[0])
    return y if bias is None else y + bias


def fp8_linear(x: torch.Tensor, weight: Fp8Weight, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x W^T (+ bias)`` with ``x`` (..., K) bf16 quantised by rows in the call; the input gradient is ``dY W`` with ``dY``
    quantised by rows in its turn, and needs the weight's transposed codes."""
    nat = native.module() if bias is None else None
    if nat is not None:
        y = nat.fp8_linear(x, weight.codes, weight.scales, weight.codes_t, weight.scales_t)
        if y is None and x.is_cuda and x.device.index not in _registered:
            _registered.add(x.device.index)
            nat.set_status_word(x.device.index, _lib.status_word(x.device).data_ptr())
            y = nat.fp8_linear(x, weight.codes, weight.scales, weight.codes_t, weight.scales_t)
        if y is not None:
            return y
    _no_trace("fp8_linear")
    _require_cuda(x, bias)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"fp8_linear takes bfloat16 activations (got {x.dtype})")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.shape[1] == 0:
        raise ValueError(f"x {tuple(x.shape)} does not fit a weight {tuple(weight.shape)}")
    if not (torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad))) and not native.followed(x, bias):
        return _forward(x, bias, weight)
    if x.requires_grad and weight.codes_t is None:
        raise ValueError("the input gradient needs the weight's transposed codes (Fp8Weight.from_weight(w, transposed=True))")
    return _Fp8Linear.apply(x, bias, weight)
