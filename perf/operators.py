"""Measured cases of three sets of operators around the fused linears: the loss at the logits, the optimizer step of
the parameters that are not fused linears, and linear products in 8-bit floating point.

  logprobs   log probability of a given token per row of logits, the row's entropy and its most likely alternatives;
             `train` adds the gradient of both with respect to the logits
  adamw      one AdamW step over a list of tensors of any sizes, moments in fp32, int8 or e4m3 (one scale for each 64
             consecutive elements), optionally with the gradients clipped by their common norm
  quantize   e4m3 codes with one fp32 scale for each 1 x 128 block of a row (activations, gradients) or each 128 x 128
             block (weights, both ways round)
  product    Y = X W^T: X (bf16) is quantised by rows in the call, W comes as codes and scales; `train` adds dX = dY W

`run` computes the plain form with elementary torch operations in fp32; where `own` is true it calls forge_b200.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LR, BETA1, BETA2, EPS, DECAY, STEP = 3e-4, 0.9, 0.95, 1e-8, 0.1, 7
IGNORE = -100


def listed():
    return [
        # one sequence decoding: the sampled token's log probability and five alternatives; latency is what counts
        {"name": "logprobs-decode", "op": "logprobs", "rows": 1, "vocab": 128256, "dtype": "bf16", "top": 5, "train": False,
         "masked": False, "temperature": 1.0},
        # a batch of sequences decoding under a grammar that masks half of the vocabulary, twenty alternatives
        {"name": "logprobs-serve", "op": "logprobs", "rows": 64, "vocab": 151936, "dtype": "f32", "top": 20, "train": False,
         "masked": True, "temperature": 0.7},
        # the next-token loss of one 512-token sequence and its gradient
        {"name": "logprobs-train", "op": "logprobs", "rows": 511, "vocab": 128256, "dtype": "bf16", "top": 0, "train": True,
         "masked": False, "temperature": 1.0},
        # a policy-gradient step over a long batch: log probabilities with an entropy bonus, an odd number of rows
        {"name": "logprobs-train-long", "op": "logprobs", "rows": 4095, "vocab": 151936, "dtype": "bf16", "top": 0,
         "train": True, "masked": False, "temperature": 0.9},
        # the norm weights of a decoder: many tiny tensors, where launches are all that there is
        {"name": "adamw-norms", "op": "adamw", "mode": "f32", "count": 65, "numel": 4096, "odd": False, "rows": 0, "cols": 0,
         "param": "bf16", "clip": 0.0},
        # norms, biases and a small embedding of odd sizes, int8 moments
        {"name": "adamw-odd-int8", "op": "adamw", "mode": "int8", "count": 129, "numel": 14336, "odd": True, "rows": 5001,
         "cols": 1025, "param": "bf16", "clip": 0.0},
        # fp32 weights and moments, clipped by the common norm
        {"name": "adamw-clip-f32", "op": "adamw", "mode": "f32", "count": 65, "numel": 5120, "odd": False, "rows": 32064,
         "cols": 4096, "param": "f32", "clip": 1.0},
        # the embedding and the norms of an 8B decoder, e4m3 moments
        {"name": "adamw-embedding-fp8", "op": "adamw", "mode": "fp8_block", "count": 65, "numel": 4096, "odd": False,
         "rows": 128256, "cols": 4096, "param": "bf16", "clip": 0.0},
        # the activations of 512 tokens in front of a projection
        {"name": "quantize-rows", "op": "quantize", "rows": 512, "cols": 4096, "block_rows": 1},
        # a projection's weight after its update, as it is and transposed (for the input gradient)
        {"name": "quantize-weight", "op": "quantize", "rows": 14336, "cols": 4096, "block_rows": 128},
        # one token through a projection: the weight's codes are all that is read
        {"name": "product-decode", "op": "product", "m": 1, "n": 14336, "k": 4096, "train": False},
        # a projection's forward product and input gradient over 4096 tokens
        {"name": "product-train", "op": "product", "m": 4096, "n": 14336, "k": 4096, "train": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "adamw", "adamw", "quantize", "product", "product"])
    if op == "logprobs":
        vocab = _log_uniform(rng, 1000, 160000)
        return {"op": op, "rows": min(_log_uniform(rng, 1, 4095), 4095 * 151936 // vocab), "vocab": vocab,
                "dtype": rng.choice(["bf16", "f32"]) if vocab < 100000 else "bf16", "top": rng.choice([0, 1, 5, 20, 32]),
                "train": rng.random() < 0.5, "masked": rng.random() < 0.3, "temperature": round(rng.uniform(0.5, 1.5), 2)}
    if op == "adamw":
        return {"op": op, "mode": rng.choice(["f32", "bf16", "int8", "fp8_block"]), "count": _log_uniform(rng, 1, 300),
                "numel": _log_uniform(rng, 64, 20000), "odd": rng.random() < 0.6, "rows": _log_uniform(rng, 1, 30000),
                "cols": _log_uniform(rng, 1, 6000), "param": rng.choice(["bf16", "f32"]), "clip": rng.choice([0.0, 0.0, 1.0])}
    if op == "quantize":
        block = rng.choice([1, 128])
        return {"op": op, "rows": _log_uniform(rng, 1, 14336), "cols": _log_uniform(rng, 16, 4096), "block_rows": block}
    return {"op": op, "m": _log_uniform(rng, 1, 4096), "n": 16 * _log_uniform(rng, 4, 896), "k": 16 * _log_uniform(rng, 8, 256),
            "train": rng.random() < 0.4}


def _sizes(case):
    """The shapes of an adamw case's tensors, the largest first."""
    shapes = [(case["rows"], case["cols"])] if case["rows"] else []
    step = 7 if case["odd"] else 0
    return shapes + [(max(1, case["numel"] - step * (i % 13)),) for i in range(case["count"])]


def _quantize_plain(x, block_rows):
    """Codes and scales of `x` in blocks of block_rows x 128: scale = absmax / 448 + 1e-12, code = e4m3(x / scale)."""
    r, c = x.shape
    rp, cp = -(-r // block_rows) * block_rows, -(-c // 128) * 128
    f = torch.zeros(rp, cp, dtype=torch.float32, device=x.device)
    f[:r, :c] = x
    blocks = f.view(rp // block_rows, block_rows, cp // 128, 128)
    scale = blocks.abs().amax(dim=(1, 3)) / E4M3_MAX + 1e-12
    q = (blocks / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(rp, cp)[:r, :c].contiguous(), scale


def _dequantize_plain(codes, scale, block_rows):
    r, c = codes.shape
    return codes.float() * scale.repeat_interleave(block_rows, 0)[:r].repeat_interleave(128, 1)[:, :c]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed * 1000003 + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = dict(case)
    if case["op"] == "logprobs":
        rows, vocab, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        logits = torch.empty(rows, vocab, dtype=dt, device=dev)
        for i in range(0, rows, 512):        # peaked rows, as a trained model's are: a few tokens far above the rest
            part = randn(min(512, rows - i), vocab) * 2.5
            part += 12.0 * (torch.rand(part.shape, generator=g, device=dev) < 3.0 / vocab)
            if case["masked"]:
                part = part.masked_fill(torch.rand(part.shape, generator=g, device=dev) < 0.5, -math.inf)
            logits[i:i + 512] = part.to(dt)
        targets = torch.randint(0, vocab, (rows,), generator=g, device=dev)
        if rows > 16:
            targets[5::16] = IGNORE          # padding
        s.update(logits=logits.requires_grad_(case["train"]), targets=targets, g_logprob=randn(rows) / rows,
                 g_entropy=randn(rows).abs() * -0.01 / rows)
    elif case["op"] == "adamw":
        pdt, mode = DTYPES[case["param"]], case["mode"]
        shapes = _sizes(case)
        params = [(randn(*n) * 0.02).to(pdt) for n in shapes]
        grads = [(randn(*n) * 1e-2).to(pdt) for n in shapes]
        if mode in ("f32", "bf16"):
            sdt = DTYPES[mode]
            s.update(m=[(randn(*n) * 1e-3).to(sdt) for n in shapes], v=[(randn(*n).square() * 1e-5).to(sdt) for n in shapes],
                     m_scale=None, v_scale=None)
        else:
            blocks = [-(-math.prod(n) // 64) for n in shapes]
            if mode == "int8":
                m = [(randn(*n) * 40).round().clamp(-127, 127).to(torch.int8) for n in shapes]
                v = [(randn(*n).abs() * 40).round().clamp(0, 127).to(torch.int8) for n in shapes]
                top = 127.0
            else:
                m = [(randn(*n) * 140).clamp(-448, 448).to(torch.float8_e4m3fn) for n in shapes]
                v = [(randn(*n).abs() * 140).clamp(0, 448).to(torch.float8_e4m3fn) for n in shapes]
                top = 448.0
            s.update(m=m, v=v, m_scale=[(1 + torch.rand(b, generator=g, device=dev)) * 2e-3 / top for b in blocks],
                     v_scale=[(1 + torch.rand(b, generator=g, device=dev)) * 2e-5 / top for b in blocks])
        s.update(params=params, grads=grads)
    elif case["op"] == "quantize":
        x = randn(case["rows"], case["cols"])
        s["x"] = (x * (0.02 if case["block_rows"] == 128 else 1.0)).bfloat16()
    else:
        m, n, k = case["m"], case["n"], case["k"]
        x = randn(m, k)
        x[:, 7::1024] *= 30.0                # a few channels with large activations
        w = (randn(n, k) * 0.02).bfloat16()
        s["x"] = x.bfloat16().requires_grad_(case["train"])
        s["w_codes"], s["w_scales"] = _quantize_plain(w, 128)
        if case["train"]:
            s["wt_codes"], s["wt_scales"] = s["w_codes"].t().contiguous(), s["w_scales"].t().contiguous()
            s["dy"] = (randn(m, n) * 1e-2).bfloat16()
    return s


def _blocks64(t):
    """A tensor's elements in blocks of 64 consecutive ones, the last filled up with zeros (fp32)."""
    flat = t.reshape(-1).float()
    out = torch.zeros(-(-flat.numel() // 64) * 64, dtype=torch.float32, device=t.device)
    out[:flat.numel()] = flat
    return out.view(-1, 64)


def _values(codes, scale):
    """What a tensor of 8-bit codes stands for, in bf16."""
    return (_blocks64(codes) * scale[:, None]).view(-1)[:codes.numel()].bfloat16().view(codes.shape)


def _run_logprobs(s):
    if own:
        from forge_b200.loss import token_logprobs
        out = token_logprobs(s["logits"], s["targets"], top_k=s["top"], temperature=s["temperature"], ignore_index=IGNORE)
        grad = None
        if s["train"]:
            (grad,) = torch.autograd.grad((out.logprobs, out.entropy), (s["logits"],), (s["g_logprob"], s["g_entropy"]))
        return {"logprobs": out.logprobs.detach(), "entropy": out.entropy.detach(), "top_logprobs": out.top_logprobs,
                "top_ids": out.top_ids, "grad": grad}
    x, t = s["logits"].detach().float(), s["targets"]
    kept = t != IGNORE
    at = torch.where(kept, t, 0)[:, None]
    z = x / s["temperature"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    z -= total.log()
    p = e.div_(total)
    logprobs = torch.where(kept, z.gather(1, at)[:, 0], 0.0)
    entropy = -torch.where(p > 0, p * z, 0.0).sum(1)
    ids = top = grad = None
    if s["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
        top = z.gather(1, ids)
    if s["train"]:
        gl, ge = torch.where(kept, s["g_logprob"], 0.0)[:, None], s["g_entropy"][:, None]
        grad = -gl * p - ge * torch.where(p > 0, p * (z + entropy[:, None]), 0.0)
        grad.scatter_add_(1, at, gl)
        grad = (grad / s["temperature"]).to(s["logits"].dtype)
    return {"logprobs": logprobs, "entropy": entropy, "top_logprobs": top, "top_ids": ids, "grad": grad}


def _adamw_plain(s):
    norm, coef = None, 1.0
    if s["clip"]:
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
        coef = torch.clamp(s["clip"] / (norm + 1e-6), max=1.0)
    quantized = s["mode"] in ("int8", "fp8_block")
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        g = g.float() * coef
        m, v = s["m"][i], s["v"][i]
        if quantized:
            g = _blocks64(g)
            mf, vf = _blocks64(m) * s["m_scale"][i][:, None], (_blocks64(v) * s["v_scale"][i][:, None]).clamp(min=1e-8)
            pf = _blocks64(p)
        else:
            mf, vf, pf = m.float(), v.float(), p.float()
        mf = mf * BETA1 + g * (1 - BETA1)
        vf = vf * BETA2 + (g * (1 - BETA2)) * g
        update = (mf / (1 - BETA1 ** STEP)) / ((vf / (1 - BETA2 ** STEP)).sqrt() + EPS)
        pf = pf * (1 - LR * DECAY) - LR * update
        p.copy_(pf.view(-1)[:p.numel()].view(p.shape))
        if not quantized:
            m.copy_(mf)
            v.copy_(vf)
            continue
        live = (torch.arange(pf.numel(), device=p.device) < p.numel()).view(-1, 64)
        for f, codes, scale in ((mf, m, s["m_scale"][i]), (vf, v, s["v_scale"][i])):
            top = 127.0 if s["mode"] == "int8" else E4M3_MAX
            f = f * live
            scale.copy_(f.abs().amax(1) / top + 1e-12)
            q = f / scale[:, None]
            q = q.round().clamp(-127, 127) if s["mode"] == "int8" else q.clamp(-top, top)
            codes.copy_(q.view(-1)[:p.numel()].view(p.shape).to(codes.dtype))
    return norm


def _run_adamw(s):
    if own:
        from forge_b200.multi_tensor import multi_tensor_adamw
        norm = multi_tensor_adamw(s["params"], s["grads"], s["m"], s["v"], s["m_scale"], s["v_scale"], lr=LR, beta1=BETA1,
                                  beta2=BETA2, eps=EPS, weight_decay=DECAY, step=STEP, max_norm=s["clip"] or None)
    else:
        norm = _adamw_plain(s)
    # the largest tensor, the first and the last of the others: 64 outputs are looked at
    some = [0, 1, len(s["params"]) - 1] if len(s["params"]) > 2 else list(range(len(s["params"])))
    out = {"norm": norm, "params": s["params"][:24]}
    for name in ("m", "v"):
        codes = [s[name][i] for i in some]
        if s["mode"] == "int8":
            codes = [_values(c, s[name + "_scale"][i]) for c, i in zip(codes, some)]
        out[name] = codes
        if s["m_scale"] is not None:
            out[name + "_scale"] = [s[name + "_scale"][i] for i in some]
    return out


def _run_quantize(s):
    x, block = s["x"], s["block_rows"]
    if own:
        from forge_b200.fp8 import quantize_fp8
        if block == 1:
            return quantize_fp8(x)
        return quantize_fp8(x, block_rows=128, transposed=True)
    codes, scale = _quantize_plain(x, block)
    return (codes, scale) if block == 1 else (codes, scale, codes.t().contiguous(), scale.t().contiguous())


def _run_product(s):
    x = s["x"]
    if own:
        from forge_b200.fp8 import Fp8Weight, fp8_linear
        y = fp8_linear(x, Fp8Weight(s["w_codes"], s["w_scales"], s.get("wt_codes"), s.get("wt_scales")))
        if not s["train"]:
            return {"y": y}
        return {"y": y.detach(), "dx": torch.autograd.grad(y, x, s["dy"])[0]}
    w = _dequantize_plain(s["w_codes"], s["w_scales"], 128)
    out = {"y": (_dequantize_plain(*_quantize_plain(x.detach(), 1), 1) @ w.t()).bfloat16()}
    if s["train"]:
        out["dx"] = (_dequantize_plain(*_quantize_plain(s["dy"], 1), 1) @ w).bfloat16()
    return out


def run(state):
    return {"logprobs": _run_logprobs, "adamw": _run_adamw, "quantize": _run_quantize, "product": _run_product}[state["op"]](state)


def work(case):
    if case["op"] == "logprobs":
        rows, n = case["rows"], case["rows"] * case["vocab"]
        b = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * b * (2 if case["train"] else 1) + rows * (8 + 8 + 12 * case["top"] + (8 if case["train"] else 0)),
                "flops": n * (10 if case["train"] else 6)}
    if case["op"] == "adamw":
        n = sum(math.prod(x) for x in _sizes(case))
        pb = 2 if case["param"] == "bf16" else 4
        sb = {"f32": 4, "bf16": 2}.get(case["mode"], 1 + 4 / 64)
        return {"bytes": n * (3 * pb + 4 * sb), "flops": n * 16}
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        if case["block_rows"] == 1:
            return {"bytes": n * 3 + case["rows"] * -(-case["cols"] // 128) * 4, "flops": n * 3}
        return {"bytes": n * 4 + 8 * -(-case["rows"] // 128) * -(-case["cols"] // 128), "flops": n * 3}
    m, n, k = case["m"], case["n"], case["k"]
    one = m * k * 2 + n * k + 4 * -(-n // 128) * -(-k // 128) + m * n * 2
    return {"bytes": one * (2 if case["train"] else 1), "flops": 2 * m * n * k * (2 if case["train"] else 1)}


def _e4m3(x):
    """Nearest e4m3 values (ties to even), in 64 bits."""
    a = x.abs().clamp(max=E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=E4M3_MAX)


def _exact_blocks(x, block_rows):
    """(codes' values, scales, what they stand for) of a matrix in 64 bits."""
    r, c = x.shape
    f = torch.nn.functional.pad(x.double(), (0, -c % 128, 0, -r % block_rows))
    b = f.unfold(0, block_rows, block_rows).unfold(1, 128, 128)           # (R, C, block_rows, 128)
    scale = b.abs().amax((2, 3)) / 448 + 1e-12
    q = _e4m3(b / scale[:, :, None, None])

    def whole(t):
        return t.permute(0, 2, 1, 3).reshape(f.shape)[:r, :c]

    return whole(q), scale, whole(q * scale[:, :, None, None])


def _exact_logprobs(s):
    logits, t = s["logits"].detach(), s["targets"]
    parts = {"logprobs": [], "entropy": [], "top_logprobs": [], "top_ids": [], "grad": []}
    for i in range(0, logits.shape[0], 256):
        x, tt = logits[i:i + 256].double(), t[i:i + 256]
        lp = torch.log_softmax(x / s["temperature"], 1)
        p, rows = lp.exp(), torch.arange(x.shape[0], device=x.device)
        kept = (tt != IGNORE).double()
        ent = -torch.nansum(p * lp.clamp(min=-1e300), 1)
        parts["logprobs"].append(torch.where(kept > 0, lp[rows, tt.clamp(min=0)], torch.zeros_like(ent)))
        parts["entropy"].append(ent)
        if s["top"]:
            v, ids = torch.sort(x, dim=1, descending=True, stable=True)
            parts["top_ids"].append(ids[:, :s["top"]])
            parts["top_logprobs"].append(torch.take_along_dim(lp, ids[:, :s["top"]], 1))
        if s["train"]:
            hot = torch.zeros_like(p)
            hot[rows, tt.clamp(min=0)] = 1
            a, b = (s["g_logprob"][i:i + 256].double() * kept)[:, None], s["g_entropy"][i:i + 256].double()[:, None]
            parts["grad"].append((a * (hot - p) - b * p * (lp.clamp(min=-1e300) + ent[:, None])) / s["temperature"])
    return {k: torch.cat(v) if v else None for k, v in parts.items()}


def _exact_adamw(s):
    coef, norm = 1.0, None
    if s["clip"]:
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))
        coef = min(1.0, s["clip"] / (norm + 1e-6))
        norm = torch.tensor(norm, dtype=torch.float64, device="cuda")
    some = [0, 1, len(s["params"]) - 1] if len(s["params"]) > 2 else list(range(len(s["params"])))
    out = {"norm": norm, "params": [], "m": [], "v": []}
    eight = s["mode"] in ("int8", "fp8_block")
    if eight:
        out.update(m_scale=[], v_scale=[])
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        if i >= 24 and i not in some:
            continue
        n = p.numel()
        g, w = g.double().view(-1) * coef, p.double().view(-1)
        m, v = s["m"][i].double().view(-1), s["v"][i].double().view(-1)
        if eight:
            m = m * s["m_scale"][i].double().repeat_interleave(64)[:n]
            v = torch.clamp_min(v * s["v_scale"][i].double().repeat_interleave(64)[:n], 1e-8)
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g ** 2
        w = w - LR * DECAY * w - LR * (m / (1 - BETA1 ** STEP)) / (torch.sqrt(v / (1 - BETA2 ** STEP)) + EPS)
        if i < 24:
            out["params"].append(w.view(p.shape))
        if i not in some:
            continue
        for name, f in (("m", m), ("v", v)):
            if eight:
                b = torch.nn.functional.pad(f, (0, -n % 64)).view(-1, 64)
                scale = b.abs().amax(1, keepdim=True) / (127 if s["mode"] == "int8" else 448) + 1e-12
                q = torch.round(b / scale) * scale if s["mode"] == "int8" else _e4m3(b / scale)
                out[name + "_scale"].append(scale[:, 0])
                f = q.reshape(-1)[:n]
            out[name].append(f.view(p.shape))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"] == "quantize":
        codes, scale, _ = _exact_blocks(s["x"], case["block_rows"])
        return (codes, scale) if case["block_rows"] == 1 else (codes, scale, codes.t(), scale.t())
    n, k = s["w_codes"].shape
    up = s["w_scales"].double()
    w = s["w_codes"].double() * torch.kron(up, torch.ones(128, 128, dtype=torch.float64, device=up.device))[:n, :k]
    out = {"y": _exact_blocks(s["x"].detach(), 1)[2] @ w.t()}
    if case["train"]:
        out["dx"] = _exact_blocks(s["dy"], 1)[2] @ w
    return out
