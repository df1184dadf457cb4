"""Bad arguments of the loss, multi-tensor and 8-bit entry points are refused by the host code before anything is launched
(no GPU is needed to see it), and CPU tensors by the wrappers; the rank exchange of a sliced vocabulary on two gloo ranks."""

import ctypes
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from forge_b200 import _lib

P = 1 << 20          # an aligned address that nothing reads


def logprobs(**kw):
    a = _lib.ForgeLogprobsArgs()
    for k, v in {**dict(logits=P, targets=P, rows=4, vocab=100, ld=100, vocab_start=0, vocab_total=100, ignore_index=-100,
                        temperature=1.0, dtype=_lib.DT_BF16, top_k=0, logprobs=P, entropy=P, lse=P), **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.FORGE_ERR_INVALID_ARG), (dict(dtype=7), _lib.FORGE_ERR_INVALID_ARG),
    (dict(top_k=33), _lib.FORGE_ERR_INVALID_ARG), (dict(top_k=2), _lib.FORGE_ERR_INVALID_ARG),
    (dict(temperature=0.0), _lib.FORGE_ERR_INVALID_ARG), (dict(temperature=float("nan")), _lib.FORGE_ERR_INVALID_ARG),
    (dict(temperature=float("inf")), _lib.FORGE_ERR_INVALID_ARG), (dict(temperature=1e-60), _lib.FORGE_ERR_INVALID_ARG),
    (dict(vocab=0), _lib.FORGE_ERR_SHAPE), (dict(ld=99), _lib.FORGE_ERR_SHAPE), (dict(vocab_start=-1), _lib.FORGE_ERR_SHAPE),
    (dict(vocab_start=1), _lib.FORGE_ERR_SHAPE), (dict(vocab_total=200), _lib.FORGE_ERR_INVALID_ARG),
    (dict(vocab_total=1 << 31, stats=P), _lib.FORGE_ERR_SHAPE), (dict(logits=None), _lib.FORGE_ERR_INVALID_ARG),
    (dict(logits=P + 1), _lib.FORGE_ERR_ALIGNMENT), (dict(targets=P + 4), _lib.FORGE_ERR_ALIGNMENT),
    (dict(entropy=P + 2), _lib.FORGE_ERR_ALIGNMENT), (dict(top_k=2, top_logprobs=P, top_ids=P + 4), _lib.FORGE_ERR_ALIGNMENT),
    (dict(top_k=2, stats=P, keys=P + 4), _lib.FORGE_ERR_ALIGNMENT), (dict(rows=1 << 31), _lib.FORGE_ERR_SHAPE),
    (dict(vocab=3, ld=3, vocab_total=3, top_k=4, top_logprobs=P, top_ids=P), _lib.FORGE_ERR_SHAPE)])
def test_logprobs_forward_refuses(kw, code):
    assert _lib.load().forge_logprobs_forward(ctypes.byref(logprobs(**kw)), None) == code
    assert _lib.last_error()


def test_logprobs_other_entries_refuse():
    lib = _lib.load()
    bad, shape = _lib.FORGE_ERR_INVALID_ARG, _lib.FORGE_ERR_SHAPE
    assert lib.forge_logprobs_forward(None, None) == bad
    assert lib.forge_logprobs_forward(ctypes.byref(logprobs(rows=0)), None) == 0
    assert lib.forge_logprobs_join(None, P, P, 2, None) == bad
    assert lib.forge_logprobs_join(ctypes.byref(logprobs()), None, P, 2, None) == bad
    assert lib.forge_logprobs_join(ctypes.byref(logprobs()), P, P, 0, None) == bad
    assert lib.forge_logprobs_join(ctypes.byref(logprobs(top_k=2)), P, P, 2, None) == bad
    assert lib.forge_logprobs_backward(None, P, P, P, 100, None) == bad
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs(lse=None)), P, P, P, 100, None) == bad
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs(entropy=None)), P, P, P, 100, None) == bad
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs()), P, P, None, 100, None) == bad
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs()), P, P, P, 99, None) == shape
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs()), P, P, P + 1, 100, None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs(lse=P + 2)), P, P, P, 100, None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs()), P + 2, P, P, 100, None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_logprobs_join(ctypes.byref(logprobs()), P + 2, P, 2, None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_logprobs_join(ctypes.byref(logprobs(top_k=2, top_logprobs=P, top_ids=P)), P, P + 4, 2, None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_logprobs_backward(ctypes.byref(logprobs(rows=0)), P, P, P, 100, None) == 0


def multi(count=1, mode=_lib.ST_F32, step=1, items=True, coef=None, device=None, **kw):
    arr = (_lib.ForgeMultiItem * max(count, 1))()
    for it in arr:
        for k, v in {**dict(param=P, grad=P, m=P, v=P, numel=64, param_dtype=1, grad_dtype=1), **kw}.items():
            setattr(it, k, v)
    a = _lib.ForgeMultiArgs()
    a.items = arr if items else None
    a.count, a.state_mode = count, mode
    a.hyper = _lib.ForgeHyper(1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, 0, step)
    a.grad_coef, a.hyper_device = coef, device
    a._keep = arr
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(count=-1), _lib.FORGE_ERR_INVALID_ARG), (dict(items=False), _lib.FORGE_ERR_INVALID_ARG),
    (dict(mode=_lib.ST_FP8_TENSOR), _lib.FORGE_ERR_UNSUPPORTED), (dict(mode=_lib.ST_NONE), _lib.FORGE_ERR_UNSUPPORTED),
    (dict(step=0), _lib.FORGE_ERR_INVALID_ARG), (dict(numel=-1), _lib.FORGE_ERR_INVALID_ARG),
    (dict(param_dtype=2), _lib.FORGE_ERR_INVALID_ARG), (dict(grad=None), _lib.FORGE_ERR_INVALID_ARG),
    (dict(mode=_lib.ST_INT8), _lib.FORGE_ERR_INVALID_ARG), (dict(param=P + 2), _lib.FORGE_ERR_ALIGNMENT),
    (dict(mode=_lib.ST_INT8, m_scale=P, v_scale=P + 2), _lib.FORGE_ERR_ALIGNMENT),
    (dict(coef=P + 1), _lib.FORGE_ERR_ALIGNMENT), (dict(device=P + 4), _lib.FORGE_ERR_ALIGNMENT),
    (dict(numel=1 << 50), _lib.FORGE_ERR_SHAPE)])
def test_multi_adamw_refuses(kw, code):
    if code == _lib.FORGE_ERR_SHAPE and not torch.cuda.is_available():
        code = (code, _lib.FORGE_ERR_CUDA)          # sized after the device has been asked for its SMs
    else:
        code = (code,)
    assert _lib.load().forge_multi_adamw(ctypes.byref(multi(**kw)), None) in code


def test_multi_norm_refuses():
    lib = _lib.load()
    bad = _lib.FORGE_ERR_INVALID_ARG
    it = (_lib.ForgeNormItem * 1)()
    it[0].grad, it[0].numel, it[0].dtype = P, 5000, _lib.DT_F32
    need = lib.forge_multi_norm_scratch_bytes(it, 1)
    assert need == 3 * 8 and lib.forge_multi_norm_scratch_bytes(None, 1) == 0
    assert lib.forge_multi_adamw(None, None) == bad and lib.forge_multi_adamw(ctypes.byref(multi(count=0)), None) == 0
    assert lib.forge_multi_norm(None, 1, 1.0, P, P, P, need, None) == bad
    assert lib.forge_multi_norm(it, 1, 1.0, None, P, P, need, None) == bad
    assert lib.forge_multi_norm(it, 1, 0.0, P, P, P, need, None) == bad
    assert lib.forge_multi_norm(it, 1, float("nan"), P, P, P, need, None) == bad
    assert lib.forge_multi_norm(it, 1, 1.0, P, P, P, need - 1, None) == _lib.FORGE_ERR_SCRATCH
    assert lib.forge_multi_norm(it, 1, 1.0, P, P, P + 4, need, None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_multi_norm(it, 1, 1.0, P + 2, P, P, need, None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_multi_norm(it, 1, 1.0, P, P + 2, P, need, None) == _lib.FORGE_ERR_ALIGNMENT
    it[0].dtype = 9
    assert lib.forge_multi_norm(it, 1, 1.0, P, P, P, need, None) == bad


def fill(cls, base, kw):
    a = cls()
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.FORGE_ERR_INVALID_ARG), (dict(dtype=5), _lib.FORGE_ERR_INVALID_ARG),
    (dict(block_rows=64), _lib.FORGE_ERR_INVALID_ARG), (dict(scales=None), _lib.FORGE_ERR_INVALID_ARG),
    (dict(codes_t=P, scales_t=P, ld_codes_t=200), _lib.FORGE_ERR_INVALID_ARG),
    (dict(codes_t=P, block_rows=128, ld_codes_t=200), _lib.FORGE_ERR_INVALID_ARG),
    (dict(codes_t=P, scales_t=P, block_rows=128, ld_codes_t=9), _lib.FORGE_ERR_INVALID_ARG),
    (dict(ld_x=99), _lib.FORGE_ERR_SHAPE), (dict(ld_codes=99), _lib.FORGE_ERR_SHAPE), (dict(x=P + 1), _lib.FORGE_ERR_ALIGNMENT),
    (dict(scales=P + 2), _lib.FORGE_ERR_ALIGNMENT),
    (dict(codes_t=P, scales_t=P + 2, block_rows=128, ld_codes_t=112), _lib.FORGE_ERR_ALIGNMENT), (dict(rows=0), 0), (dict(cols=0), 0)])
def test_quantize_refuses(kw, code):
    base = dict(x=P, rows=10, cols=100, ld_x=100, dtype=_lib.DT_BF16, block_rows=1, codes=P, ld_codes=112, scales=P)
    assert _lib.load().forge_fp8_quantize(ctypes.byref(fill(_lib.ForgeFp8QuantizeArgs, base, kw)), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), _lib.FORGE_ERR_INVALID_ARG), (dict(K=0), _lib.FORGE_ERR_SHAPE), (dict(K=1 << 32), _lib.FORGE_ERR_SHAPE),
    (dict(y=None), _lib.FORGE_ERR_INVALID_ARG), (dict(x_codes=P + 8), _lib.FORGE_ERR_ALIGNMENT),
    (dict(ld_w=264), _lib.FORGE_ERR_ALIGNMENT), (dict(ld_x=240), _lib.FORGE_ERR_SHAPE), (dict(ld_y=3), _lib.FORGE_ERR_SHAPE),
    (dict(y=P + 1), _lib.FORGE_ERR_ALIGNMENT), (dict(x_scales=P + 1), _lib.FORGE_ERR_ALIGNMENT), (dict(w_scales=P + 2), _lib.FORGE_ERR_ALIGNMENT),
    (dict(status=P + 2), _lib.FORGE_ERR_ALIGNMENT), (dict(M=0), 0), (dict(N=0), 0)])
def test_product_refuses(kw, code):
    base = dict(x_codes=P, x_scales=P, w_codes=P, w_scales=P, y=P, M=4, N=128, K=256, ld_x=256, ld_w=256, ld_y=128,
                x_scale_row=2, x_scale_col=1, w_scale_row=2, w_scale_col=1)
    assert _lib.load().forge_fp8_product(ctypes.byref(fill(_lib.ForgeFp8ProductArgs, base, kw)), None) == code
    assert _lib.load().forge_fp8_product(None, None) == _lib.FORGE_ERR_INVALID_ARG


@pytest.mark.parametrize("xkw,pkw,code", [
    (dict(block_rows=128), {}, _lib.FORGE_ERR_INVALID_ARG), (dict(rows=5), {}, _lib.FORGE_ERR_INVALID_ARG),
    (dict(cols=128), {}, _lib.FORGE_ERR_INVALID_ARG), (dict(codes=P + 256), {}, _lib.FORGE_ERR_INVALID_ARG),
    (dict(ld_codes=272), {}, _lib.FORGE_ERR_INVALID_ARG), ({}, dict(x_scale_row=1, x_scale_col=4), _lib.FORGE_ERR_INVALID_ARG),
    (dict(scales=P + 64), {}, _lib.FORGE_ERR_INVALID_ARG), ({}, dict(y=None), _lib.FORGE_ERR_INVALID_ARG),
    ({}, dict(ld_w=264), _lib.FORGE_ERR_ALIGNMENT), (dict(rows=0), dict(M=0), 0)])
def test_linear_refuses(xkw, pkw, code):
    x = dict(x=P, rows=4, cols=256, ld_x=256, dtype=_lib.DT_BF16, block_rows=1, codes=P, ld_codes=256, scales=P)
    base = dict(x_codes=P, x_scales=P, w_codes=P, w_scales=P, y=P, M=4, N=128, K=256, ld_x=256, ld_w=256, ld_y=128,
                x_scale_row=2, x_scale_col=1, w_scale_row=2, w_scale_col=1)
    a, b = fill(_lib.ForgeFp8QuantizeArgs, x, xkw), fill(_lib.ForgeFp8ProductArgs, base, pkw)
    assert _lib.load().forge_fp8_linear(ctypes.byref(a), ctypes.byref(b), None) == code
    assert _lib.load().forge_fp8_linear(None, ctypes.byref(b), None) == _lib.FORGE_ERR_INVALID_ARG


def test_wrappers_refuse_cpu_tensors():
    from forge_b200.fp8 import Fp8Weight, fp8_linear, fp8_matmul, quantize_fp8
    from forge_b200.loss import logprob_parts, token_logprobs
    from forge_b200.multi_tensor import MultiTensorAdamW, multi_tensor_adamw, multi_tensor_grad_norm
    x, t = torch.zeros(4, 16), torch.zeros(4, dtype=torch.long)
    c = torch.zeros(4, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(4, 1)
    p = torch.nn.Parameter(x.clone())
    p.grad = x
    for f in (lambda: token_logprobs(x, t), lambda: logprob_parts(x, t, 0, 16), lambda: multi_tensor_adamw([x], [x], [x], [x]),
              lambda: multi_tensor_grad_norm([x]), lambda: MultiTensorAdamW([p]).step(), lambda: quantize_fp8(x),
              lambda: fp8_matmul(c, s, c, s[:1]), lambda: fp8_linear(x.bfloat16(), Fp8Weight(c, s[:1]))):
        with pytest.raises(_lib.ForgeLibraryError):
            f()


def _gather_worker(rank, world, port, result):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from forge_b200.loss import _gather_parts
        stats = torch.arange(15.0).view(3, 5) + 100 * rank
        keys = torch.arange(6).view(3, 2) + 1000 * rank
        s, k = _gather_parts(stats, keys, dist.group.WORLD)
        for r in range(world):
            assert torch.equal(s[r], torch.arange(15.0).view(3, 5) + 100 * r)
            assert torch.equal(k[r], torch.arange(6).view(3, 2) + 1000 * r)
        _, none = _gather_parts(stats, keys[:, :0], dist.group.WORLD)
        assert none.shape == (world, 3, 0)
        result.put((rank, "ok"))
    except BaseException as e:
        result.put((rank, repr(e)))
    finally:
        dist.destroy_process_group()


def test_parts_are_gathered_in_rank_order():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ctx = mp.get_context("spawn")
    result = ctx.SimpleQueue()
    procs = [ctx.Process(target=_gather_worker, args=(r, 2, port, result)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(result.get() for _ in range(2))
    for p in procs:
        p.join(60)
    assert got == {0: "ok", 1: "ok"}, got


def test_logprobs_row_maxima_and_sums_are_checked():
    lib = _lib.load()
    for kw, code in ((dict(lse=None, row_max=P), _lib.FORGE_ERR_INVALID_ARG), (dict(lse=None, log_sum=P), _lib.FORGE_ERR_INVALID_ARG),
                     (dict(row_max=P + 2, log_sum=P), _lib.FORGE_ERR_ALIGNMENT), (dict(row_max=P, log_sum=P + 1), _lib.FORGE_ERR_ALIGNMENT)):
        assert lib.forge_logprobs_backward(ctypes.byref(logprobs(**kw)), P, P, P, 100, None) == code
    assert lib.forge_logprobs_forward(ctypes.byref(logprobs(row_max=P + 2)), None) == _lib.FORGE_ERR_ALIGNMENT
    assert lib.forge_logprobs_join(ctypes.byref(logprobs(log_sum=P + 2)), P, P, 2, None) == _lib.FORGE_ERR_ALIGNMENT


@pytest.mark.parametrize("mode", ["f32", "bf16", "int8", "fp8_block"])
def test_loading_a_checkpoint_keeps_the_moments_where_they_are(mode):
    """A captured step goes on with the tensors that it was captured with: a checkpoint is loaded into them, and those of a
    parameter that it lacks start again from what the first step begins with."""
    import copy
    from forge_b200.multi_tensor import MultiTensorAdamW
    params = [torch.nn.Parameter(torch.ones(3, 70)), torch.nn.Parameter(torch.ones(5))]
    opt = MultiTensorAdamW(params, state_mode=mode)
    fresh = [{k: v.clone() if k != "step" else v for k, v in opt._state_of(p, mode).items()} for p in params]
    for p in params:
        for k, v in opt.state[p].items():
            if k == "step":
                opt.state[p][k] = 7
            else:
                v.view(torch.uint8).fill_(9)
    before = {p: dict(opt.state[p]) for p in params}
    saved = copy.deepcopy(opt.state_dict())
    del saved["state"][1]
    opt.load_state_dict(saved)
    for p in params:
        for k, v in before[p].items():
            if k != "step":
                assert opt.state[p][k] is v
    assert opt.state[params[0]]["step"] == 7 and opt.state[params[1]]["step"] == 0
    for k, v in fresh[1].items():
        if k != "step":
            assert torch.equal(opt.state[params[1]][k].view(torch.uint8), v.view(torch.uint8))
            assert (opt.state[params[0]][k].view(torch.uint8) == 9).all()


def test_a_checkpoint_that_does_not_fit_a_captured_step_is_refused():
    import copy
    from forge_b200.multi_tensor import MultiTensorAdamW
    p = torch.nn.Parameter(torch.ones(3, 70))
    old, new = MultiTensorAdamW([p], lr=0.5, state_mode="int8"), MultiTensorAdamW([p], lr=1.0, state_mode="f32")
    old._state_of(p, "int8"), new._state_of(p, "f32")
    saved = copy.deepcopy(old.state_dict())
    new.enable_device_hyper()                          # what a captured step reads may be in use
    state = new.state[p]["exp_avg"]
    with pytest.raises(ValueError, match="exp_avg"):
        new.load_state_dict(saved)
    assert new.state[p]["exp_avg"] is state and new.param_groups[0]["lr"] == 1.0
    again = MultiTensorAdamW([p], lr=1.0, state_mode="f32")
    again._state_of(p, "f32")
    again.load_state_dict(saved)                       # without one it is taken as it is
    assert again.state[p]["exp_avg"].dtype == torch.int8 and again.param_groups[0]["state_mode"] == "int8"


@pytest.mark.parametrize("temperature", [3.4e-39, 1e-37, 1e37, 1e300])
def test_temperatures_that_leave_fp32_are_refused(temperature):
    """log2 e / temperature has to be a number, and (lowest logit) / temperature far below the exponential's range."""
    bad, a = _lib.FORGE_ERR_INVALID_ARG, logprobs(temperature=temperature)
    assert _lib.load().forge_logprobs_forward(ctypes.byref(a), None) == bad
    assert _lib.load().forge_logprobs_join(ctypes.byref(a), P, P, 2, None) == bad
    assert _lib.load().forge_logprobs_backward(ctypes.byref(a), P, P, P, 100, None) == bad
    from forge_b200.loss import token_logprobs
    with pytest.raises(ValueError, match="temperature"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long), temperature=temperature)


def test_a_refused_parameter_group_is_not_added():
    from forge_b200.multi_tensor import MultiTensorAdamW
    opt = MultiTensorAdamW([torch.nn.Parameter(torch.ones(3))], state_mode="int8")
    with pytest.raises(ValueError, match="state_mode"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(4))], state_mode="fp4"))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(4))]))
    assert [g["state_mode"] for g in opt.param_groups] == ["int8", "int8"]
