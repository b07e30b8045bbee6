"""What the norm, log-probability and AdamW operators refuse, and what the optimizer keeps: checked before any device is
asked for anything, so on the CPU."""
import ctypes
import math

import pytest
import torch

from spherical_distortion import functional as F
from spherical_distortion import nn
from sphmap import capi, optim


@pytest.mark.parametrize("call, message", [
    (lambda x: F.rms_norm(x.double()), "float32, bfloat16 or float16"),
    (lambda x: F.rms_norm(x.long()), "float32, bfloat16 or float16"),
    (lambda x: F.rms_norm(x, torch.ones(5)), r"size \(4,\)"),
    (lambda x: F.rms_norm(x, torch.ones(4).half()), "weight must be float32 or have"),
    (lambda x: F.rms_norm(x, torch.ones(8)[::2]), "weight must be contiguous"),
    (lambda x: F.rms_norm(x, dim=4), r"dim must be in \[-4, 3\]"),
    (lambda x: F.rms_norm(x, eps=-1e-3), "eps must be finite"),
    (lambda x: F.rms_norm(x, eps=math.nan), "eps must be finite"),
    (lambda x: F.rms_norm(x.transpose(0, 3)), "must be contiguous, or rows"),
    (lambda x: F.rms_norm(x[:, :, ::2]), "must be contiguous, or rows"),
    (lambda x: F.rms_norm(torch.ones(1, 4).expand(3, 4), dim=-1), "must be contiguous, or rows"),
    (lambda x: F.rms_norm(x, residual=x[:1]), "residual must have the input's size"),
    (lambda x: F.rms_norm(x, residual=x.half()), "residual must have the input's dtype"),
    (lambda x: F.rms_norm(x, residual=x.contiguous(memory_format=torch.channels_last)), "input's memory layout"),
    (lambda x: F.rms_norm(x[:, :0]), "at least one value along dim"),
    (lambda x: F.rms_norm(torch.tensor(1.0)), "at least one dimension"),
    (lambda x: F.rms_norm(x), "CUDA tensor"),
    (lambda x: F.rms_norm_quantized(x), "CUDA tensor"),
    (lambda x: F.rms_norm_quantized(x, torch.ones(3)), r"size \(4,\)"),
    (lambda x: F.token_log_probs(x, torch.zeros(2, 6, 10)), "target must be int64"),
    (lambda x: F.token_log_probs(x, torch.zeros(2, 6, 9).long()), "target must have the logits' size"),
    (lambda x: F.token_log_probs(x, torch.zeros(2, 10, 6).long().transpose(1, 2)), "target must be contiguous"),
    (lambda x: F.token_log_probs(x, torch.zeros(2, 6, 10).long(), top_k=5), r"top_k must be in \[0, 4\]"),
    (lambda x: F.token_log_probs(x, torch.zeros(2, 6, 10).long(), top_k=-1), "top_k must be in"),
    (lambda x: F.token_log_probs(x.double(), torch.zeros(2, 6, 10).long()), "float32, bfloat16 or float16"),
    (lambda x: F.token_log_probs(x, torch.zeros(2, 6, 10).long()), "CUDA tensor"),
])
def test_refusals(call, message):
    with pytest.raises(RuntimeError, match=message):
        call(torch.zeros(2, 4, 6, 10))


def _step(n=5, dtype=torch.float32, **changed):
    p = [torch.zeros(n, dtype=dtype)]
    a = dict(params=p, grads=[torch.zeros(n, dtype=dtype)], exp_avgs=[torch.zeros(n)], exp_avg_sqs=[torch.zeros(n)], step=1, lr=1e-3)
    a.update(changed)
    optim.adamw_step(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), **a)


E4 = torch.float8_e4m3fn


@pytest.mark.parametrize("changed, message", [
    (dict(grads=[]), "same length"),
    (dict(grads=[torch.zeros(4)]), "grad must have 5 values"),
    (dict(grads=[torch.zeros(5).half()]), "grad must be float32 or have"),
    (dict(grads=[torch.zeros(10)[::2]]), "grad must be contiguous"),
    (dict(exp_avgs=[torch.zeros(5).half()]), "exp_avg must be Float"),
    (dict(exp_avgs=[torch.zeros(5).to(E4)]), "exp_avg must be Float"),
    (dict(exp_avg_scales=[torch.zeros(1)]), "both moments have scales"),
    (dict(exp_avg_scales=[torch.zeros(1)], exp_avg_sq_scales=[torch.zeros(1)]), "exp_avg must be Float8_e4m3fn"),
    (dict(exp_avgs=[torch.zeros(5).to(E4)], exp_avg_sqs=[torch.zeros(5).to(E4)], exp_avg_scales=[torch.zeros(2)],
          exp_avg_sq_scales=[torch.zeros(1)]), "exp_avg_scale must have 1 values"),
    (dict(masters=[torch.zeros(5)]), "takes no master"),
    (dict(params=[torch.zeros(5).half()], masters=[torch.zeros(4)]), "master must have 5"),
    (dict(step=0), "step counts from 1"),
    (dict(lr=-1.0), "must not be negative"),
    (dict(lr=math.nan), "must not be negative"),
    (dict(lr=torch.tensor(1.0)), "lr on the device needs step"),
    (dict(betas=(1.0, 0.9)), "betas must be in"),
    (dict(params=[torch.zeros(5).double()]), "float32, bfloat16 or float16"),
    (dict(), "CUDA tensor"),
])
def test_adamw_step_refusals(changed, message):
    with pytest.raises(RuntimeError, match=message):
        _step(**changed)


@pytest.mark.parametrize("bad", [dict(state_bits=4), dict(lr=-1), dict(betas=(0.9, 1.0)), dict(eps=-1), dict(weight_decay=-0.1),
                                 dict(lr=torch.tensor(1e-3))])
def test_adamw_constructor_refusals(bad):
    with pytest.raises(ValueError):
        optim.AdamW([torch.zeros(3, requires_grad=True)], **bad)


def test_adamw_of_nothing():
    optim.adamw_step([], [], [], [], step=1, lr=1e-3)
    p = torch.zeros(3, requires_grad=True)
    o = optim.AdamW([p])
    o.step()                    # no gradient: nothing to do
    assert not o.state[p]


def test_adamw_state_dict_keeps_types():
    def filled():
        p = torch.zeros(300, dtype=torch.bfloat16, requires_grad=True)
        o = optim.AdamW([p], state_bits=8, master_weights=True)
        o._state_of(p, o.param_groups[0], False)
        return p, o
    p, o = filled()
    s = o.state[p]
    s["exp_avg"].copy_(torch.arange(300) % 7)
    s["exp_avg_scale"][1] = 0.25
    s["master"] += 1.00001
    s["step"] = 12
    q, o2 = filled()
    o2.load_state_dict(o.state_dict())
    t = o2.state[q]
    assert t["step"] == 12 and t["exp_avg"].dtype == E4 and t["master"].dtype == torch.float32
    for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "master"):
        assert torch.equal(t[k].float(), s[k].float()) and t[k].data_ptr() != s[k].data_ptr()


def test_modules_carry_their_parameters():
    m = nn.RMSNorm(7, eps=1e-5)
    assert list(m.state_dict()) == ["weight"] and torch.equal(m.weight, torch.ones(7))
    assert not list(nn.TokenLogProbs(top_k=2).parameters())


def test_c_entries_refuse_before_any_launch():
    null, one = ctypes.c_void_p(0), ctypes.c_void_p(256)
    i, d = capi._ints, ctypes.c_double
    fwd = lambda dtype=0, outer=4, C=8, inner=1, xs=8, eps=1e-6, x=one, out=one, res=null, sm=null: capi.lib.sph_rms_norm_forward(  # noqa: E731
        x, res, null, sm, out, null, null, *i(outer, C, inner, xs, 0), d(eps), dtype, 0, null)
    assert fwd(dtype=1) == 2 and fwd(dtype=9) == 2
    assert fwd(C=0) == 1 and fwd(inner=0) == 1 and fwd(outer=-1) == 1 and fwd(xs=7) == 1 and fwd(eps=-1) == 1 and fwd(x=null) == 1
    assert fwd(res=one) == 1 and fwd(sm=one) == 1 and fwd(eps=math.nan) == 1
    assert fwd(C=1 << 40) == 5 and fwd(outer=1 << 30, inner=1 << 30) == 5
    assert fwd(outer=0, x=null, out=null) == 0
    assert capi.lib.sph_rms_norm_workspace_bytes(*i(100, 64, 1)) >= 256 and capi.lib.sph_rms_norm_workspace_bytes(*i(1, 0, 1)) == 0
    lp = lambda dtype=0, outer=4, C=8, k=0, xs=8, x=one, top=null: capi.lib.sph_token_log_probs_forward(  # noqa: E731
        x, one, one, one, null, top, top, *i(outer, C, 1, xs, k, -100), dtype, null)
    assert lp(dtype=1) == 2 and lp(k=9) == 1 and lp(k=-1) == 1 and lp(C=0) == 1 and lp(xs=7) == 1 and lp(x=null) == 1 and lp(k=2) == 1
    assert lp(outer=0, x=null) == 0 and lp(outer=1 << 33) == 5
    step = lambda n=1, dtype=0, gdtype=0, bits=32, b1=0.9, step=1.0: capi.lib.sph_adamw_step(  # noqa: E731
        *i(n), null, null, null, null, null, null, null, null, dtype, gdtype, bits, d(1e-3), d(b1), d(0.999), d(1e-8), d(0.0), d(1.0),
        d(step), null, null, null)
    assert step() == 1 and step(n=0) == 0 and step(n=-1) == 1 and step(n=0, b1=1.0) == 1 and step(n=0, step=0.0) == 1
    assert step(bits=16) == 2 and step(dtype=1) == 2 and step(dtype=2, gdtype=3) == 2
