"""Traces and forward-mode differentiation of the operators around the convolutions: recorded or refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from spherical_distortion import functional as F

pytestmark = pytest.mark.gpu
EPS = 1e-6


def values(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def test_quantized_norm_refuses_tangents():
    """Of any of its arguments, as rms_norm does."""
    x, w = values((3, 4), 1), values((4,), 2)
    with fwAD.dual_level():
        for args in ((fwAD.make_dual(x, x), None, None), (x, fwAD.make_dual(w, w), None), (x, None, fwAD.make_dual(x, x))):
            with pytest.raises(NotImplementedError, match="jvp"):
                F.rms_norm_quantized(*args, EPS, 1)


@pytest.mark.parametrize("residual", [False, True])
def test_traced_quantized_norm(residual):
    w, r = values((30,), 2), values((4, 30), 4) if residual else None
    call = lambda a: F.rms_norm_quantized(a, w, r, EPS, -1)  # noqa: E731
    traced = torch.jit.trace(call, (values((4, 30), 1),), check_trace=False)
    y = values((4, 30), 3)
    for _ in range(2):
        junk = [torch.full((4, 30), 7.0, device="cuda") for _ in range(20)]   # (memory that an allocation alone would show)
        del junk
        got, want = traced(y), call(y)
        assert len(got) == len(want) == 2 + residual
        for a, b in zip(got, want):
            assert a.dtype == b.dtype and torch.equal(a.float(), b.float())


@pytest.mark.parametrize("k", [0, 3])
def test_traced_log_probs(k):
    target = torch.zeros(4, dtype=torch.int64, device="cuda")
    call = lambda a: tuple(t for t in F.token_log_probs(a, target, -1, k) if t is not None)  # noqa: E731
    traced = torch.jit.trace(call, (values((4, 30), 1),), check_trace=False)
    y = values((4, 30), 3)
    got, want = traced(y), call(y)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_quantized_norm_has_no_gradient_in_either_form():
    x = values((4, 30), 1).requires_grad_()
    for out in (F.rms_norm_quantized(x, None, x, EPS, -1), F._by_function(F._C.rms_norm_quantized, (x, None, x, EPS, -1))):
        assert not any(t.requires_grad for t in out)
        assert torch.equal(out[2], (x + x).detach())


def test_quantized_norm_refuses_transforms():
    x = values((4, 30), 1)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: F.rms_norm_quantized(q, None, None, EPS, -1)[1], (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: F.rms_norm_quantized(q, None, None, EPS, -1)[1])(x)
