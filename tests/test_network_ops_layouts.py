"""Rows whose dimension is followed by dimensions of one value only, such as (batch, channels, 1, 1), are rows like any others."""
import pytest
import torch

import _network_ops as ref
from spherical_distortion import functional as F

EPS = 1e-6
SHAPES = [(6, 40, 1, 1), (6, 40, 1), (3, 2, 40, 1)]


def values(shape, seed, device):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(device)


def mixed(shape, device):
    """(input, residual) pairs, one of the two a slice of wider rows."""
    dim = 2 if len(shape) == 4 and shape[2] == 40 else 1
    wide = [s + 9 if i == dim else s for i, s in enumerate(shape)]
    dense, cut = values(shape, 1, device), values(wide, 2, device).narrow(dim, 3, 40)
    return dim, [(cut, dense), (dense, cut), (cut, cut)]


@pytest.mark.parametrize("shape", SHAPES)
def test_a_dense_residual_of_sliced_rows_is_taken(shape):
    dim, pairs = mixed(shape, "cpu")
    for x, r in pairs:
        with pytest.raises(RuntimeError, match="CUDA tensor"):      # (and not for its layout)
            F.rms_norm(x, None, r, EPS, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_sliced_and_dense_rows_together(shape):
    dim, pairs = mixed(shape, "cuda")
    w, gout, gsum = values((40,), 3, "cuda"), values(shape, 4, "cuda"), values(shape, 5, "cuda")
    for x, r in pairs:
        leaf = [t.detach().requires_grad_() for t in (x, w, r)]
        out, s = F.rms_norm(*leaf, EPS, dim)
        gx, gw, gr = torch.autograd.grad((out, s), leaf, (gout, gsum))
        want = ref.norm(x, w, r, EPS, dim, gout, gsum)
        for name, t in (("out", out), ("sum", s), ("gx", gx), ("gx", gr), ("gw", gw)):
            value, bound = want[name]
            if name == "gw":
                value, bound = value.reshape(-1), bound.reshape(-1)
            ref.close(t, value, bound, torch.float32, name)
        q, scale, t = F.rms_norm_quantized(x, w, r, EPS, dim)
        assert torch.equal(t, s) and q.shape == x.shape and list(scale.shape) == [n for i, n in enumerate(shape) if i != dim]
        target = torch.full(scale.shape, 7, device="cuda")
        a, b = F.token_log_probs(x, target, dim, 3), F.token_log_probs(x.contiguous(), target, dim, 3)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
