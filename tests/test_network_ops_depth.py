"""The norm and log-probability kernels within bounds that follow the depth of their sums, and planted mistakes outside of them: what
a bound that grows with the number of terms would let pass at large sizes."""
import math

import pytest
import torch

import _network_depth as depth
import _network_ops as ref

EPS = 1e-6
BF, F32, F16 = torch.bfloat16, torch.float32, torch.float16


def values(shape, seed, dtype=F32, scale=1.0, device="cpu"):
    return (torch.randn(shape, generator=torch.Generator(device=device).manual_seed(seed), device=device) * scale).to(dtype)


# ---- mistakes, in the oracle -----------------------------------------------------------------------------------------
def log_probs_with(x, target, g, h, mistake):
    """(log_probs, entropy, gradient) over the last dimension in 64 bits, rounded at the end, with a mistake on the way."""
    d, n = x.double(), x.shape[-1]
    most = d.amax(-1, keepdim=True)
    away = d - most
    if mistake == "distances in 16 bits":
        away = away.to(BF).double()
    e = away.exp()
    counted = e.clone()
    if mistake == "a vector left out":
        first = n * 3 // 16 // 8 * 8                # the last one before a block's end
        counted[..., first:first + 16 // x.element_size()] = 0
    parts = torch.nn.functional.pad(counted, (0, -n % 4096)).view(*x.shape[:-1], -1, 4096).sum(-1)
    z = (parts.to(BF).double() if mistake == "partial sums in 16 bits" else parts).sum(-1, keepdim=True)
    H = z.log() - (counted * away).sum(-1, keepdim=True) / z
    p, logp = e / z, away - z.log()
    if mistake == "entropies half right":
        H = H + 1e-4
    gx = -p * (g[:, None] + h[:, None] * (logp + (0 if mistake == "gradient without the entropy" else H)))
    gx = gx.scatter_add(-1, target[:, None], g[:, None].double())
    return logp.gather(-1, target[:, None]).squeeze(-1).float(), H.squeeze(-1).float(), gx.to(x.dtype)


@pytest.mark.parametrize("shape, dtype", [((2, 131075), F32), ((3, 32000), BF), ((1, 300001), BF), ((2, 50257), F16), ((300, 4096), F32)])
def test_planted_mistakes_in_log_probs_are_outside(shape, dtype):
    x, target = values(shape, 1, dtype, 0.5), torch.arange(shape[0]) * 7
    g, h = values(shape[:1], 2).abs() + 0.5, values(shape[:1], 3).abs() + 0.5
    want = depth.log_probs(x, target, -1, 0, -100, g, h)
    names = ("log_probs", "entropy", "gx")
    kinds = (F32, F32, dtype)
    for got, name, kind in zip(log_probs_with(x, target, g, h, None), names, kinds):
        ref.close(got, *want[name], kind, name)
    caught = {"a vector left out": "log_probs", "partial sums in 16 bits": "log_probs", "distances in 16 bits": "log_probs",
              "entropies half right": "entropy", "gradient without the entropy": "gx"}
    for mistake, name in caught.items():
        got = dict(zip(names, log_probs_with(x, target, g, h, mistake)))[name]
        with pytest.raises(AssertionError, match="out of bounds"):
            ref.close(got, *want[name], F32 if name != "gx" else dtype, name)
            raise ValueError(mistake)


def norm_with(x, w, gout, mistake):
    """(out, gx, gw) over the last dimension."""
    d, n = x.double(), x.shape[-1]
    squares = d.square()
    if mistake == "a vector left out":
        squares[..., n // 2:n // 2 + 16 // x.element_size()] = 0
    rstd = (squares.mean(-1, keepdim=True) + EPS).rsqrt()
    unit, g = d * rstd, gout.double() * w.double()
    mean = (g * unit).mean(-1, keepdim=True)
    mean = mean.to(BF).double() if mistake == "means in 16 bits" else mean * 0.99 if mistake == "a hundredth of the mean left out" else mean
    gu = gout.double() * unit
    if mistake == "a row left out":
        gu[len(gu) // 2] = 0
    if mistake == "partial sums in 16 bits":
        gu = torch.stack([q.sum(0) for q in gu.split(64)]).to(BF).double()
    return (unit * w.double()).to(x.dtype), (rstd * (g - unit * mean)).to(x.dtype), gu.sum(0).float()


@pytest.mark.parametrize("shape", [(3, 40000), (60, 4096), (20000, 64), (5000, 333)])
def test_planted_mistakes_in_the_norm_are_outside(shape):
    x, w, gout = values(shape, 1), values(shape[-1:], 2) * 0.2 + 1, values(shape, 3) + 0.5
    want = depth.norm(x, w, None, EPS, -1, gout)
    names = ("out", "gx", "gw")
    for got, name in zip(norm_with(x, w, gout, None), names):
        ref.close(got, want[name][0], want[name][1], F32, name)
    caught = {"a vector left out": "out", "a hundredth of the mean left out": "gx"}
    if shape[0] > 100:
        caught |= {"a row left out": "gw", "partial sums in 16 bits": "gw"}
    if shape[1] <= 4096:        # (of 40000 the mean is about 1 / 200, and half a step of 16 bits of that, 1e-5, within the bound of 2e-5)
        caught["means in 16 bits"] = "gx"
    for mistake, name in caught.items():
        with pytest.raises(AssertionError, match="out of bounds"):
            ref.close(dict(zip(names, norm_with(x, w, gout, mistake)))[name], *want[name], F32, name)
            raise ValueError(mistake)


# ---- the kernels -----------------------------------------------------------------------------------------------------
LOGPROBS = [((1, 131072), -1), ((2, 131075), -1), ((1, 300001), -1), ((3, 32000), -1), ((300, 32000), -1), ((8, 50257), -1), ((600, 1500), -1),
            ((700, 5003), -1), ((40, 1000), -1), ((33, 130), -1), ((2, 41, 11, 13), 1), ((4, 19, 64, 64), 1), ((2, 300, 1, 8), 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape, dim", LOGPROBS)
def test_log_probs_within_their_depth(shape, dim, dtype):
    from spherical_distortion import functional as F
    for scale, k in ((0.5, 0), (0.5, 8), (2.5, 0), (2.5, 4), (6.0, 1)) + (((0.5, 40),) if shape == (2, 131075) or len(shape) > 2 and shape[1] >= 40 else ()):
        x = values(shape, 11, dtype, scale, "cuda")
        n = shape[dim]
        target = torch.randint(n, [s for i, s in enumerate(shape) if i != dim % len(shape)], generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
        target.view(-1)[-1] = -100
        g, h = values(target.shape, 12, device="cuda"), values(target.shape, 13, device="cuda")
        t = values([k if i == dim % len(shape) else s for i, s in enumerate(shape)], 14, device="cuda") if k else None
        leaf = x.detach().requires_grad_()
        r = F.token_log_probs(leaf, target, dim, k)
        outs = [(r.log_probs, g), (r.entropy, h)] + ([(r.top_log_probs, t)] if k else [])
        gx, = torch.autograd.grad([o for o, _ in outs], leaf, [q for _, q in outs])
        want = depth.log_probs(x, target, dim, k, -100, g, h, t)
        ref.close(r.log_probs, *want["log_probs"], F32, "log_probs")
        ref.close(r.entropy, *want["entropy"], F32, "entropy")
        ref.close(gx, *want["gx"], dtype, "gradient")
        if k:
            assert torch.equal(r.top_indices, want["top_indices"])
            ref.close(r.top_log_probs, *want["top"], F32, "top_log_probs")


NORMS = [((300, 4096), -1), ((2, 40000), -1), ((70, 20000), -1), ((3, 16384), -1), ((11, 4099), -1), ((5000, 333), -1), ((20000, 64), -1), ((3000, 1000), -1),
         ((999, 24), -1), ((1, 2, 70000), 1), ((2, 96, 181, 33), 1), ((1, 1030, 4, 64), 1), ((2, 700, 5, 9), 1), ((2, 256, 32, 33), 1), ((2, 256, 64, 64), 1),
         ((8, 512, 7, 7), 1), ((4, 30, 90, 91), 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape, dim", NORMS)
def test_norm_within_its_depth(shape, dim, dtype):
    from spherical_distortion import functional as F
    x, r = values(shape, 1, dtype, 1.5, "cuda"), values(shape, 2, dtype, 2.0, "cuda")
    gout, gsum = values(shape, 3, dtype, device="cuda") + 0.5, values(shape, 4, dtype, device="cuda")
    w = values((shape[dim],), 5, device="cuda") * 0.2 + 1
    for residual in (None, r):
        leaf = [t.detach().requires_grad_() for t in (x, w) + ((r,) if residual is not None else ())]
        out = F.rms_norm(leaf[0], leaf[1], leaf[2] if residual is not None else None, EPS, dim)
        outs, grads = ((out,), (gout,)) if residual is None else (out, (gout, gsum))
        gx, gw, *_ = torch.autograd.grad(outs, leaf, grads)
        want = depth.norm(x, w, residual, EPS, dim, gout, None if residual is None else gsum)
        ref.close(outs[0], *want["out"], dtype, "out")
        ref.close(gx, *want["gx"], dtype, "gx")
        ref.close(gw, want["gw"][0].reshape(-1), want["gw"][1].reshape(-1), F32, "gw")


def test_depths_are_far_below_the_number_of_terms():
    assert depth.log_probs_depths(300001, 1, 1, 0, 4)[0] < 64 and depth.norm_depths(4096, 8192, 1, 8192)[1] < 256
    assert math.prod(depth.norm_depths(2, 70000, 70000, 1)) < 1000
