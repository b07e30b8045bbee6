"""The norm, log-probability and AdamW operators in 64 bits, each value with a bound of the error that float32 arithmetic may
make (u = 2^-24 for each of its roundings, as counted at each bound) and a last rounding to the type it is held in adds."""
import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float8_e4m3fn: 0.0}


def close(got, want, bound, dtype, what):
    """|got - want| <= bound + half a step of `dtype` at want; what is not finite is alike."""
    got, want = got.detach().double().cpu(), want.cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand(want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].nan_to_num(7e30), want[~fine].nan_to_num(7e30)), what + ": infinities or NaN differ"
    over = (got - want).abs() - (bound + HALF[dtype] * want.abs() * (1 + 1e-6) + LEAST[dtype])
    over = torch.where(fine, over, -1.0)
    if over.numel() and over.max() > 0:
        at = over.argmax()
        raise AssertionError("%s: %d of %d out of bounds, worst %g against %g (bound %g)" % (
            what, (over > 0).sum(), over.numel(), got.reshape(-1)[at], want.reshape(-1)[at], bound.reshape(-1)[at]))


def norm(x, w, r, eps, dim, gout=None, gsum=None):
    """{name: (value, bound)} of out, sum and, with gout, the gradients.  Sums over n values are bounded by n roundings,
    whatever their order."""
    s = x if r is None else (x.float() + r.float()).to(x.dtype)   # the sum as it is stored
    out = {"sum": (x.double() + (0 if r is None else r.double()), 0.0)}
    d, n = s.double(), x.shape[dim]
    shape = [1] * x.dim()
    shape[dim] = n
    ww = torch.ones(shape, dtype=torch.float64, device=x.device) if w is None else w.double().view(shape)
    rstd = (d.square().mean(dim, keepdim=True) + eps).rsqrt()
    unit = d * rstd
    y = unit * ww
    rel = (n / 2 + 8) * U       # the sum's n roundings halved by the root; mean, eps, root, reciprocal, products
    out["out"] = y, rel * y.abs()
    if gout is not None:
        g = gout.double() * ww
        c = (g * unit).mean(dim, keepdim=True)
        gx = rstd * (g - unit * c)
        size = rstd * (g.abs() + unit.abs() * (g * unit).abs().mean(dim, keepdim=True))
        if gsum is not None:
            gx = gx + gsum.double()
            size = size + gsum.double().abs()
        out["gx"] = gx, (2 * n + 24) * U * size
        other = [i for i in range(x.dim()) if i != dim % x.dim()]
        rows = x.numel() // n
        gw = gout.double() * unit
        out["gw"] = (gw.sum(other), (rows + n / 2 + 12) * U * gw.abs().sum(other)) if other else (gw, (n / 2 + 12) * U * gw.abs())
    return out


def log_probs(x, target, dim, k, ignore, g=None, h=None, t=None):
    """{name: (value, bound)} and, with k, the indices; with g, h, t (any may be None) the gradient."""
    d, n = x.double(), x.shape[dim]
    most = d.amax(dim, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    e = (d - most).exp()
    z = e.sum(dim, keepdim=True)
    empty = z == 0
    lse = most + z.log()
    logp = torch.where(empty, -math.inf, d - lse)
    p = torch.where(empty, 0.0, e / z)
    plogp = torch.where(p == 0, 0.0, p * logp)
    H = -plogp.sum(dim, keepdim=True)
    # lse: n roundings of a positive sum, 8 of the exponentials and the logarithm, and 4 of the size of the numbers themselves
    size = torch.where(torch.isfinite(d), d.abs(), 0.0).amax(dim, keepdim=True)
    lse_off = (n + 8) * U + 4 * U * (size + z.log().abs().nan_to_num(0.0, 0.0, 0.0))
    given = target != ignore
    bad = given & ((target < 0) | (target >= n))
    index = torch.where(given & ~bad, target, 0).unsqueeze(dim)
    lp = logp.gather(dim, index).squeeze(dim)
    lp = torch.where(bad, math.nan, torch.where(given, lp, 0.0))
    out = {"log_probs": (lp, lse_off.squeeze(dim)),
           "entropy": (H.squeeze(dim), ((2 * n + 24) * U * (2 + math.log(n)) + lse_off).squeeze(dim))}
    if k:
        best = x.float().sort(dim=dim, descending=True, stable=True).indices.narrow(dim, 0, k)
        out["top_indices"] = best
        out["top"] = logp.gather(dim, best), lse_off.expand_as(best)
    if g is not None or h is not None or t is not None:
        zero = torch.zeros(target.shape, dtype=torch.float64, device=x.device)
        gg = torch.where(given & ~empty.squeeze(dim), zero if g is None else g.double(), 0.0)
        gg = torch.where(bad & ~empty.squeeze(dim), math.nan, gg) if g is not None else gg
        gg, hh = gg.unsqueeze(dim), (zero if h is None else h.double()).unsqueeze(dim)
        tt = torch.where(empty, 0.0, t.double()) if t is not None else None
        al = gg + (tt.sum(dim, keepdim=True) if tt is not None else 0.0)
        gx = -p * (al + hh * H) - hh * plogp
        gx = gx.scatter_add(dim, index, torch.where(bad.unsqueeze(dim), 0.0, gg))
        inner = al.abs() + hh.abs() * (H + 1 + torch.where(p == 0, 0.0, logp.abs()))
        off = p * inner * (2 * lse_off + (2 * n + 24) * U * (2 + math.log(n)) + 16 * U) + 4 * U * gg.abs() * (p * 0 + 1) + 1e-37
        if tt is not None:
            gx = gx.scatter_add(dim, best, tt)
            off = off.scatter_add(dim, best, (k + 4) * U * tt.abs()) + (k + 4) * U * p * tt.abs().sum(dim, keepdim=True)
        out["gx"] = gx, off
    return out


def adamw(w, g, m, v, step, lr, b1, b2, eps, decay):
    """(w, m, v) after a step, with bounds: four roundings of each moment's terms, twelve of the update's."""
    w, g, m, v = (t.double() for t in (w, g, m, v))
    m2 = b1 * m + (1 - b1) * g
    v2 = b2 * v + (1 - b2) * g * g
    up = lr / (1 - b1 ** step) * m2 / ((v2 / (1 - b2 ** step)).sqrt() + eps)
    up_size = lr / (1 - b1 ** step) * ((b1 * m).abs() + ((1 - b1) * g).abs()) / ((v2 / (1 - b2 ** step)).sqrt() + eps)
    w2 = w * (1 - lr * decay) - up
    return ((w2, 12 * U * up_size + 4 * U * w.abs()), (m2, 4 * U * ((b1 * m).abs() + ((1 - b1) * g).abs())), (v2, 5 * U * v2))
