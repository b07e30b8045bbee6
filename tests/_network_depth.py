"""Error bounds of the norm and log-probability operators by how deep their kernels sum: how many roundings lie one behind the other
on the way of a term, which is a few dozen where the number of terms is a hundred thousand.  Values come from _network_ops.

u = 2^-24 bounds every float32 rounding, relative to its result; first-order terms are summed, and 1 % covers the rest."""
import math

import torch

import _network_ops as ref

U = ref.U
MORE = 1.01
SMS = 148


def _cdiv(a, b):
    return -(-a // b)


# ---- norm ----------------------------------------------------------------------------------------------------------
def norm_depths(c, norms, inner, outer):
    """(roundings of a sum over the channels, of a weight gradient's sum over the norms).

    Channels.  Rows: up to 32 values a thread one after the other, five steps over a warp's lanes and five over the block's warps;
    beyond 16384 channels c / 256 a thread, five, eight warps.  Planes: all of up to 32, an eighth of up to 512 and eight warps, all.
    Norms.  At least 148 blocks share them, or as many as there are (rows in tiles of at most norms / 296 or one); then a block's
    lanes (5), its warps (8) and the partial sums, up to 37 for each of 32 threads, and a warp (5).  Planes: a lane has up to four
    pixels of each of a block's runs of 32 pixels or more.  Behind the limits: as launched."""
    if inner == 1 and c <= 16384:
        return 42, _cdiv(norms, SMS) * 2 + 8 + 5 + 8 + 37 + 5
    if inner > 1 and c <= 512:
        return (c if c <= 32 else _cdiv(c, 8) + 8), 4 * _cdiv(outer * _cdiv(inner, 32), SMS) + 5 + 8 + 14 + 5
    blocks = _cdiv(c, 32) if inner == 1 else c
    splits = max(1, min(_cdiv(SMS * 8, blocks), _cdiv(norms, 64)))
    each = _cdiv(norms, splits * 8) + 8 if inner == 1 else _cdiv(norms, splits * 256) + 13
    return (_cdiv(c, 256) + 13 if inner == 1 else c), each + _cdiv(splits, 32) + 5


def norm(x, w, r, eps, dim, gout, gsum=None):
    """{name: (value, bound)} as _network_ops.norm."""
    values = ref.norm(x, w, r, eps, dim, gout, gsum)
    dim %= x.dim()
    c, outer = x.shape[dim], math.prod(x.shape[:dim])
    inner = math.prod(x.shape[dim + 1:])
    if not x.is_contiguous():
        outer, inner = outer * inner, 1
    deep, deep_w = norm_depths(c, outer * inner, inner, outer)
    s = (x if r is None else (x.float() + r.float()).to(x.dtype)).double()
    rstd = (s.square().mean(dim, keepdim=True) + eps).rsqrt()
    unit = s * rstd
    shape = [c if i == dim else 1 for i in range(x.dim())]
    g = gout.double().abs() * (1.0 if w is None else w.double().abs().view(shape))
    # squares (1), their sum, 1 / c and its product (2), eps (1): halved by the root, then root and reciprocal
    rho = (deep + 4) / 2 + 2
    out = {"sum": values["sum"], "out": (values["out"][0], MORE * U * (rho + 2) * values["out"][0].abs())}
    # the mean's terms: rstd's own error, three products, the sum; its factor -rstd rstd / c: 2 rho, four products, 1 / c;
    # the two terms' sum, and that with gsum
    first = rstd * g
    second = rstd * unit.abs() * (g * unit.abs()).mean(dim, keepdim=True)
    off = first * (rho + 3) + second * (rho + 3 + deep + 2 * rho + 6) + values["gx"][0].abs() + (0 if gsum is None else gsum.double().abs())
    out["gx"] = values["gx"][0], MORE * U * off
    others = [i for i in range(x.dim()) if i != dim]
    size = (gout.double() * unit).abs()
    size = size.sum(others) if others else size
    out["gw"] = values["gw"][0], MORE * U * (rho + 3 + deep_w) * size
    return out


# ---- log probabilities -----------------------------------------------------------------------------------------------
def log_probs_depths(c, rows, inner, k, size):
    """(roundings of a sum over the classes, how often a sum is moved to another maximum) for elements of `size` bytes."""
    n = 16 // size
    if inner > 1:       # a thread a pixel, eight classes or more to a maximum; with k > 8 another pass, class by class
        return c + 2, (c if k > 8 else _cdiv(c, 8)) + 1
    if c <= 1024 - n:   # 32 values a lane in two sums, a warp
        return 16 + 2 + 5, 2
    if k > 32:          # class by class
        return _cdiv(c, 256) + 13, _cdiv(c, 256) + 9
    tile = 256 * 32 if k else 256 * 4 * n
    blocks = 1
    while blocks < 16 and blocks < _cdiv(c, tile) and blocks * rows < 2 * SMS:
        blocks *= 2
    if k == 0 and blocks == 1:      # 128 threads, four vectors each to a tile; five steps, three warps
        tiles = _cdiv(c + n, 128 * 4 * n)
        return 16 + 2 + tiles + 8, tiles + 4
    tiles = _cdiv(_cdiv(c + 2 * n, blocks) + n, tile)      # five steps, three over the warps, four over the cluster
    return 16 + 2 + tiles + 12, tiles + 3


def log_probs(x, target, dim, k, ignore, g=None, h=None, t=None):
    """{name: (value, bound)} as _network_ops.log_probs."""
    values = ref.log_probs(x, target, dim, k, ignore, g, h, t)
    dim %= x.dim()
    c = x.shape[dim]
    inner = math.prod(x.shape[dim + 1:]) if x.is_contiguous() else 1
    deep, moves = log_probs_depths(c, x.numel() // c // inner, inner, k, x.element_size())
    d = x.double()
    most = d.amax(dim, keepdim=True)
    most = torch.where(torch.isfinite(most), most, 0.0)
    far = torch.where(torch.isfinite(d), (most - d), 0.0)
    e = (d - most).exp()
    z = e.sum(dim, keepdim=True)
    empty = z == 0
    p = torch.where(empty, 0.0, e / z)
    a, b = (p * far).sum(dim, keepdim=True), (p * far * far).sum(dim, keepdim=True)
    ln = torch.where(empty, 0.0, z.log())
    H = values["entropy"][0].unsqueeze(dim)
    # a term 2^d: difference, factor, product (3 |d|) and the exponential (2^-22, that is 4); a move: exponential and product
    # (5; the sum of 2^d d one more product and sum, 7)
    sigma = 3 * a + 4 + 5 * moves + deep
    tau = 3 * b + a * (7 + 7 * moves + deep)
    off_h = sigma * (1 + a) + tau + 4 * ln + 5 * a + H
    out = {"entropy": (values["entropy"][0], MORE * U * off_h.squeeze(dim))}

    def of(index, value):
        return sigma + far.gather(dim, index) + 3 * ln + torch.where(torch.isfinite(value), value.abs(), 0.0)
    index = torch.where((target >= 0) & (target < c) & (target != ignore), target, 0).unsqueeze(dim)
    lp = values["log_probs"][0]
    out["log_probs"] = lp, MORE * U * of(index, lp.unsqueeze(dim)).squeeze(dim)
    if k:
        best = out["top_indices"] = values["top_indices"]
        out["top"] = values["top"][0], MORE * U * of(best, values["top"][0])
    if "gx" in values:
        gx = values["gx"][0]
        gg = torch.where(target != ignore, g.double().abs(), 0.0).unsqueeze(dim) if g is not None else 0.0
        hh = h.double().abs().unsqueeze(dim) if h is not None else 0.0
        tt = t.double().abs() if t is not None else None
        al = gg + (tt.sum(dim, keepdim=True) if tt is not None else 0.0)
        rest = hh * (H - ln).abs()
        # flat: the sum of the gradients, H - ln S, 1 / S; slope: 1 / S and two products; then e, the two's sum and product
        off = p * ((al + rest) * (sigma + 3 * far + 8) + (k + 2) * al + hh * (off_h + 4 * ln + (H - ln).abs()) + hh * far * (sigma + 3 * far + 10))
        off = off + torch.where(torch.isfinite(gx), gx.abs(), 0.0)
        if g is not None:
            off = off.scatter_add(dim, index, 2 * gg)
        if tt is not None:
            off = off.scatter_add(dim, best, (k + 2) * tt)
        out["gx"] = gx, MORE * U * off + 1e-36      # (exponentials below 2^-126 are 0)
    return out
