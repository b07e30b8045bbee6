"""Timed cases of what a training or serving step of a mapped network needs around its convolutions, each in a plain form
(elementary torch operations, 32 bits) and through the framework's own operators:

  norm      root-mean-square norm over the channels, with the residual's addition, forward and backward:
                sum = residual + input, stored in the input's type;  out = sum / sqrt(mean(sum^2) + eps) * weight
            What is normalised is the sum as it is stored, which is what the next layer reads.
  norm8     the same norm forward only, its output held in 8 bits (e4m3) with one float32 scale for each normalised row
  logprob   log probabilities of given classes (tokens, or labels of pixels), the entropy of each distribution and, with
            `top` > 0, the `top` most probable classes; with `train`, the gradient of the logits too
  adamw     an AdamW step over many tensors at once, its moments in 32 bits, or in 8 bits (e4m3) with a float32 scale for
            each 256 values (the second moment as its square root)

Two layouts: "planes" is (batch, channels, height, width), normalised over or classified by the channels; "rows" is
(rows, channels).
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "spherical-package_b200")
_API = {}

EPS = 1e-6
IGNORE = -100
BLOCK, E4M3_MAX, TINY = 256, 448.0, 2.0 ** -100
BETAS, ADAM_EPS, LR, DECAY = (0.9, 0.999), 1e-8, 1e-3, 0.01
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---- cases ---------------------------------------------------------------------------------------------------------
def _rows(rows):
    return dict(layout="rows", batch=rows, height=1, width=1)


def _planes(batch, height, width):
    return dict(layout="planes", batch=batch, height=height, width=width)


def _norm(where, channels, dtype, weight, residual):
    return dict(op="norm", **where, channels=channels, dtype=dtype, weight=weight, residual=residual)


def _norm8(where, channels, dtype, weight, residual):
    return dict(op="norm8", **where, channels=channels, dtype=dtype, weight=weight, residual=residual)


def _logprob(where, channels, dtype, train, top, masked):
    return dict(op="logprob", **where, channels=channels, dtype=dtype, train=train, top=top, masked=masked)


def _adamw(tensors, largest, dtype, bits, master, encoder=False):
    return dict(op="adamw", tensors=tensors, largest=largest, dtype=dtype, bits=bits, master=master, encoder=encoder)


def listed():
    return [
        # the activations behind the third layer of the spherical encoder, in training, with a skip connection
        dict(_norm(_planes(16, 128, 256), 256, "float32", "float32", True), name="norm train planes f32"),
        # tokens (positions of a sequence or of an image) of a wide layer, in training
        dict(_norm(_rows(8192), 4096, "bfloat16", "bfloat16", True), name="norm train rows bf16"),
        # one token of a serving step, its output quantised for the product that follows: launch latency
        dict(_norm8(_rows(1), 5120, "bfloat16", "bfloat16", True), name="norm8 one token"),
        # a small ragged image batch, quantised
        dict(_norm8(_planes(3, 181, 333), 96, "bfloat16", "float32", False), name="norm8 planes odd"),
        # the loss of a language model's step: a large vocabulary, some positions ignored, entropy regularised
        dict(_logprob(_rows(4096), 32000, "bfloat16", True, 0, False), name="logprob train rows bf16"),
        # eight sequences of a serving step, a longer vocabulary with classes masked out, the eight best alternatives
        dict(_logprob(_rows(8), 131072, "float32", False, 8, True), name="logprob serve 8 rows"),
        # semantic labels of panoramas: a loss at every pixel
        dict(_logprob(_planes(8, 512, 1024), 13, "float32", True, 0, False), name="logprob train planes f32"),
        # one small ragged image's labels with the three best alternatives of each pixel
        dict(_logprob(_planes(1, 101, 203), 41, "bfloat16", False, 3, False), name="logprob planes odd top3"),
        # the weights and biases of the four-layer spherical encoder
        dict(_adamw(8, 0, "float32", 32, False, encoder=True), name="adamw encoder f32"),
        # many tensors of all sizes, odd ones among them, in 32 bits
        dict(_adamw(160, 8 << 20, "float32", 32, False), name="adamw many f32"),
        # bf16 weights with float32 masters and 8-bit moments
        dict(_adamw(96, 16 << 20, "bfloat16", 8, True), name="adamw many bf16 8-bit"),
        # a small network's float32 weights with 8-bit moments
        dict(_adamw(24, 70001, "float32", 8, False), name="adamw small 8-bit"),
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(("norm", "norm8", "logprob", "logprob", "adamw"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    if op == "adamw":
        return _adamw(_log(rng, 1, 160), _log(rng, 64, 8 << 20), dtype, rng.choice((8, 32)), dtype != "float32" and rng.random() < 0.5)
    if rng.random() < 0.5:
        channels = _log(rng, 2, 131072 if op == "logprob" else 16384)
        where = _rows(_log(rng, 1, max(1, min(32768, (32 << 20) // channels))))
    else:
        channels = _log(rng, 2, 150 if op == "logprob" else 512)
        height = _log(rng, 1, 512)
        width = _log(rng, 1, 1024)
        where = _planes(max(1, min(_log(rng, 1, 16), (32 << 20) // (channels * height * width))), height, width)
    if op == "logprob":
        train = rng.random() < 0.5
        return _logprob(where, channels, dtype, train, 0 if train else min(channels, rng.choice((0, 1, 4, 8, 20))), rng.random() < 0.3)
    weight = rng.choice((dtype, "float32"))
    return (_norm if op == "norm" else _norm8)(where, channels, dtype, weight, rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------------------------------------------
def _dim(case):
    return 1 if case["layout"] == "planes" else -1


def _shape(case, channels=True):
    c = (case["channels"],) if channels else ()
    return (case["batch"],) + c + ((case["height"], case["width"]) if case["layout"] == "planes" else ())


def _adamw_sizes(case):
    if case["encoder"]:  # channels 3 -> 64 -> 128 -> 256 -> 256, nine slots
        chans = (3, 64, 128, 256, 256)
        return [n for a, b in zip(chans, chans[1:]) for n in (a * b * 9, b)]
    # three tensors in eight are vectors of a layer's width; the others fall from the largest in steps, a third of them odd
    n, top = case["tensors"], case["largest"]
    return [max(1, min(top, 16 + 61 * i)) if i % 8 in (1, 4, 6) else max(1, int(top * 0.97 ** i) - (i % 3 == 2)) for i in range(n)]


def _arena(tensors, unit=BLOCK):
    """(one allocation, its views): the tensors one behind the other, each from a multiple of `unit` values on, zeros between."""
    starts = [0]
    for t in tensors:
        starts.append(starts[-1] + -(-t.numel() // unit) * unit)
    flat = torch.zeros(starts[-1], dtype=tensors[0].dtype, device="cuda")
    views = [flat[i:i + t.numel()] for i, t in zip(starts, tensors)]
    for view, t in zip(views, tensors):
        view.copy_(t)
    return flat, views


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, scale=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)

    def uniform(shape, low=0.0, high=1.0):
        return torch.rand(shape, generator=g, device="cuda") * (high - low) + low

    if case["op"] == "adamw":
        dtype, sizes = TYPES[case["dtype"]], _adamw_sizes(case)
        s = dict(case=case, step=100, arenas={}, masters=None, exp_avg_scales=None, exp_avg_sq_scales=None)

        def keep(name, tensors, unit=BLOCK):
            s["arenas"][name], s[name] = _arena(tensors, unit)

        full = [normal(n, 0.05) for n in sizes]
        keep("params", [p.to(dtype) for p in full])
        if case["master"]:
            keep("masters", full)
        del full
        s["all_grads"], s["grads"] = _arena([normal(n, 1e-2, dtype) for n in sizes])
        for name, root in (("exp_avg", False), ("exp_avg_sq", True)):
            moments = [uniform(n, 0.5, 2.0).square_().mul_(1e-5) if root else normal(n, 1e-3) for n in sizes]
            if case["bits"] == 8:
                coded = [_encode(t, root) for t in moments]
                moments = [q for q, _ in coded]
                keep(name + "_scales", [c for _, c in coded], 1)  # block by block, as the moments lie
            keep(name + "s", moments)
        return s
    dtype, shape = TYPES[case["dtype"]], _shape(case)
    if case["op"] == "logprob":
        x = normal(shape, 2.5, dtype)
        target = torch.randint(case["channels"], _shape(case, False), generator=g, device="cuda")
        if case["masked"]:  # about one class in sixteen is out of the question, the first never
            gone = uniform((case["channels"],) + ((1, 1) if case["layout"] == "planes" else ())) < 1 / 16
            gone[0] = False
            x = x.masked_fill_(gone, -math.inf)
            target = torch.where(gone.reshape(-1)[target], 0, target)
        if case["train"]:  # one position in ten has no class
            target = torch.where(uniform(target.shape) < 0.1, IGNORE, target)
        s = dict(case=case, x=x.requires_grad_(case["train"]), target=target)
        if case["train"]:
            s["g_log_probs"] = torch.full(target.shape, -1.0 / target.numel(), device="cuda")
            s["g_entropy"] = torch.full(target.shape, -0.01 / target.numel(), device="cuda")
        return s
    train = case["op"] == "norm"
    s = dict(case=case, x=normal(shape, 1.5, dtype).requires_grad_(train), residual=None,
             weight=uniform(case["channels"], 0.5, 1.5).to(TYPES[case["weight"]]).requires_grad_(train))
    if case["residual"]:
        s["residual"] = normal(shape, 2.0, dtype).requires_grad_(train)
    if train:
        s["g_out"] = normal(shape, 1.0, dtype)
        s["g_sum"] = normal(shape, 1.0, dtype) if case["residual"] else None
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _encode(x, root):
    """(e4m3 values, float32 scale of each block of 256); with `root` of the square root, what is positive never as zero."""
    x = x.sqrt() if root else x
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    amax = blocks.abs().amax(1)
    amax = torch.where(amax < TINY, 0.0, amax)
    inverse = torch.where(amax > 0, E4M3_MAX / amax, 0.0)
    scaled = (blocks * inverse[:, None]).view(-1)[:n]
    if root:
        scaled = torch.where(scaled > 0, scaled.clamp(min=2.0 ** -9), scaled)
    return scaled.to(torch.float8_e4m3fn), amax / E4M3_MAX


def _decode(q, scale, root):
    x = q.float() * scale.repeat_interleave(BLOCK)[:q.numel()]
    return x * x if root else x


def _plain_adamw(s):
    """All tensors at once: they lie in arenas, whose padding stays zero."""
    (b1, b2), t, a = BETAS, s["step"], s["arenas"]
    m, v, eight = a["exp_avgs"], a["exp_avg_sqs"], s["case"]["bits"] == 8
    if eight:
        m, v = _decode(m, a["exp_avg_scales"], False), _decode(v, a["exp_avg_sq_scales"], True)
    g = s["all_grads"].float()
    p = (a["masters"] if s["case"]["master"] else a["params"]).float()
    m.mul_(b1).add_(g, alpha=1 - b1)
    v.mul_(b2).addcmul_(g, g, value=1 - b2)
    denominator = v.sqrt().div_(math.sqrt(1 - b2 ** t)).add_(ADAM_EPS)
    p.mul_(1 - LR * DECAY).addcdiv_(m, denominator, value=-LR / (1 - b1 ** t))
    if p is not a["params"]:
        a["params"].copy_(p)
    if eight:
        q, scale = _encode(m, False)
        a["exp_avgs"].copy_(q)
        a["exp_avg_scales"].copy_(scale)
        q, scale = _encode(v, True)
        a["exp_avg_sqs"].copy_(q)
        a["exp_avg_sq_scales"].copy_(scale)


def _plain_logprob(s):
    x, target, top = s["x"].detach().float(), s["target"], s["case"]["top"]
    dim = _dim(s["case"])
    most = x.amax(dim, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    e = (x - most).exp()
    z = e.sum(dim, keepdim=True)
    logp = torch.where(z > 0, x - (most + z.log()), -math.inf)
    p = torch.where(z > 0, e / z, 0.0)
    weighted = torch.where(p > 0, p * logp, 0.0)
    entropy = -weighted.sum(dim)
    given = target != IGNORE
    index = torch.where(given, target, 0).unsqueeze(dim)
    out = {"log_probs": torch.where(given, logp.gather(dim, index).squeeze(dim), 0.0), "entropy": entropy}
    if top:
        best = x.sort(dim=dim, descending=True, stable=True).indices.narrow(dim, 0, top)
        out |= {"top_log_probs": logp.gather(dim, best), "top_indices": best}
    if s["case"]["train"]:
        g = torch.where(given, s["g_log_probs"], 0.0).unsqueeze(dim)
        h = s["g_entropy"].unsqueeze(dim)
        grad = -p * (g + h * entropy.unsqueeze(dim)) - h * weighted
        out["grad"] = grad.scatter_add_(dim, index, g).to(s["x"].dtype)
    return out


def _plain_norm(s):
    case, dim = s["case"], _dim(s["case"])
    x, w = s["x"].detach(), s["weight"].detach().float()
    w = w.view(-1, 1, 1) if case["layout"] == "planes" else w
    out = {}
    if case["residual"]:
        x = (x.float() + s["residual"].detach().float()).to(x.dtype)
        out["sum"] = x
    dtype, x = x.dtype, x.float()
    rstd = (x.square().mean(dim, keepdim=True) + EPS).rsqrt()
    unit = x * rstd
    y = unit * w
    if case["op"] == "norm8":
        amax = y.abs().amax(dim, keepdim=True)
        amax = torch.where(amax < TINY, 0.0, amax)
        inverse = torch.where(amax > 0, E4M3_MAX / amax, 0.0)
        return out | {"out": (y * inverse).to(torch.float8_e4m3fn), "scale": (amax / E4M3_MAX).squeeze(dim)}
    out["out"] = y.to(dtype)
    g = s["g_out"].float()
    others = (0, 2, 3) if case["layout"] == "planes" else 0
    out["g_weight"] = (g * unit).sum(others).to(s["weight"].dtype)
    g = g * w
    gx = rstd * (g - unit * (g * unit).mean(dim, keepdim=True))
    if case["residual"]:
        gx = gx + s["g_sum"].float()
        out["g_residual"] = gx.to(dtype)
    out["g_input"] = gx.to(dtype)
    return out


# ---- the framework's operators ---------------------------------------------------------------------------------------
def _framework():
    if not _API:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        from spherical_distortion import functional
        from sphmap import optim
        _API.update(F=functional, optim=optim)
    return _API


def _own_adamw(s):
    _framework()["optim"].adamw_step(
        s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], step=s["step"], lr=LR, betas=BETAS, eps=ADAM_EPS,
        weight_decay=DECAY, masters=s["masters"], exp_avg_scales=s["exp_avg_scales"], exp_avg_sq_scales=s["exp_avg_sq_scales"])


def _own_logprob(s):
    case = s["case"]
    r = _framework()["F"].token_log_probs(s["x"], s["target"], dim=_dim(case), top_k=case["top"], ignore_index=IGNORE)
    out = {"log_probs": r.log_probs, "entropy": r.entropy}
    if case["top"]:
        out |= {"top_log_probs": r.top_log_probs, "top_indices": r.top_indices}
    if case["train"]:
        out["grad"], = torch.autograd.grad((r.log_probs, r.entropy), (s["x"],), (s["g_log_probs"], s["g_entropy"]))
    return out


def _own_norm(s):
    case, F = s["case"], _framework()["F"]
    if case["op"] == "norm8":
        r = F.rms_norm_quantized(s["x"], s["weight"], residual=s["residual"], eps=EPS, dim=_dim(case))
        out = {"out": r[0], "scale": r[1]}
        return out | {"sum": r[2]} if case["residual"] else out
    r = F.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, dim=_dim(case))
    if not case["residual"]:
        gx, gw = torch.autograd.grad((r,), (s["x"], s["weight"]), (s["g_out"],))
        return {"out": r, "g_input": gx, "g_weight": gw}
    gx, gr, gw = torch.autograd.grad(r, (s["x"], s["residual"], s["weight"]), (s["g_out"], s["g_sum"]))
    return {"out": r[0], "sum": r[1], "g_input": gx, "g_residual": gr, "g_weight": gw}


def run(state):
    op = state["case"]["op"]
    if op == "adamw":
        state["step"] += 1
        (_own_adamw if own else _plain_adamw)(state)
        return state["arenas"]  # all that was updated
    if op == "logprob":
        return (_own_logprob if own else _plain_logprob)(state)
    return (_own_norm if own else _plain_norm)(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adamw":
        size = 4 if case["dtype"] == "float32" else 2
        n = sum(_adamw_sizes(case))
        moments = 2 * (4 if case["bits"] == 32 else 1 + 4 / BLOCK)
        # gradient read; weight, master and moments read and written (a weight beside its master only written)
        per = size + (8 + size if case["master"] else 2 * size) + 2 * moments
        return {"bytes": n * per, "flops": 14 * n}
    size = 4 if case["dtype"] == "float32" else 2
    rows = case["batch"] * case["height"] * case["width"]
    n = rows * case["channels"]
    if case["op"] == "logprob":
        b = n * size * (2 if case["train"] else 1) + rows * (8 + 8 + (8 if case["train"] else 0) + 12 * case["top"])
        return {"bytes": b, "flops": n * (12 if case["train"] else 5)}
    weight = case["channels"] * (4 if case["weight"] == "float32" else 2)
    r = 1 if case["residual"] else 0
    if case["op"] == "norm8":
        return {"bytes": n * (size * (1 + 2 * r) + 1) + rows * 4 + weight, "flops": 6 * n}
    # forward reads input (and residual), writes out (and sum); backward reads both output gradients, writes one gradient
    return {"bytes": n * size * (2 + 2 * r + 2 + r) + 2 * weight, "flops": 14 * n}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    return _exact_logprob(case, s) if case["op"] == "logprob" else _exact_norm(case, s)


def _exact_adamw(case, s):
    beta1, beta2, t = BETAS[0], BETAS[1], s["step"] + 1
    out = {k: torch.zeros_like(v, dtype=torch.float64) for k, v in s["arenas"].items()}

    def put(name, i, x):
        start = s[name][i].storage_offset()
        out[name][start:start + len(x)] = x

    for i in range(len(s["params"])):
        w = (s["masters"] if case["master"] else s["params"])[i].double()
        g, m, v = s["grads"][i].double(), s["exp_avgs"][i].double(), s["exp_avg_sqs"][i].double()
        at = torch.arange(g.numel(), device=g.device) // BLOCK
        if case["bits"] == 8:
            m = m * s["exp_avg_scales"][i].double()[at]
            v = (v * s["exp_avg_sq_scales"][i].double()[at]).pow(2)
        m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
        m_hat, v_hat = m / (1 - beta1 ** t), v / (1 - beta2 ** t)
        w = w - LR * (m_hat / (v_hat.pow(0.5) + ADAM_EPS) + DECAY * w)
        put("params", i, w)
        if case["master"]:
            put("masters", i, w)
        if case["bits"] == 32:
            put("exp_avgs", i, m)
            put("exp_avg_sqs", i, v)
            continue
        for name, x in (("exp_avg", m), ("exp_avg_sq", v.pow(0.5))):
            scale = torch.zeros(int(at[-1]) + 1, dtype=torch.float64, device=g.device).scatter_reduce_(0, at, x.abs(), "amax") / 448
            put(name + "s", i, x / scale[at])
            put(name + "_scales", i, scale)
    return out


def _exact_logprob(case, s):
    dim = _dim(case)
    logits = s["x"].detach().movedim(dim, -1)
    out, whole = [], logits.reshape(-1, case["channels"])
    targets = s["target"].reshape(-1)
    for rows in torch.arange(len(whole), device="cuda").split(max(1, (64 << 20) // case["channels"])):  # a few GB at a time
        logp = torch.log_softmax(whole[rows].double(), -1)
        t = targets[rows]
        kept = t != IGNORE
        at = torch.arange(len(t), device=t.device), t.clamp(min=0)
        surprise = torch.special.entr(logp.exp())
        entropy = surprise.sum(-1)
        got = {"log_probs": torch.where(kept, logp[at], 0.0), "entropy": entropy}
        if case["top"]:
            got["top_log_probs"] = logp.topk(case["top"], -1).values
        if case["train"]:
            g = s["g_log_probs"].reshape(-1)[rows].double() * kept
            h = s["g_entropy"].reshape(-1)[rows].double()
            d = h[:, None] * (surprise - logp.exp() * entropy[:, None]) - g[:, None] * logp.exp()
            d[at] += g
            got["grad"] = d
        out.append(got)
    def joined(k):
        v = torch.cat([o[k] for o in out])
        lead = _shape(case, False)
        return v.reshape(lead) if v.dim() == 1 else v.reshape(lead + (-1,)).movedim(-1, dim).contiguous()
    r = {k: joined(k) for k in out[0]}
    if case["top"]:
        r["top_indices"] = None
    return r


def _exact_norm(case, s):
    dim = _dim(case)
    x = s["x"].detach()
    out = {}
    if case["residual"]:
        out["sum"] = x.double() + s["residual"].detach().double()
        x = out["sum"].to(x.dtype)
    w = s["weight"].detach().double()
    w = w[:, None, None] if case["layout"] == "planes" else w
    x = x.double()
    root = ((x * x).mean(dim, keepdim=True) + EPS).pow(0.5)
    y = x / root * w
    if case["op"] == "norm8":
        scale = y.abs().amax(dim, keepdim=True) / 448
        return out | {"out": y / scale, "scale": scale.squeeze(dim)}
    out["out"] = y
    g = s["g_out"].double()
    x = x / root
    out["g_weight"] = (g * x).movedim(dim, -1).reshape(-1, case["channels"]).sum(0)
    g = g * w
    gx = (g - x * (x * g).mean(dim, keepdim=True)) / root
    if case["residual"]:
        gx = gx + s["g_sum"].double()
        out["g_residual"] = gx
    out["g_input"] = gx
    return out
