"""The norm, log-probability and AdamW kernels against their formulas in 64 bits (bounds in _network_ops.py), at the sizes,
layouts, types and masks where they can go wrong, and in the ways programs call them: on streams, in graphs, together."""
import math

import pytest
import torch

import _network_ops as ref
from spherical_distortion import functional as F
from spherical_distortion import nn
from sphmap import optim

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E4 = torch.float8_e4m3fn
EPS = 1e-6


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


# ---- norm ----------------------------------------------------------------------------------------------------------
NORM_SHAPES = [  # (shape, dim)
    ((1, 1), -1), ((1, 5120), -1), ((3, 7), -1), ((65, 31), -1), ((33, 32), 1), ((5, 33), -1), ((130, 96), -1), ((7, 255), -1),
    ((9, 256), -1), ((4, 257), -1), ((70, 1000), -1), ((17, 1024), -1), ((3, 1025), -1), ((5, 2048), -1), ((11, 4099), -1),
    ((2, 8192), -1), ((3, 8200), -1), ((2, 16384), -1), ((3, 16385), -1), ((2, 40000), -1), ((300, 4096), -1), ((1100, 64), -1),
    ((1000, 8), -1), ((999, 24), -1), ((515, 72), -1), ((2049, 5), -1), ((777, 13), -1), ((50, 12), -1), ((601, 200), -1), ((2000, 333), -1),
    ((2, 3, 5, 40), -1), ((3, 40, 5), 0), ((100, 1), 1), ((2, 1, 5, 7), 1), ((1, 3, 1, 1), 1), ((2, 5, 3, 11), 1), ((1, 64, 37, 75), 1),
    ((3, 48, 16, 8), 1), ((2, 256, 32, 33), 1), ((2, 255, 8, 8), 1), ((1, 512, 9, 16), 1), ((2, 700, 5, 9), 1), ((1, 1030, 4, 64), 1),
    ((4, 16, 130), 1), ((1, 2, 70000), 1), ((2, 96, 181, 33), 1),
]


def run_norm(x, w, r, dim, gout, gsum, eps=EPS):
    leaf = [t.detach().requires_grad_() if t is not None else None for t in (x, w, r)]
    out = F.rms_norm(leaf[0], leaf[1], leaf[2], eps, dim)
    outs = (out,) if r is None else out
    wanted = [t for t in leaf if t is not None]
    got = list(torch.autograd.grad(outs, wanted, (gout,) if r is None else (gout, gsum)))
    res = {"out": outs[0], "gx": got.pop(0)}
    if w is not None:
        res["gw"] = got.pop(0)
    if r is not None:
        res["sum"], res["gr"] = outs[1], got.pop(0)
    return res


def check_norm(x, w, r, dim, gout, gsum, eps=EPS):
    got = run_norm(x, w, r, dim, gout, gsum, eps)
    want = ref.norm(x, w, r, eps, dim, gout, gsum if r is not None else None)
    for k, t in got.items():
        value, bound = want["gx" if k == "gr" else k]
        if k == "gw":
            value, bound = value.reshape(-1), bound.reshape(-1)
        ref.close(t, value, bound, t.dtype, k)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, dim", NORM_SHAPES)
def test_norm(shape, dim, dtype):
    c = shape[dim]
    x, r = normal(shape, 1, dtype, 1.5), normal(shape, 2, dtype, 2.0)
    gout, gsum = normal(shape, 3, dtype), normal(shape, 4, dtype)
    w = normal((c,), 5) * 0.2 + 1
    check_norm(x, w, r, dim, gout, gsum)
    check_norm(x, w.to(dtype), None, dim, gout, None)
    check_norm(x, None, r, dim, gout, gsum)


def check_quantized(x, w, r, dim, eps=EPS):
    q, scale, *rest = F.rms_norm_quantized(x, w, r, eps, dim)
    assert q.dtype == E4 and scale.dtype == torch.float32
    want = ref.norm(x, w, r, eps, dim)
    if r is not None:
        ref.close(rest[0], *want["sum"], x.dtype, "sum")
    value, bound = want["out"]
    amax = value.abs().amax(dim, keepdim=True)
    rel = (x.shape[dim] / 2 + 12) * ref.U
    ref.close(scale.unsqueeze(dim), amax / 448, rel * amax / 448, torch.float32, "scale")
    # e4m3: half a step relative, or half of its smallest, 2^-9; a value may lie on a border
    ref.close(q.float() * scale.unsqueeze(dim), value, 2 * bound + amax / 448 * 2.0 ** -10 * 1.01 + 2.0 ** -4 * rel * value.abs(), E4, "quantised")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, dim", NORM_SHAPES)
def test_norm_quantized(shape, dim, dtype):
    x, r = normal(shape, 1, dtype, 1.5), normal(shape, 2, dtype, 2.0)
    w = normal((shape[dim],), 5) * 0.2 + 1
    check_quantized(x, w, r, dim)
    check_quantized(x, w.to(dtype), None, dim)
    check_quantized(x, None, None, dim)


def test_results_in_a_channels_last_layout_are_written_in_place():
    """As contiguous ones are: an activation in place behind the norm, and its gradient, which is that of the one beside it."""
    img = normal((2, 24, 5, 3), 3).contiguous(memory_format=torch.channels_last)
    w, r = normal((24,), 4), normal((2, 24, 5, 3), 5).contiguous(memory_format=torch.channels_last)
    grads = []
    for relu in (torch.relu, torch.relu_):
        leaf = [t.clone().requires_grad_() for t in (img, w, r)]
        out, s = F.rms_norm(leaf[0], leaf[1], leaf[2], EPS, 1)
        grads.append(torch.autograd.grad((relu(out) * 3).sum(), leaf))
    for a, b in zip(*grads):
        assert torch.equal(a, b)
    top = F.token_log_probs(img.clone().requires_grad_(), torch.zeros((2, 5, 3), dtype=torch.int64, device="cuda"), top_k=2).top_log_probs
    top.mul_(2)
    top.sum().backward()


def saved_cases():
    """(input, dim): rows of wider rows, a channels-last image, planes."""
    return [(normal((40, 72), 6)[:, 3:60], 1), (normal((2, 24, 5, 3), 7).contiguous(memory_format=torch.channels_last), 1),
            (normal((2, 24, 5, 3), 8), 1), (normal((64, 4096), 9)[:, :2048], 1)]


@pytest.mark.parametrize("pinned", [False, True])
@pytest.mark.parametrize("case", range(4))
def test_saved_tensors_may_come_back_with_other_strides(case, pinned):
    """What a node saved is kept on the host until the backward pass, from where slices and channels-last images may come
    back dense in another order."""
    x, dim = saved_cases()[case]
    w, target = normal((x.shape[dim],), 10), torch.zeros([s for i, s in enumerate(x.shape) if i != dim], dtype=torch.int64, device="cuda")
    gout, gsum = normal(x.shape, 13), normal(x.shape, 14)
    with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
        check_norm(x, w, None, dim, gout, None)
        check_norm(x, w, x, dim, gout, gsum)
        check_log_probs(x, target, dim, 3)


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_in_the_backward_pass(reentrant):
    """Norms and log probabilities in a checkpointed block, whose forward pass runs again in the backward pass."""
    from torch.utils.checkpoint import checkpoint
    x, w = normal((2, 24, 5, 3), 15), normal((24,), 16)
    target = torch.randint(24, (2, 5, 3), generator=gen(17), device="cuda")

    def block(x, w):
        out, s = F.rms_norm(x, w, x * 0.5, EPS, 1)
        out = F.rms_norm(torch.relu_(out) + s, w, dim=1)
        p = F.token_log_probs(out, target, top_k=2)
        return p.log_probs.mean() + p.entropy.mean() + p.top_log_probs.mean()

    grads = []
    for kept in (True, False):
        leaf = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        loss = block(*leaf) if kept else checkpoint(block, *leaf, use_reentrant=reentrant)
        loss.backward()
        grads.append([t.grad for t in leaf])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_calls_from_two_threads():
    """Each on its own stream, forward and backward; the same results as alone."""
    import threading
    xs, w = [normal((300, 512), 18), normal((64, 40, 9, 7), 19)], [normal((512,), 20), normal((40,), 21)]

    def run(i):
        leaf = [xs[i].clone().requires_grad_(), w[i].clone().requires_grad_()]
        out = F.rms_norm(leaf[0], leaf[1], dim=1)
        target = torch.zeros([s for d, s in enumerate(xs[i].shape) if d != 1], dtype=torch.int64, device="cuda")
        p = F.token_log_probs(out, target, top_k=2)
        return [out, p.log_probs, p.top_indices, *torch.autograd.grad(p.log_probs.sum() + p.entropy.sum(), leaf)]

    alone, together, errors = [run(0), run(1)], [[], []], []
    torch.cuda.synchronize()

    def worker(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    together[i] = run(i)
            stream.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=worker, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for got, want in zip(together, alone):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("other", [lambda t: t.double(), lambda t: t.reshape(-1)[:1], lambda t: t.cpu()])
def test_saved_tensors_that_come_back_as_others_are_refused(other):
    x, w = normal((8, 96), 11).requires_grad_(), normal((96,), 12).requires_grad_()
    target = torch.zeros(8, dtype=torch.int64, device="cuda")
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
        out, p = F.rms_norm(x, w, dim=1), F.token_log_probs(x, target, top_k=2)
    for o in (out, p.log_probs, p.top_log_probs):
        with pytest.raises(RuntimeError, match="hooks returned another"):
            o.sum().backward(retain_graph=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [64, 65, 1000, 4096])
def test_norm_of_wider_rows_and_channels_last(c, dtype):
    """Rows that are slices of wider ones, one value behind an aligned address; channels-last images."""
    for first in (0, 1, 8):
        wide = normal((37, c + 24), 1, dtype)
        x = wide[:, first:first + c]
        gout = normal((37, c + 8), 3, dtype)[:, 1:c + 1]
        w = normal((c,), 5) * 0.2 + 1
        check_norm(x, w, None, -1, gout, None)
        check_norm(x, w, normal((37, c), 2, dtype), -1, gout, gout)
        check_quantized(x, w, None, -1)
    img = normal((2, c, 5, 3), 1, dtype).contiguous(memory_format=torch.channels_last)
    got = check_norm(img, w, img * 2, 1, normal((2, c, 5, 3), 3, dtype), normal((2, c, 5, 3), 4, dtype))
    assert got["out"].is_contiguous(memory_format=torch.channels_last)
    check_quantized(img, w, img * 2, 1)


def test_rows_that_are_a_first_dimension():
    """(C, rows) over rows of C values: dimension 0 of a transposed tensor."""
    x, r = normal((40, 72), 1).t(), normal((40, 72), 2).t()
    w = normal((72,), 5) * 0.2 + 1
    got = check_norm(x, w, r, 0, normal((72, 40), 3), normal((72, 40), 4))
    assert got["out"].stride() == x.stride()
    check_quantized(x, w, r, 0)
    check_log_probs(x, torch.randint(72, (40,), generator=gen(1), device="cuda"), 0, 3)


def test_norm_takes_shifted_addresses():
    """Contiguous tensors that start one value behind an aligned address."""
    for shape, dim in (((9, 512), -1), ((2, 64, 8, 16), 1)):
        for dtype in TYPES:
            n = math.prod(shape)
            t = [normal((n + 1,), i, dtype)[1:].view(shape) for i in range(4)]
            w = (normal((shape[dim] + 1,), 5) * 0.2 + 1)[1:]
            check_norm(t[0], w, t[1], dim, t[2], t[3])
            check_quantized(t[0], w, t[1], dim)


@pytest.mark.parametrize("shape, dim", [((5, 300), -1), ((5, 8192), -1), ((2, 20, 5, 7), 1)])
def test_norm_of_zeros_infinities_and_nan(shape, dim):
    """A row of zeros; one with an infinity; one with a NaN: each keeps to itself."""
    x = normal(shape, 1).movedim(dim, -1).contiguous()
    flat = x.view(-1, x.shape[-1])
    flat[0] = 0
    flat[1, 3], flat[2, 5], flat[3, 7] = math.inf, math.nan, -math.inf
    x = x.movedim(-1, dim).contiguous() if dim == 1 else x
    w = normal((shape[dim],), 5) * 0.2 + 1
    out = F.rms_norm(x, w, None, EPS, dim)
    value, bound = ref.norm(x, w, None, EPS, dim)["out"]
    ref.close(out, value, bound.nan_to_num(0.0), torch.float32, "out")
    q, scale = F.rms_norm_quantized(x, w, None, EPS, dim)
    rows, s = q.movedim(dim, -1).reshape(-1, shape[dim]).float(), scale.reshape(-1)
    assert s[0] == 0 and not rows[0].any()
    assert torch.isnan(rows[2]).all() and torch.isnan(s[1:4]).all()
    assert torch.isfinite(rows[4:]).all() and torch.isfinite(s[4:]).all()


@pytest.mark.parametrize("eps", [0.0, 1e-12, 0.5])
def test_norm_eps(eps):
    x, w = normal((40, 120), 1, scale=1e-4), normal((120,), 5)
    check_norm(x, w, None, -1, normal((40, 120), 3), None, eps)


def test_norm_gradients_asked_in_part():
    x, w, r = normal((6, 40), 1).requires_grad_(), normal((40,), 2).requires_grad_(), normal((6, 40), 3)
    g = normal((6, 40), 4)
    out, s = F.rms_norm(x, w, r, EPS, -1)
    want = ref.norm(x.detach(), w.detach(), r, EPS, -1, g)
    gw, = torch.autograd.grad(out, w, g, retain_graph=True)
    ref.close(gw, *want["gw"], torch.float32, "gw alone")
    gx, = torch.autograd.grad(out, x, g, retain_graph=True)
    ref.close(gx, *want["gx"], torch.float32, "gx without the sum's gradient")
    gx, = torch.autograd.grad(s, x, g, retain_graph=True)
    assert torch.equal(gx, g)
    frozen = F.rms_norm(x, w.detach(), None, EPS, -1)
    gx, = torch.autograd.grad(frozen, x, g)
    ref.close(gx, *ref.norm(x.detach(), w.detach(), None, EPS, -1, g)["gx"], torch.float32, "gx, weight without gradient")
    assert F.rms_norm(x.detach(), w.detach()[:40], None, EPS, -1).grad_fn is None


def test_norm_gradients_against_differences():
    """Central differences in float32 inputs of the 64-bit value of a smooth loss: truncation h^2 and rounding u/h."""
    x, w, r = normal((3, 5, 4), 1), normal((5,), 2), normal((3, 5, 4), 3)
    a, b = normal((3, 5, 4), 4).double(), normal((3, 5, 4), 5).double()
    leaf = [t.clone().requires_grad_() for t in (x, w, r)]
    out, s = F.rms_norm(*leaf, 1e-3, 1)
    got = torch.autograd.grad((out.double() * a).sum() + (s.double() * b).sum(), leaf)

    def loss(x, w, r):
        s = x + r
        return ((s * (s.square().mean(1, keepdim=True) + 1e-3).rsqrt() * w.view(1, -1, 1) * a).sum() + (s * b).sum()).item()
    h = 1e-5
    for i, t in enumerate((x, w, r)):
        base = [q.double() for q in (x, w, r)]
        for j in range(t.numel()):
            ends = []
            for d in (h, -h):
                moved = [q.clone() for q in base]
                moved[i].view(-1)[j] += d
                ends.append(loss(*moved))
            diff = (ends[0] - ends[1]) / (2 * h)
            assert abs(diff - got[i].reshape(-1)[j].item()) < 1e-4 * (1 + abs(diff))   # 1e-10 third derivatives, 1e-6 float32


# ---- log probabilities -----------------------------------------------------------------------------------------------
LOGPROB_SHAPES = [  # (shape, dim, ks)
    ((1, 1), -1, (0, 1)), ((3, 2), -1, (0, 2)), ((5, 31), -1, (1, 31)), ((33, 32), -1, (4,)), ((6, 33), -1, (3, 33)), ((1, 997), -1, (5,)),
    ((9, 1000), 1, (0, 8)), ((4, 1024), -1, (1, 20)), ((3, 1025), -1, (8,)), ((7, 4096), -1, (0, 2)), ((2, 4097), -1, (8,)),
    ((3, 8192), -1, (1,)), ((2, 16384), -1, (8,)), ((2, 16385), -1, (7,)), ((3, 32000), -1, (0, 20)), ((2, 50257), -1, (1, 33)),
    ((1, 131072), -1, (8,)), ((2, 131075), -1, (4,)), ((1, 300001), -1, (5,)), ((600, 1500), -1, (2,)), ((300, 70), -1, (3,)),
    ((2, 3, 50), -1, (2,)), ((3001, 10), -1, (0, 3)), ((515, 64), -1, (0, 1)), ((260, 129), -1, (0,)), ((70, 1016), -1, (0, 9)), ((70, 1023), -1, (0,)), ((1, 13, 8, 16), 1, (0, 1, 4, 13)), ((2, 41, 11, 13), 1, (3, 20)), ((3, 2, 5), 1, (0, 2)), ((1, 150, 3, 64), 1, (8,)),
    ((1, 1, 4, 5), 1, (1,)), ((2, 300, 1, 7), 1, (9,)), ((4, 19, 64, 64), 1, (0, 5)), ((7, 3, 9), 0, (2,)), ((2, 1031, 2, 3), 1, (4,)),
    ((1, 5, 70000), 1, (0, 2)), ((1, 65537, 4), 1, (3,)), ((2, 50, 3, 8), 1, (3, 8, 50)),
]


def make_logits(shape, dim, dtype, seed, masked):
    x = normal(shape, seed, dtype, 2.5)
    n = shape[dim]
    rest = [s for i, s in enumerate(shape) if i != dim % len(shape)]
    target = torch.randint(n, rest, generator=gen(seed + 1), device="cuda")
    if masked:
        gone = torch.rand(shape, generator=gen(seed + 2), device="cuda") < 0.2
        x = x.masked_fill(gone, -math.inf)
        rows = x.movedim(dim, -1).reshape(-1, n).clone()
        rows[0] = -math.inf                              # an empty distribution
        if len(rows) > 2:
            rows[2] = -math.inf
            rows[2, n // 2] = 3.0                        # one class left
        x = rows.view(rest + [n]).movedim(-1, dim).contiguous()
        flat = target.reshape(-1)
        flat[-1:] = -100
        target = flat.view(rest)
    return x, target


def check_log_probs(x, target, dim, k, ignore=-100, seed=7, parts=("g", "h", "t")):
    n = target.numel()
    g = normal(target.shape, seed) if "g" in parts else None
    h = normal(target.shape, seed + 1) if "h" in parts else None
    shape = list(x.shape)
    shape[dim] = k
    t = normal(shape, seed + 2) if k and "t" in parts else None
    leaf = x.detach().requires_grad_()
    r = F.token_log_probs(leaf, target, dim, k, ignore)
    pairs = [(o, q) for o, q in ((r.log_probs, g), (r.entropy, h), (r.top_log_probs, t)) if q is not None]
    gx, = torch.autograd.grad([o for o, _ in pairs], leaf, [q for _, q in pairs])
    want = ref.log_probs(x, target, dim, k, ignore, g, h, t)
    ref.close(r.log_probs, *want["log_probs"], torch.float32, "log_probs")
    ref.close(r.entropy, *want["entropy"], torch.float32, "entropy")
    if k:
        assert torch.equal(r.top_indices, want["top_indices"])
        ref.close(r.top_log_probs, *want["top"], torch.float32, "top_log_probs")
    ref.close(gx, *want["gx"], x.dtype, "gradient")
    with torch.no_grad():
        again = F.token_log_probs(x, target, dim, k, ignore)
    for a, b in zip(r, again):
        assert (a is None and b is None) or torch.equal(a.nan_to_num(5e30), b.nan_to_num(5e30))
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, dim, ks", LOGPROB_SHAPES)
def test_log_probs(shape, dim, ks, dtype):
    for k in ks:
        check_log_probs(*make_logits(shape, dim, dtype, 11, False), dim, k)
    if shape[dim] > 2:
        check_log_probs(*make_logits(shape, dim, dtype, 12, True), dim, ks[-1])


@pytest.mark.parametrize("parts", [("g",), ("h",), ("t",), ("g", "t"), ("h", "t")])
@pytest.mark.parametrize("shape, dim", [((5, 70), -1), ((3, 5000), -1), ((2, 17, 5, 8), 1)])
def test_log_probs_gradients_in_part(shape, dim, parts):
    x, target = make_logits(shape, dim, torch.float32, 21, True)
    check_log_probs(x, target, dim, 3, parts=parts)


@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_ties_go_to_the_lowest_index(dtype):
    for shape, dim in (((4, 500), -1), ((4, 20000), -1), ((2, 40, 3, 3), 1)):
        x = torch.randint(-2, 3, shape, generator=gen(1), device="cuda").to(dtype)
        x[x == 0] = -0.0 if dim == 1 else 0.0
        target = torch.zeros([s for i, s in enumerate(shape) if i != dim % len(shape)], dtype=torch.long, device="cuda")
        check_log_probs(x, target, dim, 20)
        check_log_probs(torch.zeros_like(x), target, dim, 9)
    zeros = torch.tensor([[0.0, -0.0, 0.0, -1.0]], device="cuda")
    assert F.token_log_probs(zeros, torch.zeros(1, dtype=torch.long, device="cuda"), -1, 3).top_indices.tolist() == [[0, 1, 2]]


@pytest.mark.parametrize("shape, dim", [((6, 90), -1), ((6, 3000), -1), ((6, 9, 2), 1)])
def test_log_probs_targets_outside(shape, dim):
    """Targets outside the classes give NaN and NaN gradients of their own distribution; ignored ones nothing."""
    x, target = make_logits(shape, dim, torch.float32, 31, False)
    rows = target.view(shape[0], -1)
    rows[0], rows[1], rows[2], rows[3] = shape[dim], -1, -100, 2 ** 40
    check_log_probs(x, target, dim, 2)
    rows[4] = 255
    check_log_probs(x, target, dim, 0, ignore=255)
    check_log_probs(x, target, dim, 0, ignore=2 ** 40)


@pytest.mark.parametrize("shape, dim", [((5, 40), -1), ((5, 6000), -1), ((5, 140000), -1), ((5, 8, 2), 1)])
def test_log_probs_infinities_nan_and_lowest(shape, dim):
    """+inf and NaN spoil their own distribution alone; a mask of the type's lowest value is no infinity."""
    x, target = make_logits(shape, dim, torch.float32, 41, False)
    x = x.movedim(dim, -1).contiguous()
    x[0, ..., 3], x[1, ..., 2] = math.inf, math.nan
    x[2] = torch.finfo(torch.float32).min
    x[3, ..., 1:] = torch.finfo(torch.float32).min
    x = x.movedim(-1, dim).contiguous()
    r = F.token_log_probs(x, target, dim, 4)
    assert torch.isnan(r.entropy[:2]).all() and torch.isfinite(r.entropy[2:]).all() and torch.isnan(r.log_probs[:2]).all()
    top = r.top_indices.movedim(dim, -1)
    assert (top[0, ..., 0] == 3).all() and (top[1, ..., 0] == 2).all()        # NaN stands before numbers
    n = shape[dim]
    uniform = math.log(n)
    assert (r.entropy[2] - uniform).abs().max() < (n + 30) * ref.U * (2 + uniform) + 4 * ref.U * uniform
    assert (r.entropy[3] == 0).all() and (r.top_log_probs.movedim(dim, -1)[3, ..., 0] == 0).all()
    check_log_probs(x[4:], target[4:], dim, 4)


@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_of_wider_rows_and_channels_last(dtype):
    for n in (33, 1000, 5000, 20000):
        for first in (0, 1, 8):
            wide = normal((6, n + 64), 51, dtype, 2.0)
            x = wide[:, first:first + n]
            target = torch.randint(n, (6,), generator=gen(2), device="cuda")
            check_log_probs(x, target, -1, 4)
    img = normal((2, 21, 6, 5), 52, dtype).contiguous(memory_format=torch.channels_last)
    r = check_log_probs(img, torch.randint(21, (2, 6, 5), generator=gen(3), device="cuda"), 1, 3)
    assert r.top_indices.shape == (2, 3, 6, 5)
    flat = normal((2 * 12 * 40 + 1,), 53, dtype)[1:].view(2, 12, 40)
    check_log_probs(flat, torch.randint(12, (2, 40), generator=gen(4), device="cuda"), 1, 2)


def test_log_probs_large_logits_keep_their_precision():
    x = normal((4, 300), 61) * 50 + 3e4
    check_log_probs(x, torch.randint(300, (4,), generator=gen(5), device="cuda"), -1, 3)


def test_log_probs_mean_loss():
    """One gradient for all positions, as a mean's backward pass gives it."""
    x, target = make_logits((64, 500), -1, torch.bfloat16, 71, False)
    target[3] = -100
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    r = F.token_log_probs(a, target, -1)
    (-r.log_probs.mean() - 0.1 * r.entropy.mean()).backward()
    g = torch.full((64,), -1 / 64, device="cuda")
    h = torch.full((64,), -0.1 / 64, device="cuda")
    r = F.token_log_probs(b, target, -1)
    torch.autograd.backward((r.log_probs, r.entropy), (g, h))
    assert torch.equal(a.grad, b.grad)


def test_empty_tensors():
    for shape, dim in (((0, 5), -1), ((2, 5, 0, 3), 1), ((0, 4, 2, 2), 1)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[dim], device="cuda", requires_grad=True)
        out, s = F.rms_norm(x, w, x * 1, EPS, dim)
        (out.sum() + s.sum()).backward()
        assert out.shape == x.shape and x.grad.shape == x.shape and not w.grad.any()
        q, scale = F.rms_norm_quantized(x, w, None, EPS, dim)
        rest = [v for i, v in enumerate(shape) if i != dim % len(shape)]
        assert q.shape == x.shape and list(scale.shape) == rest
        r = F.token_log_probs(x, torch.zeros(rest, dtype=torch.long, device="cuda"), dim, 2)
        r.log_probs.sum().backward()
        assert list(r.entropy.shape) == rest and r.top_indices.shape[dim] == 2


def test_offsets_beyond_32_bits():
    """Rows 2^31 elements apart, read by both operators."""
    wide = torch.empty((2, 2 ** 31 + 64), dtype=torch.bfloat16, device="cuda")
    x = wide[:, :1000]
    x.copy_(normal((2, 1000), 1, torch.bfloat16))
    check_norm(x, None, None, -1, normal((2, 1000), 2, torch.bfloat16), None)
    check_log_probs(x, torch.tensor([3, 999], device="cuda"), -1, 4)
    x = wide[:, 2 ** 31 - 500:2 ** 31 + 40]
    x.copy_(normal((2, 540), 3, torch.bfloat16))
    check_quantized(x, None, None, -1)


def test_dense_rows_beyond_32_bits():
    """More than 2^31 elements in all: the last rows are computed like the first."""
    rows, n = 70001, 32768
    x = torch.zeros((rows, n), dtype=torch.bfloat16, device="cuda")
    few = normal((3, n), 1, torch.bfloat16)
    x[:3], x[-3:] = few, few
    out = F.rms_norm(x, None, None, EPS, -1)
    assert torch.equal(out[:3], out[-3:])
    ref.close(out[-3:], *ref.norm(few, None, None, EPS, -1)["out"], torch.bfloat16, "out")
    del out
    x.requires_grad_()
    target = torch.full((rows,), 5, device="cuda")
    r = F.token_log_probs(x, target, -1)
    g = torch.full((rows,), 2.0, device="cuda")
    gx, = torch.autograd.grad(r.log_probs, x, g)
    assert torch.equal(gx[:3], gx[-3:]) and torch.equal(r.log_probs[:3], r.log_probs[-3:])
    want = ref.log_probs(few, target[:3], -1, 0, -100, g[:3])
    ref.close(gx[-3:], *want["gx"], torch.bfloat16, "gradient")


# ---- AdamW -----------------------------------------------------------------------------------------------------------
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SIZES = [[1], [255, 256, 257], [7, 70001, 3, 1024, 12345], [33] * 33, [5 + 3 * i for i in range(450)], [2 ** 21 + 5]]


def adam_state(sizes, dtype, grad_dtype, seed, shift=0):
    g = gen(seed)

    def make(n, scale, d=torch.float32):
        return (torch.randn(n + shift, generator=g, device="cuda") * scale).to(d)[shift:]
    return dict(p=[make(n, 0.1, dtype) for n in sizes], g=[make(n, 1e-2, grad_dtype) for n in sizes],
                m=[make(n, 1e-3) for n in sizes], v=[make(n, 1e-3).square() for n in sizes])


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype, grad_dtype, master", [
    (torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.float32, True),
    (torch.float16, torch.float16, True), (torch.float16, torch.float32, False)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%d tensors" % len(s))
def test_adamw(sizes, dtype, grad_dtype, master, shift):
    """shift: tensors that start one value behind an aligned address."""
    s = adam_state(sizes, dtype, grad_dtype, 1, shift)
    masters = [p.float() + 1e-4 for p in s["p"]] if master else None
    want = [ref.adamw(w, g, m, v, 7, HYPER["lr"], 0.9, 0.999, 1e-8, 0.1)
            for w, g, m, v in zip(masters or s["p"], s["g"], s["m"], s["v"])]
    before = [t.clone() for t in s["g"]]
    optim.adamw_step(s["p"], s["g"], s["m"], s["v"], step=7, masters=masters, **HYPER)
    for i, (w, m, v) in enumerate(want):
        if master:
            ref.close(masters[i], *w, torch.float32, "master")
            assert torch.equal(s["p"][i], masters[i].to(dtype))
        else:
            ref.close(s["p"][i], *w, dtype, "param")
        ref.close(s["m"][i], *m, torch.float32, "exp_avg")
        ref.close(s["v"][i], *v, torch.float32, "exp_avg_sq")
        assert torch.equal(s["g"][i], before[i])


def encode(x, root):
    """(codes, scales) as the operator holds them; made here so that a step has something to start from."""
    x = x.double().sqrt() if root else x.double()
    n = x.numel()
    b = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    scale = (b.abs().amax(1) / 448).float()
    q = torch.where(scale[:, None] > 0, b / scale[:, None].double(), 0.0).float().view(-1)[:n].to(E4)
    return q, scale


def decode(q, scale):
    return q.double() * scale.double().repeat_interleave(256)[:q.numel()]


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype, master", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, False)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%d tensors" % len(s))
def test_adamw_8_bit(sizes, dtype, master, shift):
    s = adam_state(sizes, dtype, dtype, 2, shift)
    masters = [p.float() + 1e-4 for p in s["p"]] if master else None
    mq, vq = [encode(t, False) for t in s["m"]], [encode(t, True) for t in s["v"]]
    codes = [[torch.cat([q.new_zeros(shift), q])[shift:] if shift else q for q, _ in c] for c in (mq, vq)]
    scales = [[c for _, c in mq], [c for _, c in vq]]
    want = [ref.adamw(w, g, decode(*a), decode(*b).square(), 7, HYPER["lr"], 0.9, 0.999, 1e-8, 0.1)
            for w, g, a, b in zip(masters or s["p"], s["g"], mq, vq)]
    optim.adamw_step(s["p"], s["g"], codes[0], codes[1], step=7, masters=masters, exp_avg_scales=scales[0], exp_avg_sq_scales=scales[1], **HYPER)
    for i, (w, m, v) in enumerate(want):
        ref.close((masters or s["p"])[i], *w, torch.float32 if master else dtype, "param")
        for q, scale, (value, bound), root in ((codes[0][i], scales[0][i], m, False), (codes[1][i], scales[1][i], v, True)):
            if root:
                value, bound = value.sqrt(), 4 * ref.U * value.sqrt()
            blocks = torch.nn.functional.pad(value.abs(), (0, -value.numel() % 256)).view(-1, 256)
            amax = blocks.amax(1)
            ref.close(scale, amax / 448, 12 * ref.U * amax / 448, torch.float32, "scale")
            step = (amax / 448 * 2.0 ** -9).repeat_interleave(256)[:value.numel()]   # the smallest value; half of it by rounding, all by never zero
            ref.close(decode(q, scale), value, 3 * bound + 12 * ref.U * value.abs() + step * (1.01 if root else 0.505), E4, "codes")
            assert not root or ((q.float() > 0) == (value > 0)).all()


def test_adamw_8_bit_zeros_tiny_and_not_finite():
    n = 256 * 4
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    g[256:512] = 1e-38
    g[512], g[513], g[514] = math.inf, math.nan, 1.0
    g[768:] = normal((256,), 1)
    m, v = torch.zeros(n, device="cuda").to(E4), torch.zeros(n, device="cuda").to(E4)
    ms, vs = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    optim.adamw_step([p], [g], [m], [v], step=1, lr=1e-2, weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    assert not p[:256].any() and not m[:512].float().any() and not v[:512].float().any() and not ms[:2].any() and not vs[:2].any()
    assert torch.isfinite(p[:512]).all() and torch.isfinite(p[514:]).all() and torch.isnan(p[512:514]).all()
    assert torch.isnan(m.float()[512:514]).all() and torch.isfinite(m.float()[514:]).all() and torch.isfinite(ms).all() and torch.isfinite(vs).all()
    assert abs(p[514].item() + 1e-2) < 1e-7 and (p[515:768] == 0).all()


def test_adamw_zero_betas_and_scaled_gradients():
    s = adam_state([1000], torch.float32, torch.float32, 3)
    want = ref.adamw(s["p"][0], s["g"][0].double() * 0.125, s["m"][0], s["v"][0], 1, 1e-2, 0.0, 0.0, 1e-8, 0.0)
    optim.adamw_step(s["p"], s["g"], s["m"], s["v"], step=1, lr=1e-2, betas=(0.0, 0.0), weight_decay=0.0, grad_scale=0.125)
    for t, w, name in zip((s["p"][0], s["m"][0], s["v"][0]), want, ("param", "exp_avg", "exp_avg_sq")):
        ref.close(t, *w, torch.float32, name)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_optimizer_with_ragged_steps(bits):
    """Parameters without a gradient stay, with their own step numbers; one tensor's noncontiguous gradient is copied."""
    ps = [normal((300, 7), 1).requires_grad_(), normal((5,), 2, torch.bfloat16).requires_grad_(), torch.zeros(0, device="cuda", requires_grad=True)]
    o = optim.AdamW(ps, state_bits=bits, master_weights=True, **HYPER)
    ps[0].grad = normal((7, 300), 3).t()
    w = ref.adamw(ps[0].detach(), ps[0].grad, torch.zeros_like(ps[0]), torch.zeros_like(ps[0]), 1, 1e-2, 0.9, 0.999, 1e-8, 0.1)
    still = ps[1].detach().clone()
    version = ps[0]._version
    o.step()
    ref.close(ps[0], *w[0], torch.float32, "param")
    assert torch.equal(ps[1], still) and ps[0]._version > version
    ps[1].grad, ps[2].grad = normal((5,), 4, torch.bfloat16), torch.zeros(0, device="cuda")
    w = ref.adamw(still, ps[1].grad, torch.zeros_like(still), torch.zeros_like(still), 1, 1e-2, 0.9, 0.999, 1e-8, 0.1)
    o.step()
    assert o.state[ps[0]]["step"] == 2 and o.state[ps[1]]["step"] == 1
    ref.close(o.state[ps[1]]["master"], *w[0], torch.float32, "master")
    assert torch.equal(ps[1], o.state[ps[1]]["master"].bfloat16())
    with pytest.raises(RuntimeError, match="twice"):
        optim.adamw_step([ps[0], ps[0]], [ps[0].grad.contiguous()] * 2, [o.state[ps[0]]["exp_avg"].float()] * 2,
                         [o.state[ps[0]]["exp_avg_sq"].float()] * 2, step=1, lr=0.1)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_continues_after_loading(bits):
    def steps(o, p, seeds):
        for i in seeds:
            p.grad = normal((1000,), i)
            o.step()
    a = normal((1000,), 0).requires_grad_()
    o = optim.AdamW([a], state_bits=bits, **HYPER)
    steps(o, a, range(1, 4))
    b = a.detach().clone().requires_grad_()
    o2 = optim.AdamW([b], state_bits=bits, **HYPER)
    o2.load_state_dict(o.state_dict())
    steps(o, a, range(4, 7))
    steps(o2, b, range(4, 7))
    assert torch.equal(a, b)


# ---- as programs call them -------------------------------------------------------------------------------------------
def test_on_another_stream():
    x, w, g = normal((500, 3000), 1), normal((3000,), 2), normal((500, 3000), 3)
    target = torch.randint(3000, (500,), generator=gen(1), device="cuda")

    def all_of_it():
        a = x.clone().requires_grad_()
        out, s = F.rms_norm(a, w, x, EPS, -1)
        r = F.token_log_probs(out, target, -1, 3)
        r.log_probs.mean().backward()
        p = out.detach().clone()
        optim.adamw_step([p], [g], [g * 0], [g * 0], step=1, lr=1e-2)
        return out.detach(), r.entropy.detach(), r.top_indices, a.grad, p
    want = all_of_it()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = all_of_it()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("capturable_bits", [8, 32])
def test_training_step_in_two_graphs(capturable_bits):
    """A whole step (norm with a residual, head, log probabilities, backward, AdamW), captured twice over the same weights and
    replayed in turn, does what eager steps do."""
    def network(seed):
        norm = nn.RMSNorm(64, dim=-1).cuda()
        head = normal((64, 211), seed, scale=0.1).requires_grad_()
        params = [norm.weight, head]
        o = optim.AdamW(params, state_bits=capturable_bits, capturable=True, lr=1e-2)

        def step(x, r, target):
            o.zero_grad(set_to_none=True)
            out, s = norm(x, r)
            logp = F.token_log_probs(out @ head, target, -1)
            loss = -logp.log_probs.mean() - 0.01 * logp.entropy.mean() + 1e-3 * s.square().mean()
            loss.backward()
            o.step()
            return loss.detach()
        return params, step, o
    data = [(normal((96, 64), 2 * i), normal((96, 64), 2 * i + 1), torch.randint(211, (96,), generator=gen(i), device="cuda")) for i in range(5)]
    torch.manual_seed(0)
    params, step, o = network(9)
    eager = [step(*d) for d in data]
    want = [p.detach().clone() for p in params]
    params, step, o = network(9)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        losses = [step(*data[0])]
    torch.cuda.current_stream().wait_stream(st)
    inputs = [[t.clone() for t in data[0]] for _ in range(2)]
    graphs, out = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(step(*inputs[i]))
        graphs.append(g)
    for n, d in enumerate(data[1:]):
        for a, b in zip(inputs[n % 2], d):
            a.copy_(b)
        graphs[n % 2].replay()
        losses.append(out[n % 2].clone())
    for a, b in zip(eager, losses):
        assert torch.allclose(a, b, rtol=1e-6, atol=0)
    for a, b in zip(params, want):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    assert o.param_groups[0]["step"].item() == 5


def test_forwards_replayed_with_new_inputs():
    """Every forward kernel family in one graph, replayed on other values: what an eager call gives."""
    rows = {n: normal((5, n), n) for n in (30, 1000, 5001, 40000)}
    planes = {c: normal((2, c, 12, 20), c) for c in (5, 64, 300)}
    odd = normal((2, 40, 33, 31), 7)
    targets = {5: torch.zeros(5, dtype=torch.long, device="cuda"), (2, 12, 20): torch.zeros((2, 12, 20), dtype=torch.long, device="cuda")}

    def everything():
        out = []
        for x in rows.values():
            out += [*F.token_log_probs(x, targets[5], -1, 4), *F.token_log_probs(x, targets[5], -1)[:2]]
            out += [F.rms_norm(x, None, None, EPS, -1), *F.rms_norm_quantized(x, None, x, EPS, -1)]
        for x in planes.values():
            out += [*F.token_log_probs(x, targets[2, 12, 20], 1, 2), F.rms_norm(x, None, x, EPS, 1)[0], *F.rms_norm_quantized(x, None, None, EPS, 1)]
        return out + [F.rms_norm(odd, None, None, EPS, 1)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        everything()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = everything()
    for x in (*rows.values(), *planes.values(), odd):
        x.copy_(torch.randn_like(x) * 2)
    g.replay()
    for a, b in zip(got, everything()):
        assert torch.equal(a.float(), b.float())


def test_mapped_network_step():
    """As they are used together: mapped convolution, norm with a skip connection, mapped head, labels of pixels, backward, AdamW;
    every gradient against the same network of plain operators."""
    from sphmap.workloads import gnomonic_map
    H, W = 16, 32
    m = gnomonic_map(H, W).cuda()
    torch.manual_seed(3)
    conv, head, norm = nn.MappedConvolution(8, 24, 9).cuda(), nn.MappedConvolution(24, 13, 9).cuda(), nn.RMSNorm(24).cuda()
    loss_of = nn.TokenLogProbs(top_k=2, ignore_index=255)
    x = normal((2, 8, H, W), 1)
    skip = normal((2, 24, H, W), 2).requires_grad_()
    labels = torch.randint(13, (2, H, W), generator=gen(3), device="cuda")
    labels[:, :2] = 255
    params = [p for q in (conv, norm, head) for p in q.parameters()]
    out, s = norm(conv(x, m), skip)
    r = loss_of(head(out, m), labels)
    loss = -r.log_probs.sum() / (labels != 255).sum()
    got = torch.autograd.grad(loss, params + [skip])
    s2 = conv(x, m) + skip
    out2 = s2 * (s2.square().mean(1, keepdim=True) + norm.eps).rsqrt() * norm.weight.view(1, -1, 1, 1)
    logp = torch.log_softmax(head(out2, m), 1)
    want = torch.autograd.grad(torch.nn.functional.nll_loss(logp, labels, ignore_index=255), params + [skip])
    assert torch.equal(r.top_indices, logp.topk(2, 1).indices)
    for a, b in zip(got, want):
        assert (a - b).norm() <= 2e-5 * b.norm()     # two float32 computations: sums of up to 9 * 24 * 1024 terms
    o = optim.AdamW(params)
    for p, g in zip(params, got):
        p.grad = g
    before = [p.detach().clone() for p in params]
    o.step()
    for p, b, g in zip(params, before, got):
        z = torch.zeros_like(b)
        ref.close(p, *ref.adamw(b, g, z, z, 1, 1e-3, 0.9, 0.999, 1e-8, 0.01)[0], torch.float32, "param")


@pytest.mark.parametrize("precision", [0, 1])
def test_encoder_stack_with_an_optimizer(precision):
    """The encoder's step ends with AdamW's update from the gradients it left in its buffers."""
    from sphmap import workloads
    from sphmap.parallel import EncoderStack, GradReducer
    cfg = workloads.config4(B=2, H=64, W=128)
    x, go = cfg["x"].cuda(), cfg["grad_output"].cuda()
    plain = EncoderStack(cfg, "cuda", precision, 2, GradReducer())
    stack = EncoderStack(cfg, "cuda", precision, 2, GradReducer(), optimizer=lambda p: optim.AdamW(p, lr=1e-3))
    loss = stack.step(x, go)
    assert torch.equal(loss, plain.step(x, go))
    for p, before, g in zip(stack.parameters(), plain.parameters(), (t for pair in zip(plain.gw, plain.gb) for t in pair)):
        z = torch.zeros_like(p)
        ref.close(p, *ref.adamw(before, g, z, z, 1, 1e-3, 0.9, 0.999, 1e-8, 0.01)[0], torch.float32, "parameter")
    assert not torch.equal(stack.step(x, go), loss)


def test_adamw_refuses_captures_that_would_not_count():
    p = normal((100,), 1).requires_grad_()
    p.grad = normal((100,), 2)
    for o, message in ((optim.AdamW([p]), "capturable"), (optim.AdamW([p], capturable=True), "has to run before")):
        with pytest.raises(RuntimeError, match=message):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                o.step()


def test_capturable_step_and_lr_on_the_device():
    a, b = normal((300,), 1).requires_grad_(), normal((300,), 1).requires_grad_()
    lr = torch.tensor(1e-2, device="cuda")
    o, o2 = optim.AdamW([a], lr=lr, capturable=True), optim.AdamW([b], lr=1e-2)
    for i in range(3):
        a.grad = b.grad = normal((300,), 10 + i)
        o.step()
        o2.step()
    assert (a - b).abs().max() <= 3 * 1e-2 * 40 * ref.U + 4 * ref.U * b.abs().max()   # three steps of at most about lr each
    c = a.detach().clone().requires_grad_()
    o3 = optim.AdamW([c], lr=lr, capturable=True)
    o3.load_state_dict(o.state_dict())
    a.grad = c.grad = normal((300,), 20)
    o.step()
    o3.step()
    assert torch.equal(a, c) and o3.param_groups[0]["step"].item() == 4 == o.param_groups[0]["step"].item()


def test_shared_weight_sums_its_gradients():
    x, y, w = normal((8, 50), 1), normal((8, 50), 2), normal((50,), 3).requires_grad_()
    (F.rms_norm(x, w, None, EPS, -1).sum() + F.rms_norm(y, w, None, EPS, -1).sum()).backward()
    a, = torch.autograd.grad(F.rms_norm(x, w, None, EPS, -1).sum(), w)
    b, = torch.autograd.grad(F.rms_norm(y, w, None, EPS, -1).sum(), w)
    assert torch.equal(w.grad, a + b)
    z = x.clone().requires_grad_()                       # one tensor as input and residual
    out, s = F.rms_norm(z, None, z, EPS, -1)
    gz, = torch.autograd.grad(out.sum() + s.sum(), z)
    leaf = x.clone().requires_grad_()
    o, t = F.rms_norm(leaf, None, x, EPS, -1)
    g1, = torch.autograd.grad(o.sum() + t.sum(), leaf)
    assert torch.equal(gz, g1 + g1)


def test_results_do_not_change_from_call_to_call():
    x, w, g = normal((2, 96, 64, 130), 1), normal((96,), 2), normal((2, 96, 64, 130), 3)
    first = run_norm(x, w, x, 1, g, g)
    for _ in range(3):
        again = run_norm(x, w, x, 1, g, g)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_changed_sum_is_noticed_and_gradients_are_not_differentiable():
    x = normal((4, 30), 1).requires_grad_()
    out, s = F.rms_norm(x, None, normal((4, 30), 2), EPS, -1)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    g, = torch.autograd.grad(F.rms_norm(x, None, None, EPS, -1).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        g.sum().backward()


def test_traced_and_transformed_calls():
    x, w = normal((4, 30), 1), normal((30,), 2)
    traced = torch.jit.trace(lambda a: F.rms_norm(a, w, None, EPS, -1), (x,), check_trace=False)
    y = normal((4, 30), 3)
    assert torch.equal(traced(y), F.rms_norm(y, w, None, EPS, -1))
    a = x.clone().requires_grad_()
    out, s = F._by_function(F._C.rms_norm_op, (a, w, y, EPS, -1))
    g1 = torch.autograd.grad((out * 2).sum() + s.sum(), a)[0]
    b = x.clone().requires_grad_()
    o, t = F.rms_norm(b, w, y, EPS, -1)
    assert torch.equal(g1, torch.autograd.grad((o * 2).sum() + t.sum(), b)[0]) and torch.equal(o, out)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: F.rms_norm(q, w, None, EPS, -1), (x,), (x,))
