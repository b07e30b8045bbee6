"""EncoderStack with an optimizer: whose weights it updates, from which gradients, with one rank and behind the exchange of two.
The convolutions are stood in for by products on the CPU, whose gradients are easy to write down."""
import contextlib
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from sphmap import capi
from sphmap.parallel import EncoderStack, GradReducer, shard_batch
from test_parallel import _free_port

CHANNELS = (3, 5, 4, 6, 2)


def config(batch=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    layers = [(ci, co, (3, 4), (3, 4), 1) for ci, co in zip(CHANNELS, CHANNELS[1:])]
    return dict(K=2, interp=1, layers=layers, maps=[torch.zeros(3, 4, 2, 2)] * 4, x=torch.rand(batch, 3, 3, 4, generator=g),
                weights=[torch.randn(co, ci, 2, generator=g) * 0.5 for ci, co, *_ in layers],
                biases=[torch.rand(co, generator=g) for _, co, *_ in layers],
                grad_output=torch.randn(batch, CHANNELS[-1], 3, 4, generator=g))


@contextlib.contextmanager
def plain_convolutions():
    """Every slot of the kernel reads the pixel itself."""
    def forward(x, smap, w, b, K, interp, iw=None, precision=0, out=None, ws=None):
        return out.copy_(torch.einsum("bihw,oik->bohw", x, w) + b.view(-1, 1, 1))

    def backward_input(go, plan, w, ih, iw_, K, precision=0, out=None, ws=None):
        return out.copy_(torch.einsum("bohw,oik->bihw", go, w))

    def backward_weight(go, x, smap, K, interp, iw=None, precision=0, ws=None, gw=None, gb=None):
        gw.copy_(torch.einsum("bohw,bihw->oi", go, x).unsqueeze(2).expand_as(gw))
        return gw, gb.copy_(go.sum((0, 2, 3)))
    fakes = dict(plan_build=lambda *a: None, conv_workspace=lambda *a, **k: None, conv_forward=forward, conv_backward_input=backward_input,
                 conv_backward_weight=backward_weight)
    before = {k: getattr(capi, k) for k in fakes}
    for k, f in fakes.items():
        setattr(capi, k, f)
    try:
        yield
    finally:
        for k, f in before.items():
            setattr(capi, k, f)


def sgd(params):
    return torch.optim.SGD(params, lr=0.01)


def stack_of(cfg, batch=4, **kwargs):
    return EncoderStack(cfg, "cpu", capi.EXACT, batch, fuse_relu=False, companions=False, **kwargs)


def stepped(cfg, steps=1):
    """Weights and biases after plain steps of the same optimizer."""
    params = [t.clone().requires_grad_() for pair in zip(cfg["weights"], cfg["biases"]) for t in pair]
    o = sgd(params)
    for _ in range(steps):
        h = cfg["x"]
        for w, b in zip(params[::2], params[1::2]):
            h = torch.relu(torch.einsum("bihw,oik->bohw", h, w) + b.view(-1, 1, 1))
        o.zero_grad()
        (h * cfg["grad_output"]).sum().backward()
        o.step()
    return [p.detach() for p in params]


def check(stack, want):
    for p, q in zip(stack.parameters(), want):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-5)     # sums of up to 48 float32 terms of about one


def test_the_callers_weights_stay():
    """Of a config that already lies where the stack does."""
    cfg = config()
    kept, want = [t.clone() for t in cfg["weights"] + cfg["biases"]], stepped(cfg)
    with plain_convolutions():
        stack = stack_of(cfg, optimizer=sgd)
        stack.step(cfg["x"], cfg["grad_output"])
    assert all(torch.equal(a, b) for a, b in zip(cfg["weights"] + cfg["biases"], kept))
    assert all(t.grad is None for t in cfg["weights"] + cfg["biases"])
    check(stack, want)


def test_two_stacks_of_one_config_do_not_share():
    cfg = config()
    want = [stepped(cfg, n) for n in range(3)]
    with plain_convolutions():
        a, b, c = stack_of(cfg, optimizer=sgd), stack_of(cfg, optimizer=sgd), stack_of(cfg)
        c.parameters()
        for _ in range(2):
            a.step(cfg["x"], cfg["grad_output"])
        check(a, want[2])
        check(b, want[0])
        check(c, want[0])
        b.step(cfg["x"], cfg["grad_output"])
        check(b, want[1])


@pytest.mark.parametrize("to_none", [False, True])
def test_cleared_gradients_do_not_end_the_updates(to_none):
    cfg = config()
    want = stepped(cfg, 3)
    with plain_convolutions():
        stack = stack_of(cfg, optimizer=sgd)
        for _ in range(3):
            stack.optimizer.zero_grad(set_to_none=to_none)
            stack.step(cfg["x"], cfg["grad_output"])
        check(stack, want)


def _rank(rank, world, port, mode, out):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    cfg = config(5)
    lo, hi = shard_batch(5, rank, world)
    want = stepped(cfg, 2)       # of the whole batch
    with plain_convolutions():
        stack = stack_of(cfg, hi - lo, reducer=GradReducer(mode=mode), optimizer=sgd)
        for _ in range(2):
            stack.step(cfg["x"][lo:hi], cfg["grad_output"][lo:hi])
        check(stack, want)
    out[rank] = [p.tolist() for p in stack.parameters()]
    dist.destroy_process_group()


@pytest.mark.parametrize("mode", ["layer", "step"])
def test_two_ranks_update_from_the_exchanged_gradients(mode):
    with mp.Manager() as manager:
        out = manager.dict()
        mp.spawn(_rank, args=(2, _free_port(), mode, out), nprocs=2, join=True)
        assert out[0] == out[1]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [0, 1])
def test_a_step_uses_the_weights_that_the_last_one_left(precision):
    """The second step's loss and gradients are those of a new stack made from the updated weights: nothing keeps a copy of the old."""
    from sphmap import optim, workloads
    cfg = workloads.config4(B=2, H=64, W=128)
    x, go = cfg["x"].cuda(), cfg["grad_output"].cuda()
    stack = EncoderStack(cfg, "cuda", precision, 2, GradReducer(), optimizer=lambda p: optim.AdamW(p, lr=1e-3))
    stack.step(x, go)
    now = dict(cfg, weights=[t.clone() for t in stack.w], biases=[t.clone() for t in stack.b])
    fresh = EncoderStack(now, "cuda", precision, 2, GradReducer())
    want, loss = fresh.step(x, go), stack.step(x, go)
    assert torch.equal(loss, want)
    for a, b in zip(stack.gw + stack.gb, fresh.gw + fresh.gb):
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(now["weights"], fresh.w))


@pytest.mark.gpu
def test_a_config_on_the_device_stays():
    from sphmap import optim, workloads
    cfg = workloads.config4(B=2, H=64, W=128)
    there = dict(cfg, weights=[t.cuda() for t in cfg["weights"]], biases=[t.cuda() for t in cfg["biases"]])
    x, go = cfg["x"].cuda(), cfg["grad_output"].cuda()
    adamw = lambda p: optim.AdamW(p, lr=1e-3)  # noqa: E731
    a, b = (EncoderStack(there, "cuda", 0, 2, optimizer=adamw) for _ in range(2))
    for _ in range(2):
        a.optimizer.zero_grad()
        a.step(x, go)
    for t, u, v in zip(there["weights"] + there["biases"], cfg["weights"] + cfg["biases"], b.w + b.b):
        assert torch.equal(t.cpu(), u) and torch.equal(v, t) and t.grad is None
    assert a.optimizer.state[a.w[0]]["step"] == 2 and not torch.equal(a.w[0], b.w[0])
