"""Calls of the AdamW step that would be lost or go wrong without a word, refused before any device is asked for."""
import random

import pytest
import torch

from sphmap import optim


def test_adamw_step_in_a_trace_is_refused():
    """A trace would hold nothing of it, and its replays would not step."""
    p = torch.zeros(5)

    def step(g):
        optim.adamw_step([p], [g], [torch.zeros(5)], [torch.zeros(5)], step=1, lr=1e-3)
        return g * 1
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(step, (torch.ones(5),), check_trace=False)


def lists(sizes, eight=False, master=False):
    """Arguments of a step over tensors that lie apart."""
    dtype = torch.bfloat16 if master else torch.float32
    state = torch.float8_e4m3fn if eight else torch.float32
    zeros = lambda d, f=lambda n: n: [torch.zeros(f(n), dtype=d) for n in sizes]  # noqa: E731
    a = dict(params=zeros(dtype), grads=zeros(dtype), exp_avgs=zeros(state), exp_avg_sqs=zeros(state))
    if master:
        a["masters"] = zeros(torch.float32)
    if eight:
        a["exp_avg_scales"], a["exp_avg_sq_scales"] = (zeros(torch.float32, lambda n: -(-n // 256)) for _ in range(2))
    return a


def step(a):
    a = dict(a)
    optim.adamw_step(a.pop("params"), a.pop("grads"), a.pop("exp_avgs"), a.pop("exp_avg_sqs"), step=1, lr=1e-3, **a)


WRITTEN = ["params", "exp_avgs", "exp_avg_sqs", "masters", "exp_avg_scales", "exp_avg_sq_scales"]


@pytest.mark.parametrize("name", WRITTEN)
def test_one_tensor_twice_in_a_list_is_refused(name):
    """Two threads would write the same values."""
    a = lists([600, 70, 600], eight=True, master=True)
    a[name][2] = a[name][0]
    with pytest.raises(RuntimeError, match="appears twice"):
        step(a)


@pytest.mark.parametrize("first", WRITTEN)
@pytest.mark.parametrize("second", WRITTEN + ["grads"])
def test_overlapping_tensors_are_refused(first, second):
    """The last byte of one is the first of another, in the same list or in two."""
    a = lists([520, 520], eight=True, master=True)
    x, y = a[first][0], a[second][1]
    one = torch.zeros(8192, dtype=torch.uint8)
    start = x.numel() * x.element_size() - y.element_size()
    start -= start % 4
    a[first][0] = one[:x.numel() * x.element_size()].view(x.dtype)
    a[second][1] = one[start:start + y.numel() * y.element_size()].view(y.dtype)
    with pytest.raises(RuntimeError, match="overlaps"):
        step(a)


def test_what_does_not_overlap_is_not_refused_for_it():
    """Neighbours of one allocation in any order, empty tensors, one gradient for two params, a gradient inside nothing written."""
    a = lists([512, 0, 512, 0], eight=True, master=True)
    for name in WRITTEN:
        unit = a[name][0].numel()
        flat = torch.zeros(2 * unit, dtype=a[name][0].dtype)
        a[name][0], a[name][2] = flat[unit:], flat[:unit]
        a[name][1], a[name][3] = flat[unit:unit], flat[:0]
    a["grads"][2] = a["grads"][0]
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        step(a)
    b = lists([300, 200], master=False)
    everything = torch.zeros(4, 500)
    for row, name in zip(everything, ("params", "exp_avgs", "grads", "exp_avg_sqs")):
        b[name] = [row[:300], row[300:]]
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        step(b)


def test_overlaps_at_random():
    """Against a look at all pairs: tensors anywhere in one allocation, in any order, of which a few or none overlap."""
    rng = random.Random(5)
    found = [0, 0]
    for _ in range(400):
        n, one = rng.randrange(1, 12), torch.zeros(1 << 14)
        starts = rng.sample(range(0, 1 << 14, 64), 4 * n)
        if rng.random() < 0.5:
            starts.sort(reverse=rng.random() < 0.5)
        a, spans = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[]), []
        for i in range(n):
            size = rng.choice((0, 1, 63, 64, 64, rng.choice((64, 65))))
            for k, name in enumerate(a):
                at = min(starts[4 * i + k], (1 << 14) - size)
                a[name].append(one[at:at + size])
                if size:
                    spans.append((at, at + size, name != "grads"))
        clash = any((p[2] or q[2]) and p[0] < q[1] and q[0] < p[1] for i, p in enumerate(spans) for q in spans[:i])
        found[clash] += 1
        with pytest.raises(RuntimeError, match="overlaps" if clash else "CUDA tensor"):
            step(a)
    assert min(found) > 40
