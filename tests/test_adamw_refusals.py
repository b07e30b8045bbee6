"""Calls of the AdamW step that would be lost or go wrong without a word, refused before any device is asked for."""
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
