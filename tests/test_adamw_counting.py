"""Where the number of an AdamW step is kept, as a param group's `capturable` changes: on from where it was, or refused."""
import pytest
import torch

from sphmap import optim


@pytest.fixture
def calls(monkeypatch):
    """The numbers of the steps that were asked for."""
    numbers = []
    monkeypatch.setattr(optim, "adamw_step", lambda *lists, step, **kwargs: numbers.append(float(step)))
    return numbers


def optimizer(n=2, **kwargs):
    params = [torch.zeros(4, requires_grad=True) for _ in range(n)]
    for p in params:
        p.grad = torch.ones(4)
    return params, optim.AdamW(params, **kwargs)


def test_counts_on_when_a_group_becomes_capturable(calls):
    params, o = optimizer()
    for _ in range(3):
        o.step()
    o.param_groups[0]["capturable"] = True
    for _ in range(2):
        o.step()
    o.param_groups[0]["capturable"] = False
    o.step()
    assert calls == [1, 2, 3, 4, 5, 6]
    assert all(o.state[p]["step"] == 6 for p in params) and "step" not in o.param_groups[0]


def test_counts_on_from_a_loaded_state_that_was_not_capturable(calls):
    _, o = optimizer()
    for _ in range(3):
        o.step()
    _, other = optimizer(capturable=True)
    other.load_state_dict(o.state_dict())
    other.param_groups[0]["capturable"] = True      # (loading takes over the saved group's options)
    other.step()
    assert calls == [1, 2, 3, 4]


def test_params_at_different_numbers_cannot_become_capturable(calls):
    params, o = optimizer()
    o.step()
    params[0].grad = None
    o.step()
    o.param_groups[0]["capturable"] = True
    with pytest.raises(RuntimeError, match="different step numbers"):
        o.step()
    assert calls == [1, 2]


def test_a_count_is_not_begun_inside_a_graph(calls, monkeypatch):
    """Every replay would begin it anew."""
    _, o = optimizer()
    o.step()
    o.param_groups[0]["capturable"] = True
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="has to run before"):
        o.step()
    assert calls == [1] and "step" not in o.param_groups[0]


def test_loading_brings_a_groups_tensors_to_its_device():
    """Both that a captured step reads, from a checkpoint that was loaded to the host."""
    def one(device):
        return optim.AdamW([torch.zeros(4, device=device, requires_grad=True)], lr=torch.tensor(1e-3, device=device), capturable=True)
    o, other = one("cpu"), one("meta")
    o.param_groups[0]["step"] = torch.tensor(3.0)
    o.add_param_group(dict(params=[]))
    other.add_param_group(dict(params=[]))
    other.load_state_dict(o.state_dict())
    group = other.param_groups[0]
    assert group["step"].device.type == "meta" and group["lr"].device.type == "meta"


def test_capturable_groups_count_from_one(calls):
    params, o = optimizer(capturable=True)
    o.step()
    params[0].grad = None
    o.step()
    assert calls == [1, 2] and o.param_groups[0]["step"].item() == 2
