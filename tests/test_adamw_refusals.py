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
