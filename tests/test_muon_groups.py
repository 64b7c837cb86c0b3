"""Parameter groups MuonHip takes and refuses (CPU)."""

from __future__ import annotations

import pytest
import sr_states
import torch


def _parameters(n=2):
    return [torch.nn.Parameter(torch.zeros(4, 4)) for _ in range(n)]


def test_a_set_of_parameters_is_refused():
    """Its order changes between runs, and with it every parameter's random stream."""
    with pytest.raises(TypeError, match="ordered collections"):
        sr_states.MuonHip([{"params": set(_parameters())}])
    opt = sr_states.MuonHip(_parameters())
    with pytest.raises(TypeError, match="ordered collections"):
        opt.add_param_group({"params": set(_parameters())})
    assert len(opt.param_groups) == 1


def test_ordered_groups_are_taken():
    a, b, c, d = _parameters(4)
    opt = sr_states.MuonHip([{"params": (p for p in (a, b))}, {"params": c}])
    opt.add_param_group({"params": [d]})
    assert [p for group in opt.param_groups for p in group["params"]] == [a, b, c, d]
