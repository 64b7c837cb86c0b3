"""Edges of the block-scaled operators: grad modes, extreme scales, results that autograd watches."""

from __future__ import annotations

import pytest
import sr_states
import torch
from sr_states import _lib

pytestmark = pytest.mark.gpu


def _values(shape, device, seed, dtype=torch.float32):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(shape, device=device, generator=gen).to(dtype)


class _Recorder:
    """The native entries, with the results of linear_forward kept."""

    def __init__(self, module):
        self.module, self.results = module, []

    def __getattr__(self, name):
        return getattr(self.module, name)

    def linear_forward(self, *args):
        self.results.append(self.module.linear_forward(*args))
        return self.results[-1]


@pytest.fixture
def recorder(monkeypatch):
    recorder = _Recorder(_lib.matrix())
    monkeypatch.setattr(_lib, "_matrix", recorder)
    return recorder


# What a forward pass makes for the backward one, by which tensors require gradients and the grad mode.
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode, torch.enable_grad])
@pytest.mark.parametrize("x_grad, w_grad", [(False, True), (True, False), (True, True), (False, False)])
def test_linear_casts_for_a_backward_pass_only_where_one_can_follow(cuda, recorder, mode, x_grad, w_grad):
    x = _values((40, 256), cuda, 1).requires_grad_(x_grad)
    w = torch.nn.Parameter(_values((30, 256), cuda, 2), requires_grad=w_grad)
    with mode():
        y = sr_states.block_linear(x, w)
    follows = mode is torch.enable_grad
    (out,) = recorder.results
    # The input's turned cast makes the weight gradient, the weight's the input gradient.
    assert [t is not None for t in out[1:]] == [follows and w_grad] * 2 + [follows and x_grad] * 2
    assert y.requires_grad == (follows and (x_grad or w_grad))
    with torch.enable_grad():
        assert torch.equal(y, sr_states.block_linear(x, w).detach())
