"""Edges of the block-scaled operators: grad modes, extreme scales, results that autograd watches.

Tolerances are those of test_gpu_block_scaled.py.
"""

from __future__ import annotations

import _matrix_oracle as oracle
import pytest
import sr_states
import torch
from sr_states import BlockScaled, _lib

pytestmark = pytest.mark.gpu
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
# Unit roundoffs: significands of 8, 11 and 24 bits.
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


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


# Exponents of the two scales and of the data.  The first pairs' scales multiply to more than FP32 holds, or to less
# than its normal numbers, although the results and their partial sums are inside; the last pairs are those where one
# scale alone takes a block's sum out of the range that the other brings it back to.
@pytest.mark.parametrize("log_a, log_b, log_data", [
    (100, 30, -6), (30, 100, -6), (64, 64, -4), (-90, -50, 7), (-50, -90, 7), (-100, -50, 14),
    (-50, -100, 14), (100, -100, 0), (-100, 100, 0), (127, -127, 0), (-127, 127, 0), (120, -120, 6), (-120, 120, 6),
])
@pytest.mark.parametrize("scale", ["e8m0", "fp32"])
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("m, n", [(5, 70), (40, 70), (300, 2000), (2100, 2000)])
def test_scales_far_apart_and_far_from_one(cuda, m, n, dtype, scale, log_a, log_b, log_data):
    if log_data > 8 and dtype == E4M3:
        pytest.skip("beyond E4M3's values")
    k = 200 if m == 40 else 208  # rows of any alignment, and rows on 16 bytes
    gen = torch.Generator(device=cuda).manual_seed(5)
    top = 1.75 * 2.0**oracle.FORMATS[dtype][2]
    data = [(_values((rows, k), cuda, rows) * 2.0**log_data).clamp(-top, top).to(dtype) for rows in (m, n)]
    data[0].view(torch.uint8)[m // 2] = 0  # sums of exactly zero

    def scales(rows, log):
        if scale == "e8m0":
            return torch.full((rows, 2), log + 127, dtype=torch.uint8, device=cuda).view(torch.float8_e8m0fnu)
        fraction = 1 + torch.rand(rows, 2, device=cuda, generator=gen)
        return torch.ldexp(torch.ldexp(fraction.cpu(), torch.tensor(log // 2)), torch.tensor(log - log // 2)).to(cuda)

    a, b = BlockScaled(data[0], scales(m, log_a)), BlockScaled(data[1], scales(n, log_b))
    want, magnitude = oracle.product(a, b)
    for out in (torch.float32, torch.bfloat16) + ((torch.float16,) if log_a + log_b + log_data == 0 else ()):
        got = sr_states.block_matmul(a, b, out_dtype=out)
        assert not got[m // 2].any()
        inner = k * 2.0**-24 + (0 if out == torch.float32 else 2.0**-13)
        limit = HALF_ULP[out] * want.abs() + inner * magnitude * (1 + HALF_ULP[out])
        if out == torch.float16:
            limit = limit + 2.0**-25
        assert float(((got.double() - want).abs() - limit).max()) <= 0


def _operands(device):
    return (sr_states.block_cast(_values((rows, 128), device, rows)) for rows in (8, 16))


def test_a_result_that_requires_a_gradient_is_refused(cuda):
    a, b = _operands(cuda)
    leaf = torch.zeros(8, 16, device=cuda, requires_grad=True)
    for out in (leaf, leaf * 1.0):
        with pytest.raises(RuntimeError, match="requires grad"):
            sr_states.block_matmul(a, b, out=out)
        assert not out.any()
    with torch.no_grad():  # as torch's own out= functions
        assert sr_states.block_matmul(a, b, out=leaf) is leaf
    assert torch.equal(leaf, sr_states.block_matmul(a, b, out_dtype=torch.float32))


def test_a_result_written_over_a_saved_tensor_is_noticed(cuda):
    a, b = _operands(cuda)
    x = torch.ones(8, 16, device=cuda, requires_grad=True)
    saved = torch.full((8, 16), 2.0, device=cuda)
    product = x * saved
    version = saved._version
    sr_states.block_matmul(a, b, out=saved)
    assert saved._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        inside = torch.empty(8, 16, device=cuda)
        sr_states.block_matmul(a, b, out=inside)
    # Nothing tracks an inference tensor.
    assert sr_states.block_matmul(a, b, out=inside) is inside
