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


@pytest.mark.parametrize("dtypes", [(torch.float16, torch.float16), (torch.float16, torch.float32),
                                    (torch.float32, torch.float16)])
@pytest.mark.parametrize("shape", [(300,), (70, 300), (2, 3, 300)])
def test_linear_of_fp16_and_of_one_row(cuda, dtypes, shape):
    seed, n = 5, 140
    x = _values(shape, cuda, 1, dtypes[0]).requires_grad_()
    w = (_values((n, 300), cuda, 2) * 0.05).to(dtypes[1]).requires_grad_()
    y = sr_states.block_linear(x, w, seed=seed)
    dy = (_values(tuple(y.shape), cuda, 3) * 0.1).to(y.dtype)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert (y.dtype, dx.dtype, dw.dtype) == (dtypes[0], *dtypes) and dx.shape == x.shape and dw.shape == w.shape
    keys = [sr_states.state_key(seed, k) for k in range(3)]
    rows, grads = x.detach().reshape(-1, 300), dy.reshape(-1, n)
    wanted = (
        oracle.product(oracle.block_cast(rows, E4M3, "nearest", False, 1, keys[0]),
                       oracle.block_cast(w.detach(), E4M3, "nearest", True, 1, keys[1])),
        oracle.product(oracle.block_cast(grads, E4M3, "stochastic", False, 1, keys[2]),
                       oracle.block_cast(w.detach(), E4M3, "nearest", True, 0, keys[1])),
        oracle.product(oracle.block_cast(grads, E4M3, "stochastic", False, 0, keys[2]),
                       oracle.block_cast(rows, E4M3, "nearest", False, 0, keys[0])),
    )
    for got, (want, magnitude), k in zip((y, dx, dw), wanted, (300, n, rows.shape[0])):
        got = got.detach().reshape(want.shape)
        inner = k * 2.0**-24 + (0 if got.dtype == torch.float32 else 2.0**-13)
        limit = HALF_ULP[got.dtype] * want.abs() + inner * magnitude * (1 + HALF_ULP[got.dtype])
        if got.dtype == torch.float16:
            limit = limit + 2.0**-25
        assert float(((got.double() - want).abs() - limit).max()) <= 0


def test_linear_gradients_of_an_expanded_and_of_a_strided_gradient(cuda):
    x, w = _values((60, 200), cuda, 1), _values((50, 200), cuda, 2)

    def gradients(dy):
        leaves = x.clone().requires_grad_(), w.clone().requires_grad_()
        return torch.autograd.grad(sr_states.block_linear(*leaves, seed=3), leaves, dy)

    for dy in (torch.ones((), device=cuda).expand(60, 50), _values((50,), cuda, 3).expand(60, 50),
               _values((50, 60), cuda, 4).t(), _values((60, 57), cuda, 5)[:, 3:53]):
        for got, want in zip(gradients(dy), gradients(dy.contiguous())):
            assert torch.equal(got, want)
    # Only one of the two is wanted.
    leaf = x.clone().requires_grad_()
    dy = _values((60, 50), cuda, 6)
    sr_states.block_linear(leaf, w, seed=3).backward(dy)
    assert torch.equal(leaf.grad, gradients(dy)[0])
    leaf = w.clone().requires_grad_()
    sr_states.block_linear(x, leaf, seed=3).backward(dy)
    assert torch.equal(leaf.grad, gradients(dy)[1])


def test_linear_under_autocast_checkpointing_and_compilation(cuda):
    from torch.utils.checkpoint import checkpoint

    x, w = _values((60, 200), cuda, 1, torch.bfloat16), _values((50, 200), cuda, 2)
    dy = _values((60, 50), cuda, 3, torch.bfloat16)

    def gradients(call):
        leaves = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = call(*leaves)
        y.backward(dy)
        return y.detach(), *(leaf.grad for leaf in leaves)

    def layer(x, w):
        return sr_states.block_linear(x, w, seed=3)

    def cast(x, w):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return layer(x, w)

    want = gradients(layer)
    for call in (cast, lambda x, w: checkpoint(layer, x, w, use_reentrant=False),
                 lambda x, w: checkpoint(layer, x, w, use_reentrant=True), torch.compile(layer, backend="eager")):
        for a, b in zip(gradients(call), want):
            assert torch.equal(a, b)


def test_linear_on_a_side_stream(cuda):
    x, w = _values((300, 512), cuda, 1, torch.bfloat16).requires_grad_(), _values((256, 512), cuda, 2).requires_grad_()
    dy = _values((300, 256), cuda, 3, torch.bfloat16)
    want = torch.autograd.grad(sr_states.block_linear(x, w, seed=1), (x, w), dy)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late = dy.clone()
        for _ in range(20):
            late = late * 1.0
        got = torch.autograd.grad(sr_states.block_linear(x, w, seed=1), (x, w), late)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_products_of_subnormal_values(cuda, dtype):
    """Zeros and the three smallest magnitudes of the format, through each kind of instruction."""
    lowest = 2.0 ** (oracle.FORMATS[dtype][1] - oracle.FORMATS[dtype][0])
    gen = torch.Generator(device=cuda).manual_seed(1)
    for m in (5, 40, 2100):
        a, b = ((torch.randint(-3, 4, (rows, 256), device=cuda, generator=gen) * lowest).to(dtype)
                for rows in (m, 2000))
        for scales in (torch.float8_e8m0fnu, torch.float32):
            operands = [BlockScaled(t, torch.ones(t.shape[0], 2, device=cuda).to(scales)) for t in (a, b)]
            want, magnitude = oracle.product(*operands)
            assert float(want.abs().max()) > 0
            for out in (torch.float32, torch.bfloat16):
                got = sr_states.block_matmul(*operands, out_dtype=out)
                inner = 256 * 2.0**-24 + (0 if out == torch.float32 else 2.0**-13)
                limit = HALF_ULP[out] * want.abs() + inner * magnitude * (1 + HALF_ULP[out])
                assert float(((got.double() - want).abs() - limit).max()) <= 0


@pytest.mark.parametrize("rule", ["nearest", "stochastic"])
def test_cast_of_many_columns_alone(cuda, rule):
    x = _values((4100, 2050), cuda, 1, torch.bfloat16)
    got = sr_states.block_cast(x, dtype=E5M2, axis=0, rounding=rule, seed=9)
    value, scale = oracle.block_cast(x, E5M2, rule, False, 0, 9)
    assert torch.equal(got.data.double(), value) and torch.equal(got.scale.double(), scale)


def test_lazily_negated_views(cuda):
    """Imaginary parts of conjugates, among others, are views whose memory holds the opposite values."""
    x, w, dy = _values((40, 60), cuda, 1), _values((30, 60), cuda, 2), _values((40, 30), cuda, 3)

    def view(t):
        negated = torch._neg_view(-t)
        assert negated.is_neg() and torch.equal(negated, t)
        return negated

    def gradients(x, dy):
        leaf = w.clone().requires_grad_()
        y = sr_states.block_linear(x, leaf, seed=1)
        return y, *torch.autograd.grad(y, leaf, dy)

    for got, want in zip(gradients(view(x), view(dy)), gradients(x, dy)):
        assert torch.equal(got, want)
    assert torch.equal(sr_states.orthogonalize(view(x)), sr_states.orthogonalize(x))
    for axis in (0, 1):
        got, want = (sr_states.block_cast(t, axis=axis, seed=1) for t in (view(x), x))
        assert torch.equal(got.dequantize(), want.dequantize())
    q = sr_states.block_cast(x)
    with pytest.raises(ValueError, match="negated"):
        sr_states.block_matmul(q, q, out=view(_values((40, 40), cuda, 4)))


@pytest.mark.parametrize("k", [128, 768, 1024, 1100])
@pytest.mark.parametrize("m, n", [(40, 70), (300, 2000), (2100, 2000)])
def test_scales_of_one_value_in_either_type_give_one_result(cuda, m, n, k):
    """Powers of two as E8M0 and as FP32, for whole and partial runs of blocks."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    operands = []
    for rows in (m, n):
        codes = torch.randint(100, 150, (rows, -(-k // 128)), device=cuda, generator=gen, dtype=torch.uint8)
        operands.append((_values((rows, k), cuda, rows).to(E4M3), codes.view(torch.float8_e8m0fnu)))
    got, want = (sr_states.block_matmul(*(BlockScaled(data, scale.to(dtype)) for data, scale in operands),
                                        out_dtype=torch.float32) for dtype in (torch.float8_e8m0fnu, torch.float32))
    assert torch.equal(got, want)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m, n, k", [(40, 70, 300), (300, 2000, 1024), (2100, 2000, 208)])
def test_one_small_scale_leaves_the_other_rows_alone(cuda, m, n, k, out):
    """A row scaled by 2^-80, as of a gradient of next to nothing, has products that are normal numbers."""
    gen = torch.Generator(device=cuda).manual_seed(4)
    data = [_values((rows, k), cuda, rows).to(E4M3) for rows in (m, n)]
    scales = [torch.rand(rows, -(-k // 128), device=cuda, generator=gen) + 0.1 for rows in (m, n)]
    b = BlockScaled(data[1], scales[1])
    plain = sr_states.block_matmul(BlockScaled(data[0], scales[0]), b, out_dtype=out)
    scales[0][7] *= 2.0**-80
    small = sr_states.block_matmul(BlockScaled(data[0], scales[0]), b, out_dtype=out)
    others = torch.arange(m, device=cuda) != 7
    assert torch.equal(small[others], plain[others])
    assert torch.equal(small[7].float() * 2.0**80, plain[7].float())
