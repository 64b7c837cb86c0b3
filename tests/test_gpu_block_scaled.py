"""block_cast, block_matmul and block_linear against 64-bit forms of their definitions.

Tolerances.  A cast has one right value per element.  A product's sums are
FP32: k terms of magnitudes adding up to S lie within k 2^-24 S of the exact
sum, which bounds FP32 results; the FP8 instructions behind BF16 and FP16
results keep at least 15 bits of a block's largest term, which adds at most
2^-13 S; the final rounding adds at most the type's unit roundoff, 2^-8, 2^-11
or 2^-24 of the result.
"""

from __future__ import annotations

import _matrix_oracle as oracle
import pytest
import sr_states
import torch
from sr_states import BlockScaled

pytestmark = pytest.mark.gpu
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
# Unit roundoffs: significands of 8, 11 and 24 bits.
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _spread(shape, device, seed, dtype=torch.float32):
    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(shape, device=device, generator=gen)
    return (x * torch.randn(shape[-1], device=device, generator=gen).exp()).to(dtype)


def _assert_cast(got, x, dtype, rule, square, axis, seed):
    value, scale = oracle.block_cast(x, dtype, rule, square, axis, seed)
    assert got.data.dtype == dtype and got.scale.dtype == torch.float8_e8m0fnu
    torch.testing.assert_close(got.scale.double(), scale, rtol=0, atol=0)
    torch.testing.assert_close(got.data.double(), value, rtol=0, atol=0, equal_nan=True)


SHAPES = [(1, 1), (1, 128), (1, 2048), (3, 127), (128, 128), (129, 257), (130, 4), (257, 5), (500, 1000)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("dtype, rule", [(E4M3, "nearest"), (E4M3, "stochastic"), (E5M2, "nearest"), (E5M2, "stochastic")])
def test_cast_equals_the_definition(cuda, shape, square, dtype, rule):
    x = _spread(shape, cuda, 3, torch.bfloat16)
    block = (128, 128) if square else (1, 128)
    by_rows, by_cols = sr_states.block_cast(x, dtype=dtype, block=block, axis=(1, 0), rounding=rule, seed=11, offset=5)
    _assert_cast(by_rows, x, dtype, rule, square, 1, 16)
    _assert_cast(by_cols, x, dtype, rule, square, 0, 16)
    for axis, both in ((1, by_rows), (0, by_cols)):
        one = sr_states.block_cast(x, dtype=dtype, block=block, axis=axis, rounding=rule, seed=16)
        assert torch.equal(one.data.view(torch.uint8), both.data.view(torch.uint8))
        assert torch.equal(one.scale.view(torch.uint8), both.scale.view(torch.uint8))
    turned = sr_states.block_cast(x, dtype=dtype, block=block, axis=(0, 1), rounding=rule, seed=16)
    assert torch.equal(turned[0].data.view(torch.uint8), by_cols.data.view(torch.uint8))


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("skip, wide", [(0, 0), (1, 3), (5, 1)])
def test_cast_reads_strided_rows_of_any_alignment(cuda, x_dtype, skip, wide):
    rows, cols = 140, 261
    flat = _spread((rows * (cols + wide) + skip,), cuda, 4, x_dtype)
    x = flat[skip:].view(rows, cols + wide)[:, :cols]
    for axis in (1, 0):
        got = sr_states.block_cast(x, axis=axis, seed=3)
        _assert_cast(got, x, E4M3, "stochastic", False, axis, 3)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("square", [False, True])
def test_cast_of_special_values(cuda, dtype, square):
    x = torch.zeros(256, 384, device=cuda)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = float("nan"), float("inf"), -float("inf"), 3.0
    x[1, 130], x[1, 131] = float("inf"), -0.0  # a block without a nonzero finite value
    x[2, 256:] = 2.0**-149  # subnormal: the scale stops at 2^-127
    x[3, 256:] = 3.4e38
    x[200, :] = torch.linspace(-1e-3, 1e-3, 384, device=cuda)
    for rule in ("nearest", "stochastic"):
        for axis in (1, 0):
            got = sr_states.block_cast(x, dtype=dtype, block=(128, 128) if square else (1, 128), axis=axis,
                                       rounding=rule, seed=1)
            _assert_cast(got, x, dtype, rule, square, axis, 1)


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype, rule", [(E4M3, "nearest"), (E4M3, "stochastic"), (E5M2, "nearest"), (E5M2, "stochastic")])
def test_cast_of_many_blocks_in_both_orientations(cuda, x_dtype, dtype, rule):
    x = torch.empty(2050, 2101, device=cuda, dtype=x_dtype).copy_(_spread((2050, 2101), cuda, 6))
    x[5, 7], x[600, 1300], x[600, 1301], x[2049, 2100] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[128:256, 256:384] = 0
    x[300:400, 100] *= 2.0**-12
    by_rows, by_cols = sr_states.block_cast(x, dtype=dtype, axis=(1, 0), rounding=rule, seed=4)
    _assert_cast(by_rows, x, dtype, rule, False, 1, 4)
    _assert_cast(by_cols, x, dtype, rule, False, 0, 4)


def test_cast_is_the_plain_cast_of_the_scaled_values(cuda):
    x = _spread((64, 256), cuda, 8)
    got = sr_states.block_cast(x, seed=21)
    factor = got.scale.float().repeat_interleave(128, 1)
    want = sr_states.cast((x / factor).contiguous(), dtype=E4M3, seed=21)
    assert torch.equal(got.data.contiguous().view(torch.uint8), want.view(torch.uint8))


def test_cast_wraps_its_counters(cuda):
    x = _spread((3, 200), cuda, 9)
    got = sr_states.block_cast(x, seed=0xFFFFFFF0, offset=7)
    _assert_cast(got, x, E4M3, "stochastic", False, 1, 0xFFFFFFF7)


def _operand(rows, k, dtype, scale, square, device, seed, pad=0, skip=0):
    """A random block-scaled matrix; its rows lie `pad` bytes apart in a buffer of NaN bytes."""
    gen = torch.Generator(device=device).manual_seed(seed)
    values = (torch.randn(rows, k, device=device, generator=gen) * oracle.FORMATS[dtype][2] * 4).to(dtype)
    buffer = torch.full((skip + rows * (k + pad) + 64,), 0x7F, dtype=torch.uint8, device=device)
    data = buffer[skip:skip + rows * (k + pad)].view(rows, k + pad)[:, :k].view(dtype)
    data.view(torch.uint8).copy_(values.view(torch.uint8))
    shape = (-(-rows // 128) if square else rows, -(-k // 128))
    if scale == "e8m0":
        factor = torch.randint(118, 130, shape, device=device, generator=gen, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    else:
        factor = torch.rand(shape, device=device, generator=gen) + 0.01
    return BlockScaled(data, factor)


def _assert_product(a, b, dtype, got=None):
    if got is None:
        got = sr_states.block_matmul(a, b, out_dtype=dtype)
    assert got.dtype == dtype and got.shape == (a.data.shape[0], b.data.shape[0])
    want, magnitude = oracle.product(a, b)
    k = a.data.shape[1]
    inner = k * 2.0**-24 if dtype == torch.float32 else k * 2.0**-24 + 2.0**-13
    limit = HALF_ULP[dtype] * want.abs() + inner * magnitude * (1 + HALF_ULP[dtype])
    if dtype == torch.float16:
        limit = limit + 2.0**-25  # half the spacing below its normal range
    excess = (got.double() - want).abs() - limit
    assert not got.isnan().any()
    assert float(excess.max()) <= 0, f"{float(excess.max())} over the bound"


SIZES = [
    (1, 16, 128), (1, 1, 1), (2, 17, 100), (16, 130, 1000), (17, 64, 128), (17, 65, 129), (33, 500, 640),
    (64, 64, 256), (100, 2305, 384), (128, 128, 2048), (300, 257, 1000), (513, 130, 127), (700, 5200, 160),
]


@pytest.mark.parametrize("m, n, k", SIZES)
@pytest.mark.parametrize("scale", ["e8m0", "fp32"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_equals_the_definition(cuda, m, n, k, scale, out):
    a = _operand(m, k, E4M3, scale, False, cuda, 1)
    b = _operand(n, k, E4M3, scale, True, cuda, 2)
    _assert_product(a, b, out)


@pytest.mark.parametrize("a_dtype", [E4M3, E5M2])
@pytest.mark.parametrize("b_dtype", [E4M3, E5M2])
@pytest.mark.parametrize("squares", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("scale", ["e8m0", "fp32"])
def test_product_formats_and_block_shapes(cuda, a_dtype, b_dtype, squares, scale):
    for m, n, k in ((5, 200, 300), (150, 270, 300)):
        a = _operand(m, k, a_dtype, scale, squares[0], cuda, 3)
        b = _operand(n, k, b_dtype, scale, squares[1], cuda, 4)
        for out in (torch.bfloat16, torch.float16, torch.float32):
            if out == torch.float16:  # inside FP16's range
                a = BlockScaled(a.data, (a.scale.float() * 2.0**-14).to(a.scale.dtype))
            _assert_product(a, b, out)


@pytest.mark.parametrize("m, n", [(3, 40), (70, 150), (2100, 2100)])
@pytest.mark.parametrize("pad, skip", [(0, 1), (1, 0), (8, 0), (16, 16), (16, 3)])
@pytest.mark.parametrize("k", [256, 272, 200])
def test_product_of_strided_rows_reads_nothing_beyond_them(cuda, m, n, pad, skip, k):
    # Everything between the rows is NaN: a value read from there would show.
    a = _operand(m, k, E4M3, "e8m0", False, cuda, 5, pad, skip)
    b = _operand(n, k, E4M3, "e8m0", True, cuda, 6, pad, skip)
    for out in (torch.bfloat16, torch.float32):
        _assert_product(a, b, out)


def test_product_into_a_strided_result(cuda):
    a = _operand(130, 256, E4M3, "e8m0", False, cuda, 1)
    b = _operand(70, 256, E4M3, "e8m0", False, cuda, 2)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        a16 = BlockScaled(a.data, (a.scale.float() * 2.0**-14).to(a.scale.dtype)) if dtype == torch.float16 else a
        whole = torch.full((131, 75), 7.0, dtype=dtype, device=cuda)
        out = whole[1:, 3:73]
        assert sr_states.block_matmul(a16, b, out=out) is out
        _assert_product(a16, b, dtype, out)
        assert (whole[0] == 7).all() and (whole[:, :3] == 7).all() and (whole[:, 73:] == 7).all()


def test_products_of_nothing(cuda):
    def empty(rows, k):
        return BlockScaled(torch.zeros(rows, k, device=cuda).to(E4M3),
                           torch.ones(rows, -(-k // 128), device=cuda))

    assert sr_states.block_matmul(empty(0, 128), empty(5, 128)).shape == (0, 5)
    assert sr_states.block_matmul(empty(5, 128), empty(0, 128)).shape == (5, 0)
    for m in (3, 40):
        assert torch.equal(sr_states.block_matmul(empty(m, 0), empty(5, 0)), torch.zeros(m, 5, device=cuda, dtype=torch.bfloat16))
    for shape in ((0, 128), (5, 0), (0, 0)):
        for q in sr_states.block_cast(torch.zeros(shape, device=cuda), axis=(1, 0)):
            assert q.data.numel() == 0


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_scales_and_values_that_are_not_finite_reach_the_result(cuda, out):
    for m in (4, 40):
        a, b = (_operand(r, 256, E4M3, "e8m0", False, cuda, 7) for r in (m, 20))
        a.data[1, 200] = float("nan")
        a.scale.view(torch.uint8)[2, 1] = 255  # E8M0's NaN
        got = sr_states.block_matmul(a, b, out_dtype=out)
        nan = got.isnan()
        assert nan[1].all() and nan[2].all() and not nan[0].any() and not nan[3:].any()


def test_offsets_beyond_32_bits(cuda):
    rows, k = (1 << 24) + 300, 256  # 4.3 GB of data
    data = torch.zeros(rows, k, dtype=torch.uint8, device=cuda)
    tail = _operand(300, k, E4M3, "e8m0", False, cuda, 1)
    data[-300:] = tail.data.view(torch.uint8)
    scale = torch.full((rows, 2), 127, dtype=torch.uint8, device=cuda)
    scale[-300:] = tail.scale.view(torch.uint8)
    b = _operand(16, k, E4M3, "e8m0", False, cuda, 2)
    got = sr_states.block_matmul(BlockScaled(data.view(E4M3), scale.view(torch.float8_e8m0fnu)), b)
    assert not got[:-300].any()
    _assert_product(tail, b, torch.bfloat16, got[-300:])
    del got
    # The large matrix on the other side: its columns of the result.
    got = sr_states.block_matmul(b, BlockScaled(data.view(E4M3), scale.view(torch.float8_e8m0fnu)))
    _assert_product(b, tail, torch.bfloat16, got[:, -300:])


def test_operators_run_on_the_current_stream(cuda):
    stream = torch.cuda.Stream()
    x = _spread((512, 512), cuda, 1, torch.bfloat16)
    want = sr_states.block_matmul(sr_states.block_cast(x), sr_states.block_cast(x))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        y = x.clone()
        for _ in range(20):
            y = y * 1.0
        got = sr_states.block_matmul(sr_states.block_cast(y), sr_states.block_cast(y))
    stream.synchronize()
    assert torch.equal(got, want)


def test_captured_products_replay(cuda):
    x = _spread((300, 512), cuda, 1, torch.bfloat16)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        warm = sr_states.block_cast(x)
        sr_states.block_matmul(warm, warm)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = sr_states.block_cast(x, seed=3)
        out = sr_states.block_matmul(q, q)
    for k in range(3):
        x.copy_(_spread((300, 512), cuda, 10 + k, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        q2 = sr_states.block_cast(x, seed=3)
        assert torch.equal(out, sr_states.block_matmul(q2, q2))


def _linear_reference(x, w, dy, seed, formats):
    keys = [sr_states.state_key(seed, k) for k in range(3)]

    def cast(t, k, square, axis):
        dtype, rule = formats[k]
        return oracle.block_cast(t, dtype, rule, square, axis, keys[k])

    y = oracle.product(cast(x, 0, False, 1), cast(w, 1, True, 1))
    dx = oracle.product(cast(dy, 2, False, 1), cast(w, 1, True, 0))
    dw = oracle.product(cast(dy, 2, False, 0), cast(x, 0, False, 0))
    return y, dx, dw


DEFAULT_FORMATS = ((E4M3, "nearest"), (E4M3, "nearest"), (E4M3, "stochastic"))
MIXED_FORMATS = ((E4M3, "stochastic"), (E4M3, "nearest"), (E5M2, "stochastic"))


@pytest.mark.parametrize("shape, n", [((3, 50, 200), 150), ((1, 64), 1), ((257, 384), 640)])
@pytest.mark.parametrize("dtypes", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("formats", [DEFAULT_FORMATS, MIXED_FORMATS])
def test_linear_equals_the_formulas(cuda, shape, n, dtypes, formats):
    seed = 77
    x = _spread(shape, cuda, 1, dtypes[0]).requires_grad_()
    w = (_spread((n, shape[-1]), cuda, 2) * 0.05).to(dtypes[1]).requires_grad_()
    dy = (_spread((*shape[:-1], n), cuda, 3) * 1e-3).to(dtypes[0])
    given = None if formats is DEFAULT_FORMATS else {
        name: sr_states.StateFormat(*fmt) for name, fmt in zip(("input", "weight", "gradient"), formats)}
    y = sr_states.block_linear(x, w, seed=seed, formats=given)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == dx.dtype == dtypes[0] and dw.dtype == dtypes[1]
    assert y.shape == dy.shape and dx.shape == x.shape and dw.shape == w.shape
    flat = [t.detach().reshape(-1, t.shape[-1]) for t in (x, dy)]
    reference = _linear_reference(flat[0], w.detach(), flat[1], seed, formats)
    for got, (want, magnitude), k in zip((y, dx, dw), reference, (shape[-1], n, flat[0].shape[0])):
        got = got.detach().reshape(want.shape)
        inner = k * 2.0**-24 + (0 if got.dtype == torch.float32 else 2.0**-13)
        limit = HALF_ULP[got.dtype] * want.abs() + inner * magnitude * (1 + HALF_ULP[got.dtype])
        assert float(((got.double() - want).abs() - limit).max()) <= 0


def test_linear_gradients_are_differences_where_fp8_is_exact(cuda):
    """Small integers survive the casts, so the layer is exactly linear there and differences are exact."""
    gen = torch.Generator(device=cuda).manual_seed(0)

    def integers(*shape):
        return torch.randint(-4, 5, shape, device=cuda, generator=gen).float()

    x, w, dy = integers(60, 140).requires_grad_(), integers(70, 140).requires_grad_(), integers(60, 70)
    dx, dw = torch.autograd.grad(sr_states.block_linear(x, w), (x, w), dy)

    def loss(x, w):
        return float((sr_states.block_linear(x, w).double() * dy.double()).sum())

    with torch.no_grad():
        start = loss(x, w)
        for _ in range(8):
            r, c = (int(torch.randint(0, s, ())) for s in x.shape)
            moved = x.clone()
            moved[r, c] += 1
            assert loss(moved, w) - start == float(dx[r, c])
            r, c = (int(torch.randint(0, s, ())) for s in w.shape)
            moved = w.clone()
            moved[r, c] += 1
            assert loss(x, moved) - start == float(dw[r, c])


def test_linear_gradients_that_are_not_wanted_are_not_computed(cuda):
    x, w = _spread((40, 128), cuda, 1), _spread((30, 128), cuda, 2)
    y = sr_states.block_linear(x.clone().requires_grad_(), w)
    y.sum().backward()
    leaf = w.clone().requires_grad_()
    # An expanded gradient and a transposed input.
    out = sr_states.block_linear(x.t().contiguous().t(), leaf)
    out.sum().backward()
    assert leaf.grad.shape == w.shape
    assert not sr_states.block_linear(x, w).requires_grad


def test_linear_over_no_tokens(cuda):
    x = torch.zeros(0, 3, 128, device=cuda, requires_grad=True)
    w = torch.ones(20, 128, device=cuda, requires_grad=True)
    y = sr_states.block_linear(x, w)
    assert y.shape == (0, 3, 20)
    y.sum().backward()
    assert x.grad.shape == x.shape and torch.equal(w.grad, torch.zeros_like(w))


def test_refusals(cuda):
    x = torch.zeros(8, 256, device=cuda)
    q = sr_states.block_cast(x)
    cases = [
        (TypeError, "expected FP32, BF16 or FP16", lambda: sr_states.block_cast(x.double())),
        (TypeError, "expected a tensor", lambda: sr_states.block_cast([1.0])),
        (ValueError, "block casts give", lambda: sr_states.block_cast(x, dtype=torch.bfloat16)),
        (ValueError, "no rounding", lambda: sr_states.block_cast(x, rounding="up")),
        (ValueError, "block must be", lambda: sr_states.block_cast(x, block=(1, 64))),
        (ValueError, "axis must be", lambda: sr_states.block_cast(x, axis=2)),
        (ValueError, "takes a matrix", lambda: sr_states.block_cast(x[0])),
        (ValueError, "consecutive columns", lambda: sr_states.block_cast(x.t())),
        (ValueError, "consecutive columns", lambda: sr_states.block_cast(x[:1].expand(8, 256))),
        (TypeError, "data must be FP8", lambda: sr_states.block_matmul(BlockScaled(x, q.scale), q)),
        (TypeError, "scales must be", lambda: sr_states.block_matmul(BlockScaled(q.data, q.scale.half()), q)),
        (ValueError, "scales of a 8 x 256", lambda: sr_states.block_matmul(BlockScaled(q.data, q.scale[:, :1]), q)),
        (TypeError, "scales of one type", lambda: sr_states.block_matmul(BlockScaled(q.data, q.scale.float()), q)),
        (ValueError, "contract 256 and 128", lambda: sr_states.block_matmul(q, sr_states.block_cast(x[:, :128]))),
        (TypeError, "out_dtype must be", lambda: sr_states.block_matmul(q, q, out_dtype=E4M3)),
        (ValueError, "out must be", lambda: sr_states.block_matmul(q, q, out=torch.zeros(8, 9, device=cuda))),
        (TypeError, "out has dtype", lambda: sr_states.block_matmul(q, q, out_dtype=torch.float16, out=torch.zeros(8, 8, device=cuda))),
        (ValueError, "must not overlap", lambda: sr_states.block_matmul(q, q, out=q.data.view(torch.uint8).flatten()[:256].view(torch.float32).view(8, 8))),
        (ValueError, "do not match", lambda: sr_states.block_linear(x, x[:, :128].contiguous())),
        (ValueError, "must be FP8", lambda: sr_states.block_linear(x, x, formats=sr_states.StateFormat(torch.bfloat16))),
        (ValueError, "same GPU", lambda: sr_states.block_linear(x, x.cpu())),
    ]
    for error, message, call in cases:
        with pytest.raises(error, match=message):
            call()
