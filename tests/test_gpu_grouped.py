"""grouped_block_cast, grouped_block_matmul and grouped_block_linear against 64-bit forms of their definitions.

Tolerances are those of test_gpu_block_scaled.py: a cast has one right value
per element; a product of k terms whose magnitudes add up to S is off by at most
k 2^-24 S where it is summed in FP32, 2^-13 S more on the FP8 instructions, and by
the result's unit roundoff.
"""

from __future__ import annotations

import _grouped_oracle as grouped
import _matrix_oracle as oracle
import pytest
import sr_states
import torch
from sr_states import BlockScaled
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
FORMATS = [(E4M3, "nearest"), (E4M3, "stochastic"), (E5M2, "nearest"), (E5M2, "stochastic")]


def _spread(shape, device, seed, dtype=torch.float32):
    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(shape, device=device, generator=gen)
    return (x * torch.randn(shape[-1], device=device, generator=gen).exp()).to(dtype)


def _sizes(counts, device, dtype=torch.int32):
    return torch.tensor(counts, dtype=dtype, device=device)


def _assert_pair(got, want):
    value, scale = want
    assert got.scale.dtype == torch.float8_e8m0fnu and got.data.shape == value.shape
    torch.testing.assert_close(got.scale.double(), scale, rtol=0, atol=0)
    torch.testing.assert_close(got.data.double(), value, rtol=0, atol=0, equal_nan=True)


def _assert_near(got, want, magnitude, k):
    inner = k * 2.0**-24 + (0 if got.dtype == torch.float32 else 2.0**-13)
    limit = HALF_ULP[got.dtype] * want.abs() + inner * magnitude * (1 + HALF_ULP[got.dtype])
    if got.dtype == torch.float16:
        limit = limit + 2.0**-25
    assert got.shape == want.shape and not got.isnan().any()
    # Results of 65520 = 2^16 - 2^4 or more round to FP16's infinities: half a step of 2^5 above its largest number.
    top = 65520.0 if got.dtype == torch.float16 else float("inf")
    high = want.abs() >= top
    assert not (got.isinf() & (want.abs() + limit < top)).any()
    got = torch.where(got.isinf() & (want.abs() + limit >= top) & (got.sign() == want.sign()), want, got.double())
    assert not (high & (want.abs() - limit >= top) & (got != want)).any()
    if got.numel():
        assert float(((got.double() - want).abs() - limit).max()) <= 0


# Groups that are empty, of one row, that end at, before and behind a block's end; rows behind the last group; sizes that
# are negative or lead beyond the matrix; more groups than a wave has lanes.
GROUPS = [
    (1, [1]),
    (1, [0]),
    (5, [0, 5, 0]),
    (300, [1, 127, 128, 44]),
    (300, [129, 0, 0, 100]),
    (300, [0, 0, 0]),
    (300, [-7, 100, 1000, 5]),
    (200, [1, 2] * 50 + [0] * 20),
    (517, [3] * 64 + [0, 200, 1]),
]


@pytest.mark.parametrize("rows, counts", GROUPS)
@pytest.mark.parametrize("cols", [1, 130, 256])
@pytest.mark.parametrize("dtype, rule", FORMATS)
def test_cast_of_groups_equals_the_definition(cuda, rows, counts, cols, dtype, rule):
    x = _spread((rows, cols), cuda, 3, torch.bfloat16)
    sizes = _sizes(counts, cuda)
    live = grouped.counts_of(counts, rows)
    by_rows, by_cols = sr_states.grouped_block_cast(x, sizes, dtype=dtype, axis=(1, 0), rounding=rule, seed=11, offset=5)
    _assert_pair(by_rows, oracle.block_cast(x, dtype, rule, False, 1, 16))
    _assert_pair(by_cols, grouped.cast_columns(x, live, dtype, rule, 16))
    alone = sr_states.grouped_block_cast(x, sizes.long(), dtype=dtype, axis=0, rounding=rule, seed=16)
    assert torch.equal(alone.data.view(torch.uint8), by_cols.data.view(torch.uint8))
    assert torch.equal(alone.scale.view(torch.uint8), by_cols.scale.view(torch.uint8))
    rows_alone = sr_states.grouped_block_cast(x, sizes, dtype=dtype, rounding=rule, seed=16)
    assert torch.equal(rows_alone.data.view(torch.uint8), by_rows.data.view(torch.uint8))


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype, rule", FORMATS)
def test_cast_of_many_blocks_of_groups(cuda, x_dtype, dtype, rule):
    """Enough blocks for workgroups that do both orientations of a tile."""
    x = torch.empty(2050, 2101, device=cuda, dtype=x_dtype).copy_(_spread((2050, 2101), cuda, 6))
    x[5, 7], x[600, 1300], x[600, 1301], x[2049, 2100] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[128:256, 256:384] = 0
    for counts in ([700, 0, 129, 1, 900], [2050], [0] * 70 + [1000, 1050]):
        by_rows, by_cols = sr_states.grouped_block_cast(x, _sizes(counts, cuda), dtype=dtype, axis=(1, 0), rounding=rule, seed=4)
        _assert_pair(by_rows, oracle.block_cast(x, dtype, rule, False, 1, 4))
        _assert_pair(by_cols, grouped.cast_columns(x, counts, dtype, rule, 4))


@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 130, 4), (5, 7, 300), (2, 128, 128), (9, 700, 800)])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("dtype, rule", FORMATS)
def test_cast_of_a_stack_equals_the_definition(cuda, shape, square, dtype, rule):
    x = _spread(shape, cuda, 5)
    block = (128, 128) if square else (1, 128)
    by_cols, by_rows = sr_states.grouped_block_cast(x, dtype=dtype, block=block, axis=(0, 1), rounding=rule, seed=9)
    _assert_pair(by_rows, grouped.cast_stack(x, dtype, rule, square, 1, 9))
    _assert_pair(by_cols, grouped.cast_stack(x, dtype, rule, square, 0, 9))
    for axis, both in ((1, by_rows), (0, by_cols)):
        one = sr_states.grouped_block_cast(x, dtype=dtype, block=block, axis=axis, rounding=rule, seed=9)
        assert torch.equal(one.data.view(torch.uint8), both.data.view(torch.uint8))
        for i in range(shape[0]):
            alone = sr_states.block_cast(x[i], dtype=dtype, block=block, axis=axis, rounding=rule, seed=9, offset=i * x[i].numel())
            assert torch.equal(alone.data.view(torch.uint8), one.data[i].view(torch.uint8))
            assert torch.equal(alone.scale.view(torch.uint8), one.scale[i].view(torch.uint8))


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_casts_read_strided_rows(cuda, x_dtype):
    flat = _spread((3 * 150 * 270 + 5,), cuda, 4, x_dtype)
    x = flat[5:].view(3, 150, 270)[:, 3:143, 1:262]  # matrices, rows and columns apart
    for axis in (1, 0):
        got = sr_states.grouped_block_cast(x, axis=axis, seed=3)
        _assert_pair(got, grouped.cast_stack(x, E4M3, "stochastic", False, axis, 3))
    got = sr_states.grouped_block_cast(x[0], _sizes([40, 60], cuda), axis=0, seed=3)
    _assert_pair(got, grouped.cast_columns(x[0], [40, 60], E4M3, "stochastic", 3))
    same = x[1:2].expand(3, 140, 261)  # one matrix three times
    _assert_pair(sr_states.grouped_block_cast(same, seed=3), grouped.cast_stack(same, E4M3, "stochastic", False, 1, 3))


def _operand(shape, dtype, scale, square, device, seed, pad=0, skip=0):
    """Random block-scaled matrices; rows lie `pad` bytes apart in a buffer of NaN bytes."""
    gen = torch.Generator(device=device).manual_seed(seed)
    *stack, rows, k = shape
    count = stack[0] if stack else 1
    values = (torch.randn(count, rows, k, device=device, generator=gen) * oracle.FORMATS[dtype][2] * 4).to(dtype)
    buffer = torch.full((skip + count * rows * (k + pad) + 64,), 0x7F, dtype=torch.uint8, device=device)
    data = buffer[skip:skip + count * rows * (k + pad)].view(count, rows, k + pad)[..., :k].view(dtype)
    data.view(torch.uint8).copy_(values.view(torch.uint8))
    grid = (count, -(-rows // 128) if square else rows, -(-k // 128))
    if scale == "e8m0":
        factor = torch.randint(118, 130, grid, device=device, generator=gen, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    else:
        factor = torch.rand(grid, device=device, generator=gen) + 0.01
    return BlockScaled(data, factor) if stack else BlockScaled(data[0], factor[0])


@pytest.mark.parametrize("rows, counts", GROUPS + [(700, [300, 0, 17, 250]), (2600, [1300, 1, 1200]), (40, [20, 20]), (1200, [8] * 130)])
@pytest.mark.parametrize("n, k, pad, skip", [(1, 1, 0, 0), (70, 200, 0, 0), (130, 256, 16, 0), (200, 384, 3, 1), (2000, 144, 0, 0)])
@pytest.mark.parametrize("scale, out", [("e8m0", torch.bfloat16), ("fp32", torch.float16), ("e8m0", torch.float32)])
def test_product_equals_the_definition(cuda, rows, counts, n, k, pad, skip, scale, out):
    if len(counts) * n * k > 1 << 24:
        counts = counts[:60]
    live = grouped.counts_of(counts, rows)
    a = _operand((rows, k), E4M3, scale, False, cuda, 1, pad, skip)
    b = _operand((len(counts), n, k), E4M3, scale, True, cuda, 2, pad, skip)
    got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out_dtype=out)
    want, magnitude = grouped.product(a, b, live)
    assert got.dtype == out
    _assert_near(got, want, magnitude, k)
    assert not got[sum(live):].any()
    kept = torch.full((rows, n + 3), 7.0, device=cuda, dtype=out)
    assert sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda, torch.int64), out=kept[:, :n]) is not None
    assert torch.equal(kept[:sum(live), :n], got[:sum(live)])
    assert (kept[sum(live):] == 7).all() and (kept[:, n:] == 7).all()


@pytest.mark.parametrize("a_dtype", [E4M3, E5M2])
@pytest.mark.parametrize("b_dtype", [E4M3, E5M2])
@pytest.mark.parametrize("a_square, b_square", [(False, False), (True, True)])
@pytest.mark.parametrize("scale", ["e8m0", "fp32"])
@pytest.mark.parametrize("rows, counts", [(150, [3, 100, 47]), (20, [3, 9, 8])])
def test_product_of_every_format(cuda, a_dtype, b_dtype, a_square, b_square, scale, rows, counts):
    a = _operand((rows, 272), a_dtype, scale, False, cuda, 3)
    if a_square:  # a scale that 128 rows share: the same for each of them
        a = BlockScaled(a.data, a.scale.view(torch.uint8 if scale == "e8m0" else torch.float32)[::128].repeat_interleave(128, 0)[:rows].view(a.scale.dtype))
    b = _operand((3, 140, 272), b_dtype, scale, b_square, cuda, 4)
    for out in (torch.bfloat16, torch.float32):
        got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out_dtype=out)
        _assert_near(got, *grouped.product(a, b, counts), 272)


# The 16-row kernel, 64 x 64 tiles in one, two and four groups of waves, aligned and not, 128 x 128 tiles, and those of one
# stage: groups start inside blocks of 128 rows, at their ends, and behind an empty group.
@pytest.mark.parametrize("rows, counts, n, k, pad", [
    (20, [3, 9, 8], 140, 272, 0), (300, [40] * 7, 33, 130, 3), (330, [1, 127, 0, 128, 44], 140, 272, 0),
    (700, [300, 0, 17, 250], 200, 384, 3), (700, [300, 0, 17, 250], 70, 1408, 16), (2600, [1300, 1, 1200], 1000, 256, 0),
    (3100, [1500, 0, 129, 1, 900, 60], 3001, 384, 0), (2600, [130] * 20, 2000, 200, 1),
])
@pytest.mark.parametrize("a_dtype, scale, out", [
    (E4M3, "e8m0", torch.bfloat16), (E5M2, "fp32", torch.float16), (E4M3, "e8m0", torch.float32), (E4M3, "fp32", torch.float32),
])
def test_groups_of_rows_that_share_scales(cuda, rows, counts, n, k, pad, a_dtype, scale, out):
    a = _operand((rows, k), a_dtype, scale, True, cuda, 5, pad)
    assert a.scale.shape[0] == -(-rows // 128)
    b = _operand((len(counts), n, k), E4M3, scale, True, cuda, 6, pad)
    got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out_dtype=out)
    _assert_near(got, *grouped.product(a, b, grouped.counts_of(counts, rows)), k)
    shared = a.scale.view(torch.uint8 if scale == "e8m0" else torch.float32).repeat_interleave(128, 0)[:rows].view(a.scale.dtype)
    same = sr_states.grouped_block_matmul(BlockScaled(a.data, shared), b, _sizes(counts, cuda), out_dtype=out)
    assert torch.equal(got, same)  # a scale for each row: the same values


@pytest.mark.parametrize("counts", [[100, 7, 93], [0, 200]])
def test_groups_of_a_cast_in_square_blocks(cuda, counts):
    x, w = _spread((200, 300), cuda, 1, torch.bfloat16), _spread((2, 90, 300), cuda, 2)
    w = torch.cat((w, w[:1] * 3))[:len(counts)]
    a = sr_states.block_cast(x, block=(128, 128), rounding="nearest")
    b = sr_states.grouped_block_cast(w, block=(128, 128), rounding="nearest")
    got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out_dtype=torch.float32)
    _assert_near(got, *grouped.product(a, b, counts), 300)


def test_shared_scales_that_are_far_from_one(cuda):
    """Factors whose products leave FP32's normal range on the way to a result: a tile's sums are taken once more."""
    counts = [100, 0, 300, 112]
    a = _operand((512, 512), E4M3, "fp32", True, cuda, 7)
    b = _operand((4, 200, 512), E4M3, "fp32", False, cuda, 8)
    a.scale[1:3] = 2.0**100
    b.scale[:] = b.scale.clamp(0.25, 1) * 2.0**-120
    for out in (torch.bfloat16, torch.float32):
        got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out_dtype=out)
        _assert_near(got, *grouped.product(a, b, counts), 512)


def _padded(rows, counts, width, dtype, scale, device, seed):
    """An operand of a contraction: random values in the groups' columns, zeros in the others."""
    q = _operand((rows, width), dtype, scale, False, device, seed)
    keep = torch.zeros(width, dtype=torch.bool, device=device)
    for at, n in zip(grouped.starts(counts), counts):
        keep[at:at + n] = True
    data = torch.empty_strided((rows, width), (width, 1), dtype=torch.uint8, device=device)
    data.copy_(torch.where(keep, q.data.view(torch.uint8), 0))
    return BlockScaled(data.view(dtype), q.scale)


@pytest.mark.parametrize("tokens, counts", [(1, [1]), (300, [1, 127, 128, 44]), (300, [0, 0, 129, 0, 100]), (90, [1] * 70),
                                            (1500, [1200, 0, 300]), (6000, [6000]), (100, [0, 0])])
@pytest.mark.parametrize("m, n", [(1, 1), (70, 130), (300, 2000), (2100, 2000)])
@pytest.mark.parametrize("scale, out", [("e8m0", torch.bfloat16), ("fp32", torch.bfloat16), ("e8m0", torch.float32), ("fp32", torch.float32)])
def test_contraction_equals_the_definition(cuda, tokens, counts, m, n, scale, out):
    if len(counts) * m * n > 1 << 24:
        counts = counts[:3]
    width = grouped.columns(tokens, len(counts))
    a = _padded(m, counts, width, E4M3, scale, cuda, 1)
    b = _padded(n, counts, width, E5M2, scale, cuda, 2)
    got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out_dtype=out)
    assert got.dtype == out
    _assert_near(got, *grouped.contract(a, b, counts), max(counts))
    kept = torch.full((len(counts), m + 1, n + 2), 7.0, device=cuda, dtype=out)
    sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out=kept[:, :m, :n])
    assert torch.equal(kept[:, :m, :n], got)
    assert (kept[:, m:] == 7).all() and (kept[:, :, n:] == 7).all()


@pytest.mark.parametrize("a_dtype, b_dtype", [(E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2)])
@pytest.mark.parametrize("k", [128, 640, 2048 + 384])
@pytest.mark.parametrize("counts", [[1500, 0, 129, 1, 900, 60], [0, 3000], [1] * 80 + [2500], [0, 0]])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
def test_products_of_more_tiles_than_the_chip_holds(cuda, a_dtype, b_dtype, k, counts, out):
    rows, n = 3100, 3001
    counts = counts if k == 128 else counts[-6:]
    a = _operand((rows, k), a_dtype, "e8m0", False, cuda, 1)
    b = _operand((len(counts), n, k), b_dtype, "e8m0", True, cuda, 2)
    got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out_dtype=out)
    _assert_near(got, *grouped.product(a, b, counts), k)
    kept = torch.full((rows, n), 7.0, device=cuda, dtype=out)
    sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda), out=kept)
    assert torch.equal(kept[:sum(counts)], got[:sum(counts)]) and (kept[sum(counts):] == 7).all()


@pytest.mark.parametrize("tokens, counts", [(3000, [300, 0, 129, 1, 2300, 60]), (100, [1] * 90)])
@pytest.mark.parametrize("a_dtype, b_dtype", [(E4M3, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
def test_contractions_of_more_tiles_than_the_chip_holds(cuda, tokens, counts, a_dtype, b_dtype):
    m, n = (1300, 1281) if len(counts) < 10 else (130, 500)
    width = grouped.columns(tokens, len(counts))
    a, b = _padded(m, counts, width, a_dtype, "e8m0", cuda, 1), _padded(n, counts, width, b_dtype, "e8m0", cuda, 2)
    got = sr_states.grouped_block_matmul(a, b, _sizes(counts, cuda))
    _assert_near(got, *grouped.contract(a, b, counts), max(counts))


def test_sizes_that_lead_beyond_the_columns_end_there(cuda):
    counts = [100, 10**9, -5, 3]
    a = _operand((20, 512), E4M3, "e8m0", False, cuda, 1)
    got = sr_states.grouped_block_matmul(a, a, _sizes(counts, cuda), out_dtype=torch.float32)
    _assert_near(got, *grouped.contract(a, a, [100, 384, 0, 0]), 512)
    wide = sr_states.grouped_block_matmul(a, a, _sizes([100, 1 << 40, -(1 << 40), 3], cuda, torch.int64), out_dtype=torch.float32)
    assert torch.equal(wide, got)


def _linear_reference(x, w, dy, counts, seed, formats):
    keys = [sr_states.state_key(seed, k) for k in range(3)]
    (fx, rx), (fw, rw), (fg, rg) = formats
    y = grouped.product(oracle.block_cast(x, fx, rx, False, 1, keys[0]), grouped.cast_stack(w, fw, rw, True, 1, keys[1]), counts)
    dx = grouped.product(oracle.block_cast(dy, fg, rg, False, 1, keys[2]), grouped.cast_stack(w, fw, rw, True, 0, keys[1]), counts)
    dw = grouped.contract(grouped.cast_columns(dy, counts, fg, rg, keys[2]), grouped.cast_columns(x, counts, fx, rx, keys[0]), counts)
    return y, dx, dw


DEFAULT_FORMATS = ((E4M3, "nearest"), (E4M3, "nearest"), (E4M3, "stochastic"))
MIXED_FORMATS = ((E4M3, "stochastic"), (E4M3, "nearest"), (E5M2, "stochastic"))


@pytest.mark.parametrize("rows, counts", [(1, [0, 1]), (300, [129, 0, 100]), (150, [2] * 70), (640, [200, 440]), (9, [0, 0])])
@pytest.mark.parametrize("n, k", [(1, 64), (150, 200), (640, 384)])
@pytest.mark.parametrize("dtypes", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("formats", [DEFAULT_FORMATS, MIXED_FORMATS])
def test_linear_equals_the_formulas(cuda, rows, counts, n, k, dtypes, formats):
    seed = 77
    x = _spread((rows, k), cuda, 1, dtypes[0]).requires_grad_()
    w = (_spread((len(counts), n, k), cuda, 2) * 0.05).to(dtypes[1]).requires_grad_()
    dy = (_spread((rows, n), cuda, 3) * 1e-3).to(dtypes[0])
    given = None if formats is DEFAULT_FORMATS else {
        name: sr_states.StateFormat(*fmt) for name, fmt in zip(("input", "weight", "gradient"), formats)}
    y = sr_states.grouped_block_linear(x, w, _sizes(counts, cuda), seed=seed, formats=given)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == dx.dtype == dtypes[0] and dw.dtype == dtypes[1]
    reference = _linear_reference(x.detach(), w.detach(), dy, counts, seed, formats)
    for got, (want, magnitude), terms in zip((y, dx, dw), reference, (k, n, max(max(counts), 1))):
        _assert_near(got.detach(), want, magnitude, terms)
    live = sum(counts)
    assert not y[live:].any() and not dx[live:].any()


def test_one_group_of_all_rows_is_the_plain_layer(cuda):
    x = _spread((200, 256), cuda, 1, torch.bfloat16).requires_grad_()
    w = _spread((130, 256), cuda, 2, torch.bfloat16).requires_grad_()
    dy = _spread((200, 130), cuda, 3, torch.bfloat16)
    y = sr_states.grouped_block_linear(x, w[None], _sizes([200], cuda), seed=5)
    plain = sr_states.block_linear(x, w, seed=5)
    assert torch.equal(y, plain)
    for got, want in zip(torch.autograd.grad(y, (x, w), dy), torch.autograd.grad(plain, (x, w), dy)):
        assert torch.equal(got, want)


def test_linear_gradients_are_differences_where_fp8_is_exact(cuda):
    """Small integers survive the casts, so the layer is exactly linear there and differences are exact."""
    gen = torch.Generator(device=cuda).manual_seed(0)

    def integers(*shape):
        return torch.randint(-4, 5, shape, device=cuda, generator=gen).float()

    sizes = _sizes([20, 0, 35], cuda)
    x, w, dy = integers(60, 140).requires_grad_(), integers(3, 70, 140).requires_grad_(), integers(60, 70)
    dx, dw = torch.autograd.grad(sr_states.grouped_block_linear(x, w, sizes), (x, w), dy)

    def loss(x, w):
        return float((sr_states.grouped_block_linear(x, w, sizes).double() * dy.double()).sum())

    with torch.no_grad():
        start = loss(x, w)
        for tensor, gradient in ((x, dx), (w, dw)):
            for _ in range(12):
                at = tuple(int(torch.randint(0, s, ())) for s in tensor.shape)
                moved = tensor.clone()
                moved[at] += 1
                assert loss(*((moved, w) if tensor is x else (x, moved))) - start == float(gradient[at])


def test_linear_without_rows_groups_or_values(cuda):
    for rows, groups, n, k in ((0, 3, 20, 128), (7, 0, 20, 128), (7, 3, 0, 128), (7, 3, 20, 0)):
        x = torch.ones(rows, k, device=cuda, requires_grad=True)
        w = torch.ones(groups, n, k, device=cuda, requires_grad=True)
        y = sr_states.grouped_block_linear(x, w, torch.zeros(groups, dtype=torch.int32, device=cuda))
        assert y.shape == (rows, n) and not y.any()
        y.sum().backward()
        assert x.grad.shape == x.shape and not x.grad.any()
        assert w.grad.shape == w.shape and not w.grad.any()


def test_linear_casts_only_what_its_gradients_need(cuda):
    x, w, sizes = _spread((40, 128), cuda, 1), _spread((2, 30, 128), cuda, 2), _sizes([10, 30], cuda)
    y = sr_states.grouped_block_linear(x.clone().requires_grad_(), w, sizes)
    y.sum().backward()
    leaf = w.clone().requires_grad_()
    # An expanded gradient, a transposed input and a transposed weight.
    out = sr_states.grouped_block_linear(x.t().contiguous().t(), leaf.mT.contiguous().mT, sizes)
    out.sum().backward()
    assert leaf.grad.shape == w.shape and torch.equal(out, sr_states.grouped_block_linear(x, w, sizes))
    assert not sr_states.grouped_block_linear(x, w, sizes).requires_grad
    with torch.no_grad():
        assert not sr_states.grouped_block_linear(x, leaf, sizes).requires_grad


def test_sizes_changed_before_the_backward_pass_are_noticed(cuda):
    x, sizes = _spread((40, 128), cuda, 1).requires_grad_(), _sizes([10, 30], cuda)
    y = sr_states.grouped_block_linear(x, _spread((2, 30, 128), cuda, 2), sizes)
    sizes.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_sizes_of_a_replayed_graph_are_read_when_it_runs(cuda):
    x, w = _spread((300, 256), cuda, 1, torch.bfloat16).requires_grad_(), _spread((5, 130, 256), cuda, 2, torch.bfloat16).requires_grad_()
    dy, sizes = _spread((300, 130), cuda, 3, torch.bfloat16), _sizes([60] * 5, cuda)

    def step():
        y = sr_states.grouped_block_linear(x, w, sizes, seed=3)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for counts in ([60] * 5, [300, 0, 0, 0, 0], [0, 1, 128, 129, 2], [0] * 5, [17, 100, 3, 150, 30]):
        sizes.copy_(_sizes(counts, cuda))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)
        torch.cuda.synchronize()


def test_calls_on_two_streams_at_once(cuda):
    x, w = _spread((900, 256), cuda, 1, torch.bfloat16), _spread((5, 130, 256), cuda, 2, torch.bfloat16)
    sizes = [_sizes(c, cuda) for c in ([180] * 5, [900, 0, 0, 0, 0])]
    want = [sr_states.grouped_block_linear(x, w, s) for s in sizes]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    got = [[], []]
    for _ in range(10):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(sr_states.grouped_block_linear(x, w, sizes[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(y, want[k]) for y in got[k])


def test_a_refused_call_leaves_its_result_alone(cuda):
    x, sizes = torch.ones(8, 256, device=cuda), _sizes([3, 5], cuda)
    q, w = sr_states.block_cast(x), sr_states.grouped_block_cast(torch.ones(2, 16, 256, device=cuda))
    out = torch.full((8, 16), 7.0, device=cuda)
    version = out._version
    for error, a, b in ((ValueError, q, BlockScaled(w.data, w.scale[:, :, :1])), (ValueError, q, BlockScaled(w.data, w.scale[:, :15])),
                        (TypeError, q, BlockScaled(w.data, w.scale.view(torch.uint8))), (TypeError, q, BlockScaled(w.data.float(), w.scale)),
                        (TypeError, BlockScaled(q.data, q.scale.float()), w)):
        with pytest.raises(error):
            sr_states.grouped_block_matmul(a, b, sizes, out=out)
        assert out._version == version
    assert (out == 7).all()
    sr_states.grouped_block_matmul(q, w, sizes, out=out)
    assert out._version > version and (out == 256).all()


def test_tangents_are_refused(cuda):
    x, w, sizes = torch.randn(8, 256, device=cuda), torch.randn(2, 16, 256, device=cuda), _sizes([3, 5], cuda)
    with forward_ad.dual_level():
        for operands in ((forward_ad.make_dual(x, torch.ones_like(x)), w), (x, forward_ad.make_dual(w, torch.ones_like(w)))):
            for mode in (True, False):
                with torch.set_grad_enabled(mode), pytest.raises(NotImplementedError, match="forward-mode"):
                    sr_states.grouped_block_linear(*operands, sizes)


def test_refusals(cuda):
    x, sizes = torch.zeros(8, 256, device=cuda), _sizes([3, 5], cuda)
    q, w = sr_states.block_cast(x), sr_states.grouped_block_cast(torch.zeros(2, 16, 256, device=cuda))
    turned = sr_states.grouped_block_cast(x, sizes, axis=0)
    matmul, cast, linear = sr_states.grouped_block_matmul, sr_states.grouped_block_cast, sr_states.grouped_block_linear
    weight = torch.zeros(2, 16, 256, device=cuda)
    cases = [
        (TypeError, "expected FP32, BF16 or FP16", lambda: cast(x.double(), sizes)),
        (TypeError, "expected FP32, BF16 or FP16", lambda: cast(weight.double())),
        (ValueError, "rows of a matrix", lambda: cast(weight, sizes)),
        (ValueError, "three dimensions", lambda: cast(x)),
        (ValueError, "blocks of one row", lambda: cast(x, sizes, block=(128, 128))),
        (ValueError, "consecutive columns", lambda: cast(x.t(), sizes, axis=0)),
        (ValueError, "consecutive columns", lambda: cast(weight.mT)),
        (TypeError, "sizes must be", lambda: cast(x, sizes.float(), axis=0)),
        (ValueError, "one row of consecutive", lambda: cast(x, sizes[None], axis=0)),
        (ValueError, "one row of consecutive", lambda: cast(x, _sizes([1, 2, 3, 4], cuda)[::2], axis=0)),
        (ValueError, "same GPU", lambda: cast(x, sizes.cpu(), axis=0)),
        (ValueError, "at most 4096", lambda: cast(x, torch.zeros(4097, dtype=torch.int32, device=cuda), axis=0)),
        (ValueError, "2 matrices for 3", lambda: matmul(q, w, _sizes([1, 2, 3], cuda))),
        (ValueError, "contract 256 and 128", lambda: matmul(q, cast(weight[..., :128]), sizes)),
        (ValueError, "stack of as many scales", lambda: matmul(q, BlockScaled(w.data, w.scale[0]), sizes)),
        (ValueError, "scales of a 16 x 256", lambda: matmul(q, BlockScaled(w.data, w.scale[:, :, :1]), sizes)),
        (TypeError, "scales of one type", lambda: matmul(BlockScaled(q.data, q.scale.float()), w, sizes)),
        (TypeError, "out_dtype must be", lambda: matmul(q, w, sizes, out_dtype=E4M3)),
        (ValueError, "out must be a 8 x 16", lambda: matmul(q, w, sizes, out=torch.zeros(8, 17, device=cuda))),
        (ValueError, "out must be a 2 x 256 x 256", lambda: matmul(turned, turned, sizes, out=torch.zeros(256, 256, device=cuda))),
        (ValueError, "matrices that do not overlap", lambda: matmul(turned, turned, sizes, out=torch.zeros(1, 256, 256, device=cuda).expand(2, 256, 256))),
        (ValueError, "must not overlap", lambda: matmul(q, w, sizes, out=w.data.view(torch.uint8).flatten()[:512].view(torch.float32).view(8, 16))),
        (ValueError, "multiple of 128", lambda: matmul(BlockScaled(q.data[:, :200], q.scale), BlockScaled(q.data[:, :200], q.scale), sizes)),
        (ValueError, "16 bytes", lambda: matmul(BlockScaled(turned.data[:, 8:136], turned.scale[:, :1]), BlockScaled(turned.data[:, 8:136], turned.scale[:, :1]), sizes)),
        (ValueError, "do not match", lambda: linear(x, x, sizes)),
        (ValueError, "2 weights take as many sizes", lambda: linear(x, weight, _sizes([8], cuda))),
        (ValueError, "same GPU", lambda: linear(x, weight, sizes.cpu())),
        (ValueError, "must be FP8", lambda: linear(x, weight, sizes, formats=sr_states.StateFormat(torch.bfloat16))),
    ]
    for error, message, call in cases:
        with pytest.raises(error, match=message):
            call()
    leaf = torch.zeros(8, 16, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="grouped_block_matmul records no gradients"):
        matmul(q, w, sizes, out=leaf)
