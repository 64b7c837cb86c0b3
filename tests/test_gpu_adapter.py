"""adapter_add and its gradients against their definition in 64 bits.

Tolerances.  Every result is a sum of products of two sums.  A sum of m FP32
terms on the matrix instructions is off by at most m 2^-23 of the sum of their
magnitudes (an addition may truncate), a BF16 call's value between the two sums
by 2^-15 (its truncated part leaves 2^-7 of it, which rounds to BF16 by 2^-8), and
the final rounding by the type's unit roundoff.  With S the sum over all
magnitudes, m the terms of both sums and 16 more for scales, joins of partial sums and
the addition of base, the bound is u |result| + (1 + u) (m 2^-23 + 2^-15) S.
"""

from __future__ import annotations

import _adapter_oracle as oracle
import pytest
import sr_states
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _assert_near(got, pair, terms):
    want, size = (t.reshape(got.shape) for t in pair)
    u = HALF_ULP[got.dtype]
    inner = (terms + 16) * 2.0**-23 + (2.0**-15 if got.dtype == torch.bfloat16 else 0)
    limit = u * want.abs() + (1 + u) * inner * size
    if got.dtype == torch.float16:
        limit = limit + 2.0**-25  # half the spacing below its normal range
    assert not got.isnan().any()
    if got.numel():
        assert float(((got.double() - want).abs() - limit).max()) <= 0


def _inputs(device, rows, k, n, count, rank, dtype, index, seed=1):
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(shape, std):
        return (torch.randn(shape, device=device, generator=gen) * std).to(dtype)

    lead = rows if isinstance(rows, tuple) else (rows,)
    base, x = normal((*lead, n), 1.0), normal((*lead, k), 1.0)
    a, b = normal((count, rank, k), max(k, 1) ** -0.5), normal((count, n, rank), rank**-0.5)
    if index == "mixed":
        index = torch.randint(-1, count, lead, device=device, generator=gen)
    elif index == "one":
        index = torch.full(lead, count - 1, device=device)
    elif index == "runs":
        index = (torch.arange(lead[0], device=device) * (count + 1) // max(lead[0], 1) - 1)
    else:
        index = torch.full(lead, -1, device=device)
    scaling = torch.rand(count, device=device, generator=gen) * 3 - 1
    return base, x, a, b, index, scaling


# (rows, k, n, adapters, rank)
SHAPES = [
    (1, 1, 1, 1, 1),
    (1, 2048, 70, 3, 8),
    (5, 63, 65, 2, 4),
    (16, 128, 64, 16, 16),
    (17, 200, 130, 40, 17),
    (64, 515, 33, 30, 12),
    (130, 64, 1000, 3, 33),
    (300, 1000, 257, 5, 64),
    (300, 96, 300, 2, 65),
    (1500, 130, 300, 4, 128),
    (5000, 200, 320, 3, 20),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, k, n, count, rank", SHAPES)
@pytest.mark.parametrize("index", ["mixed", "one", "runs", "none"])
def test_equals_the_definition(cuda, rows, k, n, count, rank, dtype, index):
    base, x, a, b, index, scaling = _inputs(cuda, rows, k, n, count, rank, dtype, index)
    for t in (base, x, a, b):
        t.requires_grad_()
    dy = torch.randn(rows, n, device=cuda).to(dtype)
    y = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
    assert y.dtype == dtype and y.shape == base.shape
    _assert_near(y.detach(), oracle.add(base, x, a, b, index, scaling), k + rank)
    dbase, dx, da, db = torch.autograd.grad(y, (base, x, a, b), dy)
    assert torch.equal(dbase, dy)
    assert [g.dtype for g in (dx, da, db)] == [dtype] * 3
    for got, want, terms in zip((dx, da, db), oracle.gradients(dy, x, a, b, index, scaling), (n + rank, n + rows, k + rows)):
        _assert_near(got, want, terms)
    with torch.no_grad():
        assert torch.equal(y, sr_states.adapter_add(base, x, a, b, index.int(), scaling=scaling))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, k, n, rank", [(1, 2048, 2048, 8), (1, 100, 37, 16), (2, 1000, 300, 16), (2, 2048, 130, 20),
                                              (1, 4096, 64, 3), (3, 512, 64, 16), (1, 64, 64, 128)])
def test_single_tokens(cuda, dtype, rows, k, n, rank):
    """One launch or two, whichever the rows and ranks take, and the gradients that follow."""
    base, x, a, b, _, scaling = _inputs(cuda, rows, k, n, 3, rank, dtype, "none")
    dy = torch.randn(rows, n, device=cuda).to(dtype)
    for t in (x, a, b):
        t.requires_grad_()
    for index in ([0, 2, 1], [1, 1, 1], [2, -1, 0], [-1, 0, 2], [-1, -1, -1]):
        index = torch.tensor(index[:rows], device=cuda)
        y = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
        _assert_near(y.detach(), oracle.add(base, x, a, b, index, scaling), k + rank)
        got = torch.autograd.grad(y, (x, a, b), dy)
        for g, want, terms in zip(got, oracle.gradients(dy, x, a, b, index, scaling), (n + rank, n + rows, k + rows)):
            _assert_near(g, want, terms)
        with torch.no_grad():
            into = base.clone()
            sr_states.adapter_add(into, x, a, b, index, scaling=scaling, out=into)
            assert torch.equal(into, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("rank", [8, 32])
def test_many_rows(cuda, dtype, order, rank):
    """Rows of several parts, tiles that share an adapter's registers, 64 columns a wave."""
    rows, k, n, count = 9000, 400, 500, 5
    base, x, a, b, index, _ = _inputs(cuda, rows, k, n, count, rank, dtype, order)
    for t in (x, a, b):
        t.requires_grad_()
    dy = torch.randn(rows, n, device=cuda).to(dtype)
    y = sr_states.adapter_add(base, x, a, b, index, scaling=0.5)
    _assert_near(y.detach(), oracle.add(base, x, a, b, index, 0.5), k + rank)
    got = torch.autograd.grad(y, (x, a, b), dy)
    for g, want, terms in zip(got, oracle.gradients(dy, x, a, b, index, 0.5), (n + rank, n + rows, k + rows)):
        _assert_near(g, want, terms)
    again = torch.autograd.grad(sr_states.adapter_add(base, x, a, b, index, scaling=0.5), (x, a, b), dy)
    assert all(torch.equal(g, h) for g, h in zip(got, again))


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_of_an_adapter_reaches_other_rows(cuda, dtype):
    base, x, a, b, index, scaling = _inputs(cuda, 200, 130, 150, 6, 12, dtype, "mixed")
    base[3], index[3] = -float("inf"), -1
    base[4, 0], index[4] = float("nan"), 99
    keep = (index != 2) & (index != 4)

    def run(x, a, b, scaling, dy):
        x, a, b = (t.clone().requires_grad_() for t in (x, a, b))
        y = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
        return (y.detach(), *torch.autograd.grad(y, (x, a, b), dy))

    dy = torch.randn(200, 150, device=cuda).to(dtype)
    clean = run(x, a, b, scaling, dy)
    a[2], b[2], scaling[4] = float("nan"), float("inf"), float("inf")
    x[(index == 2).nonzero()[0]] = float("inf")
    dy[(index == 4).nonzero()[0]] = float("nan")
    dirty = run(x, a, b, scaling, dy)
    for got, want in zip(dirty[:2], clean[:2]):  # y and dx, by rows
        torch.testing.assert_close(got[keep], want[keep], rtol=0, atol=0, equal_nan=True)
    for got, want in zip(dirty[2:], clean[2:]):  # da and db, by adapters
        others = [0, 1, 3, 5]
        assert torch.equal(got[others], want[others])
    assert dirty[0][index == 2].isnan().all()
    assert torch.equal(clean[0][3], base[3]) and clean[0][4, 0].isnan() and torch.equal(clean[0][4, 1:], base[4, 1:])


@pytest.mark.parametrize("rows", [1, 64, 4096])
@pytest.mark.parametrize("dtype, x, a, b", [
    (torch.float16, -20, 5, 10), (torch.float16, 0, -20, 10), (torch.float16, 0, 8, -20),
    (torch.bfloat16, -130, 100, 20), (torch.bfloat16, 100, -130, 20), (torch.bfloat16, 50, 60, -130), (torch.bfloat16, -60, -70, 100),
    (torch.float32, -140, 100, 20), (torch.float32, 60, 50, -140), (torch.float32, -60, -75, 100),
])
def test_subnormal_values_count(cuda, rows, dtype, x, a, b):
    """Powers of two, so that every product and sum is exact; each case has an operand or a value between below the normal range."""
    def full(shape, log):
        return torch.full(shape, 2.0**log, device=cuda, dtype=dtype)

    index = torch.zeros(rows, dtype=torch.int32, device=cuda)
    y = sr_states.adapter_add(torch.zeros(rows, 80, device=cuda, dtype=dtype), full((rows, 64), x), full((1, 16, 64), a),
                              full((1, 80, 16), b), index)
    assert (y.double() == 2.0 ** (6 + 4 + x + a + b)).all()


# One launch for a row, 16 columns a wave, 64 columns a wave and rows in parts.
@pytest.mark.parametrize("rows, n, rank", [(1, 40, 16), (60, 80, 1), (60, 80, 40), (300, 70, 128), (2500, 900, 20)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("infinite", ["base", "x", "a", "b", "dy", "scaling"])
def test_infinities_are_the_definitions(cuda, rows, n, rank, dtype, infinite):
    """Where the definition multiplies an infinity by zero or adds two of them, NaN, and nowhere else: not where BF16
    holds a sum between the products, as it does those of x and a here, small multiples of a power of two."""
    gen = torch.Generator().manual_seed(5)

    def powers(shape, log, signed=False):
        t = 2.0 ** torch.randint(log, log + 2, shape, generator=gen)
        return (t * (1 - 2 * torch.randint(0, 2, shape, generator=gen)) if signed else t).to(dtype)

    k, count = 8, 3
    base, x, dy = powers((rows, n), 0, True), powers((rows, k), 0), powers((rows, n), -9)
    a, b = powers((count, rank, k), -1), powers((count, n, rank), -4)
    b[2] *= 1 - 2 * torch.randint(0, 2, (n, rank), generator=gen).to(dtype)
    index = torch.arange(rows) % (count + 1)  # the last has no adapter
    scaling = torch.tensor([1.0, -2.0, 0.5])
    if rows > 1:
        x[1::7] = 0
    operands = {"base": base, "x": x, "a": a, "b": b, "dy": dy}
    if infinite == "scaling":
        scaling[0] = float("inf")
    else:
        t = operands[infinite]
        flat = t.view(-1)
        flat[::max(flat.numel() // 5, 7)] = float("inf")
        flat[3::max(flat.numel() // 3, 11)] = -float("inf")
    want = [oracle.add(base, x, a, b, index, scaling), *oracle.gradients(dy, x, a, b, index, scaling)]
    assert any(value.isinf().any() for value, _ in want)
    leaves = [t.to(cuda).requires_grad_() for t in (x, a, b)]
    y = sr_states.adapter_add(base.to(cuda), *leaves, index.to(cuda), scaling=scaling.to(cuda))
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy.to(cuda))]
    for result, (value, size), terms in zip(got, want, (k + rank, n + rank, n + rows, k + rows)):
        result, value = result.cpu(), value.reshape(result.shape)
        special = ~value.isfinite()
        assert torch.equal(result.isnan(), value.isnan())
        assert torch.equal(result[value.isinf()].double(), value[value.isinf()])
        clean = [torch.where(special, 0, t.reshape(result.shape)) for t in (value, size)]
        _assert_near(torch.where(special, 0, result), clean, terms)


def test_indices_outside_the_adapters_are_none(cuda):
    base, x, a, b, _, scaling = _inputs(cuda, 6, 64, 64, 3, 8, torch.bfloat16, "none")
    index = torch.tensor([0, 3, -1, 1 << 40, -(1 << 40), 2], device=cuda)
    y = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
    assert torch.equal(y[1:5], base[1:5])
    _assert_near(y, oracle.add(base, x, a, b, index, scaling), 72)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_any_layout(cuda, dtype):
    flat = _inputs(cuda, (3, 50), 80, 90, 4, 10, dtype, "mixed")
    base, x, a, b, index, scaling = flat
    wide = torch.full((3, 50, 95), 7.0, device=cuda, dtype=dtype)[..., 2:92]
    wide.copy_(base)
    odd = torch.empty(3 * 50 * 83 + 1, device=cuda, dtype=dtype)[1:].view(3, 50, 83)[..., :80]
    odd.copy_(x)
    want = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
    _assert_near(want, oracle.add(base, x, a, b, index, scaling), 90)
    got = sr_states.adapter_add(wide, odd, a.mT.contiguous().mT, b.mT.contiguous().mT, index.t().contiguous().t(),
                                scaling=scaling.repeat_interleave(2)[::2])
    assert torch.equal(got, want)
    turned = x.transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()
    y = sr_states.adapter_add(base, turned, a, b, index, scaling=scaling)
    assert torch.equal(y, want)
    y.sum().backward()  # an expanded gradient
    assert turned.grad.shape == turned.shape
    one = sr_states.adapter_add(base[0, 0], x[0, 0], a, b, index[0, 0], scaling=scaling)
    assert one.shape == (90,)
    _assert_near(one, oracle.add(base[0, 0], x[0, 0], a, b, index[0, 0], scaling), 90)


def test_results_into_given_tensors(cuda):
    base, x, a, b, index, scaling = _inputs(cuda, 100, 80, 90, 4, 10, torch.bfloat16, "mixed")
    want = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
    out = torch.full((100, 95), 7.0, device=cuda, dtype=torch.bfloat16)
    assert sr_states.adapter_add(base, x, a, b, index, scaling=scaling, out=out[:, :90]) is not None
    assert torch.equal(out[:, :90], want) and (out[:, 90:] == 7).all()
    version = base._version
    assert sr_states.adapter_add(base, x, a, b, index, scaling=scaling, out=base) is base
    assert torch.equal(base, want) and base._version > version


def test_gradients_are_differences_where_sums_are_exact(cuda):
    """Small integers in FP32: the result is linear in each operand alone, and differences are exact."""
    gen = torch.Generator(device=cuda).manual_seed(0)

    def integers(*shape):
        return torch.randint(-4, 5, shape, device=cuda, generator=gen).float()

    operands = [integers(40, 30).requires_grad_(), integers(40, 20).requires_grad_(), integers(3, 5, 20).requires_grad_(),
                integers(3, 30, 5).requires_grad_()]
    index, dy = torch.randint(-1, 3, (40,), device=cuda, generator=gen), integers(40, 30)
    gradients = torch.autograd.grad(sr_states.adapter_add(*operands, index, scaling=2.0), operands, dy)

    def loss(*t):
        return float((sr_states.adapter_add(*t, index, scaling=2.0).double() * dy.double()).sum())

    with torch.no_grad():
        start = loss(*operands)
        for k, gradient in enumerate(gradients):
            for _ in range(12):
                at = tuple(int(torch.randint(0, s, ())) for s in operands[k].shape)
                moved = [t.clone() if j == k else t for j, t in enumerate(operands)]
                moved[k][at] += 1
                assert loss(*moved) - start == float(gradient[at])


def test_gradients_that_are_not_wanted_are_not_made(cuda):
    base, x, a, b, index, scaling = _inputs(cuda, 60, 80, 90, 4, 10, torch.float32, "mixed")
    dy = torch.randn(60, 90, device=cuda)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    whole = torch.autograd.grad(sr_states.adapter_add(base, *leaves, index, scaling=scaling), leaves, dy)
    for wanted in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(wanted >> k & 1)) for k, t in enumerate((x, a, b))]
        y = sr_states.adapter_add(base, *leaves, index, scaling=scaling)
        y.backward(dy)
        for k, leaf in enumerate(leaves):
            assert leaf.grad is None if not wanted >> k & 1 else torch.equal(leaf.grad, whole[k])
    assert not sr_states.adapter_add(base, x, a, b, index).requires_grad
    leaf = base.clone().requires_grad_()
    sr_states.adapter_add(leaf, x, a, b, index).backward(dy)
    assert torch.equal(leaf.grad, dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k, n, rank, count", [(201, 333, 20, 3), (7, 2, 1, 1)])
def test_some_gradients_of_rows_in_parts(cuda, dtype, k, n, rank, count):
    """The parts' sums are joined by 256 threads at a time, more than either gradient alone has use for."""
    base, x, a, b, index, scaling = _inputs(cuda, 2500, k, n, count, rank, dtype, "mixed")
    assert (count * -(-k // 4) * rank) % 256 and (count * n * -(-rank // 4)) % 256
    dy = torch.randn(2500, n, device=cuda).to(dtype)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    whole = torch.autograd.grad(sr_states.adapter_add(base, *leaves, index, scaling=scaling), leaves, dy)
    for got, want, terms in zip(whole, oracle.gradients(dy, x, a, b, index, scaling), (n + rank, n + 2500, k + 2500)):
        _assert_near(got, want, terms)
    for wanted in range(1, 7):
        leaves = [t.clone().requires_grad_(bool(wanted >> j & 1)) for j, t in enumerate((x, a, b))]
        sr_states.adapter_add(base, *leaves, index, scaling=scaling).backward(dy)
        for j, leaf in enumerate(leaves):
            assert leaf.grad is None if not wanted >> j & 1 else torch.equal(leaf.grad, whole[j])


def test_without_rows_adapters_or_values(cuda):
    for rows, k, n, count in ((0, 20, 30, 3), (7, 20, 30, 0), (7, 0, 30, 3), (7, 20, 0, 3)):
        base, x, a, b, index, scaling = _inputs(cuda, rows, k, n, count, 4, torch.float32, "none")
        index.fill_(1)
        for t in (x, a, b):
            t.requires_grad_()
        y = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
        assert torch.equal(y, base)
        y.sum().backward()
        for t in (x, a, b):
            assert t.grad.shape == t.shape and not t.grad.any()


def test_a_replayed_graph_reads_its_index_when_it_runs(cuda):
    base, x, a, b, index, scaling = _inputs(cuda, 2500, 200, 150, 5, 12, torch.bfloat16, "mixed")
    for t in (x, a, b):
        t.requires_grad_()
    dy = torch.randn(2500, 150, device=cuda).bfloat16()

    def step():
        y = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
        return (y.detach(), *torch.autograd.grad(y, (x, a, b), dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        index.copy_(_inputs(cuda, 2500, 200, 150, 5, 12, torch.bfloat16, ("mixed", "runs", "one", "none")[seed])[4])
        scaling.mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)
        torch.cuda.synchronize()


def test_calls_on_two_streams_at_once(cuda):
    cases = [_inputs(cuda, 700, 200, 150, 5, 12, torch.bfloat16, order, seed) for seed, order in enumerate(("mixed", "runs"))]
    want = [sr_states.adapter_add(*case[:5], scaling=case[5]) for case in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(sr_states.adapter_add(*cases[k][:5], scaling=cases[k][5]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(y, want[k]) for y in got[k])


def test_an_operand_changed_before_the_backward_pass_is_noticed(cuda):
    base, x, a, b, index, scaling = _inputs(cuda, 60, 80, 90, 4, 10, torch.float32, "mixed")
    a.requires_grad_()
    for t in (x, index, scaling):
        y = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_tangents_are_refused(cuda):
    """Forward-mode differentiation, in every grad mode; a tangent would be lost without a word."""
    base, x, a, b, index, scaling = _inputs(cuda, 20, 80, 90, 4, 10, torch.float32, "mixed")
    want = sr_states.adapter_add(base, x, a, b, index, scaling=scaling)
    operands = {"base": base, "x": x, "a": a, "b": b, "scaling": scaling, "out": base.clone()}
    with forward_ad.dual_level():
        for name, t in operands.items():
            dual = {**operands, name: forward_ad.make_dual(t, torch.ones_like(t))}
            if name != "out":
                dual.pop("out")
            for mode in (True, False):
                with torch.set_grad_enabled(mode), pytest.raises(NotImplementedError, match="forward-mode"):
                    sr_states.adapter_add(index=index, **dual)
            with forward_ad._set_fwd_grad_enabled(False):  # nothing is lost where nothing is differentiated
                assert torch.equal(sr_states.adapter_add(index=index, **dual), want)
        assert torch.equal(sr_states.adapter_add(base, x, a, b, index, scaling=scaling), want)


def test_refusals(cuda):
    base, x, a, b, index, scaling = _inputs(cuda, 20, 80, 90, 4, 10, torch.float32, "mixed")
    add = sr_states.adapter_add
    cases = [
        (TypeError, "FP32, BF16 or FP16", lambda: add(base.double(), x.double(), a.double(), b.double(), index)),
        (TypeError, "a must have x's dtype", lambda: add(base, x, a.half(), b, index)),
        (TypeError, "b must have x's dtype", lambda: add(base, x, a, b.half(), index)),
        (TypeError, "base must have x's dtype", lambda: add(base.half(), x, a, b, index)),
        (TypeError, "index must be", lambda: add(base, x, a, b, index.float())),
        (TypeError, "scaling must be", lambda: add(base, x, a, b, index, scaling=scaling.half())),
        (ValueError, "number for each adapter", lambda: add(base, x, a, b, index, scaling=scaling[:3])),
        (ValueError, "scaling gets no gradient", lambda: add(base, x, a, b, index, scaling=scaling.clone().requires_grad_())),
        (ValueError, "stack of matrices", lambda: add(base, x, a[0], b, index)),
        (ValueError, "do not match", lambda: add(base, x, a[:3], b, index)),
        (ValueError, "do not match", lambda: add(base, x, a[:, :9], b, index)),
        (ValueError, "do not match", lambda: add(base, x[:, :79], a, b, index)),
        (ValueError, "rank 1 to 128", lambda: add(base, x, a[:, :0], b[..., :0], index)),
        (ValueError, "rank 1 to 128", lambda: add(base, x, a.repeat(1, 13, 1), b.repeat(1, 1, 13), index)),
        (ValueError, "an adapter for each row", lambda: add(base, x, a, b, index[:19])),
        (ValueError, "base must be 20 x 90", lambda: add(base[:, :89], x, a, b, index)),
        (ValueError, "x's device", lambda: add(base, x, a, b, index.cpu())),
        (ValueError, "x's device", lambda: add(base, x, a.cpu(), b, index)),
        (ValueError, "x's device", lambda: add(base.cpu(), x, a, b, index)),
        (ValueError, "out must be", lambda: add(base, x, a, b, index, out=base[:19].clone())),
        (TypeError, "out has dtype", lambda: add(base, x, a, b, index, out=base.half())),
        (ValueError, "must not overlap", lambda: add(base[:10], x[:10], a, b, index[:10], out=base[5:15])),
        (ValueError, "consecutive columns", lambda: add(base, x, a, b, index, out=torch.zeros(90, 20, device=cuda).t())),
        (RuntimeError, "records no gradients", lambda: add(base, x.clone().requires_grad_(), a, b, index, out=base.clone())),
        (RuntimeError, "records no gradients", lambda: add(base, x, a, b, index, out=base.clone().requires_grad_())),
    ]
    for error, message, call in cases:
        with pytest.raises(error, match=message):
            call()
