"""orthogonalize, hip_muon_step_ and MuonHip against 64-bit forms of their definitions.

Tolerance of an orthogonalised matrix, in the 2-norm relative to the result.
Rounding a value to FP16 costs at most 2^-11 / sqrt(3) = 2.8e-4 of it (rms).
A step rounds X's copy, G and P; with |P| <= 3, |P + 1.5| <= 3 and
|b + 2 c G| <= 4.8 these add at most 6.4 * 2.8e-4 = 1.8e-3 in quadrature, and
a step's map contracts errors around the fixed range, so that no more than two
steps' worth survives: 2.6e-3.  With BF16's own 1.7e-3 (rms) that is 3.1e-3;
the limit is 4e-3.
"""

from __future__ import annotations

import copy

import _matrix_oracle as oracle
import pytest
import sr_states
import torch
from conftest import POLICIES

pytestmark = pytest.mark.gpu
LIMIT = 4e-3


def _matrix(shape, device, seed, dtype=torch.float32, std=1e-3):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, device=device, generator=gen) * std).to(dtype)


SHAPES = [
    (1, 1), (1, 300), (300, 1), (2, 2), (16, 16), (31, 65), (64, 64), (64, 576), (65, 63), (100, 1000), (129, 128),
    (257, 130), (500, 300), (768, 2304), (1100, 1030), (2048, 700),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize_equals_the_definition(cuda, shape, x_dtype):
    x = _matrix(shape, cuda, 1, x_dtype)
    got = sr_states.orthogonalize(x)
    assert got.dtype == torch.bfloat16 and got.shape == x.shape
    assert oracle.relative(got, oracle.orthogonalize(x)) < LIMIT


@pytest.mark.parametrize("shape", [(2003, 2101), (2101, 2003), (8, 1101, 2050), (8, 2050, 1101), (24, 640, 700)])
def test_orthogonalize_of_many_tiles(cuda, shape):
    x = _matrix(shape, cuda, 2, torch.bfloat16)
    got = sr_states.orthogonalize(x, dtype=torch.float32)
    for g, one in zip(got.view(-1, *shape[-2:])[::5], x.view(-1, *shape[-2:])[::5]):
        assert oracle.relative(g, oracle.orthogonalize(one)) < LIMIT


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_orthogonalize_result_types(cuda, dtype):
    for shape in ((96, 130), (130, 96), (50, 20)):
        x = _matrix(shape, cuda, 2)
        got = sr_states.orthogonalize(x, dtype=dtype)
        assert got.dtype == dtype and oracle.relative(got, oracle.orthogonalize(x)) < 2.6e-3


@pytest.mark.parametrize("shape", [(3, 40, 70), (2, 5, 90, 30), (70, 33, 20), (5, 200, 200)])
def test_orthogonalize_batches(cuda, shape):
    x = _matrix(shape, cuda, 3) * torch.arange(1, shape[0] + 1, device=cuda).view(-1, *[1] * (len(shape) - 1))
    got = sr_states.orthogonalize(x)
    want = oracle.orthogonalize(x)
    for g, w in zip(got.flatten(0, -3), want.flatten(0, -3)):
        assert oracle.relative(g, w) < LIMIT
    # A matrix's result does not depend on the batch around it, up to the tile it was computed in.
    assert oracle.relative(got[1], sr_states.orthogonalize(x[1].contiguous())) < LIMIT


def test_orthogonalize_small_singular_values(cuda):
    """A few strong directions over weak noise: the noise's directions grow by 3.4 a step."""
    for rows, cols in ((512, 512), (64, 64), (40, 300), (300, 1500)):
        gen = torch.Generator(device=cuda).manual_seed(4)
        rank = max(1, rows // 32)
        x = torch.randn(rows, rank, device=cuda, generator=gen) @ torch.randn(rank, cols, device=cuda, generator=gen)
        x += 1e-3 * torch.randn(rows, cols, device=cuda, generator=gen)
        assert oracle.relative(sr_states.orthogonalize(x), oracle.orthogonalize(x)) < LIMIT


def test_orthogonalize_scales_and_zeros(cuda):
    x = _matrix((70, 90), cuda, 5)
    want = sr_states.orthogonalize(x)
    for scale in (2.0**40, 2.0**-8):
        assert oracle.relative(sr_states.orthogonalize(x * scale), oracle.orthogonalize(x * scale)) < LIMIT
    assert oracle.relative(sr_states.orthogonalize(x * 2.0**-60), oracle.orthogonalize(x * 2.0**-60)) < LIMIT
    zero = torch.zeros(70, 90, device=cuda)
    assert not sr_states.orthogonalize(zero).any()
    batch = torch.stack([zero, x])
    got = sr_states.orthogonalize(batch)
    assert not got[0].any() and torch.equal(got[1], want)
    rowless = x.clone()
    rowless[3] = 0
    rowless[:, 7] = 0
    got = sr_states.orthogonalize(rowless)
    assert not got[3].any() and not got[:, 7].any()


def test_orthogonalize_keeps_what_is_not_a_number(cuda):
    x = _matrix((2, 70, 90), cuda, 6)
    x[0, 5, 5] = float("nan")
    got = sr_states.orthogonalize(x)
    assert got[0].isnan().all() and not got[1].isnan().any()


def test_orthogonalize_strides_steps_and_coefficients(cuda):
    x = _matrix((90, 70), cuda, 7)
    assert torch.equal(sr_states.orthogonalize(x.t()), sr_states.orthogonalize(x.t().contiguous()))
    view = _matrix((100, 80), cuda, 8)[3:93, 5:75]
    assert torch.equal(sr_states.orthogonalize(view), sr_states.orthogonalize(view.contiguous()))
    flat = _matrix((90 * 70 + 1,), cuda, 9)
    odd = flat[1:].view(90, 70)  # four bytes off the allocation's alignment
    assert torch.equal(sr_states.orthogonalize(odd), sr_states.orthogonalize(odd.clone()))
    for steps, coefficients in ((1, oracle.COEFFICIENTS), (2, oracle.COEFFICIENTS), (9, (1.5, -0.5, 0.0)), (6, (15 / 8, -10 / 8, 3 / 8))):
        got = sr_states.orthogonalize(x, steps=steps, coefficients=coefficients)
        assert oracle.relative(got, oracle.orthogonalize(x, steps, coefficients)) < LIMIT


def test_orthogonalize_replays_and_streams(cuda):
    x = _matrix((200, 130), cuda, 1)
    sr_states.orthogonalize(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sr_states.orthogonalize(x)
    for k in range(3):
        x.copy_(_matrix((200, 130), cuda, 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sr_states.orthogonalize(x))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        other = sr_states.orthogonalize(x * 1.0)
    stream.synchronize()
    assert torch.equal(out, other)


HYPER = {"lr": 0.02, "momentum_factor": 0.95, "weight_decay": 0.1}


def _expected(p, g, m, lr, momentum_factor, weight_decay, nesterov=True, update_scale="spectral"):
    """(momentum before rounding in FP32, parameter in 64 bits, the size of its update)."""
    u = m.float() * momentum_factor + g.float()
    v = u * momentum_factor + g.float() if nesterov else u
    rows, cols = p.shape[0], p[0].numel()
    o = oracle.orthogonalize(v.view(rows, cols)).view(p.shape)
    s = max(1.0, rows / cols) ** 0.5 if update_scale == "spectral" else 0.2 * max(rows, cols) ** 0.5
    return u, p.double() * (1 - lr * weight_decay) - lr * s * o, lr * s * float(o.norm())


def _assert_parameter(got, want, size):
    """Within LIMIT of the update's size, and the parameter's own rounding."""
    half_ulp = 2.0**-9 if got.dtype == torch.bfloat16 else 2.0**-22  # FP32: a few operations
    limit = LIMIT * size + half_ulp * float(want.norm())
    assert float((got.double() - want).norm()) <= limit


@pytest.mark.parametrize("policy", sorted(POLICIES))
@pytest.mark.parametrize("shape", [(70, 130), (130, 65)])
def test_step_stores_every_momentum_format(cuda, policy, shape):
    dtype, rule = POLICIES[policy]
    fmt = sr_states.StateFormat(dtype, rule)
    p, g = _matrix(shape, cuda, 1, std=0.05), _matrix(shape, cuda, 2, std=0.1)
    m = _matrix(shape, cuda, 3, std=0.3).to(dtype)
    u, want, size = _expected(p, g, m, **HYPER)
    stored = sr_states.cast(u, dtype=dtype, rounding=rule, seed=sr_states.state_key(99, 0), offset=12)
    sr_states.hip_muon_step_(p, g, m, **HYPER, seed=99, offset=12, formats=(fmt,))
    assert torch.equal(m.view(torch.uint8), stored.view(torch.uint8))
    _assert_parameter(p, want, size)


@pytest.mark.parametrize("p_dtype, g_dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("shape", [(1, 1), (1, 77), (64, 64), (33, 3, 5, 5), (300, 129)])
@pytest.mark.parametrize("nesterov, update_scale", [(True, "spectral"), (False, "rms")])
def test_step_types_shapes_and_options(cuda, p_dtype, g_dtype, shape, nesterov, update_scale):
    p, g = _matrix(shape, cuda, 1, p_dtype, 0.05), _matrix(shape, cuda, 2, g_dtype, 0.1)
    m = _matrix(shape, cuda, 3, torch.bfloat16, 0.3)
    u, want, size = _expected(p, g, m, **HYPER, nesterov=nesterov, update_scale=update_scale)
    stored = sr_states.cast(u, dtype=torch.bfloat16, seed=sr_states.state_key(5, 0))
    sr_states.hip_muon_step_(p, g, m, **HYPER, nesterov=nesterov, update_scale=update_scale, seed=5)
    assert torch.equal(m, stored)
    _assert_parameter(p, want, size)


@pytest.mark.parametrize("p_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1023, 767), (767, 1023), (4099, 4170), (4170, 4099)])
def test_step_of_large_tensors(cuda, p_dtype, shape):
    p, g = _matrix(shape, cuda, 1, p_dtype, 0.05), _matrix(shape, cuda, 2, p_dtype, 0.1)
    m = _matrix(shape, cuda, 3, torch.bfloat16, 0.3)
    u, want, size = _expected(p, g, m, **HYPER, nesterov=True, update_scale="spectral")
    stored = sr_states.cast(u, dtype=torch.bfloat16, seed=sr_states.state_key(5, 0))
    sr_states.hip_muon_step_(p, g, m, **HYPER, nesterov=True, update_scale="spectral", seed=5)
    assert torch.equal(m, stored)
    _assert_parameter(p, want, size)


def test_step_of_unaligned_views(cuda):
    shape = (65, 33)
    buffers = [_matrix((65 * 33 + 1,), cuda, k, std=0.1) for k in range(2)] + [_matrix((65 * 33 + 3,), cuda, 3).bfloat16()]
    views = [b[-65 * 33:].view(shape) for b in buffers]
    copies = [v.clone() for v in views]
    sr_states.hip_muon_step_(*views, **HYPER, seed=1)
    sr_states.hip_muon_step_(*copies, **HYPER, seed=1)
    for v, c in zip(views, copies):
        assert torch.equal(v, c)


def _model(device, p_dtype=torch.float32):
    shapes = [(96, 64), (64, 96), (96, 64), (40, 3, 3, 3), (64, 96), (0, 5), (96, 64)]
    return [torch.nn.Parameter(_matrix(s, device, k, p_dtype, 0.05)) for k, s in enumerate(shapes)]


@pytest.mark.parametrize("cls, rule", [(sr_states.MuonHip, "stochastic"), (sr_states.MuonHipRN, "nearest")])
def test_optimizer_equals_functional_steps(cuda, cls, rule):
    params = _model(cuda)
    opt = cls(params, lr=0.02, weight_decay=0.1, seed=17)
    mirror = [p.detach().clone() for p in params]
    momenta = [torch.zeros_like(p, dtype=torch.bfloat16) for p in mirror]
    for step in range(1, 4):
        for k, p in enumerate(params):
            p.grad = None if k == 1 and step == 2 else _matrix(p.shape, cuda, 100 * step + k, std=0.1)
        opt.step()
        for k, (p, m) in enumerate(zip(mirror, momenta)):
            if params[k].grad is not None and p.numel():
                u, want, size = _expected(p, params[k].grad, m, **HYPER)
                m.copy_(sr_states.cast(u, dtype=torch.bfloat16, rounding=rule,
                                       seed=sr_states.state_key(sr_states.update_key(17, step, k), 0)))
                _assert_parameter(params[k].detach(), want, size)
                assert torch.equal(opt.state[params[k]]["momentum_buffer"], m)
            p.copy_(params[k].detach())
    assert "momentum_buffer" in opt.state[params[1]]


def test_optimizer_resumes_from_a_checkpoint(cuda):
    def run(params, opt, steps):
        for step in steps:
            for k, p in enumerate(params):
                p.grad = _matrix(p.shape, cuda, 10 * step + k, std=0.1)
            opt.step()

    params = _model(cuda)
    opt = sr_states.MuonHip(params, state_dtype=torch.float8_e4m3fn, seed=3)
    run(params, opt, (1, 2))
    saved = copy.deepcopy(opt.state_dict())  # its tensors are the live states
    resumed = [torch.nn.Parameter(p.detach().clone()) for p in params]
    run(params, opt, (3,))
    other = sr_states.MuonHip(resumed, state_dtype=torch.float8_e4m3fn, seed=0)
    other.load_state_dict(saved)
    run(resumed, other, (3,))
    for a, b in zip(params, resumed):
        assert torch.equal(a, b)


def test_optimizer_lowers_a_loss_with_fp8_products(cuda):
    """The operators together: a two-layer regression with FP8 linear layers, updated by Muon."""
    gen = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(512, 64, device=cuda, generator=gen)
    target = torch.tanh(x @ torch.randn(64, 32, device=cuda, generator=gen) / 8)
    w1 = torch.nn.Parameter(torch.randn(128, 64, device=cuda, generator=gen) / 8)
    w2 = torch.nn.Parameter(torch.randn(32, 128, device=cuda, generator=gen) / 11)
    opt = sr_states.MuonHip([w1, w2], lr=0.02, seed=1)
    losses = []
    for step in range(30):
        seeds = [sr_states.update_key(9, step, k) for k in range(2)]
        hidden = torch.relu(sr_states.block_linear(x, w1, seed=seeds[0]))
        loss = (sr_states.block_linear(hidden, w2, seed=seeds[1]) - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.5 * losses[0]


def test_optimizer_refuses_capture(cuda):
    params = _model(cuda)[:1]
    opt = sr_states.MuonHip(params)
    params[0].grad = torch.ones_like(params[0])
    opt.step()
    torch.cuda.synchronize()
    before = params[0].detach().clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(before, params[0])


def test_refusals(cuda):
    p = torch.zeros(8, 16, device=cuda)
    g, m = torch.zeros_like(p), torch.zeros_like(p, dtype=torch.bfloat16)

    def step(*tensors, **options):
        return lambda: sr_states.hip_muon_step_(*tensors, **{"lr": 0.1, "momentum_factor": 0.9, "seed": 0, **options})

    cases = [
        (TypeError, "expected FP32", lambda: sr_states.orthogonalize(p.double())),
        (TypeError, "dtype must be", lambda: sr_states.orthogonalize(p, dtype=torch.float8_e5m2)),
        (ValueError, "takes matrices", lambda: sr_states.orthogonalize(p[0])),
        (ValueError, "positive integer", lambda: sr_states.orthogonalize(p, steps=0)),
        (ValueError, "three finite", lambda: sr_states.orthogonalize(p, coefficients=(1.0, 2.0))),
        (ValueError, "out of range", lambda: sr_states.orthogonalize(p, coefficients=(3.0, 0.0, 0.0))),
        (ValueError, "invalid eps", lambda: sr_states.orthogonalize(p, eps=-1.0)),
        (ValueError, "learning rate", step(p, g, m, lr=-1.0)),
        (ValueError, "invalid momentum", step(p, g, m, momentum_factor=1.0)),
        (ValueError, "weight_decay", step(p, g, m, weight_decay=-1.0)),
        (ValueError, "update_scale", step(p, g, m, update_scale="none")),
        (ValueError, "identical shapes", step(p, g[:4], m)),
        (ValueError, "contiguous", step(p.t(), g.t(), m.t())),
        (ValueError, "must not overlap", step(p, g, p)),
        (TypeError, "FP32 or BF16", step(p.half(), g, m)),
        (ValueError, "matrices", step(p[0], g[0], m[0])),
        (ValueError, "same GPU", step(p, g.cpu(), m)),
    ]
    for error, message, call in cases:
        with pytest.raises(error, match=message):
            call()
    shared = torch.nn.Parameter(p), torch.nn.Parameter(p[:4])
    opt = sr_states.MuonHip(shared)
    for parameter in shared:
        parameter.grad = torch.ones_like(parameter)
    with pytest.raises(ValueError, match="must not overlap"):
        opt.step()
    assert not p.any()
