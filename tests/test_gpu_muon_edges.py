"""Edges of the orthogonalised updates: norms at the ends of FP32's range, steps that are refused.

Tolerances are those of test_gpu_muon.py.
"""

from __future__ import annotations

import _matrix_oracle as oracle
import pytest
import sr_states
import torch

pytestmark = pytest.mark.gpu
LIMIT = 4e-3


def _matrix(shape, device, seed, dtype=torch.float32, std=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, device=device, generator=gen) * std).to(dtype)


# Sums of squares from 1e-66 to beyond 1e77, in one workgroup, in tiles, tall and in a batch.
@pytest.mark.parametrize("shape", [(50, 70), (200, 300), (300, 200), (2, 150, 90)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("std", [6e37, 1e25, 1e19, 1e-19, 1e-25, 1e-35])
def test_orthogonalize_over_the_range_of_norms(cuda, shape, dtype, std):
    x = _matrix(shape, cuda, 1, torch.float64, std).to(dtype)
    assert x.isfinite().all()
    eps = 1e-7 if std > 1 else 0.0
    got = sr_states.orthogonalize(x, eps=eps)
    want = oracle.orthogonalize(x, eps=eps)
    assert float(want.abs().max()) > 0.01
    assert oracle.relative(got, want) < LIMIT


def test_a_norm_of_zero_or_beyond_every_number(cuda):
    for shape in ((50, 70), (200, 300)):
        zero = torch.zeros(shape, device=cuda)
        assert torch.equal(sr_states.orthogonalize(zero, eps=0.0), zero.bfloat16())
        infinite = _matrix(shape, cuda, 1)
        infinite[3, 4] = float("inf")
        assert sr_states.orthogonalize(infinite).isnan().any()


@pytest.mark.parametrize("shape", [(50, 70), (200, 300), (300, 200)])
@pytest.mark.parametrize("std", [1e30, 1e-30])
def test_step_over_the_range_of_norms(cuda, shape, std):
    p, g, m = _matrix(shape, cuda, 1), _matrix(shape, cuda, 2, std=std), _matrix(shape, cuda, 3, std=std)
    u = m * 0.9 + g
    update = oracle.orthogonalize(u * 0.9 + g, eps=0.0) * max(1.0, shape[0] / shape[1]) ** 0.5
    want = p.double() - 0.5 * update
    fmt = sr_states.StateFormat(torch.float32, "nearest")
    sr_states.hip_muon_step_(p, g, m, lr=0.5, momentum_factor=0.9, eps=0.0, seed=1, formats=(fmt,))
    assert torch.equal(m, u)
    assert float((p.double() - want).norm()) <= LIMIT * float((0.5 * update).norm()) + 2.0**-22 * float(want.norm())


def _optimizer(shapes, device):
    """An optimizer after a first step over the matrices that are not too large, with gradients for a second one."""
    params = [torch.nn.Parameter(_matrix(shape, device, k)) for k, shape in enumerate(shapes)]
    opt = sr_states.MuonHip(params, seed=3)
    for step in range(2):
        for k, p in enumerate(params):
            p.grad = _matrix(p.shape, device, 10 * step + k) if step or p.shape[0] <= 1 << 20 else None
        if not step:
            opt.step()
    return params, opt


def _unchanged(params, opt, step):
    before = [(p.detach().clone(), opt.state[p]["momentum_buffer"].clone()) for p in params[:2]]
    with pytest.raises((RuntimeError, ValueError)) as error:
        step()
    for p, (value, momentum) in zip(params, before):
        assert torch.equal(p, value) and torch.equal(opt.state[p]["momentum_buffer"], momentum)
    return str(error.value)


def test_a_step_with_a_matrix_that_is_too_large_changes_nothing(cuda):
    params, opt = _optimizer([(64, 96), (130, 70), ((1 << 20) + 1, 2)], cuda)
    assert "too large" in _unchanged(params, opt, opt.step)
    with pytest.raises((RuntimeError, ValueError), match="too large"):
        sr_states.orthogonalize(params[2].detach())


def test_a_step_without_memory_for_a_workspace_changes_nothing(cuda, monkeypatch):
    params, opt = _optimizer([(64, 96), (130, 70), (900, 900)], cuda)
    empty = torch.empty

    def small_only(*args, **options):
        if options.get("dtype") == torch.uint8 and args[0] > 900 * 900 * 4:
            raise torch.OutOfMemoryError("no memory for a workspace")
        return empty(*args, **options)

    monkeypatch.setattr(torch, "empty", small_only)
    assert "no memory" in _unchanged(params, opt, opt.step)


# Both sides of the lines between tile shapes: 256 and 512 tiles of 64 x 64 on a triangle, and 256 of 128 x 128.
@pytest.mark.parametrize("shape", [
    (1410, 1500), (1472, 1480), (1984, 2050), (2040, 2100), (2112, 2150), (2170, 2180), (2816, 2900), (2890, 2900),
    (12, 570, 600), (3, 1150, 1200), (7, 760, 790), (2, 1400, 1450), (25, 380, 400),
])
def test_orthogonalize_on_both_sides_of_the_tile_shapes(cuda, shape):
    x = _matrix(shape, cuda, 1, torch.bfloat16)
    got = sr_states.orthogonalize(x)
    for g, one in zip(got.view(-1, *shape[-2:])[::6], x.view(-1, *shape[-2:])[::6]):
        assert oracle.relative(g, oracle.orthogonalize(one)) < LIMIT


def test_batches_beyond_a_launch(cuda):
    """More matrices than a launch takes, too large for one workgroup each."""
    x = _matrix((70, 90, 130), cuda, 1)
    got = sr_states.orthogonalize(x)
    for k in (0, 63, 64, 69):
        assert oracle.relative(got[k], oracle.orthogonalize(x[k])) < LIMIT
    params = [torch.nn.Parameter(t.clone()) for t in x]
    grads = _matrix((70, 90, 130), cuda, 2)
    for p, g in zip(params, grads):
        p.grad = g.clone()
    sr_states.MuonHip(params, lr=0.5, momentum=0.9, seed=1).step()
    for k in (0, 63, 64, 69):
        update = 0.5 * oracle.orthogonalize(grads[k] * 0.9 + grads[k])
        off = float((params[k].detach().double() - (x[k].double() - update)).norm())
        assert off <= LIMIT * float(update.norm()) + 2.0**-22 * float(x[k].norm())


def test_step_on_a_side_stream(cuda):
    params = [_matrix((200, 300), cuda, k) for k in range(3)]
    momentum = params[2].bfloat16()
    copies = params[0].clone(), momentum.clone()
    sr_states.hip_muon_step_(copies[0], params[1], copies[1], lr=0.1, momentum_factor=0.9, seed=1)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late = params[1].clone()
        for _ in range(20):
            late = late * 1.0
        sr_states.hip_muon_step_(params[0], late, momentum, lr=0.1, momentum_factor=0.9, seed=1)
    stream.synchronize()
    assert torch.equal(params[0], copies[0]) and torch.equal(momentum, copies[1])
