"""Expert layers and adapters as a program uses them together, and under what torch wraps around a call."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import sr_states
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "train_fp8_experts.py"
    spec = importlib.util.spec_from_file_location("train_fp8_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_trains_and_serves(cuda):
    example = _example()
    network, adapters, x, task, losses, adapted = example.train(steps=3, rows=200, device=cuda)
    assert len(losses) == len(adapted) == 3
    assert all(torch.isfinite(torch.tensor(values)).all() for values in (losses, adapted))
    assert all(p.grad is not None and p.grad.isfinite().all() for p in adapters.parameters())
    answers = example.serve(network, adapters, x, task)
    assert answers.shape == (200, 1) and answers.isfinite().all() and not answers.requires_grad


def test_gradients_reach_every_parameter_of_the_example(cuda):
    example = _example()
    torch.manual_seed(1)
    network = example.Network(128, 2, 3, cuda)
    adapters = torch.nn.ModuleList(example.Adapters(128, 4, 2, cuda) for _ in range(2))
    for adapter in adapters:
        torch.nn.init.normal_(adapter.b)
    x, task = torch.randn(90, 128, device=cuda, requires_grad=True), torch.arange(90, device=cuda) % 3 - 1
    network(x, 1, adapters, task).sum().backward()
    for name, tensor in [("x", x), *network.named_parameters(), *adapters.named_parameters()]:
        assert tensor.grad is not None and tensor.grad.isfinite().all() and tensor.grad.any(), name


def _inputs(device, rows=300, width=256, hidden=384, experts=4, tasks=3):
    gen = torch.Generator(device=device).manual_seed(4)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device=device, generator=gen) * std).bfloat16()

    tensors = dict(x=normal(rows, width), shared=normal(width, width, std=width**-0.5), a=normal(tasks, 8, width, std=width**-0.5),
                   b=normal(tasks, width, 8, std=0.3), up=normal(experts, hidden, width, std=width**-0.5),
                   down=normal(experts, width, hidden, std=hidden**-0.5))
    expert = torch.randint(0, experts, (rows,), device=device, generator=gen).sort().values
    sizes = torch.bincount(expert, minlength=experts)
    index = torch.randint(-1, tasks, (rows,), device=device, generator=gen)
    return tensors, sizes, index, normal(rows, width, std=1e-2)


def _layer(x, shared, a, b, up, down, sizes, index):
    y = sr_states.adapter_add(sr_states.block_linear(x, shared, seed=3), x, a, b, index, scaling=0.5)
    h = sr_states.grouped_block_linear(torch.relu(y), up, sizes, seed=4)
    return x + sr_states.grouped_block_linear(torch.relu(h), down, sizes, seed=5)


def _gradients(call, tensors, sizes, index, dy):
    leaves = {name: t.clone().requires_grad_() for name, t in tensors.items()}
    y = call(**leaves, sizes=sizes, index=index)
    y.backward(dy)
    return [y.detach(), *(leaf.grad for leaf in leaves.values())]


def test_layer_under_autocast_checkpointing_and_compilation(cuda):
    from torch.utils.checkpoint import checkpoint

    arguments = _inputs(cuda)
    want = _gradients(_layer, *arguments)

    def cast(**tensors):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return _layer(**tensors)

    def again(reentrant):
        return lambda **tensors: checkpoint(lambda *t: _layer(**dict(zip(tensors, t))), *tensors.values(), use_reentrant=reentrant)

    for call in (cast, again(False), again(True), torch.compile(_layer, backend="eager")):
        for got, expected in zip(_gradients(call, *arguments), want):
            assert torch.equal(got, expected)


def test_a_captured_step_of_the_layer_follows_its_routing(cuda):
    tensors, sizes, index, dy = _inputs(cuda)
    leaves = {name: t.clone().requires_grad_() for name, t in tensors.items()}

    def step():
        y = _layer(**leaves, sizes=sizes, index=index)
        return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for counts in ([300, 0, 0, 0], [75, 75, 75, 75], [1, 128, 129, 42], [10, 0, 0, 20]):
        sizes.copy_(torch.tensor(counts))
        index.copy_(index.roll(7))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)
        torch.cuda.synchronize()


def test_a_step_on_a_side_stream_that_is_still_at_work(cuda):
    tensors, sizes, index, dy = _inputs(cuda)
    want = _gradients(_layer, tensors, sizes, index, dy)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late, late_sizes, late_index = dy.clone(), sizes.clone(), index.clone()
        for _ in range(20):
            late = late * 1.0
            late_sizes, late_index = late_sizes + 0, late_index + 0
        got = _gradients(_layer, tensors, late_sizes, late_index, late)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_the_layer_in_inference_mode(cuda):
    tensors, sizes, index, _ = _inputs(cuda)
    want = _layer(**tensors, sizes=sizes, index=index)
    with torch.inference_mode():
        got = _layer(**tensors, sizes=sizes, index=index)
        base = sr_states.block_linear(tensors["x"], tensors["shared"], seed=3)
        into = torch.empty_like(base)
        sr_states.adapter_add(base, tensors["x"], tensors["a"], tensors["b"], index, out=into)
        assert torch.equal(into, sr_states.adapter_add(base, tensors["x"], tensors["a"], tensors["b"], index))
    assert torch.equal(got, want)


def test_optimizers_update_what_the_layer_learns(cuda):
    tensors, sizes, index, dy = _inputs(cuda)
    parameters = {name: torch.nn.Parameter(t) for name, t in tensors.items() if name != "x"}
    before = {name: p.detach().clone() for name, p in parameters.items()}
    optimizer = sr_states.AdamWHip(list(parameters.values()), lr=1e-2, seed=7)
    for _ in range(2):
        optimizer.zero_grad()
        _layer(tensors["x"], **parameters, sizes=sizes, index=index).backward(dy)
        optimizer.step()
    for name, p in parameters.items():
        assert p.isfinite().all() and not torch.equal(p, before[name]), name


def test_gradients_are_not_differentiated_again(cuda):
    tensors, sizes, index, dy = _inputs(cuda)
    x = tensors["x"].clone().requires_grad_()
    up = tensors["up"].clone().requires_grad_()
    a = tensors["a"].clone().requires_grad_()
    for y, leaves in ((sr_states.grouped_block_linear(x, up, sizes), (x, up)),
                      (sr_states.adapter_add(x * 1.0, x, a, tensors["b"], index), (x, a))):
        scale = torch.ones_like(y).requires_grad_()
        plain = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
        again = torch.autograd.grad(y, leaves, scale, create_graph=True)
        for got, want in zip(again, plain):
            assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            again[1].sum().backward()


def test_gradients_through_saved_tensor_hooks(cuda):
    """Saved tensors that move to the host and back, as activation offloading has it."""
    tensors, sizes, index, dy = _inputs(cuda)
    want = _gradients(_layer, tensors, sizes, index, dy)

    def offloaded(**arguments):
        with torch.autograd.graph.save_on_cpu():
            return _layer(**arguments)

    for got, expected in zip(_gradients(offloaded, tensors, sizes, index, dy), want):
        assert torch.equal(got, expected)


@pytest.mark.parametrize("operator", ["adapters", "experts"])
def test_a_node_called_by_itself_runs_on_the_callers_stream(cuda, operator):
    """Beside the engine, which sets the stream of the forward pass: a call from another one, and a captured call."""
    tensors, sizes, index, dy = _inputs(cuda)
    names = ("x", "a", "b") if operator == "adapters" else ("x", "up")
    x, *weights = (tensors[name].requires_grad_() for name in names)
    if operator == "adapters":
        y = sr_states.adapter_add(tensors["shared"][:1].expand(300, -1), x, *weights, index)
    else:
        y, dy = sr_states.grouped_block_linear(x, *weights, sizes), dy.repeat(1, 2)[:, :384].contiguous()

    def node():
        with torch.no_grad():
            return [g for g in y.grad_fn(dy) if g is not None]

    def engine():
        return torch.autograd.grad(y, (x, *weights), dy, retain_graph=True)

    first = engine()
    torch.cuda.synchronize()
    side, work = torch.cuda.Stream(), torch.randn(4096, 4096, device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            work = work @ work * 1e-2
        dy.mul_(2)
        got = node()
    torch.cuda.synchronize()
    want = engine()
    assert len(got) == len(want) and not torch.equal(want[0], first[0])
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = node()
    for factor in (0.25, 4.0, -1.0):
        dy.mul_(factor)
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(captured, engine()):
            assert torch.equal(g, w)
        torch.cuda.synchronize()


def test_nodes_refuse_gradients_and_kept_tensors_of_other_shapes(cuda):
    """What the engine would not pass: a node called by itself, and a hook that puts other tensors in place of saved ones."""
    tensors, sizes, index, dy = _inputs(cuda)
    x, a, up = (tensors[name].requires_grad_() for name in ("x", "a", "up"))

    def calls():
        return ((sr_states.adapter_add(x * 1.0, x, a, tensors["b"], index), dy),
                (sr_states.grouped_block_linear(x, up, sizes), dy.repeat(1, 2)[:, :384].contiguous()))

    for y, grad in calls():
        for other in (grad[:1], grad[:, :128], grad.float(), grad.cpu(), grad[None]):
            with torch.no_grad(), pytest.raises(RuntimeError, match="the gradient must be"):
                y.grad_fn(other)
    for change in (lambda t: t[:1], lambda t: t.double(), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.dtype == torch.float32 else t):
            y = sr_states.adapter_add(tensors["shared"][:1].expand(300, -1), x, a, tensors["b"], index)
        with pytest.raises(RuntimeError, match="kept for the backward pass"):
            torch.autograd.grad(y, a, dy)
