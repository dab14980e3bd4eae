"""The learner step's two transitions, Muon's of the matrices and AdamW's of the rest, as one."""

import pytest
import torch

from test_gpu_learner_step_optimizers import _step

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _state(step):
    return [t.clone() for t in (step.flat.master, step.muon.momentum, step.adam.first, step.adam.second, step.adam.step_count)]


@pytest.mark.parametrize("where,value", [("matrix", float("inf")), ("matrix", float("nan")), ("rest", -float("inf")),
                                         ("rest", float("nan")), ("rest", 3e30)])
def test_a_gradient_that_is_not_finite_stops_both(gold, where, value):
    """3e30: finite, but its square is not, so AdamW's guard stops it."""
    step, batches = _step(gold, sorted_embeddings=True, muon=dict(lr=0.02))
    step(batches)
    before = _state(step)
    step.gradient(batches)
    good = step.grad.clone()
    assert bool(good.isfinite().all()) and step.flat.split > 100
    step.grad[step.flat.split - 9 if where == "matrix" else step.flat.split + 9] = value
    if where == "matrix":  # an element of the last matrix, not of the few that lie between the parts
        at, r, c = step.muon.matrices[-1]
        step.grad[at + r * c - 1] = value
    step.transition()
    assert int(step.muon.skipped) == 1 and float(step.adam.report[0]) == 0.0
    for a, b in zip(before, _state(step)):
        assert torch.equal(a, b)
    assert bool((step.grad[step.flat.split:] == 0).all())
    for at, r, c in step.muon.matrices:
        assert bool((step.grad[at:at + r * c] == 0).all())
    step.grad.copy_(good)
    step.transition()
    assert int(step.muon.skipped) == 0 and float(step.adam.report[0]) == 1.0
    assert not torch.equal(before[0][:step.flat.split], step.flat.master[:step.flat.split])
    assert not torch.equal(before[0][step.flat.split:], step.flat.master[step.flat.split:])


def test_the_whole_transition_replays_in_a_graph(gold):
    step, batches = _step(gold, sorted_embeddings=True, muon={})
    twin, _ = _step(gold, sorted_embeddings=True, muon={})
    step.gradient(batches)
    twin.grad.copy_(step.grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        twin.transition()
    for stop in (False, True, False):
        for s in (step, twin):
            s.grad.copy_(s.grad if not stop else torch.full_like(s.grad, float("nan")))
        step.transition()
        graph.replay()
        for a, b in zip(_state(step), _state(twin)):
            assert torch.equal(a, b)
        assert int(step.muon.skipped) == int(twin.muon.skipped) == int(stop)
        grad = torch.randn(step.grad.shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
        step.grad.copy_(grad), twin.grad.copy_(grad)


def test_without_muon_the_transition_is_adamw(gold):
    step, batches = _step(gold)
    twin, _ = _step(gold)
    step(batches)
    twin.gradient(batches)
    twin.adam.step()
    assert torch.equal(step.adam.grad, twin.adam.grad) and torch.equal(step.flat.master, twin.flat.master)


def test_adamw_takes_the_rest_of_the_gradient(gold):
    """A first AdamW step against float64 of the gradient that it was given: about 16 fp32 roundings of the
    direction (of size 1, times lr) and two of the master."""
    lr, decay, clip = 3e-4, 0.1, 1.0
    step, batches = _step(gold, sorted_embeddings=True, muon={}, lr=lr, weight_decay=decay, grad_clip=clip)
    step.gradient(batches)
    split = step.flat.split
    before, g = step.flat.master[split:].double(), step.grad[split:].double()
    step.transition()
    g = g * min(1.0, clip / float(g.norm()))
    want = before * (1 - lr * decay) - lr * g / (g.abs() + 1e-8)
    bar = lr * 32 * 2.0 ** -24 + 2.0 ** -23 * before.abs()
    assert bool(((step.flat.master[split:].double() - want).abs() <= bar).all())
    assert float((want - before).abs().max()) > 0.9 * lr and int((g != 0).sum()) > g.numel() // 4
