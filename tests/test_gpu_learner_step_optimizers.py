"""The cfg2 learner step with sorted embeddings and with Muon for its matrices, as they are used together.

The tables' gradients by sorted tokens and by one-hot products are fp32 sums of the same terms in other
orders: they differ by at most n 2^-24 of the terms' magnitudes, compared here with the gradients' largest
value.  The transition is checked against float64 of the same gradient: an update's error is at most 2e-5
of its norm (the bar of the orthogonalisation's own tests) and the master's rounding 2^-23 of its norm.
"""

import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
sys.path.insert(0, os.path.join(os.path.dirname(__file__), "golden"))


def _step(gold, **options):
    from pbg_b200.model_train import ModelLearnerStep
    from test_gpu_model_backward import _learner_batch
    from test_gpu_queued_model import _model

    d = gold("queued_model")
    step = ModelLearnerStep(_model(d), **options)
    return step, [_learner_batch(step.model, d, "pre", 1), _learner_batch(step.model, d, "post_2", 2)]


def test_sorted_embeddings_give_the_one_hot_gradient(gold):
    plain, batches = _step(gold)
    other, _ = _step(gold, sorted_embeddings=True)
    a, b = plain.gradient(batches), other.gradient(batches)
    for x, y in zip(a, b):  # the forward is the same bits: one nonzero term per one-hot product
        assert torch.equal(x.total, y.total)
    tables = [n for n in plain.flat.names if "embedding" in n]
    assert len(tables) >= 9
    for n in plain.flat.names:
        g, h = plain.flat.view(plain.grad, n), other.flat.view(other.grad, n)
        # at most 2^16 tokens a row: their sum's rounding, relative to the largest row sum's terms
        torch.testing.assert_close(h, g, rtol=1e-3, atol=2.0 ** -24 * 2 ** 8 * float(g.abs().max()) + 1e-12)


def test_muon_takes_the_matrices_and_adam_the_rest(gold):
    from pbg_b200.model_train import is_hidden_matrix
    from test_gpu_orthogonalize import FP32_BAR, _reference

    lr, mu, decay = 0.02, 0.9, 0.1
    step, batches = _step(gold, sorted_embeddings=True, muon=dict(lr=lr, momentum=mu, decay=decay))
    plain, _ = _step(gold)
    flat = step.flat
    matrices = [n for n in flat.names if is_hidden_matrix(n, flat.shapes[n])]
    assert flat.names[:len(matrices)] == matrices and len(step.muon.matrices) == len(matrices) > 20
    assert flat.split % 4 == 0 and flat.offsets[flat.names[len(matrices)]] == flat.split
    assert sorted(flat.names) == sorted(plain.flat.names)
    for n in flat.names:  # the same weights, wherever they lie
        assert torch.equal(flat.leaves[n].detach(), plain.flat.leaves[n].detach())
    before = flat.master.clone()
    results = step(batches)
    assert all(bool(torch.isfinite(r.total).all()) for r in results) and int(step.muon.skipped) == 0
    # the matrices: float64 of the gradient that the step left in place
    for n in matrices:
        w, g = flat.view(before, n).double(), flat.view(step.grad, n).double()
        u = (mu * (1 - mu) + (1 - mu)) * g
        f = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        want = w * (1 - lr * decay) - lr * f * _reference(u)
        bar = lr * f * FP32_BAR * 1.3 * math.sqrt(min(w.shape)) + 2.0 ** -23 * float(want.norm())
        assert float((flat.view(flat.master, n).double() - want).norm()) <= bar, n
    # the rest: AdamW over the slice from the gradient of another step over the same batches
    plain.gradient(batches)
    for n in flat.names[len(matrices):]:
        moved = flat.view(flat.master, n) - flat.view(before, n)
        touched = plain.flat.view(plain.grad, n) != 0
        assert float(moved.abs().max()) <= 3e-4 * 1.01  # a first AdamW step moves at most lr
        assert bool((moved[~touched] == 0).all())
    # a second step from the moved weights, and inference with them
    results = step(batches)
    assert all(bool(torch.isfinite(r.total).all()) for r in results)
    step.model.eval()


def test_the_transitions_replay_in_one_graph(gold):
    step, batches = _step(gold, sorted_embeddings=True, muon={})
    twin, _ = _step(gold, sorted_embeddings=True, muon={})
    step.gradient(batches)
    twin.grad.copy_(step.grad)
    graph = torch.cuda.CUDAGraph()
    kept = twin.flat.master.clone()
    with torch.cuda.graph(graph):
        twin.muon.step()
        twin.adam.step()
    assert torch.equal(twin.flat.master, kept)  # capturing runs nothing
    graph.replay()
    step.muon.step()
    step.adam.step()
    assert torch.equal(step.flat.master, twin.flat.master)
    assert torch.equal(step.muon.momentum, twin.muon.momentum) and torch.equal(step.adam.first, twin.adam.first)
