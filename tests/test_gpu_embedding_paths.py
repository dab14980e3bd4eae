"""The embedding gradient at sizes that the dispatch sends to the sort and to the narrow-row kernel, against float64.

The dispatch (csrc/embedding.cu): a block per row takes up to 4,096 tokens where rows x column tiles are at most
eight an SM, the kept tables up to 52 rows of 32 columns or more, ranges of narrow rows tables of 1,024 rows or
more; the rest is sorted, in one block up to 2,048 tokens.
"""

import pytest
import torch

from test_gpu_embedding import BF16, DEV, F16, F32, _check_gradient, _index

pytestmark = pytest.mark.gpu

CASES = [
    # sorted: 1,000 rows in two column tiles
    (2048, 1000, 200, F32, F32, "uniform"),   # the last size that one block sorts
    (2049, 1000, 200, F32, F32, "uniform"),   # the first that several do
    (2049, 1000, 200, BF16, F32, "half"),
    (30000, 1000, 200, F32, F32, "one"),      # one run over every share
    (30001, 900, 264, BF16, BF16, "one"),
    (100003, 600, 17, F16, F32, "half"),      # one column a lane
    # ranges of narrow rows
    (5000, 2000, 17, F32, F32, "zipf"),       # the last column tile has one column
    (5000, 2000, 33, BF16, F32, "half"),
    (60001, 1024, 15, F32, F32, "one"),       # one warp's row
    (150001, 2047, 1, BF16, BF16, "uniform"),
]


@pytest.mark.parametrize("tokens,rows,width,gtype,otype,law", CASES)
def test_gradient_matches_float64(tokens, rows, width, gtype, otype, law):
    from pbg_b200.embedding import embedding_backward, index_error

    gen = torch.Generator(device=DEV).manual_seed(tokens + rows)
    index = _index(law, tokens, rows, gen)
    grad = torch.randn(tokens, width, generator=gen, device=DEV).to(gtype)
    got = embedding_backward(grad, index, rows, 0.375, out_dtype=otype)
    _check_gradient(got, grad, index, rows, 0.375)
    assert torch.equal(got, embedding_backward(grad, index.int(), rows, 0.375, out_dtype=otype))
    old = torch.randn(rows, width, generator=gen, device=DEV).to(otype)
    into = old.clone()
    embedding_backward(grad, index, rows, 0.375, out=into, accumulate=True)
    _check_gradient(into, grad, index, rows, 0.375, old=old)
    padded = embedding_backward(grad, index, rows, padding_index=rows // 2)
    _check_gradient(padded, grad, index, rows, 1.0, padding=rows // 2)
    assert index_error(DEV) == 0
