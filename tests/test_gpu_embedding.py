"""Embedding rows and their gradient against float64, at the sizes and indices where they can go wrong.

Tolerances, from the arithmetic: the forward is one fp32 product and one rounding, so it equals the same
two torch operations.  The gradient's fp32 sums of n terms are off by at most n 2^-24 times the sum of the
terms' magnitudes (any order), the product with the scale and an added old value by 2^-24 each of the
result's magnitude, and the rounding to the output's type by half a step, eps / 2.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _index(law, tokens, rows, gen, dtype=torch.int64):
    if law == "one":
        return torch.full((tokens,), rows // 2, device=DEV, dtype=dtype)
    if law == "ordered":
        return (torch.arange(tokens, device=DEV) * rows // max(tokens, 1)).to(dtype)
    if law == "half":  # half of the tokens on one row, the rest spread
        i = torch.randint(0, rows, (tokens,), generator=gen, device=DEV)
        return torch.where(torch.rand(tokens, generator=gen, device=DEV) < 0.5, rows - 1, i).to(dtype)
    if law == "zipf":
        u = torch.rand(tokens, generator=gen, device=DEV, dtype=torch.float64)
        return torch.exp(u * math.log(rows + 1)).long().sub_(1).clamp_(0, rows - 1).to(dtype)
    return torch.randint(0, rows, (tokens,), generator=gen, device=DEV).to(dtype)


def _check_gradient(got, grad, index, rows, scale, old=None, padding=None):
    n = torch.zeros(rows, dtype=torch.float64, device=DEV)
    keep = (index >= 0) & (index < rows)
    if padding is not None:
        keep &= index != padding
    i = index[keep].long()
    g = grad[keep].double()
    n.index_add_(0, i, torch.ones(len(i), dtype=torch.float64, device=DEV))
    ref = torch.zeros(rows, grad.shape[-1], dtype=torch.float64, device=DEV).index_add_(0, i, g)
    mag = torch.zeros_like(ref).index_add_(0, i, g.abs())
    ref, mag = ref * scale, mag * abs(scale)
    tol = (n[:, None] + 2) * 2.0 ** -24 * mag
    if old is not None:
        ref = ref + old.double()
        tol = tol + 2.0 ** -23 * (old.double().abs() + mag)
    tol = tol + torch.finfo(got.dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(got.dtype).tiny
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - ref).abs().max()))
    if old is None:
        assert bool((got[n == 0] == 0).all())
    else:
        assert torch.equal(got[n == 0], old[n == 0])


CASES = [
    # tokens, rows, width, grad type, out type, law
    (1, 1, 1, F32, F32, "uniform"),
    (1, 300, 128, BF16, F32, "uniform"),
    (7, 5, 3, F16, F16, "uniform"),
    (512, 169, 32, F32, F32, "uniform"),
    (2048, 13, 128, F32, F32, "uniform"),
    (2049, 13, 128, BF16, F32, "half"),       # the first size that sorts in several blocks
    (4096, 4, 256, F32, F32, "one"),          # one run over every share
    (5000, 511, 65, F32, F32, "zipf"),        # 9 key bits: one pass
    (5000, 512, 66, BF16, BF16, "zipf"),      # 10 key bits: two passes, 4-byte vectors
    (20000, 70001, 36, BF16, F32, "zipf"),    # 17 bits; 8-byte vectors
    (3000, 300000, 8, F32, F32, "uniform"),   # 120 ranges of rows
    (65537, 1000, 100, F32, F32, "half"),
    (81920, 13, 128, F32, F32, "uniform"),
    (150001, 4, 17, F16, F32, "uniform"),
    (100000, 100000, 64, BF16, F32, "ordered"),
    (4099, 33, 2050, BF16, F32, "zipf"),      # nine column tiles, odd pairs
    (700, 40, 8192, F32, F32, "half"),        # 64 column tiles
    (300007, 3, 8, BF16, BF16, "one"),
    (90000, 50021, 264, F32, BF16, "zipf"),
    (256, 40, 33, F32, F32, "zipf"),          # the last size of a warp per row, the first of a block per row
    (257, 40, 33, F32, F32, "zipf"),
    (200, 100003, 12, F16, F32, "half"),
    (4096, 1000, 64, BF16, F32, "half"),      # the last size that is not sorted
    (4096, 3, 2000, F32, F16, "one"),
    (1000, 5000, 64, F32, F32, "zipf"),       # few tokens, but too many rows for a block each
    (5000, 52, 32, F32, F32, "uniform"),      # the largest table that is kept whole, the smallest width
    (5000, 53, 32, F32, F32, "uniform"),
    (5000, 52, 31, F32, F32, "uniform"),
    (9000, 40, 4102, BF16, F32, "zipf"),      # 65 column tiles of a kept table, odd pairs
    (5000, 1, 130, F16, BF16, "one"),
    (20011, 21, 100, BF16, F32, "half"),
    # rows in ranges of 22,528 sums, columns by 16, tokens in shares of 1,024 or more
    (300, 1408, 16, F32, F32, "zipf"),        # one range of rows, one share
    (2047, 1409, 16, F16, F16, "uniform"),    # two ranges; the last size of one share
    (2048, 1409, 16, BF16, F32, "half"),      # two shares
    (2049, 22529, 1, F32, F32, "zipf"),
    (150001, 363, 1, BF16, BF16, "uniform"),
    (97299, 3549, 8, BF16, BF16, "zipf"),
    (60001, 1, 15, F32, F32, "one"),          # one warp's row
    (30000, 17, 17, F32, BF16, "zipf"),       # a column tile of one column
    (19180, 329, 57, BF16, F32, "uniform"),
    (40000, 120730, 13, BF16, F32, "zipf"),
    (5000, 2, 24, F16, F32, "half"),
    (5000, 2000, 57, F32, BF16, "half"),      # four column tiles, the last of nine columns
    (300000, 4000, 7, BF16, F32, "zipf"),
    (30000, 1024, 16, F32, F32, "one"),
    # few rows of many columns
    (169, 4, 1752, F16, F16, "uniform"),
    (256, 1, 9000, F32, F32, "one"),
    (3, 700, 5000, BF16, F32, "uniform"),
    # sorted tokens
    (1500, 200003, 700, BF16, F32, "half"),   # in one block
    (300007, 3000, 300, BF16, F32, "half"),
    (400000, 90001, 8, F32, F32, "zipf"),
    (1000000, 700000, 4, F16, F32, "uniform"),  # 20 bits: three passes
    (70000, 3000, 1000, F32, F32, "one"),
    (70001, 400, 1500, BF16, BF16, "zipf"),
]


@pytest.mark.parametrize("tokens,rows,width,gtype,otype,law", CASES)
def test_gradient_matches_float64(tokens, rows, width, gtype, otype, law):
    from pbg_b200.embedding import embedding_backward, index_error

    gen = torch.Generator(device=DEV).manual_seed(tokens + width)
    index = _index(law, tokens, rows, gen)
    grad = torch.randn(tokens, width, generator=gen, device=DEV).to(gtype)
    got = embedding_backward(grad, index, rows, 0.375, out_dtype=otype)
    _check_gradient(got, grad, index, rows, 0.375)
    again = embedding_backward(grad, index.int(), rows, 0.375, out_dtype=otype)
    assert torch.equal(got, again)  # the same bits, and for int32 indices too
    old = torch.randn(rows, width, generator=gen, device=DEV).to(otype)
    into = old.clone()
    assert embedding_backward(grad, index, rows, 0.375, out=into, accumulate=True) is into
    _check_gradient(into, grad, index, rows, 0.375, old=old)
    assert index_error(DEV) == 0


@pytest.mark.parametrize("tokens,rows,width,ttype,otype", [
    (1, 1, 1, F32, F32), (16, 4096, 1024, BF16, BF16), (5, 9, 8192, F32, BF16), (1000, 13, 128, F32, F32),
    (33, 7, 65, BF16, F32), (129, 50, 2046, F16, F16), (3, 5, 36, F32, F16), (70001, 169, 32, F32, F32),
    (4097, 3000, 200, F16, BF16), (40000, 77, 6, BF16, BF16), (19000, 5, 128, F32, F32), (100003, 40, 250, BF16, F32)])
@pytest.mark.parametrize("scale", [1.0, 11.3137085])
def test_forward_is_one_product_and_one_rounding(tokens, rows, width, ttype, otype, scale):
    from pbg_b200.embedding import embedding

    gen = torch.Generator(device=DEV).manual_seed(tokens)
    table = torch.randn(rows, width, generator=gen, device=DEV).to(ttype)
    index = torch.randint(0, rows, (tokens,), generator=gen, device=DEV)
    ref = (table.float()[index] * torch.tensor(scale, dtype=F32, device=DEV)).to(otype)
    assert torch.equal(embedding(table, index, scale, out_dtype=otype), ref)
    assert torch.equal(embedding(table, index.int().view(1, -1), scale, out_dtype=otype), ref[None])


def test_strides_offsets_and_shapes():
    from pbg_b200.embedding import embedding, embedding_backward

    gen = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.randn(40, 300, generator=gen, device=DEV)
    for a, b in ((0, 128), (1, 129), (2, 34), (4, 260)):  # column slices: every vector width
        table = wide[:, a:b]
        index = torch.randint(0, 40, (3, 700), generator=gen, device=DEV)
        assert torch.equal(embedding(table, index.t(), 2.0), 2.0 * table[index.t()])
        grad = torch.randn(3, 700, 300, generator=gen, device=DEV)[..., a:b]
        flat = torch.randn(40 * 300 + 1, generator=gen, device=DEV)
        out = flat[1:].view(40, 300)[:, a:b]  # a slice of an unaligned flat gradient
        before = flat.clone()
        old = out.clone()
        embedding_backward(grad, index, 40, out=out, accumulate=True)
        _check_gradient(out, grad.reshape(-1, b - a), index.reshape(-1), 40, 1.0, old=old)
        mask = torch.ones(40, 300, dtype=torch.bool, device=DEV)
        mask[:, a:b] = False
        assert torch.equal(flat[1:].view(40, 300)[mask], before[1:].view(40, 300)[mask]) and flat[0] == before[0]
    row = torch.randn(64, generator=gen, device=DEV)
    index = torch.randint(0, 9, (5000,), generator=gen, device=DEV)
    _check_gradient(embedding_backward(row.expand(5000, 64), index, 9), row.expand(5000, 64), index, 9, 1.0)
    one = embedding_backward(row, torch.tensor(3, device=DEV), 9)  # a scalar index
    assert torch.equal(one[3], row) and int((one != 0).any(1).sum()) == 1
    assert torch.equal(embedding(wide[:, :64], torch.tensor(3, device=DEV)), wide[3, :64])


def test_empty_sizes():
    from pbg_b200.embedding import embedding, embedding_backward

    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    table = torch.randn(5, 8, device=DEV)
    assert embedding(table, none).shape == (0, 8)
    assert torch.equal(embedding_backward(torch.zeros(0, 8, device=DEV), none, 5), torch.zeros(5, 8, device=DEV))
    into = table.clone()
    embedding_backward(torch.zeros(0, 8, device=DEV), none, 5, out=into, accumulate=True)
    assert torch.equal(into, table)
    some = torch.zeros(3, dtype=torch.int64, device=DEV)
    assert embedding(table[:, :0], some).shape == (3, 0)
    assert embedding_backward(torch.zeros(3, 0, device=DEV), some, 5).shape == (5, 0)


@pytest.mark.parametrize("tokens,rows", [(100, 50), (3000, 50), (9000, 50), (9000, 500)])
def test_padding_and_indices_outside_the_table(tokens, rows):
    from pbg_b200 import embedding as E

    gen = torch.Generator(device=DEV).manual_seed(tokens)
    index = torch.randint(0, rows, (tokens,), generator=gen, device=DEV)
    grad = torch.randn(tokens, 40, generator=gen, device=DEV)
    assert E.index_error(DEV) == 0
    _check_gradient(E.embedding_backward(grad, index, rows, padding_index=7), grad, index, rows, 1.0, padding=7)
    assert E.index_error(DEV) == 0
    index[::3] = rows
    index[1::17] = -1
    index[2::17] = 2 ** 40
    try:
        _check_gradient(E.embedding_backward(grad, index, rows), grad, index, rows, 1.0)
        assert E.index_error(DEV) == 1
        E._error_word(DEV).zero_()
        table = torch.randn(rows, 40, generator=gen, device=DEV)
        out = E.embedding(table, index, 3.0)
        inside = (index >= 0) & (index < rows)
        assert bool((out[~inside] == 0).all()) and torch.equal(out[inside], 3.0 * table[index[inside]])
        assert E.index_error(DEV) == 1
        all_out = torch.full((tokens,), rows + 27, device=DEV)
        assert bool((E.embedding_backward(grad, all_out, rows) == 0).all())
    finally:
        E._error_word(DEV).zero_()


@pytest.mark.parametrize("tokens,width", [(200, 24), (4000, 24), (6000, 24), (6000, 40)])
def test_non_finite_rows_stay_in_their_rows(tokens, width):
    from pbg_b200.embedding import embedding_backward

    index = torch.arange(tokens, device=DEV) % 20
    grad = torch.ones(tokens, width, device=DEV)
    grad[100] = float("nan")   # row 0
    grad[103] = float("inf")   # row 3
    got = embedding_backward(grad, index, 20)
    assert bool(got[0].isnan().all()) and bool(got[3].isinf().all())
    rest = torch.ones(20, dtype=torch.bool, device=DEV)
    rest[[0, 3]] = False
    assert bool((got[rest] == tokens // 20).all())


def test_graph_replay_other_stream_and_two_graphs():
    from pbg_b200.embedding import embedding, embedding_backward

    gen = torch.Generator(device=DEV).manual_seed(5)
    table = torch.randn(300, 96, generator=gen, device=DEV)
    index = torch.randint(0, 300, (20000,), generator=gen, device=DEV)
    grad = torch.randn(20000, 96, generator=gen, device=DEV)
    embedding_backward(grad, index, 300)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = embedding(table, index, 0.5)
            back = embedding_backward(grad, index, 300, 0.5)
        graphs.append((g, out, back))
    index.copy_(torch.randint(0, 300, (20000,), generator=gen, device=DEV))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, (g, _, _) in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    want = embedding_backward(grad, index, 300, 0.5)
    for _, out, back in graphs:
        assert torch.equal(out, 0.5 * table[index]) and torch.equal(back, want)


def test_autograd_function_matches_differences():
    from pbg_b200.model_train import embedding_train

    gen = torch.Generator(device=DEV).manual_seed(9)
    table = torch.randn(11, 16, generator=gen, device=DEV).requires_grad_(True)
    index = torch.randint(0, 11, (4, 50), generator=gen, device=DEV)
    weight = torch.randn(4, 50, 16, generator=gen, device=DEV)

    def loss(t):
        return (embedding_train(t, index, 1.5).square() * weight).sum()

    (g,) = torch.autograd.grad(loss(table), table)
    ref = table.detach().double().requires_grad_(True)
    (r,) = torch.autograd.grad((((1.5 * ref)[index]).square() * weight.double()).sum(), ref)
    terms = 200 * 2.0 ** -22 * 9.0 * float(weight.abs().max()) * float(table.detach().abs().max())
    assert float((g.double() - r).abs().max()) <= terms
    # central differences of the quadratic in float64 of the outputs: exact but for fp32 rounding of the rows
    v = torch.randn(11, 16, generator=gen, device=DEV)
    h = 2.0 ** -6
    f = lambda t: (embedding_train(t, index, 1.5).detach().double().square() * weight.double()).sum()  # noqa: E731
    with torch.no_grad():
        slope = (f(table + h * v) - f(table - h * v)) / (2 * h)
    rounding = 3200 * 2.0 ** -23 * 2.25 * 4 * float((table.detach().abs().max() + h * v.abs().max()) ** 2 * weight.abs().max()) / (2 * h)
    assert abs(float(slope - (g.double() * v.double()).sum())) <= rounding


def test_refusals():
    from pbg_b200._native import NativeError
    from pbg_b200.embedding import embedding, embedding_backward

    table = torch.zeros(4, 8, device=DEV)
    index = torch.zeros(3, dtype=torch.int64, device=DEV)
    grad = torch.zeros(3, 8, device=DEV)
    for call in (lambda: embedding(table.double(), index), lambda: embedding(table[0], index),
                 lambda: embedding(table, index.float()), lambda: embedding(table, index.cpu()),
                 lambda: embedding(table, index, out=torch.zeros(3, 9, device=DEV)),
                 lambda: embedding(table, index, out_dtype=torch.int32),
                 lambda: embedding_backward(grad, index[:2], 4), lambda: embedding_backward(grad, index, -1),
                 lambda: embedding_backward(grad, index, 4, padding_index=4),
                 lambda: embedding_backward(grad, index, 4, accumulate=True),
                 lambda: embedding_backward(grad, index, 4, out=torch.zeros(8, 4, device=DEV).t()),
                 lambda: embedding_backward(grad.double(), index, 4)):
        with pytest.raises(NativeError):
            call()


def test_capture_with_an_eager_graph_of_the_table():
    """A captured backward of a leaf whose older graph lives on another stream is refused, and works once it is gone."""
    from pbg_b200._native import NativeError
    from pbg_b200.model_train import embedding_train

    gen = torch.Generator(device=DEV).manual_seed(12)
    table = torch.randn(30, 64, generator=gen, device=DEV, requires_grad=True)
    index = torch.randint(30, (500,), generator=gen, device=DEV)
    weight = torch.randn(500, 64, generator=gen, device=DEV)
    eager = (embedding_train(table, index) * weight).sum()
    eager.backward()
    want = table.grad.clone()
    table.grad.zero_()
    refused = False
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            embedding_train(table, index)
        except NativeError:
            refused = True
    assert refused
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (embedding_train(table, index) * weight).sum().backward()
    table.grad.zero_()
    for _ in range(2):
        graph.replay()
    assert torch.equal(table.grad, want + want)
    # twice differentiable it is not
    g = torch.autograd.grad((embedding_train(table, index) * weight).square().sum(), table, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()
