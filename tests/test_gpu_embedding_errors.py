"""What the embedding and orthogonalisation kernels report of failures, and who reads it."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("tokens,rows,width", [(3, 50, 24), (40000, 50, 24), (3000, 50, 40), (9000, 50, 40), (9000, 2000, 16),
                                               (9000, 500, 40)])
def test_errors_are_bits_that_stay(tokens, rows, width):
    """An index outside the table does not wipe out an earlier barrier's failure."""
    from pbg_b200 import embedding as E

    gen = torch.Generator(device=DEV).manual_seed(tokens)
    table = torch.randn(rows, width, generator=gen, device=DEV)
    index = torch.randint(0, rows, (tokens,), generator=gen, device=DEV)
    index[1] = rows
    grad = torch.randn(tokens, width, generator=gen, device=DEV)
    try:
        for call in (lambda: E.embedding(table, index), lambda: E.embedding_backward(grad, index, rows)):
            E._error_word(DEV).fill_(2)
            call()
            assert E.index_error(DEV) == 3
            E._error_word(DEV).zero_()
            call()
            assert E.index_error(DEV) == 1
    finally:
        E._error_word(DEV).zero_()


def test_the_learner_steps_checks_report_them():
    """What a one-hot lookup refused, an index outside the table, and a wait that gave up reach the caller."""
    from pbg_b200 import checks, optim
    from pbg_b200.model_train import embedding_train

    table = torch.randn(9, 16, device=DEV, requires_grad=True)
    checks.input_errors(DEV)
    embedding_train(table, torch.tensor([0, 8, 3], device=DEV)).sum().backward()
    optim.orthogonalize(torch.ones(3, 4, device=DEV))
    assert checks.input_errors(DEV) == []
    embedding_train(table, torch.tensor([0, 9, 3], device=DEV))
    with pytest.raises(ValueError, match="outside its table"):
        checks.raise_input_errors(DEV)
    checks.raise_input_errors(DEV)
    optim._error_word(DEV).fill_(4)
    with pytest.raises(ValueError, match="gave up"):
        checks.raise_input_errors(torch.device("cuda"))
    assert optim.orthogonalize_error(DEV) == 0


def test_the_first_call_on_a_busy_stream_keeps_other_streams_errors(monkeypatch):
    """The error word is clear before any call on another stream can set it."""
    from pbg_b200 import embedding as E

    table = torch.randn(9, 16, device=DEV)
    good, bad = torch.tensor([0, 8, 3], device=DEV), torch.tensor([0, 9, 3], device=DEV)
    torch.cuda.synchronize()
    monkeypatch.setattr(E, "_ERROR", {})
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        E.embedding(table, good)
    E.embedding(table, bad)
    torch.cuda.synchronize()
    assert E.index_error(DEV) == 1
