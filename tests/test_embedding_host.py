"""Refusals of the embedding operators that need no GPU: CPU tensors and the C entries' argument checks."""

import pytest
import torch


def test_cpu_tensors_are_refused():
    from pbg_b200._native import NativeError
    from pbg_b200.embedding import embedding, embedding_backward

    index = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(NativeError):
        embedding(torch.zeros(4, 8), index)
    with pytest.raises(NativeError):
        embedding_backward(torch.zeros(3, 8), index, 4)


def test_entry_points_refuse_bad_arguments():
    from pbg_b200 import _native

    lib = _native.lib()
    one = 256  # a non-null, aligned address that no refused call follows
    assert lib.pbg_embedding(-1, 4, 8, one, 1, one, 0, 8, 1.0, one, 0, one, None) == -1
    assert lib.pbg_embedding(1, 4, 8, one, 1, one, 3, 8, 1.0, one, 0, one, None) == -1
    assert lib.pbg_embedding(1, 4, 8, one, 1, one, 0, 7, 1.0, one, 0, one, None) == -1
    assert b"stride" in lib.pbg_last_error()
    assert lib.pbg_embedding(1, 4, 8, None, 1, one, 0, 8, 1.0, one, 0, one, None) == -1
    back = lib.pbg_embedding_backward
    size = lib.pbg_embedding_backward_workspace(10, 8)
    assert size > 0 and lib.pbg_embedding_backward_workspace(-1, 8) < 0
    assert back(10, 4, 8, one, 0, 8, one, 1, -1, 1.0, one, 0, 8, 0, one, size - 1, one, None) == -1
    assert b"workspace" in lib.pbg_last_error()
    assert back(10, 4, 8, one, 0, 8, one, 1, 4, 1.0, one, 0, 8, 0, one, size, one, None) == -1
    assert b"padding" in lib.pbg_last_error()
    assert back(1 << 31, 4, 8, one, 0, 8, one, 1, -1, 1.0, one, 0, 8, 0, one, size, one, None) == -1
    assert back(10, 4, 8, one, 0, 4, one, 1, -1, 1.0, one, 0, 8, 0, one, size, one, None) == -1
    assert back(0, 4, 8, None, 0, 8, None, 1, -1, 1.0, one, 0, 8, 1, None, 0, one, None) == 0
    assert lib.pbg_embedding(0, 4, 8, None, 1, None, 0, 8, 1.0, None, 0, None, None) == 0
