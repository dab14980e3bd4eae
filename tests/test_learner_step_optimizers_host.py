"""Host logic of the learner step's optimizers, on CPU: which parameters come first in the flat master, and
the constructors' refusals."""

import pytest
import torch


def test_chosen_parameters_come_first_and_the_rest_is_aligned():
    from pbg_b200.model_train import FlatParameters, is_hidden_matrix

    gen = torch.Generator().manual_seed(0)
    params = {"a.bias": torch.randn(5, generator=gen), "a.weight": torch.randn(3, 5, generator=gen),
              "seat_embedding.weight": torch.randn(4, 6, generator=gen), "b.weight": torch.randn(2, 3, generator=gen),
              "head.weight": torch.randn(1, 7, generator=gen), "tokens": torch.randn(2, 2, generator=gen)}
    flat = FlatParameters(params, "cpu", first=is_hidden_matrix)
    assert flat.names == ["a.weight", "b.weight", "a.bias", "seat_embedding.weight", "head.weight", "tokens"]
    assert flat.split == 24 and flat.offsets["a.bias"] == 24 and flat.numel == 24 + 5 + 24 + 7 + 4
    for n, v in params.items():
        assert torch.equal(flat.leaves[n].detach(), v)
    assert bool((flat.master[21:24] == 0).all())
    same = FlatParameters(params, "cpu")
    assert same.names == list(params) and same.split == 0 and same.numel == sum(v.numel() for v in params.values())


def test_optimizers_refuse_cpu_masters():
    from pbg_b200._native import NativeError
    from pbg_b200.optim import FlatAdam, FlatMuon, orthogonalize

    with pytest.raises(ValueError):
        FlatMuon(torch.zeros(16), [(0, 4, 4)])
    with pytest.raises(ValueError):
        FlatAdam(torch.zeros(16))
    with pytest.raises(NativeError):
        orthogonalize(torch.zeros(4, 4))


def test_entry_points_refuse_bad_arguments():
    import ctypes

    import numpy as np
    from pbg_b200 import _native

    lib = _native.lib()
    one = 256  # a non-null, aligned address that no refused call follows
    f = lib.pbg_orthogonalize
    size = lib.pbg_orthogonalize_workspace(1, 200, 300)
    ok = (3.4445, -4.775, 2.0315, 1e-7)
    assert f(1, 200, 300, one, 0, one, 0, 5, *ok, one, size - 1, one, None) == -1 and b"workspace" in lib.pbg_last_error()
    assert f(1, 200, 300, one, 3, one, 0, 5, *ok, one, size, one, None) == -1
    assert f(1, 200, 70000, one, 0, one, 0, 5, *ok, one, size, one, None) == -1
    assert f(1, 200, 300, one, 0, one, 0, 0, *ok, one, size, one, None) == -1 and b"steps" in lib.pbg_last_error()
    for a, b, c in ((16.0, 0.0, 0.0), (3.0, 0.0, 0.0), (3.4445, -4.775, 0.1), (float("nan"), 0.0, 0.0)):
        assert f(1, 200, 300, one, 0, one, 0, 5, a, b, c, 1e-7, one, size, one, None) == -1, (a, b, c)
    # polynomials in use pass, and empty calls touch nothing
    for a, b, c in ((3.4445, -4.775, 2.0315), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)):
        assert f(0, 200, 300, None, 0, None, 0, 10, a, b, c, 1e-7, None, 0, None, None) == 0
    ints = lambda *v: np.array(v, dtype=np.int64)  # noqa: E731
    p = lambda v: v.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    adjust, words = np.ones(2, dtype=np.float32), np.zeros(int(lib.pbg_muon_plan_words(2)), dtype=np.int64)
    desc = np.zeros(2 * int(lib.pbg_muon_descriptor_bytes()), dtype=np.uint8)
    assert lib.pbg_muon_plan(2, p(ints(0, 64)), p(ints(8, 0)), p(ints(8, 4)), p(adjust), p(desc), p(words)) == -1
    assert lib.pbg_muon_plan(2, p(ints(0, 64)), p(ints(8, 70)), p(ints(8, 4)), p(adjust), p(desc), p(words)) == 0
    assert words[0] > 0 and words[2] == 0 and words[7] == 2  # no general matrix; two blocks of teams
