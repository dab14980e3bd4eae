"""Kernels' error words among the device-side checks, on CPU tensors in the words' place."""

import pytest
import torch


def test_watched_words_are_reported_and_reset(monkeypatch):
    from pbg_b200 import checks

    words = {}
    monkeypatch.setattr(checks, "_WATCHED", [])
    checks.watch(words, {1: "first", 6: "second"})
    device = torch.device("cuda", 3)
    assert checks.input_errors(device) == []  # no call made on the device yet
    words[3] = torch.zeros(1, dtype=torch.int32)
    words[4] = torch.ones(1, dtype=torch.int32)
    assert checks.input_errors(device) == []
    words[3].fill_(4)
    assert checks.input_errors(device, reset=False) == ["second"]
    assert checks.input_errors("cuda:3") == ["second"] and int(words[3]) == 0
    words[3].fill_(3)
    with pytest.raises(ValueError, match="first; second"):
        checks.raise_input_errors(device)
    assert checks.input_errors(device) == [] and int(words[4]) == 1
    assert checks.input_errors("cpu") == []


def test_the_embedding_and_optimizer_words_are_watched():
    from pbg_b200 import checks, embedding, optim

    watched = [id(words) for words, _ in checks._WATCHED]
    assert id(embedding._ERROR) in watched and id(optim._ERROR) in watched
