"""Refusals of the operators and options behind decoding with drafted tokens that
need no GPU."""
from types import SimpleNamespace

import pytest
import torch


def choice(vocab=9, **options):
    from cacheblend.generate import _Choice
    lw = SimpleNamespace(device=torch.device("cpu"), model=SimpleNamespace(config=SimpleNamespace(vocab_size=vocab)))
    options = {**dict(repetition_penalty=1.0, presence_penalty=0.0, frequency_penalty=0.0, logit_bias=None,
                      allowed_tokens=None), **options}
    return _Choice(lw, [], 4, **options, status=None)


def test_a_vocabulary_with_nothing_allowed_is_refused():
    allowed = torch.zeros((9,), dtype=torch.bool)
    with pytest.raises(ValueError):
        choice(allowed_tokens=allowed)
    allowed[8] = True
    assert choice(allowed_tokens=allowed).mask.tolist() == [256]
