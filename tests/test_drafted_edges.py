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


def test_numbers_beyond_their_field_are_refused():
    """A number that its field of the argument struct cannot hold is a ValueError, as
    any other bad argument is."""
    from cacheblend import ops
    dev = torch.device("cuda:0")               # (refused before the device is looked at)
    with pytest.raises(ValueError):
        ops._tree_attn(dev, *[16] * 8, *[128, 1, 100, 1 << 40], 4, 4, 2, 64, 0, 1e39)
    with pytest.raises(ValueError):
        ops._tree_attn(dev, *[16] * 8, *[128, 1, 100, 1 << 40], 4, 1 << 31, 2, 64, 0, 0.1)
    with pytest.raises(ValueError):
        ops._process_logits(dev, *[16] * 12, *[100] * 12, 0, 0, 2, 1.1, 1e39, 0.0)
    with pytest.raises(ValueError):
        ops._norm_rope_scatter(dev, *[16] * 12, *[128] * 7, 4, 2, 64, 64, 0, 0, 1, -1e300)
