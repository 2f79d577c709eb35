"""Decode over the blended cache at its edges: how keys are rotated, a model
without a vocabulary size in its configuration, ends inside an accepted path, and
how many steps run."""
import pytest
import torch

import drafted_ref as ref
from test_gpu_fusor import _setup
from test_gpu_generate_drafted import CFG128, oracle_draft

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafted", [False, True])
def test_decode_rotates_in_the_mode_asked_for(drafted, monkeypatch):
    """rope_mode "fp32": the K row of every decoded token is within one rounding of
    the rotation, as the prompt's are ("ref" rounds cos, sin and each product)."""
    cb, lw, model, chunks, store = _setup(CFG128, n_chunks=4, chunk_len=100, q_len=20, seed=4)
    name = "norm_rope_scatter" if drafted else "rope_scatter"
    plain, rows_seen = getattr(cb.ops, name), []

    def spy(q, k, v, pos, *args, **kw):
        out = plain(q, k, v, pos, *args, **kw)
        if q.shape[0] <= 8:                                   # a decode step, not the prefill
            if drafted:
                rows, hq, hkv, d, rope, kc, _ = args
            else:
                rows, (_, _, hq, hkv, d, rope, kc, _) = pos, args
            on = rows >= 0
            z, mag = ref.norm_rope(k[on], hkv, d, None, 0.0, rope, pos[on], False)
            bound = ref.norm_rope_bound(z, mag, k.dtype, "fp32")
            rows_seen.append(bool(((kc[rows[on]].double() - z).abs() <= bound).all()))
        return out

    monkeypatch.setattr(cb.ops, name, spy)
    run = cb.generate_drafted if drafted else cb.generate_greedy
    kw = dict(max_nodes=8) if drafted else {}
    run(lw, chunks, store, 5, rope_mode="fp32", use_graph=False, **kw)
    assert len(rows_seen) >= lw.num_layers and all(rows_seen)
    rows_seen.clear()
    run(lw, chunks, store, 5, use_graph=False, **kw)          # the default differs, or this test shows nothing
    assert rows_seen and not all(rows_seen)


class BareConfig:
    """A model configuration without vocab_size (as of a model around a language model)."""

    def __init__(self, config):
        self.__dict__["_config"] = config

    def __getattr__(self, name):
        if name == "vocab_size":
            raise AttributeError(name)
        return getattr(self._config, name)


def test_decode_without_a_vocabulary_size(monkeypatch):
    cb, lw, model, chunks, store = _setup()
    vocab = model.config.vocab_size
    base = [run(lw, chunks, store, 5) for run in (cb.generate_greedy, cb.generate_drafted)]
    only = torch.zeros((vocab,), dtype=torch.bool)
    only[5] = True
    monkeypatch.setattr(model, "config", BareConfig(model.config))
    assert [run(lw, chunks, store, 5) for run in (cb.generate_greedy, cb.generate_drafted)] == base
    for run in (cb.generate_greedy, cb.generate_drafted):     # the head's rows are the vocabulary
        assert run(lw, chunks, store, 3, allowed_tokens=only) == [5, 5, 5]
        with pytest.raises(ValueError):
            run(lw, chunks, store, 3, logit_bias=torch.zeros(3))
    with pytest.raises(ValueError):
        cb.generate_drafted(lw, chunks, store, 3, draft=lambda ids, n: ([vocab], [-1]))


def test_every_step_runs_once(monkeypatch):
    """A run of k decoder steps after the prefill: the first eagerly, the others as
    k - 1 replays of its capture; none is run again for its result."""
    cb, lw, model, chunks, store = _setup()
    replays = []
    replay = torch.cuda.CUDAGraph.replay
    monkeypatch.setattr(torch.cuda.CUDAGraph, "replay", lambda g: (replays.append(g), replay(g))[1])
    for length in (2, 3, 6):
        replays.clear()
        none = lambda ids, k: ([], [])
        tokens, rows, steps = cb.generate_drafted(lw, chunks, store, length, draft=none, return_logits=True,
                                                  return_steps=True)
        assert len(tokens) == len(rows) == length == steps and len(replays) == length - 2
        eager, eager_rows = cb.generate_drafted(lw, chunks, store, length, draft=none, return_logits=True,
                                                use_graph=False)
        assert tokens == eager and all(torch.equal(a, b) for a, b in zip(rows, eager_rows))


def test_draft_parents_outside_the_tree_are_refused():
    cb, lw, model, chunks, store = _setup()
    for below in ([-2], [1], [-1, -2], [-1, 1]):
        with pytest.raises(ValueError):
            cb.generate_drafted(lw, chunks, store, 3, draft=lambda ids, n: ([4] * len(below), below))


def forced(vocab, n, first=100):
    """(tokens, options) such that every decode chooses these n tokens in turn: biases
    100 apart, far above any logit, and a presence penalty that takes a token out once
    it is made."""
    tokens = [first + 3 * i for i in range(n)]
    bias = torch.zeros((vocab,))
    bias[tokens] = 4000.0 + 100.0 * n - 100.0 * torch.arange(n)
    return tokens, dict(logit_bias=bias, presence_penalty=20000.0)


@pytest.mark.parametrize("use_graph", [True, False])
def test_ends_inside_an_accepted_path(use_graph):
    """15 drafted nodes with two wrong siblings before each right one are 5 right
    nodes, so a step gives 6 tokens: ends by count and by EOS at each place of a path."""
    cb, lw, model, chunks, store = _setup(CFG128, n_chunks=4, chunk_len=100, q_len=20, seed=6)
    answer, options = forced(CFG128["vocab_size"], 24)
    n = sum(c.length for c in chunks)
    kw = dict(return_logits=True, return_steps=True, use_graph=use_graph, max_nodes=16,
              draft=oracle_draft(answer, n, [1, 7]), **options)
    for length in (1, 2, 6, 7, 8, 10, 13, 14, 20):
        tokens, rows, steps = cb.generate_drafted(lw, chunks, store, length, **kw)
        assert tokens == answer[:length] and steps == 1 + (length - 1 + 5) // 6
        assert [int(r.argmax()) for r in rows] == tokens
    for at in (0, 1, 3, 6, 7, 9, 12, 17):
        tokens, rows, steps = cb.generate_drafted(lw, chunks, store, 20, eos_token_id=answer[at], **kw)
        assert tokens == answer[:at + 1] and steps == 1 + (at + 5) // 6
        assert [int(r.argmax()) for r in rows] == tokens
    assert cb.generate_greedy(lw, chunks, store, 20, eos_token_id=answer[9], **options) == answer[:10]
