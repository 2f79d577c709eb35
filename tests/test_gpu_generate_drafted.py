"""Decode with drafted tokens and with penalties over the blended cache: held to
the HF decode of the same tokens (as ``test_gpu_generate`` holds the plain
decode), to generate_greedy, and to themselves under a captured step."""
import pytest
import torch

import drafted_ref as ref
from test_gpu_fusor import _setup

pytestmark = pytest.mark.gpu

CFG128 = dict(vocab_size=2000, hidden_size=1024, intermediate_size=2048, num_hidden_layers=4, num_attention_heads=8,
              num_key_value_heads=2, head_dim=128, rope_theta=1e6, rms_norm_eps=1e-5, max_position_embeddings=8192,
              sliding_window=None)


def reference_rows(cb, lw, model, chunks, store, tokens, ratio, ck):
    """Logits rows of the HF decode over the blended cache, fed the given tokens."""
    with torch.inference_mode():
        out = cb.fuse_selective(lw, chunks, store, recompute_ratio=ratio, check_layer=ck, return_layerwise_output=True)
        cache, rows = out.past_key_values, [out.logits[0, -1]]
        for t in tokens[:-1]:
            step = model(input_ids=torch.tensor([[t]], device=lw.device), past_key_values=cache, use_cache=True)
            cache = step.past_key_values
            rows.append(step.logits[0, -1])
    return rows


def check(cb, lw, model, chunks, store, tokens, rows, ratio=0.15, ck=1, repetition=1.0, presence=0.0, frequency=0.0,
          bias=None, allowed=None):
    """Every row within the mixed-shape bound of the HF row with the same
    processing (in fp32), scaled by what the penalties scale it by; the choice
    the same wherever the reference's two best are further apart than that."""
    prompt = torch.tensor([t for c in chunks for t in c.token_ids])
    bound = 5e-2 * max(1.0, repetition, 1.0 / repetition)
    for i, (ours, hf) in enumerate(zip(rows, reference_rows(cb, lw, model, chunks, store, tokens, ratio, ck))):
        history = torch.cat([prompt, torch.tensor(tokens[:i], dtype=torch.int64)])
        exp, _ = ref.logits(hf.view(1, -1), history=history, n_prompt=torch.tensor([len(prompt)]),
                            repetition=repetition, presence=presence, frequency=frequency, bias=bias,
                            mask=None if allowed is None else cb.ops.mask_words(allowed))
        exp, got = exp[0], ours.float().cpu()
        ok = torch.isfinite(exp)
        assert torch.equal(ok, torch.isfinite(got))
        # half a step of the row's own 16-bit rounding beside the bound on the logits themselves
        diff = (got[ok] - exp[ok]).abs() - exp[ok].abs() * ref.EPS[torch.bfloat16]
        assert diff.max().item() < bound, (i, diff.max().item())
        top = torch.topk(exp, 2).values
        if (top[0] - top[1]).item() > 2 * bound:
            assert tokens[i] == int(exp.argmax()), i


def test_drafted_decode_mock_config():
    cb, lw, model, chunks, store = _setup()
    tokens, rows, steps = cb.generate_drafted(lw, chunks, store, 12, return_logits=True, return_steps=True)
    assert len(tokens) == len(rows) == 12 and 1 <= steps <= 12
    check(cb, lw, model, chunks, store, tokens, rows)


def test_drafted_decode_head_dim_128_gqa4():
    cb, lw, model, chunks, store = _setup(CFG128, n_chunks=6, chunk_len=300, q_len=40, seed=3)
    tokens, rows = cb.generate_drafted(lw, chunks, store, 9, recompute_ratio=0.2, check_layer=2, return_logits=True,
                                       max_nodes=40)
    check(cb, lw, model, chunks, store, tokens, rows, 0.2, 2)


def oracle_draft(answer, prompt_len, wrong):
    """Drafts the answer's own continuation, with wrong siblings before each right node."""
    def draft(ids, n):
        tokens, parents, node = [], [], -1
        for t in answer[len(ids) - prompt_len:]:
            for w in wrong:
                if w != t and len(tokens) < n:
                    tokens.append(w)
                    parents.append(node)
            if len(tokens) == n:
                break
            tokens.append(t)
            parents.append(node)
            node = len(tokens) - 1
        return tokens, parents
    return draft


@pytest.mark.parametrize("use_graph", [True, False])
def test_good_drafts_take_fewer_steps_and_change_nothing(use_graph):
    """A draft that knows the answer (with wrong branches to reject) is accepted;
    accepted rows are moved together in the cache, so later tokens still agree."""
    cb, lw, model, chunks, store = _setup(CFG128, n_chunks=5, chunk_len=200, q_len=40, seed=5)
    base, _, n0 = cb.generate_drafted(lw, chunks, store, 20, max_nodes=1, return_logits=True, return_steps=True,
                                      use_graph=use_graph)
    assert n0 == 20
    n = sum(c.length for c in chunks)
    tokens, rows, steps = cb.generate_drafted(lw, chunks, store, 20, max_nodes=16, return_logits=True,
                                              return_steps=True, use_graph=use_graph,
                                              draft=oracle_draft(base, n, [1, 7]))
    check(cb, lw, model, chunks, store, tokens, rows)
    if tokens == base:                         # (a near tie may fall the other way over 16 rows)
        assert steps <= 1 + 5                  # 19 tokens, at least 5 right nodes of 15 a step and the one after
    none, _, n2 = cb.generate_drafted(lw, chunks, store, 6, max_nodes=8, return_logits=True, return_steps=True,
                                      draft=lambda ids, k: ([], []))
    assert n2 == 6 and len(none) == 6


def test_captured_steps_equal_eager_ones():
    cb, lw, model, chunks, store = _setup()
    kw = dict(return_logits=True, repetition_penalty=1.2, presence_penalty=0.1)
    t1, r1 = cb.generate_drafted(lw, chunks, store, 10, use_graph=True, **kw)
    t2, r2 = cb.generate_drafted(lw, chunks, store, 10, use_graph=False, **kw)
    assert t1 == t2 and all(torch.equal(a, b) for a, b in zip(r1, r2))


@pytest.mark.parametrize("drafted", [False, True])
def test_decode_with_penalties_bias_and_allowed_tokens(drafted):
    cb, lw, model, chunks, store = _setup(CFG128, n_chunks=5, chunk_len=200, q_len=40, seed=7)
    vocab = CFG128["vocab_size"]
    g = torch.Generator().manual_seed(2)
    bias = torch.randn((vocab,), generator=g) * 0.3
    allowed = torch.rand((vocab,), generator=g) < 0.5
    run = cb.generate_drafted if drafted else cb.generate_greedy
    tokens, rows = run(lw, chunks, store, 8, return_logits=True, repetition_penalty=1.3, presence_penalty=0.2,
                       frequency_penalty=0.1, logit_bias=bias, allowed_tokens=allowed)
    assert all(bool(allowed[t]) for t in tokens)
    check(cb, lw, model, chunks, store, tokens, rows, repetition=1.3, presence=0.2, frequency=0.1, bias=bias,
          allowed=allowed)
    # one token alone allowed: it is chosen every time, whatever the penalties
    only = torch.zeros((vocab,), dtype=torch.bool)
    only[77] = True
    assert run(lw, chunks, store, 4, allowed_tokens=only, frequency_penalty=0.5) == [77] * 4


def test_shortcut_path_eos_and_refusals():
    cb, lw, model, chunks, store = _setup()
    plain = cb.generate_greedy(lw, chunks, store, 4, recompute_ratio=1.0)
    assert cb.generate_drafted(lw, chunks, store, 4, recompute_ratio=1.0) == plain
    only = torch.zeros((model.config.vocab_size,), dtype=torch.bool)
    only[5] = True
    for run in (cb.generate_greedy, cb.generate_drafted):
        assert run(lw, chunks, store, 3, recompute_ratio=1.0, allowed_tokens=only) == [5, 5, 5]
        assert run(lw, chunks, store, 3, allowed_tokens=only, eos_token_id=5) == [5]
        assert run(lw, chunks, store, 0) == []
        for bad in (dict(repetition_penalty=0.0), dict(logit_bias=torch.zeros(3)), dict(allowed_tokens=only[:9]),
                    dict(allowed_tokens=only.int())):
            with pytest.raises(ValueError):
                run(lw, chunks, store, 3, **bad)
    first = cb.generate_drafted(lw, chunks, store, 1)
    assert cb.generate_drafted(lw, chunks, store, 5, eos_token_id=first[0]) == first
    for bad in (dict(max_nodes=0), dict(max_nodes=2000), dict(draft=lambda ids, n: ([1], [0])),
                dict(draft=lambda ids, n: ([1 << 40], [-1])), dict(draft=lambda ids, n: ([-1], [-1])),
                dict(draft=lambda ids, n: ([1] * (n + 1), [-1] * (n + 1))), dict(draft=lambda ids, n: ([1], []))):
        with pytest.raises(ValueError):
            cb.generate_drafted(lw, chunks, store, 3, **bad)
