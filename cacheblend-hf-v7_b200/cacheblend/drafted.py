"""Greedy decode over the blended cache that checks a tree of drafted tokens per
step (no counterpart in cacheblend-hf-v7, whose decode loop, ``runners.py:106-152``,
takes one token at a time).

A RAG answer copies much of its chunks, so the continuation of an earlier
occurrence of the last few tokens is a good guess.  A step runs the decoder once
for the last chosen token (the tree's root) and the drafted tokens under it:
``norm_rope_scatter`` rotates every node to its depth's position and writes its
K/V into a cache row of its own, ``tree_attn`` attends over the cache and each
node's ancestors, ``process_logits`` (with each node's own path as history)
chooses a token after every node.  From the root on, a child that holds the token
its parent chose is accepted; the accepted nodes' cache rows move together, the
rest are overwritten by the next step.  A step yields one token at least, so the
result is the greedy decode's, in fewer steps.
"""
from __future__ import annotations

from typing import Callable, Sequence

import numpy as np
import torch

from cacheblend import ops
from cacheblend.chunker import Chunk
from cacheblend.fusor import _fused_w, _mlp, _norm, _qkv, _selective_prefill
from cacheblend.generate import _Choice, generate_greedy
from cacheblend.kv_store import KVStore


def prompt_lookup_tree(ids: Sequence[int], max_nodes: int, ngram: int = 3, depth: int = 10
                       ) -> tuple[list[int], list[int]]:
    """Draft by look-up in the tokens so far: (tokens, parents) of at most
    ``max_nodes`` drafted nodes, parents[i] = -1 for a continuation of ``ids``
    itself, else an earlier node.  The latest occurrences of the last ``ngram``
    tokens (then of fewer, down to one) each give up to ``depth`` tokens that
    followed them; continuations that start alike share their nodes."""
    tokens: list[int] = []
    parents: list[int] = []
    children: dict[tuple[int, int], int] = {}
    ids = np.asarray(ids, dtype=np.int64)
    n = len(ids)
    for size in range(min(ngram, n - 1), 0, -1):
        match = np.ones((n - size,), dtype=bool)            # by first token; the tail itself is not one
        for k in range(size):
            match &= ids[k:n - size + k] == ids[n - size + k]
        for start in np.flatnonzero(match)[::-1].tolist():
            if len(tokens) >= max_nodes:
                break
            node = -1
            for t in ids[start + size:start + size + depth].tolist():
                nxt = children.get((node, t))
                if nxt is None:
                    if len(tokens) >= max_nodes:
                        break
                    nxt = len(tokens)
                    children[(node, t)] = nxt
                    tokens.append(t)
                    parents.append(node)
                node = nxt
        if tokens:
            break                               # a longer match beats many short ones
    return tokens, parents


class _TreeState:
    """Static device buffers of the steps: the nodes' tokens, positions, cache rows
    and bit words, n_ctx, the attention workspace and the chosen tokens."""

    def __init__(self, lw, pre, nodes: int, keep_rows: bool):
        device, geo = lw.device, pre.geo
        self.n = nodes
        self.width = (nodes + 31) // 32
        # one pinned block, one copy a step: tokens, positions, rows, n_ctx, then the words in pairs
        self.words_at = 3 * nodes + 1
        size = self.words_at + (nodes * self.width + 1) // 2
        self.host = torch.zeros((size,), dtype=torch.int64).pin_memory()
        self.dev = torch.zeros((size,), dtype=torch.int64, device=device)
        self.token = self.dev[:nodes].view(1, nodes)
        self.pos, self.rows = self.dev[nodes:2 * nodes], self.dev[2 * nodes:3 * nodes]
        self.n_ctx = self.dev[3 * nodes:3 * nodes + 1]
        self.words = self.dev[self.words_at:].view(torch.int32)[:nodes * self.width].view(nodes, self.width)
        self.ws = ops.tree_workspace(nodes, pre.fused_k.shape[1], geo.n_q, geo.n_kv, geo.head_dim, device)
        self.chosen = torch.zeros((nodes,), dtype=torch.int64, device=device)
        self.keep_rows = keep_rows
        self.logits = None

    def load(self, n_ctx: int, tokens: list[int], parents: list[int]) -> None:
        """Nodes of the next step: the root first; unused nodes are padding (no
        cache row, context only)."""
        n, used = self.n, len(tokens)
        words, depth = ops.tree_words(parents, self.width)
        h = self.host
        h.zero_()
        h[:used] = torch.tensor(tokens, dtype=torch.int64)
        h[n:n + used] = n_ctx + depth
        h[2 * n:2 * n + used] = n_ctx + torch.arange(used)
        h[2 * n + used:3 * n] = -1
        h[3 * n] = n_ctx
        h[self.words_at:].view(torch.int32)[:used * self.width] = words.reshape(-1)
        self.dev.copy_(h, non_blocking=True)


def _tree_step(lw, pre, st: _TreeState, choice: _Choice, rope_mode: str, status) -> None:
    """The decoder over the nodes in st: their K/V into their cache rows, the token
    after each of them into st.chosen -- all on the device."""
    inner, geo = lw._inner, pre.geo
    h = inner.embed_tokens(st.token)
    m = None
    for li, layer in enumerate(inner.layers):
        attn = layer.self_attn
        w_qkv, w_gu = _fused_w(lw, li, st.n)
        hn = _norm(layer.input_layernorm, h, delta=m, sum_out=h if m is not None else None, status=status)
        q, k, v = _qkv(attn, hn, w_qkv)
        q_rot = ops.norm_rope_scatter(q[0], k[0], v[0], st.pos, st.rows, geo.n_q, geo.n_kv, geo.head_dim, pre.rope,
                                      pre.fused_k[li], pre.fused_v[li], mode=rope_mode, status=status)
        a = ops.tree_attn(q_rot, pre.fused_k[li], pre.fused_v[li], st.n_ctx, st.words, geo.n_q, geo.n_kv, geo.head_dim,
                          geo.scaling, workspace=st.ws, status=status)
        o = attn.o_proj(a.unsqueeze(0))
        m = _mlp(layer, _norm(layer.post_attention_layernorm, h, delta=o, sum_out=h, status=status), w_gu)
    logits = lw.model.lm_head(_norm(inner.norm, h, delta=m, status=status))[0]
    tree = dict(tree_tokens=st.token.view(-1), tree_words=st.words) if choice.counted else {}
    st.logits, chosen = choice(logits, st.keep_rows, **tree)
    st.chosen.copy_(chosen)


def _accept(tokens: list[int], parents: list[int], chosen: list[int]) -> list[int]:
    """Nodes from the root (node 0) on that hold the token their parent chose."""
    path = [0]
    while True:
        node = path[-1]
        for i in range(node + 1, len(tokens)):
            if parents[i] == node and tokens[i] == chosen[node]:
                path.append(i)
                break
        else:
            return path


def generate_drafted(layerwise_model, chunks: list[Chunk], kv_store: KVStore, max_new_tokens: int,
                     recompute_ratio: float = 0.15, check_layer: int = 1, eos_token_id: int | None = None,
                     rope_mode: str = "ref", status: torch.Tensor | None = None, return_logits: bool = False,
                     use_graph: bool = True, repetition_penalty: float = 1.0, presence_penalty: float = 0.0,
                     frequency_penalty: float = 0.0, logit_bias: torch.Tensor | None = None,
                     allowed_tokens: torch.Tensor | None = None, max_nodes: int = 16,
                     draft: Callable[[Sequence[int], int], tuple[list[int], list[int]]] = prompt_lookup_tree,
                     return_steps: bool = False):
    """``generate_greedy`` with a tree of drafted tokens checked per step.

    ``draft(ids, n)`` gets the tokens so far and returns at most n drafted tokens
    and their parents (-1: follows ``ids``; else an earlier drafted token);
    ``max_nodes`` (1 to 1024) counts the tree's root too.  The tokens are those of
    ``generate_greedy`` with the same options, up to the rounding of GEMMs over
    more rows.  ``return_steps`` appends the number of decoder steps to the result.
    The shortcut cases of fuse_selective run ``generate_greedy``."""
    if not 1 <= max_nodes <= 1024:
        raise ValueError(f"max_nodes must be 1 to 1024, got {max_nodes}")
    lw = layerwise_model
    options = dict(repetition_penalty=repetition_penalty, presence_penalty=presence_penalty,
                   frequency_penalty=frequency_penalty, logit_bias=logit_bias, allowed_tokens=allowed_tokens)
    if max_new_tokens <= 0 or not 0 < recompute_ratio < 1 or len(chunks) <= 1:
        out = generate_greedy(lw, chunks, kv_store, max_new_tokens, recompute_ratio, check_layer, eos_token_id,
                              rope_mode, status, return_logits, use_graph, **options)
        n = len(out[0] if return_logits else out)
        return ((*out, n) if return_logits else (out, n)) if return_steps else out
    out_rows: list[torch.Tensor] = []
    with torch.inference_mode():
        choice = _Choice(lw, chunks, max_new_tokens + max_nodes, **options, status=status)
        # the last step may check nodes past the last token asked for
        pre = _selective_prefill(lw, chunks, kv_store, recompute_ratio, check_layer, rope_mode, status, None,
                                 extra_tokens=max_new_tokens + max_nodes, logits_rows="last")
        # what a drafted token may be: it is embedded, and may be chosen
        vocab = pre.logits.shape[-1]
        vocab = min(vocab, getattr(lw._inner.embed_tokens, "num_embeddings", vocab))
        row, first = choice(pre.logits[0, -1:], return_logits)
        out = [int(first.item())]
        if return_logits:
            out_rows.append(row[0].clone())
        ids = [t for c in chunks for t in c.token_ids]
        st = _TreeState(lw, pre, max_nodes, return_logits)
        n_ctx, steps, graph = pre.S, 1, None
        while len(out) < max_new_tokens and out[-1] != eos_token_id:
            drafted, below = draft(ids + out, max_nodes - 1) if max_nodes > 1 else ([], [])
            if len(drafted) > max_nodes - 1 or len(drafted) != len(below):
                raise ValueError(f"draft returned {len(drafted)} tokens and {len(below)} parents for {max_nodes - 1} "
                                 "nodes")
            if any(p < -1 for p in below):
                raise ValueError(f"draft returned parent {min(below)} (-1 or an earlier drafted token)")
            if any(not 0 <= t < vocab for t in drafted):
                raise ValueError(f"draft returned a token outside the vocabulary of {vocab}")
            tokens, parents = [out[-1], *drafted], [-1, *(p + 1 for p in below)]
            st.load(n_ctx, tokens, parents)
            if use_graph and steps > 1 and graph is None:
                graph = _capture(lw, pre, st, choice, rope_mode, status)
            if graph is not None:
                graph.replay()
            else:
                _tree_step(lw, pre, st, choice, rope_mode, status)     # eager: first use sets up every kernel
            chosen = st.chosen.tolist()
            path = _accept(tokens, parents, chosen)
            _keep(pre, choice, n_ctx, path, tokens)
            for node in path:
                out.append(chosen[node])
                if return_logits:
                    out_rows.append(st.logits[node].clone())
                if len(out) == max_new_tokens or out[-1] == eos_token_id:
                    break
            n_ctx += len(path)
            steps += 1
        del graph
    result = (out, out_rows) if return_logits else out
    if not return_steps:
        return result
    return (*result, steps) if return_logits else (result, steps)


def _capture(lw, pre, st, choice, rope_mode, status):
    cur = torch.cuda.current_stream(lw.device)
    side = torch.cuda.Stream(device=lw.device)
    side.wait_stream(cur)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            _tree_step(lw, pre, st, choice, rope_mode, status)
    cur.wait_stream(side)
    return graph


def _keep(pre, choice: _Choice, n_ctx: int, path: list[int], tokens: list[int]) -> None:
    """The accepted nodes' K/V into the rows after the context, their tokens into
    the history."""
    device = pre.fused_k.device
    src = [i for k, i in enumerate(path) if i != k]
    if src:
        # (indices in one block; index_select copies before index_copy_ writes)
        at = torch.tensor([src, [k for k, i in enumerate(path) if i != k]], dtype=torch.int64).pin_memory()
        at = at.to(device, non_blocking=True) + n_ctx
        for cache in (pre.fused_k, pre.fused_v):
            cache.index_copy_(1, at[1], cache.index_select(1, at[0]))
    if choice.counted:
        new = torch.tensor([tokens[i] for i in path], dtype=torch.int64).pin_memory()
        choice.history[n_ctx:n_ctx + len(path)].copy_(new, non_blocking=True)
        choice.length.fill_(n_ctx + len(path))
