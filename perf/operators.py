"""Workloads of the operators behind decoding with drafted tokens.

Three operators run, in this order, each time a model checks drafted tokens
against a cache:

  write   per-head RMSNorm of Q and K, rotation to each token's position, K and V
          into their cache rows (``ops.norm_rope_scatter``);
  attend  attention of a tree of drafted tokens over the cache rows before them
          and, in the tree, over their ancestors (``ops.tree_attn``);
  choose  penalties for repeated tokens, bias and grammar mask on the logits rows,
          and the token each row chooses (``ops.process_logits``).

``run`` computes a case in elementary torch operations in 32 bits, or, where
``own`` is true, with the package's kernels; ``exact`` computes it in 64 bits.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@functools.cache
def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cacheblend-hf-v7_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from cacheblend import ops
    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _write(name, n, q_heads, kv_heads, dim, rotary, dtype, norm=True, interleaved=False, order="run"):
    return {"name": name, "op": "write", "n": n, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "dtype": dtype, "norm": norm, "interleaved": interleaved, "order": order}


def _attend(name, nodes, context, q_heads, kv_heads, dim, dtype):
    return {"name": name, "op": "attend", "nodes": nodes, "context": context, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def _choose(name, rows, vocab, history, dtype, out, shared=True, tree=False, bias=False, mask=False,
            repetition=1.1, presence=0.25, frequency=0.125):
    return {"name": name, "op": "choose", "rows": rows, "vocab": vocab, "history": history, "dtype": dtype,
            "out": out, "shared": shared, "tree": tree, "bias": bias, "mask": mask, "repetition": repetition,
            "presence": presence, "frequency": frequency}


def listed():
    return [
        # one decoded token of a 7B model: a launch's latency
        _write("write 1 token", 1, 32, 8, 128, 128, "bf16"),
        # a tree of drafted tokens, pairs interleaved, half of each head rotated
        _write("write 63 drafted", 63, 32, 8, 128, 64, "f16", interleaved=True, order="tree"),
        # a whole prompt: bound by memory
        _write("write 32768 prompt", 32768, 32, 8, 128, 128, "bf16"),
        # plain decoding: one token after a 6K blend
        _attend("attend 1 over 6208", 1, 6208, 32, 8, 128, "bf16"),
        # a small draft after a 6K blend
        _attend("attend 16 over 6208", 16, 6208, 32, 8, 128, "bf16"),
        # a small model with narrow heads, an odd tree and a context that ends inside a tile
        _attend("attend 37 over 1029", 37, 1029, 4, 2, 64, "f16"),
        # a wide draft over a long prompt: as much arithmetic as memory
        _attend("attend 64 over 32768", 64, 32768, 32, 8, 128, "bf16"),
        # a draft over the longest prompt: bound by reading the cache
        _attend("attend 24 over 131072", 24, 131072, 32, 8, 128, "bf16"),
        # one decoded token with a repetition penalty over the whole prompt
        _choose("choose 1 of 32000", 1, 32000, 6208, "bf16", "f32"),
        # an odd vocabulary, per-row histories of other requests, half precision kept
        _choose("choose 5 of 32003", 5, 32003, 777, "f16", "f16", shared=False, bias=True),
        # every node of a small draft, each with its own path as history, under a grammar
        _choose("choose 16 of 128256", 16, 128256, 6208, "bf16", "f32", tree=True, mask=True),
        # a wide draft over a long prompt: bound by memory
        _choose("choose 64 of 128256", 64, 128256, 32768, "bf16", "bf16", tree=True, bias=True, mask=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "attend", "choose"])
    if op == "write":
        dim = rng.choice([64, 96, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        q_heads = kv_heads * rng.choice([1, 2, 4, 7])
        n = _log_int(rng, 1, max(1, 32768 * 48 * 128 // ((q_heads + 2 * kv_heads) * dim * 2)))
        c = _write("", n, q_heads, kv_heads, dim, rng.choice([dim, dim // 2]), rng.choice(["bf16", "f16"]),
                   rng.random() < 0.7, rng.random() < 0.5,
                   rng.choice(["run", "tree", "scattered"] if n <= 1024 else ["run", "scattered"]))
    elif op == "attend":
        kv_heads = rng.choice([1, 2, 4, 8])
        q_heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
        nodes = _log_int(rng, 1, max(1, min(256, 1536 // q_heads)))
        c = _attend("", nodes, _log_int(rng, 1, 65536) - 1, q_heads, kv_heads, rng.choice([64, 128, 128]),
                    rng.choice(["bf16", "bf16", "f16"]))
    else:
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        tree = rng.random() < 0.5
        c = _choose("", _log_int(rng, 1, 48), rng.choice([2000, 32000, 32000 + rng.randrange(1000), 128256]),
                    _log_int(rng, 1, 16384), dtype, rng.choice([dtype, "f32"]), tree or rng.random() < 0.5, tree,
                    rng.random() < 0.5, rng.random() < 0.5, rng.choice([1.0, 1.1, 1.3]),
                    rng.choice([0.0, 0.25, 0.5]), rng.choice([0.0, 0.125, 0.3]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generators(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    return g, h


def _parents(n, h):
    """A random tree: node 0 is the root, each other node hangs off an earlier
    one, mostly off a recent one (chains with some branches)."""
    back = (torch.rand(n, generator=h) ** 2 * 6).long() + 1
    return [-1] + [max(0, i - int(back[i])) for i in range(1, n)]


def _tree(n, h):
    """Bit words (n, ceil(n/32)) int32 of each node's visible nodes: itself and
    its ancestors."""
    width = (n + 31) // 32
    masks = []
    for i, p in enumerate(_parents(n, h)):
        masks.append((masks[p] if p >= 0 else 0) | (1 << i))
    words = torch.tensor([[(m >> (32 * w)) & 0xFFFFFFFF for w in range(width)] for m in masks], dtype=torch.int64)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).cuda()


def _depths(n, h):
    depth = []
    for p in _parents(n, h):
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return torch.tensor(depth, dtype=torch.int64)


def _rope_table(n_pos, rotary, g):
    inv = 1.0 / (1e6 ** (torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary))
    angle = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def prepare(case, seed):
    g, h = _generators(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "write":
        n, hq, hk, d = case["n"], case["q_heads"], case["kv_heads"], case["dim"]
        context = 100 + seed % 50
        qkv = randn(n, (hq + 2 * hk) * d, scale=2.0)          # one stacked projection's output
        s["q"], s["k"], s["v"] = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
        cap = n + 182
        if case["order"] == "scattered":                      # a selection of a prompt's tokens
            cap = 2 * n + 150
            rows = torch.randperm(cap, generator=h)[:n].sort().values
            pos = rows
        elif case["order"] == "tree":                         # siblings share a position, not a row
            rows = context + torch.arange(n)
            pos = context + _depths(n, h)
        else:
            rows = context + torch.arange(n)
            pos = rows
        s["rows"], s["positions"] = rows.cuda(), pos.cuda()
        s["rope"] = _rope_table(cap, case["rotary"], g)
        s["k_cache"], s["v_cache"] = randn(cap, hk * d), randn(cap, hk * d)
        s["q_weight"] = (1 + 0.2 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
        s["k_weight"] = (1 + 0.2 * randn(d, dtype=torch.float32)).to(dt) if case["norm"] else None
    elif case["op"] == "attend":
        n, context, hq, hk, d = case["nodes"], case["context"], case["q_heads"], case["kv_heads"], case["dim"]
        cap = context + n + 64                                # rows after the tree hold rejected drafts
        s["q"] = randn(n, hq * d, scale=1.5)
        s["k_cache"], s["v_cache"] = randn(cap, hk * d), randn(cap, hk * d)
        s["n_ctx"] = torch.tensor([context], dtype=torch.int64, device="cuda")
        s["words"] = _tree(n, h)
    else:
        r, vocab, length = case["rows"], case["vocab"], case["history"]
        s["logits"] = randn(r, vocab, scale=2.5)
        sets = 1 if case["shared"] else r
        u = torch.rand((sets, length), generator=g, device="cuda", dtype=torch.float64)
        s["history"] = (u ** 3 * vocab).long().clamp_(max=vocab - 1)       # a few frequent tokens, many rare
        # the likely tokens are among the repeated ones
        top = s["logits"][:sets].float().topk(4, dim=1).indices
        k = min(4, length)
        s["history"][:, :k] = top[:, :k]
        s["lengths"] = torch.randint((length + 1) // 2, length + 1, (sets,), generator=g, device="cuda")
        s["n_prompt"] = s["lengths"] // 3
        if case["tree"]:
            s["tree_words"] = _tree(r, h)
            s["tree_tokens"] = s["logits"].float().topk(2, dim=1).indices[:, 1].contiguous()
        if case["bias"]:
            s["bias"] = randn(vocab, scale=0.5, dtype=torch.float32)
        if case["mask"]:
            allowed = torch.randint(-2 ** 31, 2 ** 31, (2, r, (vocab + 31) // 32), generator=g, device="cuda")
            s["mask"] = (allowed[0] | allowed[1]).to(torch.int32)          # three tokens in four allowed
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        return {"write": _run_write, "attend": _run_attend, "choose": _run_choose}[c["op"]](s, c)
    return {"write": _plain_write, "attend": _plain_attend, "choose": _plain_choose}[c["op"]](s, c)


def _run_write(s, c):
    q = _ops().norm_rope_scatter(s["q"], s["k"], s["v"], s["positions"], s["rows"], c["q_heads"], c["kv_heads"],
                                 c["dim"], s["rope"], s["k_cache"], s["v_cache"], q_weight=s["q_weight"],
                                 k_weight=s["k_weight"], eps=1e-6, interleaved=c["interleaved"], mode="fp32")
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_attend(s, c):
    return _ops().tree_attn(s["q"], s["k_cache"], s["v_cache"], s["n_ctx"], s["words"], c["q_heads"],
                            c["kv_heads"], c["dim"], c["dim"] ** -0.5)


def _run_choose(s, c):
    out, tokens = _ops().process_logits(
        s["logits"], history=s["history"], lengths=s["lengths"], n_prompt=s["n_prompt"],
        repetition=c["repetition"], presence=c["presence"], frequency=c["frequency"], bias=s.get("bias"),
        mask_words=s.get("mask"), tree_tokens=s.get("tree_tokens"), tree_words=s.get("tree_words"),
        out_dtype=DTYPES[c["out"]])
    return {"logits": out, "tokens": tokens}


# -- the same in elementary operations, in 32 bits ---------------------------
def _bits(words, n):
    """Truth values (rows, n) of bit words (rows, ceil(n / 32))."""
    at = torch.arange(n, device=words.device)
    return ((words[:, at // 32] >> (at % 32)) & 1).bool()


def _plain_write(s, c):
    n, d, rotary = c["n"], c["dim"], c["rotary"]
    table = s["rope"][s["positions"]][:, None]                 # (n, 1, rotary / 2, 2)
    cos, sin = table[..., 0], table[..., 1]

    def head_rows(x, heads, weight):
        x = x.float().reshape(n, heads, d)
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        turned, rest = x[..., :rotary], x[..., rotary:]
        if c["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, rest], -1).reshape(n, heads * d)

    q = head_rows(s["q"], c["q_heads"], s["q_weight"]).to(s["q"].dtype)
    s["k_cache"][s["rows"]] = head_rows(s["k"], c["kv_heads"], s["k_weight"]).to(s["k"].dtype)
    s["v_cache"][s["rows"]] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s, c):
    n, context, hq, hk, d = c["nodes"], c["context"], c["q_heads"], c["kv_heads"], c["dim"]
    g = hq // hk
    k = s["k_cache"][:context + n].float().reshape(-1, hk, d).permute(1, 2, 0)
    v = s["v_cache"][:context + n].float().reshape(-1, hk, d).transpose(0, 1)
    q = s["q"].float().reshape(n, hk, g, d).permute(1, 2, 0, 3).reshape(hk, g * n, d)
    score = (q @ k) * d ** -0.5                                # (hk, g n, context + n)
    hidden = ~_bits(s["words"], n)
    score.view(hk, g, n, context + n)[..., context:].masked_fill_(hidden, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.reshape(hk, g, n, d).permute(2, 0, 1, 3).reshape(n, hq * d).to(s["q"].dtype)


def _plain_choose(s, c):
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(s["history"].shape[1], device=x.device)
    valid = at < s["lengths"][:, None]
    made = valid & (at >= s["n_prompt"][:, None])
    zeros = x.new_zeros((s["history"].shape[0], vocab))
    count = zeros.scatter_add(1, s["history"], made.float())
    seen = zeros.scatter_add(1, s["history"], valid.float())
    if c["tree"]:
        path = _bits(s["tree_words"], rows).float()
        own_path = torch.zeros_like(x).scatter_add_(1, s["tree_tokens"].expand(rows, rows), path)
        count, seen = count + own_path, seen + own_path
    repetition = torch.full((), c["repetition"], device=x.device)
    x = torch.where(seen > 0, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - c["frequency"] * count
    x = x - c["presence"] * (count > 0).float()
    if c["bias"]:
        x = x + s["bias"]
    if c["mask"]:
        x = x.masked_fill(~_bits(s["mask"], vocab), -math.inf)
    return {"logits": x.to(DTYPES[c["out"]]), "tokens": x.argmax(-1)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(c):
    if c["op"] == "write":
        heads = c["q_heads"] + 2 * c["kv_heads"]
        table = c["n"] * c["rotary"] * 4
        flops = c["n"] * (c["q_heads"] + c["kv_heads"]) * (3 * c["rotary"] + (4 * c["dim"] if c["norm"] else 0))
        return {"bytes": 2 * c["n"] * heads * c["dim"] * 2 + table + 16 * c["n"], "flops": flops}
    if c["op"] == "attend":
        keys = c["context"] + c["nodes"]
        rows = 2 * c["nodes"] * c["q_heads"] + 2 * keys * c["kv_heads"]
        return {"bytes": rows * c["dim"] * 2 + c["nodes"] * ((c["nodes"] + 31) // 32) * 4,
                "flops": 4 * c["nodes"] * c["q_heads"] * c["dim"] * (c["context"] + (c["nodes"] + 1) / 2)}
    size = {"bf16": 2, "f16": 2, "f32": 4}
    cells = c["rows"] * c["vocab"]
    history = (1 if c["shared"] else c["rows"]) * c["history"] * 8 * 3 // 4      # lengths are uniform over the upper half
    extra = (4 * c["vocab"] if c["bias"] else 0) + (cells // 8 if c["mask"] else 0)
    return {"bytes": cells * (size[c["dtype"]] + size[c["out"]]) + history + extra, "flops": cells}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "attend": _exact_attend, "choose": _exact_choose}[case["op"]](s, case)


def _exact_write(s, c):
    """Each rotated pair as a complex number times exp(i angle)."""
    d, rotary = c["dim"], c["rotary"]
    turn = torch.view_as_complex(s["rope"].double())[s["positions"]]          # (n, rotary / 2)
    i = torch.arange(rotary // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rotary // 2)

    def heads(x, weight):
        y = x.double().unflatten(1, (-1, d)).clone()
        if weight is not None:
            y = weight.double() * y / (y.pow(2).sum(2, keepdim=True) / d + 1e-6).sqrt()
        z = torch.complex(y[:, :, first], y[:, :, second]) * turn[:, None]
        y[:, :, first], y[:, :, second] = z.real, z.imag
        return y.flatten(1)

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k_cache.index_copy_(0, s["rows"], heads(s["k"], s["k_weight"]))
    v_cache.index_copy_(0, s["rows"], s["v"].double())
    return {"q": heads(s["q"], s["q_weight"]), "k_cache": k_cache, "v_cache": v_cache}


def _exact_attend(s, c):
    """Head by head, through the logarithm of each row's sum of exponentials."""
    n, context, d = c["nodes"], c["context"], c["dim"]
    group = c["q_heads"] // c["kv_heads"]
    j = torch.arange(n, device="cuda")
    sees = torch.ones((n, context + n), dtype=torch.bool, device="cuda")
    sees[:, context:] = (s["words"].long()[:, j // 32] & (1 << (j % 32))) != 0
    out = []
    for head in range(c["q_heads"]):
        at = slice(head // group * d, (head // group + 1) * d)
        k, v = s["k_cache"][:context + n, at].double(), s["v_cache"][:context + n, at].double()
        score = torch.where(sees, s["q"][:, head * d:(head + 1) * d].double() @ k.T / math.sqrt(d), -math.inf)
        out.append((score - score.logsumexp(1, keepdim=True)).exp() @ v)
    return torch.cat(out, 1)


def _exact_choose(s, c):
    """Row by row, from the tokens' own counts."""
    out = []
    for r in range(c["rows"]):
        h = 0 if c["shared"] else r
        length, prompt = int(s["lengths"][h]), int(s["n_prompt"][h])
        made = s["history"][h, prompt:length]
        if c["tree"]:
            j = torch.arange(c["rows"], device="cuda")
            on_path = (s["tree_words"][r].long()[j // 32] & (1 << (j % 32))) != 0
            made = torch.cat([made, s["tree_tokens"][on_path]])
        x = s["logits"][r].double().clone()
        every = torch.cat([s["history"][h, :prompt], made]).unique()
        x[every] = torch.where(x[every] > 0, x[every] / c["repetition"], x[every] * c["repetition"])
        ids, times = made.unique(return_counts=True)
        x[ids] -= c["frequency"] * times + c["presence"]
        if c["bias"]:
            x += s["bias"].double()
        if c["mask"]:
            j = torch.arange(c["vocab"], device="cuda")
            x[(s["mask"][r].long()[j // 32] & (1 << (j % 32))) == 0] = -math.inf
        out.append(x)
    return {"logits": torch.stack(out), "tokens": None}
