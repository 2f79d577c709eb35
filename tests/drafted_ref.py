"""64-bit (or, for the logits, step-by-step 32-bit) references of the operators
behind decoding with drafted tokens, on the CPU, and the error bounds that the
kernels are held to."""
from __future__ import annotations

import numpy as np
import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step, relative
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}            # half a subnormal step


def rope_table(n_pos: int, rotary: int, theta: float = 1e4) -> torch.Tensor:
    inv = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def norm_rope(x, heads, dim, weight, eps, table, positions, interleaved):
    """(z, mag): normalised and rotated rows of x in 64 bits, and for every element
    the sum of the magnitudes of the terms it was formed from."""
    n = x.shape[0]
    y = x.double().reshape(n, heads, dim)
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    rotary = 2 * table.shape[1]
    t = table.double()[positions]
    c, s = t[:, None, :, 0], t[:, None, :, 1]
    z, mag = y.clone(), y.abs()
    first = torch.arange(0, rotary, 2) if interleaved else torch.arange(rotary // 2)
    second = first + (1 if interleaved else rotary // 2)
    a, b = y[..., first], y[..., second]
    z[..., first], z[..., second] = a * c - b * s, b * c + a * s
    mag[..., first], mag[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return z.reshape(n, -1), mag.reshape(n, -1)


def norm_rope_bound(z, mag, dtype, mode):
    """|got - z| allowed.  fp32 mode: one rounding of the result; in fp32 the sum of
    squares takes 13 roundings (8 in a lane, 5 across lanes; half of that through
    the root), the mean and root 5, weight, scale and rotation 5 more: under
    2^-19 of the terms.  ref mode: four 16-bit roundings on each term (normalised
    value, weight, cos or sin, product) and one on the sum."""
    e = EPS[dtype]
    terms = 2.0 ** -19 * mag * (1 + e) + 8 * TINY[dtype]
    if mode == "fp32":
        return e * z.abs() + terms
    return e * z.abs() + (1 + e) * ((1 + e) ** 4 - 1) * mag + terms * (1 + e) ** 5


def visible(words, n):
    w = words.cpu().numpy().astype(np.uint32)
    j = np.arange(n)
    return torch.from_numpy(((w[:, j // 32] >> (j % 32).astype(np.uint32)) & 1).astype(bool))


def tree_attention(q, k, v, n_ctx, words, hq, hkv, dim, scale):
    """(out, A) in 64 bits: attention of every node, and the same weights applied
    to |v|; rows that see nothing are zero."""
    t = words.shape[0]
    g = hq // hkv
    n = n_ctx + t
    kk = k[:n].double().reshape(n, hkv, dim)
    vv = v[:n].double().reshape(n, hkv, dim)
    sees = torch.ones((t, n), dtype=torch.bool)
    sees[:, n_ctx:] = visible(words, t)
    out = torch.zeros((t, hq, dim), dtype=torch.float64)
    A = torch.zeros_like(out)
    for i in range(t):
        at = sees[i].nonzero()[:, 0]                # a masked row's values take no part at all
        if not len(at):
            continue
        for h in range(hq):
            s = kk[at, h // g] @ q[i].double().reshape(hq, dim)[h] * scale
            p = torch.softmax(s, 0)
            out[i, h] = p @ vv[at, h // g]
            A[i, h] = p @ vv[at, h // g].abs()
    return out.reshape(t, -1), A.reshape(t, -1)


def tree_bound(out, A, n_keys, dtype, v_max):
    """|got - out| allowed: each weight rounded to the 16-bit type (half a step of
    A), the result rounded once (half a step of |out|), and in fp32 the
    exponentials to 2^-13 (and the sums far below that).  fp16 weights under 2^-14
    are held in steps of 2^-24, off by 2^-25 each against a row sum of at least 1."""
    e = EPS[dtype]
    return (e + 2.0 ** -12) * A * (1 + e) + e * out.abs() + (n_keys * v_max + 1) * TINY[dtype]


def logits(x, history=None, lengths=None, n_prompt=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
           mask=None, tree_tokens=None, tree_words=None):
    """Row by row and step by step in fp32 (numpy rounds every operation once):
    (processed fp32 rows, chosen tokens)."""
    f = np.float32
    x = x.float().cpu().numpy().astype(f)
    rows, vocab = x.shape
    out = np.empty_like(x)
    tokens = np.empty((rows,), np.int64)

    def of(t, r):
        return None if t is None else int(t.reshape(-1)[r if t.numel() > 1 else 0])

    with np.errstate(all="ignore"):
        for r in range(rows):
            count = np.zeros((vocab,), np.int64)
            seen = np.zeros((vocab,), bool)
            if history is not None:
                h2 = history.cpu() if history.dim() == 2 else history.cpu()[None]
                h = h2[r if h2.shape[0] > 1 else 0].numpy()
                n = len(h) if lengths is None else min(max(of(lengths, r), 0), len(h))
                p = 0 if n_prompt is None else of(n_prompt, r)
                h, made = h[:n], np.arange(n) >= p
                ok = (h >= 0) & (h < vocab)
                np.add.at(count, h[ok & made], 1)
                seen[h[ok]] = True
            if tree_tokens is not None:
                on = visible(tree_words[r:r + 1], tree_tokens.numel())[0].numpy()
                t = tree_tokens.cpu().numpy()[on]
                np.add.at(count, t, 1)
            seen |= count > 0
            y = x[r].copy()
            y[seen] = np.where(y[seen] > 0, y[seen] / f(repetition), y[seen] * f(repetition))
            c = count > 0
            y[c] = (y[c] - f(frequency) * count[c].astype(f)) - f(presence)
            if bias is not None:
                b = bias.cpu().numpy()
                y = y + (b if b.ndim == 1 else b[r if b.shape[0] > 1 else 0])[:vocab]
            if mask is not None:
                m = mask if mask.dim() == 2 else mask[None]
                y[~visible(m[r if m.shape[0] > 1 else 0][None], vocab)[0].numpy()] = -np.inf
            out[r] = y
            nan = np.isnan(y)
            tokens[r] = np.argmax(nan) if nan.any() else np.argmax(y)
    return torch.from_numpy(out), torch.from_numpy(tokens)
