"""Refusals of the operators behind decoding with drafted tokens, and tree words.
CPU only."""
import numpy as np
import pytest
import torch

# the fields of the three argument structs after `size`, with values that pass every check but the one under test
NR = dict(q=16, k=16, v=16, pos=16, rows=16, qw=16, kw=16, table=16, q_out=16, kc=16, vc=16, st=0, qs=256, ks=128,
          vs=128, kvs=128, n=4, t_rows=10, cap=10, hq=4, hkv=2, d=64, r=64, il=0, dt=0, mode=1, eps=1e-6)
TA = dict(q=16, k=16, v=16, n_ctx=16, words=16, out=16, ws=256, st=0, kvs=128, ws_=1, cap=100, bytes_=1 << 40, t=4,
          hq=4, hkv=2, d=64, dt=0, scale=0.1)
PL = dict(x=16, h=16, ln=0, np_=0, bias=0, mask=0, tt=0, tw=0, out=16, tok=16, st=0, ws=16, xs=100, rows=2, vocab=100, hs=0,
          hc=5, ls=0, nps=0, bs=0, ms=0, ts=0, os=100, wb=0, nt=0, dt=0, odt=2, rep=1.1, pres=0.0, freq=0.0)


def call(name, fields, **change):
    from cacheblend import _native as N
    fmt = N.PACK["cbk_" + name]
    values = {**fields, **change}
    size = values.pop("size", fmt.size)
    rc = getattr(N.LIB, "cbk_" + name)(fmt.pack(size, *values.values()), None)
    assert N.last_error() or rc == 0
    return rc


@pytest.mark.parametrize("name,fields", [("norm_rope_scatter", NR), ("tree_attn", TA), ("process_logits", PL)])
def test_argument_struct_size_is_checked(name, fields):
    from cacheblend import _native as N
    assert call(name, fields, size=N.PACK["cbk_" + name].size - 8) == -1
    assert getattr(N.LIB, "cbk_" + name)(None, None) == -1


@pytest.mark.parametrize("change,code", [
    (dict(dt=2), -2), (dict(d=72), -2), (dict(d=272), -2), (dict(d=8), -2), (dict(r=8), -2), (dict(r=24), -2),
    (dict(r=80), -2), (dict(mode=2), -1), (dict(hq=0), -1), (dict(hkv=-1), -1), (dict(n=-1), -1), (dict(cap=-1), -1),
    (dict(q=0), -1), (dict(rows=0), -1), (dict(table=0), -1), (dict(vc=0), -1), (dict(kw=0), -1),
    (dict(qs=248), -1), (dict(ks=132), -1), (dict(kvs=64), -1), (dict(q_out=24), -1), (dict(qw=24), -1),
    (dict(n=0), 0), (dict(n=0, q=0, rows=0), 0),
])
def test_norm_rope_scatter_refusals(change, code):
    assert call("norm_rope_scatter", NR, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(dt=2), -2), (dict(d=96), -2), (dict(hq=5), -1), (dict(hkv=0), -1), (dict(t=1025), -2), (dict(t=-1), -1 - 1),
    (dict(cap=3), -1), (dict(cap=1 << 31), -1), (dict(kvs=64), -1), (dict(kvs=132), -1), (dict(ws_=0), -1),
    (dict(t=33, ws_=1), -1), (dict(q=0), -1), (dict(n_ctx=0), -1), (dict(words=0), -1), (dict(out=24), -1),
    (dict(k=24), -1), (dict(ws=16), -1), (dict(scale=0.0), -1),
    (dict(scale=-0.1), -1), (dict(scale=float("inf")), -1), (dict(scale=float("nan")), -1), (dict(bytes_=16), -4), (dict(t=0), 0),
])
def test_tree_attn_refusals(change, code):
    assert call("tree_attn", TA, **change) == code


def test_tree_attn_workspace_refusals():
    from cacheblend import _native as N, ops
    f = N.LIB.cbk_tree_attn_workspace_bytes
    assert f(16, 6240, 32, 8, 128) > 0 and f(16, 6240, 32, 8, 128) % 16 == 0
    assert f(16, 6240, 32, 8, 96) == 0 and f(16, 8, 32, 8, 128) == 0 and f(16, 6240, 32, 5, 128) == 0


@pytest.mark.parametrize("change,code", [
    (dict(dt=3), -2), (dict(odt=1), -2), (dict(dt=2, odt=0), -2), (dict(vocab=0), -2), (dict(vocab=1 << 20), -2),
    (dict(rows=-1), -1), (dict(x=0), -1), (dict(tok=0), -1), (dict(rep=0.0), -1), (dict(rep=-1.0), -1),
    (dict(rep=float("nan")), -1), (dict(rep=float("inf")), -1), (dict(pres=float("nan")), -1), (dict(xs=99), -1), (dict(os=99), -1),
    (dict(mask=16, ms=3), -1), (dict(bias=16, bs=99), -1), (dict(hc=-1), -1), (dict(nt=2), -1), (dict(nt=1025), -1),
    (dict(nt=33, tt=16, tw=16, ts=1), -1), (dict(rows=64, wb=511), -4), (dict(rows=64, ws=0, wb=512), -1),
    (dict(rows=64, ws=8, wb=512), -1), (dict(rows=0), 0),
])
def test_process_logits_refusals(change, code):
    assert call("process_logits", PL, **change) == code


def test_cpu_tensors_are_refused():
    from cacheblend import ops
    z = torch.zeros((2, 128), dtype=torch.bfloat16)
    i = torch.zeros((2,), dtype=torch.int64)
    with pytest.raises(RuntimeError):
        ops.norm_rope_scatter(z, z, z, i, i, 2, 2, 64, torch.zeros((4, 32, 2)), z, z)
    with pytest.raises(RuntimeError):
        ops.tree_attn(z, z, z, i[:1], torch.ones((2, 1), dtype=torch.int32), 2, 2, 64, 0.1)
    with pytest.raises(RuntimeError):
        ops.process_logits(z)


def test_tree_words():
    from cacheblend import ops
    #      0
    #    1   2        a second root: 5
    #   3     4
    words, depth = ops.tree_words([-1, 0, 0, 1, 2, -1])
    assert words.dtype == torch.int32 and words.tolist() == [[1], [3], [5], [11], [21], [32]]
    assert depth.tolist() == [0, 1, 1, 2, 2, 0]
    words, depth = ops.tree_words(list(range(-1, 69)))            # a chain over three words
    assert words.shape == (70, 3) and depth.tolist() == list(range(70))
    assert words[69].tolist() == [-1, -1, 63] and words[31].tolist() == [-1, 0, 0] and words[0].tolist() == [1, 0, 0]
    assert ops.tree_words([-1], width=4)[0].tolist() == [[1, 0, 0, 0]]
    assert ops.tree_words([])[0].shape == (0, 1)
    for bad in ([0], [-1, 1], [-1, 2, 0], [-2]):
        with pytest.raises(ValueError):
            ops.tree_words(bad)
    with pytest.raises(ValueError):
        ops.tree_words([-1] * 33, width=1)


def test_reference_bounds_catch_mistakes():
    """The references themselves: a rotation with the wrong sign, a key too many
    and a count too few each leave the bounds."""
    import drafted_ref as ref
    g = torch.Generator().manual_seed(1)
    x = torch.randn((5, 2 * 64), generator=g).to(torch.bfloat16)
    tab, pos = ref.rope_table(50, 64), torch.tensor([3, 9, 11, 20, 49])
    z, mag = ref.norm_rope(x, 2, 64, None, 1e-6, tab, pos, False)
    b = ref.norm_rope_bound(z, mag, torch.bfloat16, "fp32")
    assert ((z.to(torch.bfloat16).double() - z).abs() <= b).all()
    flip = tab.clone()
    flip[..., 1] *= -1
    assert ((ref.norm_rope(x, 2, 64, None, 1e-6, flip, pos, False)[0] - z).abs() > b).any()
    assert ((ref.norm_rope(x, 2, 64, None, 1e-6, tab, pos, True)[0] - z).abs() > b).any()
    q, k, v = (torch.randn((n, 64), generator=g).to(torch.bfloat16) for n in (3, 40, 40))
    w = torch.tensor([[1], [3], [5]], dtype=torch.int32)
    out, A = ref.tree_attention(q, k, v, 30, w, 1, 1, 64, 0.125)
    b = ref.tree_bound(out, A, 33, torch.bfloat16, float(v.abs().max()))
    more, _ = ref.tree_attention(q, k, v, 30, torch.tensor([[3], [3], [5]], dtype=torch.int32), 1, 1, 64, 0.125)
    assert ((more - out).abs() > b)[0].any() and ((more - out).abs() <= b)[1:].all()
    row, tok = ref.logits(torch.tensor([[1.0, 3.0, 2.9, -1.0]]), history=torch.tensor([1, 3]), repetition=1.5)
    assert np.allclose(row.numpy(), [[1.0, 2.0, 2.9, -1.5]]) and tok.tolist() == [2]


def test_mask_words():
    from cacheblend import ops
    a = torch.zeros((2, 70), dtype=torch.bool)
    a[0, [0, 31, 32, 69]] = True
    a[1] = True
    w = ops.mask_words(a)
    assert w.dtype == torch.int32 and w.tolist() == [[1 - (1 << 31), 1, 32], [-1, -1, 63]]
    assert ops.mask_words(a[1]).tolist() == [-1, -1, 63]
    with pytest.raises(ValueError):
        ops.mask_words(a.int())


def test_prompt_lookup_tree():
    from cacheblend import prompt_lookup_tree as look
    #      0  1  2  3  4  5  6  7  8  9
    ids = [5, 6, 7, 8, 9, 6, 7, 1, 6, 7]
    # the tail (6, 7) is followed by 1, 6, 7 (latest first), then by 8, 9, 6, 7, 1, 6, 7
    tokens, parents = look(ids, 20)
    assert tokens == [1, 6, 7, 8, 9, 6, 7, 1, 6, 7] and parents == [-1, 0, 1, -1, 3, 4, 5, 6, 7, 8]
    assert look(ids, 4) == ([1, 6, 7, 8], [-1, 0, 1, -1])
    assert look(ids, 5, depth=2) == ([1, 6, 8, 9], [-1, 0, -1, 2])
    assert look(ids, 0) == ([], [])
    # alike beginnings share their nodes
    assert look([1, 2, 3, 4, 1, 2, 3, 5, 1], 9, depth=3) == ([2, 3, 5, 4], [-1, 0, 1, 1])
    # nothing repeats; one token; none
    assert look([1, 2, 3], 5) == ([], []) and look([4], 5) == ([], []) and look([], 5) == ([], [])
    assert look([3, 3], 5) == ([3], [-1])


def test_accepted_path():
    from cacheblend.drafted import _accept
    tokens, parents = [9, 4, 5, 6, 7, 5], [-1, 0, 0, 1, 3, 1]
    assert _accept(tokens, parents, [1, 0, 0, 0, 0, 0]) == [0]
    assert _accept(tokens, parents, [4, 6, 0, 7, 2, 0]) == [0, 1, 3, 4]
    assert _accept(tokens, parents, [4, 5, 0, 7, 2, 0]) == [0, 1, 5]
    assert _accept(tokens, parents, [5, 5, 0, 0, 0, 0]) == [0, 2]
    assert _accept([9], [-1], [3]) == [0]
