"""The operators behind decoding with drafted tokens against 64-bit references
(``drafted_ref``, which derives the bounds): sizes and masks where they can go
wrong, captured and replayed calls, other streams, and a run of the three."""
import numpy as np
import pytest
import torch

import drafted_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from cacheblend import ops as o
    return o


def status_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------
# norm_rope_scatter
# ---------------------------------------------------------------------------
NR_CASES = [  # n, Hq, Hkv, D, R, dtype, norm, interleaved
    (1, 32, 8, 128, 128, BF, True, False),
    (7, 4, 2, 64, 64, HF, True, True),
    (33, 3, 1, 80, 32, BF, True, False),
    (5, 5, 5, 96, 96, HF, True, False),
    (13, 7, 1, 256, 64, BF, True, True),
    (2, 1, 1, 16, 16, HF, True, False),
    (19, 9, 3, 48, 16, BF, False, True),
    (64, 28, 4, 128, 64, HF, False, False),
    (301, 32, 8, 128, 128, BF, True, False),
    (40, 2, 2, 240, 208, BF, True, False),
]


def nr_inputs(n, hq, hkv, d, r, dt, norm, seed=0, cap=None):
    g = gen(seed + n + d)
    cap = cap or 2 * n + 11
    qkv = (torch.randn((n, (hq + 2 * hkv) * d), generator=g) * 2).to(dt)
    rows = torch.randperm(cap, generator=g)[:n]
    pos = torch.randint(0, 4000, (n,), generator=g)
    w = [(1 + 0.3 * torch.randn((d,), generator=g)).to(dt) for _ in range(2)] if norm else [None, None]
    kc, vc = (torch.randn((cap, hkv * d), generator=g).to(dt) for _ in range(2))
    return qkv, rows, pos, w, kc, vc, ref.rope_table(4000, r)


def nr_split(qkv, hq, hkv, d):
    return qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]


@pytest.mark.parametrize("mode", ["fp32", "ref"])
@pytest.mark.parametrize("case", NR_CASES, ids=str)
def test_norm_rope_scatter(ops, case, mode):
    n, hq, hkv, d, r, dt, norm, il = case
    qkv, rows, pos, w, kc, vc, tab = nr_inputs(n, hq, hkv, d, r, dt, norm)
    qs, ks, vs = nr_split(qkv, hq, hkv, d)
    dev_qkv, dk, dv = qkv.to(DEV), kc.to(DEV), vc.to(DEV)
    st = status_word()
    got = ops.norm_rope_scatter(*nr_split(dev_qkv, hq, hkv, d), pos.to(DEV), rows.to(DEV), hq, hkv, d, tab.to(DEV), dk,
                                dv, *[None if x is None else x.to(DEV) for x in w], eps=1e-5, interleaved=il,
                                mode=mode, status=st)
    assert int(st.item()) == 0 and got.shape == (n, hq * d)
    for x, heads, weight, out in ((qs, hq, w[0], got.cpu()), (ks, hkv, w[1], dk.cpu()[rows])):
        z, mag = ref.norm_rope(x, heads, d, weight, 1e-5, tab, pos, il)
        err = (out.double() - z).abs()
        bound = ref.norm_rope_bound(z, mag, dt, mode)
        assert (err <= bound).all(), float((err / bound).max())
    assert torch.equal(dv.cpu()[rows], vs)
    rest = torch.ones(kc.shape[0], dtype=torch.bool)
    rest[rows] = False
    assert torch.equal(dk.cpu()[rest], kc[rest]) and torch.equal(dv.cpu()[rest], vc[rest])


def test_norm_rope_ref_mode_has_rope_scatter_bits(ops):
    """Without weights, position == row and the whole head rotated, the kernel is
    rope_scatter: the same bits, in both modes."""
    n, hq, hkv, d = 21, 8, 2, 128
    qkv, rows, _, _, kc, vc, tab = nr_inputs(n, hq, hkv, d, d, BF, False)
    rows = rows.sort().values.to(DEV)
    q, k, v = (t.contiguous().to(DEV) for t in nr_split(qkv, hq, hkv, d))
    tab = tab.to(DEV)
    for mode in ("ref", "fp32"):
        a, b = [kc.to(DEV), vc.to(DEV)], [kc.to(DEV), vc.to(DEV)]
        x = ops.rope_scatter(q, k, v, rows, False, kc.shape[0], hq, hkv, d, tab, *a, mode=mode)
        y = ops.norm_rope_scatter(q, k, v, rows, rows, hq, hkv, d, tab, *b, mode=mode)
        if mode == "ref":
            assert torch.equal(x, y) and torch.equal(a[0], b[0])
        else:                              # the fp32 rotations may contract differently: one rounding apart
            assert ((x.float() - y.float()).abs() <= 2.0 ** -7 * x.float().abs() + 1e-5).all()
        assert torch.equal(a[1], b[1])


def test_norm_rope_padding_and_bad_tokens(ops):
    n, hq, hkv, d = 6, 4, 2, 64
    qkv, _, _, w, _, _, tab = nr_inputs(n, hq, hkv, d, d, BF, True, cap=20)
    q, k, v = (t.to(DEV) for t in nr_split(qkv, hq, hkv, d))
    w = [x.to(DEV) for x in w]
    tab = tab[:50].contiguous().to(DEV)

    def call(pos, rows):
        kc, vc = torch.full((20, hkv * d), 7.0, dtype=BF, device=DEV), torch.full((20, hkv * d), 7.0, dtype=BF, device=DEV)
        out = torch.full((n, hq * d), 7.0, dtype=BF, device=DEV)
        st = status_word()
        ops.norm_rope_scatter(q, k, v, torch.tensor(pos, device=DEV), torch.tensor(rows, device=DEV), hq, hkv, d, tab,
                              kc, vc, *w, q_out=out, status=st)
        return out, kc, vc, int(st.item())

    good = call([0, 1, 2, 3, 4, 49], [0, 5, 6, 7, 8, 19])
    assert good[3] == 0 and not (good[0] == 7).all(1).any()
    pad = call([0, 1, 2, 3, 4, 49], [0, 5, -1, 7, -1, 19])
    assert pad[3] == 0
    bad = call([0, 1, -1, 50, 4, 49], [0, 5, 6, 7, 20, -2])
    assert bad[3] & 1
    for got, lost in ((pad, [2, 4]), (bad, [2, 3, 4, 5])):
        for j in range(n):
            row = [0, 5, 6, 7, 8, 19][j]
            if j in lost:
                assert (got[0][j] == 7).all() and (got[1][row] == 7).all() and (got[2][row] == 7).all()
            else:
                assert torch.equal(got[0][j], good[0][j]) and torch.equal(got[1][row], good[1][row])
                assert torch.equal(got[2][row], good[2][row])


def test_norm_rope_strides_sources_and_refusals(ops):
    """Caches that are column views, sources that need a copy, no tokens; what is refused."""
    n, hq, hkv, d = 9, 4, 2, 64
    qkv, rows, pos, w, kc, vc, tab = nr_inputs(n, hq, hkv, d, d, HF, True)
    args = [t.to(DEV) for t in nr_split(qkv, hq, hkv, d)]
    rows, pos, tab, w = rows.to(DEV), pos.to(DEV), tab.to(DEV), [x.to(DEV) for x in w]
    a = [kc.to(DEV), vc.to(DEV)]
    q = ops.norm_rope_scatter(*args, pos, rows, hq, hkv, d, tab, *a, *w)
    both = torch.zeros((kc.shape[0], 2 * hkv * d + 8), dtype=HF, device=DEV)
    both[:, :hkv * d], both[:, hkv * d:2 * hkv * d] = kc.to(DEV), vc.to(DEV)
    b = [both[:, :hkv * d], both[:, hkv * d:2 * hkv * d]]
    odd = torch.zeros((n, args[0].shape[1] + 3), dtype=HF, device=DEV)[:, 3:]      # rows off 16-byte boundaries
    odd.copy_(args[0])
    q2 = ops.norm_rope_scatter(odd, args[1], args[2].t().contiguous().t(), pos, rows, hq, hkv, d, tab, *b, *w)
    assert torch.equal(q, q2) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert (both[:, 2 * hkv * d:] == 0).all()
    none = ops.norm_rope_scatter(*[t[:0] for t in args], pos[:0], rows[:0], hq, hkv, d, tab, *a, *w)
    assert none.shape == (0, hq * d)
    for change, err in [(dict(mode="x"), ValueError), (dict(q_weight=w[0], k_weight=None), ValueError),
                        (dict(q_weight=w[0].float(), k_weight=w[1].float()), ValueError),
                        (dict(q_out=torch.empty((n, 8), dtype=HF, device=DEV)), ValueError)]:
        with pytest.raises(err):
            ops.norm_rope_scatter(*args, pos, rows, hq, hkv, d, tab, *a, **change)
    with pytest.raises(ValueError):
        ops.norm_rope_scatter(*args, pos[:-1], rows, hq, hkv, d, tab, *a)
    with pytest.raises(ValueError):
        ops.norm_rope_scatter(*args, pos.int(), rows, hq, hkv, d, tab, *a)
    with pytest.raises(ValueError):
        ops.norm_rope_scatter(*args, pos, rows, hq, hkv, d, tab.double(), *a)
    with pytest.raises(ValueError):
        ops.norm_rope_scatter(*args, pos, rows, hq, hkv, d, tab, a[0].to(BF), a[1])
    with pytest.raises(NotImplementedError):
        ops.norm_rope_scatter(*[t.float() for t in args], pos, rows, hq, hkv, d, tab, a[0].float(), a[1].float())
    with pytest.raises(NotImplementedError):
        ops.norm_rope_scatter(*args, pos, rows, hq, hkv, d, tab[:, :12].contiguous(), *a)


# ---------------------------------------------------------------------------
# tree_attn
# ---------------------------------------------------------------------------
TA_CASES = [  # T, n_ctx, Hq, Hkv, D, dtype, tree
    (1, 0, 4, 2, 64, BF, "tree"),
    (1, 1, 8, 8, 128, HF, "tree"),
    (1, 700, 32, 8, 128, BF, "tree"),
    (2, 127, 4, 1, 128, BF, "tree"),
    (5, 128, 4, 2, 64, HF, "tree"),
    (9, 120, 7, 1, 128, BF, "tree"),          # the tree crosses a tile edge; 63 rows per KV head
    (16, 300, 32, 8, 128, BF, "tree"),
    (31, 257, 6, 2, 64, BF, "sparse"),        # some nodes see nothing of the tree
    (33, 0, 8, 2, 128, BF, "sparse"),         # ... and there is no context: nothing at all
    (32, 31, 16, 1, 64, HF, "tree"),          # 512 rows of one KV head
    (64, 500, 8, 2, 128, HF, "full"),
    (65, 1000, 2, 2, 128, BF, "tree"),
    (130, 64, 4, 2, 64, BF, "sparse"),
    (100, 1250, 10, 2, 128, BF, "tree"),      # 500 rows: an odd number of row tiles would be 4
    (3, 2000, 64, 1, 128, BF, "tree"),        # 192 rows of one head
]


def ta_inputs(t, n_ctx, hq, hkv, d, dt, tree, seed=0, spare=70, scale=1.5):
    g = gen(seed + 7 * t + n_ctx)
    cap = n_ctx + t + spare
    q = (torch.randn((t, hq * d), generator=g) * scale).to(dt)
    k, v = (torch.randn((cap, hkv * d), generator=g).to(dt) for _ in range(2))
    width = (t + 31) // 32
    if tree == "tree":
        parents = [-1] + [max(-1, i - 1 - int(torch.randint(0, 4, (1,), generator=g))) for i in range(1, t)]
        from cacheblend import ops
        words = ops.tree_words(parents)[0]
    elif tree == "full":
        words = torch.full((t, width), -1, dtype=torch.int32)
    else:
        words = torch.randint(-2 ** 31, 2 ** 31, (t, width), generator=g).to(torch.int32)
        words[::3] = 0
    return q, k, v, words, cap


def ta_check(got, q, k, v, n_ctx, words, hq, hkv, d, scale):
    out, A = ref.tree_attention(q, k, v, n_ctx, words, hq, hkv, d, scale)
    bound = ref.tree_bound(out, A, n_ctx + words.shape[0], q.dtype, float(v[:n_ctx + words.shape[0]].abs().max()))
    err = (got.cpu().double() - out).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("case", TA_CASES, ids=str)
def test_tree_attn(ops, case):
    t, n_ctx, hq, hkv, d, dt, tree = case
    q, k, v, words, cap = ta_inputs(*case)
    k[n_ctx + t:], v[n_ctx + t:] = float("nan"), float("inf")         # behind the tree: anything
    st = status_word()
    got = ops.tree_attn(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([n_ctx], device=DEV), words.to(DEV), hq, hkv, d,
                        d ** -0.5, status=st)
    assert int(st.item()) == 0
    ta_check(got, q, k, v, n_ctx, words, hq, hkv, d, d ** -0.5)


@pytest.mark.parametrize("t,n_ctx,hq,hkv,d,dt", [(16, 6208, 32, 8, 128, BF), (40, 9001, 8, 2, 128, HF),
                                                 (64, 20000, 32, 8, 128, BF), (7, 30011, 4, 2, 64, BF)])
def test_tree_attn_long(ops, t, n_ctx, hq, hkv, d, dt):
    """Long contexts, split over many CTAs, peaked and flat, against 64 bits on the GPU."""
    q, k, v, words, cap = ta_inputs(t, n_ctx, hq, hkv, d, dt, "tree")
    q[::2] *= 4                                                        # every other node peaked
    n = n_ctx + t
    got = ops.tree_attn(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([n_ctx], device=DEV), words.to(DEV), hq, hkv, d,
                        d ** -0.5)
    sees = torch.ones((t, n), dtype=torch.bool)
    sees[:, n_ctx:] = ref.visible(words, t)
    for h in range(hq):
        at = slice(h // (hq // hkv) * d, (h // (hq // hkv) + 1) * d)
        kk, vv = k[:n, at].to(DEV).double(), v[:n, at].to(DEV).double()
        s = (q[:, h * d:(h + 1) * d].to(DEV).double() @ kk.T * d ** -0.5).masked_fill(~sees.to(DEV), -torch.inf)
        p = torch.softmax(s, 1)
        out, A = (p @ vv).cpu(), (p @ vv.abs()).cpu()
        bound = ref.tree_bound(out, A, n, dt, float(v.abs().max()))
        err = (got[:, h * d:(h + 1) * d].cpu().double() - out).abs()
        assert (err <= bound).all(), (h, float((err / bound).max()))


def test_tree_attn_masked_places_may_hold_anything(ops):
    """NaN and infinities in a node's own K or V reach the nodes that see it and no other."""
    t, n_ctx, hq, hkv, d = 12, 250, 8, 2, 128
    q, k, v, _, _ = ta_inputs(t, n_ctx, hq, hkv, d, BF, "full")
    words, _ = ops.tree_words([-1, 0, 0, 1, 1, 2, 2, 3, 5, -1, 9, 10])
    args = (torch.tensor([n_ctx], device=DEV), words.to(DEV), hq, hkv, d, d ** -0.5)
    clean = ops.tree_attn(q.to(DEV), k.to(DEV), v.to(DEV), *args)
    for value in (float("nan"), float("inf"), -float("inf")):
        for node, which in ((1, "k"), (5, "v"), (9, "v"), (2, "k")):
            k2, v2 = k.clone(), v.clone()
            if which == "k":
                k2[n_ctx + node, :d] = value
            else:
                v2[n_ctx + node, 3:5] = value
            got = ops.tree_attn(q.to(DEV), k2.to(DEV), v2.to(DEV), *args)
            sees = ref.visible(words, t)[:, node]
            assert torch.equal(got[~sees.to(DEV)], clean[~sees.to(DEV)]), (value, node, which)
            if which == "v":
                hit = got.view(t, hkv, hq // hkv, d)[sees.to(DEV)][:, 0, :, 3:5]
                assert not torch.isfinite(hit).any(), (value, node)
                assert torch.isfinite(got.view(t, hkv, -1)[:, 1]).all()
            elif value != value:
                assert torch.isnan(got.view(t, hkv, -1)[sees.to(DEV)][:, 0]).all()


def test_tree_attn_bad_context_leaves_the_output(ops):
    q, k, v, words, cap = ta_inputs(4, 20, 4, 2, 64, BF, "tree")
    for n_ctx, bad in ((-1, True), (cap - 3, True), (1 << 40, True), (-(1 << 40), True), (cap - 4, False), (0, False)):
        out = torch.full((4, 256), 7.0, dtype=BF, device=DEV)
        st = status_word()
        ops.tree_attn(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([n_ctx], device=DEV), words.to(DEV), 4, 2, 64, 0.1,
                      out=out, status=st)
        assert (int(st.item()) & 1 == 1) == bad and bool((out == 7).all()) == bad


def test_tree_attn_refusals_and_layouts(ops):
    q, k, v, words, cap = ta_inputs(6, 100, 4, 2, 64, BF, "tree")
    n = torch.tensor([100], device=DEV)
    q, k, v, words = (x.to(DEV) for x in (q, k, v, words))
    base = ops.tree_attn(q, k, v, n, words, 4, 2, 64, 0.125)
    wide = torch.zeros((cap, 304), dtype=BF, device=DEV)[:, 8:8 + 256]              # K and V side by side
    wide[:, :128], wide[:, 128:] = k, v
    pad = torch.zeros((6, 3), dtype=torch.int32, device=DEV)
    pad[:, :1] = words
    pad[:, 1:] = -1                                                                  # bits past the tree: ignored
    ws = ops.tree_workspace(6, cap, 4, 2, 64, DEV)
    odd = torch.zeros((6 * 256 + 3,), dtype=BF, device=DEV)[3:].view(6, 256)
    odd.copy_(q)
    got = ops.tree_attn(odd, wide[:, :128], wide[:, 128:], n, pad, 4, 2, 64, 0.125, workspace=ws,
                        out=torch.empty_like(base))
    assert torch.equal(got, base)
    same = ops.tree_attn(q, k, v, n, words[:1].expand(6, 1), 4, 2, 64, 0.125)       # one row of words for every node
    assert torch.equal(same, ops.tree_attn(q, k, v, n, words[:1].repeat(6, 1), 4, 2, 64, 0.125))
    assert ops.tree_attn(q[:0], k, v, n, words[:0], 4, 2, 64, 0.125).shape == (0, 256)
    for bad in (lambda: ops.tree_attn(q, k, v, n, words.long(), 4, 2, 64, 0.1),
                lambda: ops.tree_attn(q[:5], k, v, n, words, 4, 2, 64, 0.1),
                lambda: ops.tree_attn(q, k, v[:-1], n, words, 4, 2, 64, 0.1),
                lambda: ops.tree_attn(q, k, v, n.int(), words, 4, 2, 64, 0.1),
                lambda: ops.tree_attn(q, k.to(HF), v, n, words, 4, 2, 64, 0.1),
                lambda: ops.tree_attn(q, k, v, n, words, 4, 2, 64, 0.1, workspace=ws[:16]),
                lambda: ops.tree_attn(q, k[:5], v[:5], n, words, 4, 2, 64, 0.1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        ops.tree_attn(q, k, v, n, words, 8, 4, 32, 0.1)


def test_tree_attn_captured_context_advances(ops):
    """A captured call follows n_ctx, the words and the cache as they change."""
    t, hq, hkv, d = 8, 8, 2, 128
    q, k, v, words, cap = ta_inputs(t, 900, hq, hkv, d, BF, "tree")
    dq, dk, dv, dw = (x.to(DEV) for x in (q, k, v, words))
    n = torch.tensor([0], device=DEV)
    out = torch.zeros((t, hq * d), dtype=BF, device=DEV)
    ops.tree_attn(dq, dk, dv, n, dw, hq, hkv, d, d ** -0.5, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        ops.tree_attn(dq, dk, dv, n, dw, hq, hkv, d, d ** -0.5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for n_ctx in (0, 1, 119, 120, 128, 500, 895, 900):
        n.fill_(n_ctx)
        graph.replay()
        ta_check(out, q, k, v, n_ctx, words, hq, hkv, d, d ** -0.5)


def on_gpu_check(got, q, k, v, n_ctx, words, hq, hkv, d, scale, heads=None):
    """ta_check in 64 bits on the GPU, head by head (finite caches)."""
    t, n = words.shape[0], n_ctx + words.shape[0]
    sees = torch.ones((t, n), dtype=torch.bool, device=DEV)
    sees[:, n_ctx:] = ref.visible(words, t).to(DEV)
    for h in range(hq) if heads is None else heads:
        at = slice(h // (hq // hkv) * d, (h // (hq // hkv) + 1) * d)
        kk, vv = k[:n, at].to(DEV).double(), v[:n, at].to(DEV).double()
        s = (q[:, h * d:(h + 1) * d].to(DEV).double() @ kk.T * scale).masked_fill(~sees, -torch.inf)
        p = torch.softmax(s, 1).nan_to_num(0.0)              # (a row that sees nothing: zeros)
        out, A = p @ vv, p @ vv.abs()
        bound = ref.tree_bound(out, A, n, q.dtype, float(vv.abs().max()))
        err = (got[:, h * d:(h + 1) * d].double() - out).abs()
        assert (err <= bound).all(), (h, float((err / bound).max()))


@pytest.mark.parametrize("t,n_ctx,hq,hkv,d,dt", [(1024, 300, 4, 1, 128, BF), (999, 0, 6, 2, 64, HF),
                                                 (640, 5000, 3, 3, 128, BF)])
def test_tree_attn_many_nodes(ops, t, n_ctx, hq, hkv, d, dt):
    """Many Q tiles, odd counts of them, and key tiles of the tree alone."""
    q, k, v, words, cap = ta_inputs(t, n_ctx, hq, hkv, d, dt, "sparse", spare=3)
    got = ops.tree_attn(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([n_ctx], device=DEV), words.to(DEV), hq, hkv, d,
                        d ** -0.5)
    on_gpu_check(got, q, k, v, n_ctx, words, hq, hkv, d, d ** -0.5)


def test_offsets_past_32_bits(ops):
    """A cache of more than 2^31 elements: rows written and read behind that."""
    t, hq, hkv, d, n_ctx = 5, 8, 8, 128, 2_200_000
    cap = n_ctx + t + 4
    g = torch.Generator(device=DEV).manual_seed(4)
    k = torch.randn((cap, hkv * d), generator=g, device=DEV, dtype=BF)
    v = torch.randn((cap, hkv * d), generator=g, device=DEV, dtype=BF)
    assert k.numel() > 2 ** 31
    qkv, _, pos, w, _, _, tab = nr_inputs(t, hq, hkv, d, d, BF, True)
    rows = n_ctx + torch.arange(t)
    q = ops.norm_rope_scatter(*nr_split(qkv.to(DEV), hq, hkv, d), pos.to(DEV), rows.to(DEV), hq, hkv, d, tab.to(DEV), k, v,
                              *[x.to(DEV) for x in w], mode="fp32")
    z, mag = ref.norm_rope(nr_split(qkv, hq, hkv, d)[1], hkv, d, w[1], 1e-6, tab, pos, False)
    assert ((k[rows.to(DEV)].cpu().double() - z).abs() <= ref.norm_rope_bound(z, mag, BF, "fp32")).all()
    assert torch.equal(v[rows.to(DEV)].cpu(), nr_split(qkv, hq, hkv, d)[2])
    q = q * 8                                           # peaked: single far rows count
    words, _ = ops.tree_words([-1, 0, 0, 1, 2])
    got = ops.tree_attn(q, k, v, torch.tensor([n_ctx], device=DEV), words.to(DEV), hq, hkv, d, d ** -0.5)
    on_gpu_check(got, q, k, v, n_ctx, words, hq, hkv, d, d ** -0.5, heads=[0, 7])


# ---------------------------------------------------------------------------
# process_logits
# ---------------------------------------------------------------------------
def pl_check(ops, x, out_dtype=None, **kw):
    st = status_word()
    dev = {n: (t.to(DEV) if isinstance(t, torch.Tensor) else t) for n, t in kw.items()}
    got, tok = ops.process_logits(x.to(DEV), out_dtype=out_dtype, status=st, **dev)
    names = {"mask_words": "mask"}
    exp, exp_tok = ref.logits(x, **{names.get(n, n): t for n, t in kw.items()})
    exp = exp.to(out_dtype or x.dtype)
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(exp))
    assert torch.equal(torch.nan_to_num(got.cpu().float(), 0.5, 1e38, -1e38),
                       torch.nan_to_num(exp.float(), 0.5, 1e38, -1e38))
    assert torch.equal(tok.cpu(), exp_tok)
    only, tok2 = ops.process_logits(x.to(DEV), return_logits=False, **dev)
    assert only is None and torch.equal(tok2, tok)
    return int(st.item())


def pl_inputs(rows, vocab, length, dt, seed=0, shared=True):
    g = gen(seed + rows + vocab)
    x = (torch.randn((rows, vocab), generator=g) * 3).to(dt)
    sets = 1 if shared else rows
    h = (torch.rand((sets, length), generator=g) ** 3 * vocab).long().clamp_(max=vocab - 1)
    k = min(3, length)
    h[:, :k] = x[:sets].float().topk(min(3, vocab), dim=1).indices[:, :k]
    return x, h, g


@pytest.mark.parametrize("rows,vocab,length,dt,out,shared", [
    (1, 32000, 500, BF, torch.float32, True),
    (1, 1, 3, torch.float32, None, True),
    (3, 7, 20, BF, None, False),
    (5, 1009, 64, HF, None, False),               # rows off every boundary
    (4, 1009, 64, HF, torch.float32, True),
    (2, 50001, 3000, BF, torch.float32, True),
    (17, 2048, 1, torch.float32, None, True),
    (6, 4100, 5000, BF, None, True),
    (2, 128256, 40, BF, None, False),
    (1, 458752, 10, BF, None, True),
    (3, 300001, 100, torch.float32, None, False),
])
def test_process_logits(ops, rows, vocab, length, dt, out, shared):
    x, h, g = pl_inputs(rows, vocab, length, dt, shared=shared)
    sets = h.shape[0]
    lengths = torch.randint(0, length + 1, (sets,), generator=g)
    prompt = torch.randint(0, length + 1, (sets,), generator=g)
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g).to(torch.int32)
    bias = torch.randn((vocab,), generator=g)
    assert pl_check(ops, x, out, history=h, lengths=lengths, n_prompt=prompt, repetition=1.3, presence=0.4,
                    frequency=0.1, bias=bias, mask_words=mask) == 0
    pl_check(ops, x, out, history=h, repetition=0.7, frequency=-0.2)                # rewards, the whole history made
    pl_check(ops, x, out, bias=bias.repeat(rows, 1) * torch.arange(1, rows + 1)[:, None])
    pl_check(ops, x, out, mask_words=mask[0])                                       # one mask for every row
    pl_check(ops, x, out)


@pytest.mark.parametrize("dt,out", [(BF, None), (BF, torch.float32), (HF, None), (torch.float32, None)])
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (3, 4104), (30, 4096)])
def test_process_logits_long_history(ops, rows, vocab, dt, out):
    """A history long for its vocabulary: magnitudes from 0 to infinity among seen
    and unseen tokens, every penalty's extremes, a path on top; and the same rows
    with their tokens at the front of a history with much more or no more room."""
    x, h, g = pl_inputs(rows, vocab, 4000, dt, seed=7)
    odd = torch.tensor([0.0, -0.0, 1e-45, 1e-40, 1e-30, 9e-21, 1.1e-20, 1e20, 3e38, -1e-30, -3e38, float("inf"),
                        -float("inf"), float("nan")])
    at = torch.randperm(vocab - 8, generator=g)[:4 * len(odd)].view(4, -1)
    x[:, at[0]] = odd.to(dt)
    x[:, at[1]] = odd.to(dt)
    h[0, 100:100 + len(odd)] = at[0]                  # at[1] unseen but for chance
    words, _ = ops.tree_words([-1] + [i // 2 for i in range(rows - 1)])
    toks = torch.cat([at[2], at[0], h[0, :8]])[:rows]
    for kw in (dict(repetition=1.1, presence=0.25, frequency=0.125), dict(repetition=0.3, presence=-2.0, frequency=-0.7),
               dict(repetition=3.0), dict(frequency=0.3), dict(presence=0.7), dict(repetition=2.0 ** 41, presence=1.0),
               dict(repetition=1e-30), dict(repetition=1.2, frequency=float("inf")),
               dict(repetition=1.2, presence=-float("inf"))):
        assert pl_check(ops, x, out, history=h, n_prompt=torch.tensor([1500]), **kw) == 0
        assert pl_check(ops, x, out, history=h, n_prompt=torch.tensor([3990]), tree_tokens=toks, tree_words=words,
                        **kw) == 0
    kw = dict(repetition=1.1, presence=0.25, frequency=0.125, out_dtype=out)
    few = h[:, :vocab // 16 - 1].contiguous().to(DEV)
    a, t = ops.process_logits(x.to(DEV), history=h.to(DEV), lengths=torch.tensor([few.shape[1]], device=DEV), **kw)
    b, u = ops.process_logits(x.to(DEV), history=few, **kw)
    assert torch.equal(a.nan_to_num(0.5), b.nan_to_num(0.5)) and torch.equal(t, u)


@pytest.mark.parametrize("dt", [BF, HF, torch.float32])
def test_process_logits_every_alignment(ops, dt):
    """Rows of a wider buffer from every first element, and odd output strides."""
    for off in range(9):
        for vocab in (64, 65, 71):
            x, h, g = pl_inputs(3, vocab, 9, dt, seed=off)
            wide = torch.zeros((3, 90), dtype=dt, device=DEV)
            view = wide[:, off:off + vocab]
            view.copy_(x)
            exp, tok = ref.logits(x, history=h, repetition=1.2, presence=0.1)
            out = torch.full((3, 97), 7.0, dtype=dt, device=DEV)
            got, t = ops.process_logits(view, history=h.to(DEV), repetition=1.2, presence=0.1,
                                        out=out[:, 8 - off:8 - off + vocab])
            assert torch.equal(got.cpu(), exp.to(dt)) and torch.equal(t.cpu(), tok)
            assert (out[:, :8 - off] == 7).all() and (out[:, 8 - off + vocab:] == 7).all()


def test_process_logits_tree_rows(ops):
    """Row r's path counts as made tokens; every node has its own."""
    rows, vocab = 37, 5003
    x, h, g = pl_inputs(rows, vocab, 300, BF)
    parents = [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, rows)]
    words, _ = ops.tree_words(parents)
    toks = torch.randint(0, 40, (rows,), generator=g)                 # few tokens: the same one twice on a path
    x[:, :40] += 8
    for kw in (dict(history=h, n_prompt=torch.tensor([250])), {}):
        assert pl_check(ops, x, torch.float32, tree_tokens=toks, tree_words=words, repetition=1.1, presence=0.5,
                        frequency=0.25, **kw) == 0


def test_process_logits_edges(ops):
    x = torch.randn((4, 1000), generator=gen(3)).to(BF)
    x[0, 17], x[0, 400] = float("nan"), float("nan")
    x[1, 3], x[1, 900], x[1, 5] = float("inf"), float("inf"), -float("inf")
    x[2] = 1.5                                                        # every value ties: the lowest index
    x[3] = torch.finfo(BF).min
    allowed = torch.full((4, 32), -1, dtype=torch.int32)
    h = torch.tensor([17, 3, 0, 0, 5])
    pl_check(ops, x, None, history=h, repetition=2.0, presence=1.0, frequency=0.5, mask_words=allowed)
    allowed[0, 0] = 0                                                 # the NaN at 17 is masked, the one at 400 not
    allowed[1, 0], allowed[1, 28] = 0, 0                              # both infinities masked
    allowed[2] = 0                                                    # nothing left
    allowed[3] = 0
    allowed[3, 31] = 1 << 7                                           # the last token, 999, alone
    pl_check(ops, x, torch.float32, history=h, repetition=2.0, mask_words=allowed)
    _, tok = ops.process_logits(x.to(DEV), mask_words=allowed.to(DEV))
    assert tok.tolist() == [400, int(x[1].float().masked_fill(~ref.visible(allowed[1:2], 1000)[0], -np.inf).argmax()), 0, 999]
    z = torch.tensor([[-0.0, 0.0, -1.0], [-2.0, -0.0, 0.0]])
    assert ops.process_logits(z.to(DEV))[1].tolist() == [0, 1]        # -0 ties with +0
    bias = torch.zeros(1000)
    bias[999], bias[0] = float("inf"), -float("inf")
    pl_check(ops, x, torch.float32, bias=bias)
    same = x.to(DEV)
    out, _ = ops.process_logits(same, repetition=1.5, history=h.to(DEV), out=same)       # in place
    assert out is same and torch.equal(torch.nan_to_num(same.cpu()), torch.nan_to_num(ref.logits(x, history=h, repetition=1.5)[0].to(BF)))
    none, t = ops.process_logits(x[:0].to(DEV))
    assert none.shape == (0, 1000) and t.shape == (0,)
    flat, t = ops.process_logits(x[0].to(DEV), out_dtype=torch.float32)
    assert flat.shape == (1000,) and t.shape == () and int(t) == 17
    pl_check(ops, x, None, history=torch.zeros((1, 0), dtype=torch.int64), repetition=1.5)


@pytest.mark.parametrize("rows,vocab,dt", [(24, 5000, BF), (31, 3001, HF), (67, 4096, BF), (150, 1000, torch.float32)])
def test_process_logits_many_rows(ops, rows, vocab, dt):
    """More rows than clusters: a shared history counted once, one per row, none, and a tree."""
    x, h, g = pl_inputs(rows, vocab, 700, dt)
    own = (torch.rand((rows, 90), generator=g) ** 3 * vocab).long().clamp_(max=vocab - 1)
    n = torch.tensor([300])
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g).to(torch.int32)
    words, _ = ops.tree_words([-1] + [int(torch.randint(max(0, i - 3), i, (1,), generator=g)) for i in range(1, rows)])
    toks = torch.randint(0, 60, (rows,), generator=g)
    x[:, :60] += 6
    kw = dict(repetition=1.15, presence=0.2, frequency=0.3)
    assert pl_check(ops, x, torch.float32, history=h, n_prompt=n, mask_words=mask, **kw) == 0
    assert pl_check(ops, x, None, history=h, lengths=n, tree_tokens=toks, tree_words=words, **kw) == 0
    assert pl_check(ops, x, None, history=own, lengths=torch.randint(0, 91, (rows,), generator=g),
                    tree_tokens=toks, tree_words=words, **kw) == 0
    assert pl_check(ops, x, None, history=h, lengths=torch.randint(0, 701, (rows,), generator=g), **kw) == 0
    assert pl_check(ops, x, None, tree_tokens=toks, tree_words=words, **kw) == 0
    assert pl_check(ops, x, torch.float32, bias=torch.randn((vocab,), generator=g)) == 0


def test_process_logits_offsets_past_32_bits(ops):
    rows, vocab = 17000, 128256
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn((rows, vocab), generator=g, device=DEV, dtype=BF)
    assert x.numel() > 2 ** 31
    h = torch.randint(0, vocab, (500,), generator=g, device=DEV)
    out, tok = ops.process_logits(x, history=h, repetition=1.2, frequency=0.1)
    at = torch.tensor([0, 65, 66, 16743, 16744, 16999], device=DEV)
    exp, exp_tok = ref.logits(x[at], history=h, repetition=1.2, frequency=0.1)
    assert torch.equal(out[at].cpu(), exp.to(BF)) and torch.equal(tok[at].cpu(), exp_tok)


def test_process_logits_division_is_the_rounded_quotient(ops):
    """x / repetition for many mantissas and exponents, penalties in and out of the
    range of the fast way, to the bit."""
    g = gen(17)
    n = 1 << 18
    x = (1 + torch.rand((1, n), generator=g, dtype=torch.float64)).float()
    x[0, :9] = torch.tensor([1e-40, 1e-38, 9e-21, 1.1e-20, 1e20, 2e20, 3e38, float("inf"), 1.0])
    x[0, 9:n // 2] *= torch.exp2(torch.randint(-30, 30, (n // 2 - 9,), generator=g).float())
    x[0, n // 2:n // 2 + 1000] = 2 - torch.arange(1, 1001) * 2.0 ** -23          # mantissas near 2
    h = torch.arange(n)
    below_two = float(np.nextafter(np.float32(2), np.float32(0)))
    for rep in (1.1, 1.3, 0.7, 3.0, below_two, float(np.nextafter(np.float32(1), np.float32(2))), 1.0 / 3, 1e-12, 1e11,
                1e-20, 1e30, 3e-39):
        pl_check(ops, x, None, history=h, repetition=rep, bias=torch.zeros(n))


def test_process_logits_bad_tokens_are_skipped_and_reported(ops):
    x = torch.randn((2, 100), generator=gen(5)).to(BF)
    h = torch.tensor([[1, 2, -1, 100, 5], [7, 7, 1 << 40, 8, 9]])
    assert pl_check(ops, x, None, history=h, repetition=1.4, presence=0.3) & 1
    assert pl_check(ops, x, None, history=h[:, :2], lengths=torch.tensor([1, 9]), repetition=1.4) & 1
    assert pl_check(ops, x, None, history=h[:, :2], lengths=torch.tensor([-4, 2]), repetition=1.4) & 1
    assert pl_check(ops, x, None, history=h[:, :2], lengths=torch.tensor([1, 2]), repetition=1.4) == 0
    # a tree's token outside the vocabulary, on one row's path; and with the history counted once
    words = torch.tensor([[1], [3]], dtype=torch.int32)
    st = status_word()
    _, tok = ops.process_logits(x.to(DEV), tree_tokens=torch.tensor([5, 100], device=DEV), tree_words=words.to(DEV),
                                repetition=1.4, status=st)
    exp, exp_tok = ref.logits(x, tree_tokens=torch.tensor([5, 5]), tree_words=torch.ones_like(words), repetition=1.4)
    assert int(st.item()) & 1 and torch.equal(tok.cpu(), exp_tok)
    many = torch.randn((40, 100), generator=gen(6)).to(BF)
    assert pl_check(ops, many, None, history=h[0], repetition=1.4, presence=0.3) & 1
    assert pl_check(ops, many, None, history=h[0, :2], lengths=torch.tensor([9]), repetition=1.4) & 1
    assert pl_check(ops, many, None, history=h[0, :2], repetition=1.4) == 0


def test_process_logits_refusals(ops):
    x = torch.zeros((2, 64), dtype=BF, device=DEV)
    h = torch.zeros((5,), dtype=torch.int64, device=DEV)
    for bad in (dict(lengths=h[:1]), dict(history=h.int()), dict(history=h.expand(3, 5)), dict(tree_tokens=h),
                dict(history=h, lengths=h[:3]), dict(bias=x[0]), dict(bias=x.float()[:, :5]), dict(mask_words=h),
                dict(mask_words=h[:1].int()), dict(repetition=0.0), dict(repetition=float("inf")), dict(presence=float("nan")),
                dict(tree_tokens=h, tree_words=h.int().view(1, 5)), dict(out=x[:1]),
                dict(out=x, out_dtype=torch.float32)):
        with pytest.raises(ValueError):
            ops.process_logits(x, **bad)
    for bad in (dict(out=x.to(HF)), dict(out_dtype=HF), dict(out_dtype=torch.float64)):
        with pytest.raises(NotImplementedError):
            ops.process_logits(x, **bad)
    with pytest.raises(NotImplementedError):
        ops.process_logits(x.double())


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_a_step_of_the_three(ops):
    """Norm, rotation and write of a drafted tree, attention over the cache, and
    the choice of every node, on another stream, against 64 bits: the attention
    of the operators' own Q and cache, the choice from its output's logits."""
    t, n_ctx, hq, hkv, d, vocab = 23, 333, 8, 2, 128, 3001
    qkv, _, _, w, kc, vc, tab = nr_inputs(t, hq, hkv, d, d, BF, True, cap=n_ctx + t + 9)
    g = gen(11)
    parents = [-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, t)]
    words, depth = ops.tree_words(parents)
    head = (torch.randn((hq * d, vocab), generator=g) * 0.2).to(BF)
    draft = torch.randint(0, vocab, (t,), generator=g)
    prompt = torch.randint(0, vocab, (n_ctx,), generator=g)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        dk, dv, dn = kc.to(DEV), vc.to(DEV), torch.tensor([n_ctx], device=DEV)
        dw = words.to(DEV)
        q = ops.norm_rope_scatter(*nr_split(qkv.to(DEV), hq, hkv, d), n_ctx + depth.to(DEV),
                                  n_ctx + torch.arange(t, device=DEV), hq, hkv, d, tab.to(DEV), dk, dv,
                                  *[x.to(DEV) for x in w], mode="fp32")
        a = ops.tree_attn(q, dk, dv, dn, dw, hq, hkv, d, d ** -0.5)
        raw = a @ head.to(DEV)
        x, tok = ops.process_logits(raw, history=prompt.to(DEV), n_prompt=dn, repetition=1.2, presence=0.1,
                                    tree_tokens=draft.to(DEV), tree_words=dw, out_dtype=torch.float32)
    side.synchronize()
    z, mag = ref.norm_rope(nr_split(qkv, hq, hkv, d)[1], hkv, d, w[1], 1e-6, tab, n_ctx + depth, False)
    assert ((dk.cpu()[n_ctx:n_ctx + t].double() - z).abs() <= ref.norm_rope_bound(z, mag, BF, "fp32")).all()
    ta_check(a, q.cpu(), dk.cpu(), dv.cpu(), n_ctx, words, hq, hkv, d, d ** -0.5)
    exp, exp_tok = ref.logits(raw.cpu(), history=prompt, n_prompt=torch.tensor([n_ctx]), repetition=1.2, presence=0.1,
                              tree_tokens=draft, tree_words=words)
    assert torch.equal(x.cpu(), exp) and torch.equal(tok.cpu(), exp_tok)


def test_calls_on_two_streams_at_once(ops):
    """Calls that overlap on the GPU, each with its own workspace, give what they give alone."""
    cases = [ta_inputs(16, 6000, 32, 8, 128, BF, "tree", seed=s) for s in (0, 1)]
    logits = [pl_inputs(40, 20000, 3000, BF, seed=s) for s in (0, 1)]
    n = torch.tensor([6000], device=DEV)

    def work(i):
        q, k, v, words, _ = (x.to(DEV) if isinstance(x, torch.Tensor) else x for x in cases[i])
        x, h = logits[i][0].to(DEV), logits[i][1].to(DEV)
        torch.cuda.synchronize()
        return lambda: [(ops.tree_attn(q, k, v, n, words, 32, 8, 128, 0.09),
                         *ops.process_logits(x, history=h, repetition=1.2, frequency=0.1)) for _ in range(10)]

    calls = [work(0), work(1)]
    alone = [c()[0] for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    out = []
    for c, st in zip(calls, streams):
        with torch.cuda.stream(st):
            out.append(c())
    torch.cuda.synchronize()
    for i in (0, 1):
        for got in out[i]:
            for a, b in zip(got, alone[i]):
                assert torch.equal(a, b)


def test_two_captured_graphs_interleaved(ops):
    """Each captured call keeps its own workspace; lengths that advance on the device are followed."""
    x, h, _ = pl_inputs(30, 5000, 400, BF)
    dx, dh, n = x.to(DEV), h.to(DEV), torch.tensor([0], device=DEV)
    y, h2, _ = pl_inputs(3, 5000, 400, BF, seed=5)
    dy = y.to(DEV)

    def capture(f):
        f()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            out = f()
        torch.cuda.current_stream().wait_stream(side)
        return graph, out

    kw = dict(repetition=1.3, presence=0.1, frequency=0.2)
    g1, o1 = capture(lambda: ops.process_logits(dx, history=dh, lengths=n, **kw))
    g2, o2 = capture(lambda: ops.process_logits(dy, history=dh, lengths=n, **kw))
    for length in (0, 1, 57, 400):
        n.fill_(length)
        g1.replay()
        g2.replay()
        for (got, tok), z in ((o1, x), (o2, y)):
            exp, exp_tok = ref.logits(z, history=h, lengths=torch.tensor([length]), **kw)
            assert torch.equal(got.cpu(), exp.to(BF)) and torch.equal(tok.cpu(), exp_tok)


def test_the_three_repeat_bit_for_bit(ops):
    q, k, v, words, cap = ta_inputs(20, 3000, 32, 8, 128, BF, "tree")
    args = [x.to(DEV) for x in (q, k, v)] + [torch.tensor([3000], device=DEV), words.to(DEV), 32, 8, 128, 0.09]
    x, h, _ = pl_inputs(20, 32000, 900, BF)
    first = ops.tree_attn(*args), *ops.process_logits(x.to(DEV), history=h.to(DEV), repetition=1.1, frequency=0.1)
    for _ in range(5):
        again = ops.tree_attn(*args), *ops.process_logits(x.to(DEV), history=h.to(DEV), repetition=1.1, frequency=0.1)
        for a, b in zip(first, again):
            assert torch.equal(a, b)
