"""The operators behind decoding with drafted tokens where the cache itself holds
NaN or infinities in places that are visible, held to the same 64-bit formulas
and bounds as ``test_gpu_drafted_ops``."""
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


@pytest.mark.parametrize("t,n_ctx,hq,hkv,d,dt", [
    (5, 300, 16, 4, 128, BF),           # one Q tile, a key tile per CTA
    (5, 300, 16, 4, 64, HF),
    (33, 300, 16, 4, 128, BF),          # two Q tiles
    (2, 520, 76, 76, 64, BF),           # one CTA takes all key tiles of a head, one Q tile ...
    (70, 520, 152, 76, 64, BF),         # ... and two
])
def test_tree_attn_nonfinite_context_keys(ops, t, n_ctx, hq, hkv, d, dt):
    """A visible context row whose K holds NaN makes every row of its head NaN; one
    whose score is +inf makes the row NaN (inf - inf), one whose score is -inf has
    weight 0 exactly, whatever finite value its V holds -- at every column of a key
    tile that is all context."""
    g = torch.Generator().manual_seed(t + hq)
    cap, group = n_ctx + t + 5, hq // hkv
    q = (torch.randn((t, hq * d), generator=g) * 1.5).to(dt)
    q[q == 0] = 1
    k, v = (torch.randn((cap, hkv * d), generator=g).to(dt) for _ in range(2))
    words = ops.tree_words([-1] + [max(0, i - 2) for i in range(1, t)])[0]
    n = n_ctx + t
    sees = torch.ones((t, n), dtype=torch.bool)
    sees[:, n_ctx:] = ref.visible(words, t)
    sees = sees.to(DEV)[None, :, None, :]
    q, words, n_dev = q.to(DEV), words.to(DEV), torch.tensor([n_ctx], device=DEV)
    huge = 3e38 if dt == BF else 6e4
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")])
    for col in range(32):
        row = 128 + 32 * (col % 4) + col
        k2, v2 = k.clone(), v.clone()
        for h in range(hkv):
            if h % 4 < 3:                                    # every fourth head stays as it is
                k2[row, h * d + 5] = bad[h % 4]
                v2[row, h * d:(h + 1) * d] = huge
        k2, v2 = k2.to(DEV), v2.to(DEV)
        got = ops.tree_attn(q, k2, v2, n_dev, words, hq, hkv, d, d ** -0.5)
        kk = k2[:n].double().view(n, hkv, d).permute(1, 2, 0)
        vv = v2[:n].double().view(n, hkv, d).transpose(0, 1)
        qq = q.double().view(t, hkv, group * d).transpose(0, 1).reshape(hkv, t * group, d)
        s = (qq @ kk * d ** -0.5).view(hkv, t, group, n).masked_fill(~sees, -torch.inf)
        p = torch.softmax(s, -1).view(hkv, t * group, n)
        out, A = ((p @ x).view(hkv, t, group * d).transpose(0, 1).reshape(t, hq * d) for x in (vv, vv.abs()))
        assert torch.equal(torch.isnan(got), torch.isnan(out)), col
        ok = ~torch.isnan(out)
        assert ok.any() and not ok.all()
        bound = ref.tree_bound(out, A, n, dt, huge)
        assert ((got.double() - out).abs() <= bound)[ok].all(), col


@pytest.mark.parametrize("t,n_ctx,hq,hkv,d,dt", [
    (6, 0, 8, 2, 64, BF), (6, 3, 8, 2, 128, HF),      # one key tile: the attention kernel writes the output
    (6, 300, 8, 2, 128, BF),                          # several splits, merged
    (6, 900, 76, 76, 64, BF),                         # one CTA for all tiles, both slots joined
    (50, 300, 8, 2, 64, HF),                          # two Q tiles
])
def test_tree_attn_rows_of_infinitely_low_scores(ops, t, n_ctx, hq, hkv, d, dt):
    """A row that sees keys, all with a score of -inf, is 0 / 0 as in the formula; one
    that sees nothing is 0; one finite score among them has all the weight."""
    g = torch.Generator().manual_seed(t + n_ctx)
    cap = n_ctx + t + 5
    q = (torch.rand((t, hq * d), generator=g) + 0.5).to(dt)
    k = torch.full((cap, hkv * d), -float("inf"), dtype=dt)
    v = torch.randn((cap, hkv * d), generator=g).to(dt)
    k[n_ctx + 2] = 0.25                                # node 2's own key
    words = torch.zeros((t, (t + 31) // 32), dtype=torch.int32)
    words[0, 0], words[2, 0], words[3, 0], words[5, 0] = 1, 4, 0b1110, -1 << (t % 32) if t < 32 else 0
    got = ops.tree_attn(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([n_ctx], device=DEV), words.to(DEV), hq, hkv, d,
                        0.1).cpu()
    low = torch.full((t,), n_ctx > 0)                  # the context alone
    low[0], low[2], low[3] = True, False, False
    assert torch.isnan(got[low]).all()
    one = v[n_ctx + 2].view(hkv, 1, d).expand(hkv, hq // hkv, d).reshape(-1)
    assert torch.equal(got[2], one) and torch.equal(got[3], one)
    rest = ~low
    rest[2:4] = False
    assert (got[rest] == 0).all()                      # (bits behind the tree are no rows)
