"""``norm_rope_scatter`` over a whole prompt: a warp takes all heads of a token, so
its copies go several times around their ring, and from Q's chunks on to K's and V's
(with few tokens a warp has one chunk)."""
import pytest
import torch

import drafted_ref as ref
from test_gpu_drafted_ops import BF, DEV, HF, nr_inputs, nr_split, status_word

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["fp32", "ref"])
@pytest.mark.parametrize("n,hq,hkv,d,r,dt,norm,il", [
    (3607, 32, 8, 128, 128, BF, True, False),     # 12 chunks of a token for one warp
    (3600, 32, 8, 128, 128, BF, False, False),
    (4001, 28, 4, 80, 64, HF, True, True),
    (3559, 5, 2, 256, 64, BF, True, False),
    (3553, 64, 1, 16, 16, HF, False, True),
    (1999, 32, 8, 128, 128, BF, True, True),      # two warps share a token
    (1301, 7, 7, 128, 96, HF, True, False),       # three
])
def test_norm_rope_scatter_prompt(n, hq, hkv, d, r, dt, norm, il, mode):
    """Against 64 bits, with padding tokens (row -1) and tokens whose position or
    row lies outside among the others: nothing of those is written."""
    from cacheblend import ops
    qkv, rows, pos, w, kc, vc, tab = (x.to(DEV) if isinstance(x, torch.Tensor) else x
                                      for x in nr_inputs(n, hq, hkv, d, r, dt, norm))
    w = [None if x is None else x.to(DEV) for x in w]
    cap = kc.shape[0]
    call_rows, call_pos = rows.clone(), pos.clone()
    call_rows[3::7] = -1
    call_rows[5::700], call_rows[6::700], call_pos[8::700], call_pos[9::700] = cap, -2, 4000, -1
    lost = torch.zeros(n, dtype=torch.bool, device=DEV)
    for k, step in ((3, 7), (5, 700), (6, 700), (8, 700), (9, 700)):
        lost[k::step] = True
    kept = ~lost
    dk, dv = kc.clone(), vc.clone()
    out = torch.full((n, hq * d), 7.0, dtype=dt, device=DEV)
    for give_bad in (False, True):
        st = status_word()
        use_pos = call_pos if give_bad else pos
        use_rows = call_rows if give_bad else torch.where(lost, -1, rows)
        ops.norm_rope_scatter(*nr_split(qkv, hq, hkv, d), use_pos, use_rows, hq, hkv, d, tab, dk, dv, *w, eps=1e-5,
                              interleaved=il, q_out=out, mode=mode, status=st)
        assert int(st.item()) == (1 if give_bad else 0)
        assert (out[lost] == 7).all()
        qs, ks, vs = nr_split(qkv, hq, hkv, d)
        for x, heads, weight, got in ((qs, hq, w[0], out), (ks, hkv, w[1], dk[rows])):
            z, mag = ref.norm_rope(x[kept], heads, d, weight, 1e-5, tab, pos[kept], il)
            err = (got[kept].double() - z).abs()
            assert (err <= ref.norm_rope_bound(z, mag, dt, mode)).all()
        assert torch.equal(dv[rows[kept]], vs[kept])
        rest = torch.ones(cap, dtype=torch.bool, device=DEV)
        rest[rows[kept]] = False
        assert torch.equal(dk[rest], kc[rest]) and torch.equal(dv[rest], vc[rest])
        dk.copy_(kc), dv.copy_(vc), out.fill_(7.0)
