"""Sequences of one key: softmax has nothing to distribute, so dq and dk are zero, not rounding of dP - delta."""
import pytest
import torch

from apla_amd import ops
from test_attn_mod_gpu import DT, SCALE, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("S,nq,Hq,Hkv", [(1, 1, 1, 1), (31, 1, 2, 2), (40, 3, 6, 2), (2, 150, 4, 1)])
def test_scores_of_a_single_key_have_no_gradient(S, nq, Hq, Hkv, cap, dtype):
    dt = DT[dtype]
    q, k, v, do = rnd((S * nq, Hq * 64), dt, 1, 2.0).cuda(), rnd((S, Hkv * 64), dt, 2).cuda(), rnd((S, Hkv * 64), dt, 3).cuda(), rnd((S * nq, Hq * 64), dt, 4).cuda()
    mod = ops.ScoreMod(softcap=cap, slopes=torch.ones(Hq, device="cuda"))
    with ops.use_half(dt):
        o, lse = ops.attn_mod_fwd(q, k, v, Hq, Hkv, SCALE, mod, batch=S)
        dq, dk, dv = ops.attn_mod_bwd(q, k, v, o, do, lse, Hq, Hkv, SCALE, mod, batch=S)
        assert bool((dq == 0).all()) and bool((dk == 0).all())
        want = do.double().view(S, nq, Hkv, Hq // Hkv, 64).sum((1, 3)).view(S, Hkv * 64)
        size = do.double().abs().view(S, nq, Hkv, Hq // Hkv, 64).sum((1, 3)).view(S, Hkv * 64)
        # weights of 1, to 2^-20 from lse; 16 products at a time are added in fp32; one rounding of the result
        assert bool(((dv.double() - want).abs() <= torch.finfo(dt).eps / 2 * want.abs() + (2.0 ** -20 + nq * Hq * 2.0 ** -24) * size).all())
        v[0, 5] = float("nan")
        o, lse = ops.attn_mod_fwd(q, k, v, Hq, Hkv, SCALE, mod, batch=S)
        dq, dk, _ = ops.attn_mod_bwd(q, k, v, o, do, lse, Hq, Hkv, SCALE, mod, batch=S)
        assert bool(torch.isnan(dq[0, :64]).all()) and bool(torch.isnan(dk[0, :64]).all()) and bool((dq[nq:] == 0).all())
