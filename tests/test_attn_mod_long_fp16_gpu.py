"""fp16 over many keys: weights far below fp16's normal range (2^-14) keep its relative precision, forward and backward.

u = 2^-11: half a step.  A weight or score gradient is rounded once (u), the result once more (u, 2^-25 absolute where it is below the normal range).  fp32 sums go by
16 products at a time: n / 16 additions of half a step 2^-24 relative to their partial sums, statistics and exponentials 2^-18."""
import pytest
import torch

from apla_amd import _lib, ops
from test_attn_mod_gpu import SCALE, rnd, within

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -11, torch.float16


def f_of(n):
    return (n / 16 + 64) * 2.0 ** -24 + 2.0 ** -18


def backward(q, k, v, do, H=1):
    with ops.use_half(HALF):
        c = [t.to(HALF).cuda() for t in (q, k, v, do)]
        o, lse = ops.attn_mod_fwd(*c[:3], H, 1, SCALE, batch=1)
        return (t.cpu().double() for t in ops.attn_mod_bwd(*c[:3], o, c[3], lse, H, 1, SCALE, batch=1))


@pytest.mark.parametrize("n", [50000, 70002, 300008])
def test_gradients_of_uniform_weights(n):
    """q and k use other columns, so every weight is 1 / n; v = +-2^-9 by halves, so o = 0, dS = +-(dO.v) / n and every sum below has terms of one sign: rounding errors of
    equal numbers do not average out."""
    g, nq = torch.Generator().manual_seed(1), 100
    sign = torch.ones(n, 1).double()
    sign[n // 2:] = -1
    q, k, a = torch.zeros(nq, 64).double(), torch.zeros(n, 64).double(), torch.randint(1, 3, (32,), generator=g).double()
    q[:, 32:] = torch.randint(8, 16, (nq, 32), generator=g).double()
    k[:, :32] = sign * a
    v, do = sign.expand(n, 64) * 2.0 ** -9, torch.randint(1, 9, (nq, 64), generator=g).double()
    x = do.sum(1, keepdim=True) * 2.0 ** -9
    dq, dk, dv = backward(q, k, v, do)
    want = torch.zeros(nq, 64).double()
    want[:, :32] = SCALE * x * a
    within(dq, want, (2 * U + f_of(n)) * want.abs() + 2.0 ** -25, "dq")
    want = SCALE / n * sign * (x * q).sum(0)
    within(dk, want, (2 * U + f_of(nq)) * want.abs() + 2.0 ** -25, "dk")
    want = (do.sum(0) / n).expand(n, 64)
    within(dv, want, (2 * U + f_of(nq)) * want.abs() + 2.0 ** -25, "dv")


@pytest.mark.parametrize("nq,n,H", [(100, 70002, 1), (600, 20000, 2)])
def test_score_gradients_near_the_end_of_the_range(nq, n, H):
    """Two keys share one row's weight, with score gradients of +-10240: results as finite as they are over few keys."""
    q, k, v, do = torch.zeros(nq, H * 64).double(), torch.zeros(n, 64).double(), torch.zeros(n, 64).double(), torch.zeros(nq, H * 64).double()
    q[:, 40:48] = k[:2, 40:48] = 16
    k[0, 0], k[1, 0], v[0], v[1], do[5, :64] = 1, -1, 16, -16, 20
    dq, dk, dv = backward(q, k, v, do, H)
    wq, wk, wv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    wq[5, 0] = 2 * SCALE * 10240
    wk[0, 40:48], wk[1, 40:48] = SCALE * 10240 * 16, -SCALE * 10240 * 16
    wv[:2] = 10
    for got, want, size in ((dq, wq, SCALE * 20480 * 16), (dk, wk, SCALE * 10240 * 16), (dv, wv, 20)):
        within(got, want, 2 * U * want.abs() + f_of(n) * size * (want != 0) + (want == 0) * 2.0 ** -18 * size, "gradient")


@pytest.mark.parametrize("nq,n,H", [(300, 9000, 2), (600, 20000, 1)])
def test_gradients_of_random_rows(nq, n, H):
    """Every element, weights of all sizes: relative precision down to a quarter of 1 / n, below that steps of that size."""
    q, k, v, do = rnd((nq, H * 64), HALF, 1, 2.0), rnd((n, 64), HALF, 2), rnd((n, 64), HALF, 3), rnd((nq, H * 64), HALF, 4)
    dq, dk, dv = backward(q, k, v, do, H)
    K, V = k.double(), v.double()
    wk, wv, bk, bv = (torch.zeros(n, 64).double() for _ in range(4))
    step, f = U * 2.0 ** -14 * 4096 / n, f_of(n) + 2.0 ** -17
    for h in range(H):
        c = slice(64 * h, 64 * h + 64)
        Q, D = q[:, c].double(), do[:, c].double()
        P = torch.softmax(Q @ K.t() * SCALE, 1)
        W = P @ V
        dP = D @ V.t()
        dS = P * (dP - (D * W).sum(1, keepdim=True))
        E = (D.abs() * ((U + f) * (P @ V.abs()) + U * W.abs())).sum(1, keepdim=True) + f * (D.abs() @ V.abs().t())       # of dP - delta
        eds = (U + f) * dS.abs() + P * E + step
        want = SCALE * dS @ K
        within(dq[:, c], want, SCALE * (eds @ K.abs()) + (U + f) * want.abs() + 2.0 ** -25, f"dq of head {h}")
        wk, bk = wk + SCALE * dS.t() @ Q, bk + SCALE * eds.t() @ Q.abs()
        wv, bv = wv + P.t() @ D, bv + ((U + f) * P + step).t() @ D.abs()
    within(dk, wk, bk + U * wk.abs() + 2.0 ** -25, "dk")
    within(dv, wv, bv + U * wv.abs() + 2.0 ** -25, "dv")


@pytest.mark.parametrize("H,nq", [(1, 1), (66, 1), (66, 3)])
def test_forward_of_many_small_weights_next_to_a_large_one(H, nq):
    """One key of weight 1 (value 0) and n of weight w = 2^-20.6 (value 1): o = n w / (1 + n w) though w is ten and a half of fp16's smallest steps."""
    n = 1 << 18
    q, k, v = torch.zeros(nq, H * 64), torch.zeros(n + 1, 64), torch.ones(n + 1, 64)
    q[:, ::64], k[0, 0], v[0] = 16, 7.140625, 0
    w = torch.exp(torch.tensor(-16 * 7.140625 * SCALE, dtype=torch.float64))
    a = _lib.AttnMod()
    a.S, a.Hq, a.Hkv, a.max_q, a.max_k = 1, H, 1, nq, n + 1
    with ops.use_half(HALF):
        assert _lib.lib().apla_attn_mod_few_rows(a) == (H == 1)
        o, lse = ops.attn_mod_fwd(*(t.to(HALF).cuda() for t in (q, k, v)), H, 1, SCALE, batch=1)
    want = float(n * w / (1 + n * w))
    # a lane adds n / 2 weights one by one: half a step 2^-24 each, relative to the sum so far
    assert float((o.double() - want).abs().max()) <= (2 * U + n / 2 * 2.0 ** -25 + f_of(n)) * want
    assert float((lse.double() - float(torch.log1p(n * w)) - 16 * 7.140625 * SCALE).abs().max()) <= 2.0 ** -19 * 16 + n / 2 * 2.0 ** -25
