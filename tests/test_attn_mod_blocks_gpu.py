"""The 128-row forward of attention with modified scores, and lists of key tiles that take more than one pass, against the 64-bit restatement.

The forward takes few rows or few blocks through another kernel (apla_attn_mod_few_rows), so every case here has enough sequences or heads, and asks.  Bounds: those
of test_attn_mod_gpu.py, whose run_case compares every output."""
import pytest
import torch

from apla_amd import _lib, ops
from oracle import mod_oracle as O
from test_attn_mod_gpu import DT, SCALE, rnd, run_case, within

pytestmark = pytest.mark.gpu
SHORT = [2, 1, 3, 1] * 9        # one block each: with them the longer sequences of a case run in 128-row blocks


def in_blocks(S, Hq, Hkv, max_q, max_k):
    a = _lib.AttnMod()
    a.S, a.Hq, a.Hkv, a.max_q, a.max_k = S, Hq, Hkv, max_q, max_k
    return _lib.lib().apla_attn_mod_few_rows(a) == 0


def case(dt, lq, lk, Hq, Hkv, **kw):
    assert in_blocks(len(lq), Hq, Hkv, max(lq), kw.get("cap_k") or max(lk))
    return run_case(dt, lq, lk, Hq, Hkv, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("bias", [0, 1, 2, 3])
@pytest.mark.parametrize("mask", ["none", "causal", "prefix", "docs", "causal_docs", "mixed_docs"])
def test_every_modification(mask, bias, cap, dtype):
    kw = dict(causal="causal" in mask or mask == "prefix", prefix=70 if mask == "prefix" else None,
              docs="mixed" if "mixed" in mask else "sorted" if "docs" in mask else None)
    case(DT[dtype], [150, 33] + SHORT, [150, 33] + SHORT, 4, 2, cap=cap, bias=bias, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens", [[64], [65, 31], [127, 128, 129], [1, 300, 17], [0, 70, 0, 5]], ids=str)
def test_lengths(lens, dtype):
    case(DT[dtype], lens + SHORT, lens + SHORT, 2, 2)
    case(DT[dtype], lens + SHORT, lens + SHORT, 3, 1, causal=True, bias=1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nq,nk,Hq,Hkv", [(40, 300, 4, 2), (20, 5, 4, 2), (130, 65, 3, 1), (33, 1, 2, 2)])
def test_queries_and_keys_of_different_lengths(nq, nk, Hq, Hkv, dtype):
    S = 18 if Hq > 2 else 34
    for kw in (dict(), dict(causal=True, bias=1, cap=20.0), dict(causal=True, prefix=min(nk, 9))):
        case(DT[dtype], [nq] * S, [nk] * S, Hq, Hkv, packed=False, train=kw == {}, **kw)


@pytest.mark.parametrize("docs", [None, "sorted"])
def test_cache_with_used_lengths(docs):
    """Keys past len_k hold NaN / inf; caches may hold nothing yet."""
    lk = [290, 70, 64, 40, 41, 128, 129] + [40] * 3
    case(torch.bfloat16, [40] * 10, lk, 8, 2, cap=30.0, bias=1, causal=True, cap_k=300, docs=docs, poison=True)
    case(torch.float16, [40] * 10, lk, 8, 2, cap_k=300, docs=docs, poison=True, train=False)
    case(torch.bfloat16, [35] * 17, [0, 70, 0, 64, 1] + [36] * 12, 4, 2, causal=True, cap_k=100, poison=True, train=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_non_finite_values_in_masked_places(dtype):
    case(DT[dtype], [150, 200] + SHORT, [150, 200] + SHORT, 2, 1, docs="sorted", causal=True, poison=True)
    case(DT[dtype], [150, 200] + SHORT, [150, 200] + SHORT, 2, 2, docs="mixed", cap=5.0, bias=2, poison=True)
    dt, n, H = DT[dtype], 100, 66
    q, k, v = (rnd((n, H * 64), dt, s).cuda() for s in range(3))
    bad_k, bad_v = k.clone(), v.clone()
    bad_v[60, 3::64], bad_v[70, 9::64], bad_k[80] = float("inf"), float("nan"), float("-inf")
    assert in_blocks(1, H, H, n, n)
    mod = ops.ScoreMod(causal=True)
    with ops.use_half(dt):
        o, lse = ops.attn_mod_fwd(q, k, v, H, H, SCALE, mod, batch=1)
        ob, lb = ops.attn_mod_fwd(q, bad_k, bad_v, H, H, SCALE, mod, batch=1)
    assert torch.equal(o[:60], ob[:60]) and torch.equal(lse[:, :80], lb[:, :80])
    a, b = o.view(n, H, 64), ob.view(n, H, 64)
    assert not torch.isfinite(b[60:, :, 3]).any() and not torch.isfinite(b[70:, :, 9]).any() and torch.equal(a[60:80, :, 20:], b[60:80, :, 20:])


@pytest.mark.parametrize("cap", [300.0, 9e5])
def test_caps_far_above_the_scores_change_nothing(cap):
    """As the test of that name for few rows: cap tanh(s / cap) to the fp32 rounding of the scores (2^-16 in all, derived there), in whole and masked tiles."""
    T, H = 512, 20
    q, k, v = (rnd((T, H * 64), torch.bfloat16, 40 + i).cuda() for i in range(3))
    s = torch.stack([q[:, 64 * h:64 * h + 64].double() @ k[:, 64 * h:64 * h + 64].double().t() * 0.125 for h in range(H)])
    assert float(s.abs().max()) <= 12 and in_blocks(1, H, H, T, T)
    want = torch.logsumexp(cap * torch.tanh(s / cap), 2)
    for mod in (ops.ScoreMod(softcap=cap), ops.ScoreMod(softcap=cap, slopes=torch.zeros(H, device="cuda"))):
        _, lse = ops.attn_mod_fwd(q, k, v, H, H, 0.125, mod, batch=1)
        assert float((lse.double() - want).abs().max()) <= 2.0 ** -16


def test_row_strides_up_to_their_limit():
    """Rows 2^24 - 8 elements apart: the same bits as from dense rows."""
    T, ld, H = 70, (1 << 24) - 8, 66
    wide = torch.as_strided(torch.empty(T * ld, dtype=torch.bfloat16, device="cuda"), (T, 3 * H * 64), (ld, 1))
    wide.copy_(rnd((T, 3 * H * 64), torch.bfloat16, 50))
    flat = wide.contiguous()
    assert in_blocks(1, H, H, T, T)
    res = [ops.attn_mod_fwd(*x.chunk(3, 1), H, H, 0.125, ops.ScoreMod(causal=True, slopes=torch.ones(H, device="cuda")), batch=1) for x in (wide, flat)]
    assert all(torch.equal(a, b) for a, b in zip(*res))


def documents_past_the_list(n):
    """Ids of n tokens: ordinary documents, one that lies on both sides of key 16384 (the 256 tiles of one pass), one of two pieces thousands of tokens apart, one
    behind key 16384 only, padding between and at the end."""
    r = torch.Generator().manual_seed(7)
    d = torch.repeat_interleave(torch.arange(n), torch.randint(1, 600, (n,), generator=r))[:n] + 10
    d[16000:16700] = 3
    d[100:400] = d[16900:17100] = 4
    d[17100:17200] = 5
    d[17200:17300] = -2
    d[-50:] = -1
    return d.int()


@pytest.mark.parametrize("dtype,Hq,Hkv,causal,cap,bias", [("bf16", 2, 1, False, 0.0, 0), ("fp16", 2, 2, True, 20.0, 1), ("bf16", 4, 4, True, 0.0, 1)])
def test_documents_over_more_tiles_than_one_list_holds(dtype, Hq, Hkv, causal, cap, bias):
    """Every row and key of a packed row of 17 600 tokens, document by document; a few heads have their blocks' tiles split as well, four heads do not."""
    dt, n, G = DT[dtype], 17600, Hq // Hkv
    doc = documents_past_the_list(n)
    q, k, v, do = rnd((n, Hq * 64), dt, 1, 2.0), rnd((n, Hkv * 64), dt, 2), rnd((n, Hkv * 64), dt, 3), rnd((n, Hq * 64), dt, 4)
    k[doc < 0], v[doc < 0], do[doc < 0] = float("nan"), float("inf"), float("nan")
    slopes = 0.5 ** (torch.arange(Hq) + 6.0)
    mod = ops.ScoreMod(softcap=cap, slopes=slopes.cuda() if bias else None, doc_q=doc.cuda(), doc_k=doc.cuda(), causal=causal)
    assert in_blocks(1, Hq, Hkv, n, n)
    with ops.use_half(dt):
        c = [t.cuda() for t in (q, k, v, do)]
        runs = []
        for _ in range(2):
            o, lse = ops.attn_mod_fwd(*c[:3], Hq, Hkv, SCALE, mod, batch=1)
            runs.append((o, lse, *ops.attn_mod_bwd(*c[:3], o, c[3], lse, Hq, Hkv, SCALE, mod, batch=1)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    o, lse, dq, dk, dv = (t.cpu().double() for t in runs[0])
    u, floor = torch.finfo(dt).eps / 2, (2.0 ** -24 if dt == torch.float16 else 2.0 ** -126)
    assert all(bool((t[doc < 0] == 0).all()) for t in (o, dq, dk, dv)) and bool((lse[:, doc < 0] == -float("inf")).all())
    for i in doc[doc >= 0].unique():
        at = (doc == i).nonzero().flatten()
        m = at.numel()
        f = (m * (G + 1) + 64) * 2.0 ** -24 + 2.0 ** -18
        see = torch.ones(m, m, dtype=torch.float64)
        see = see.tril() if causal else see
        for hk in range(Hkv):
            K, V = (t[at, hk * 64:hk * 64 + 64].double() for t in (k, v))
            sums = [torch.zeros(m, 64, dtype=torch.float64) for _ in range(4)]
            for h in range(hk * G, hk * G + G):
                at_h = slice(h * 64, h * 64 + 64)
                Q, D = q[at, at_h].double(), do[at, at_h].double()
                raw = Q @ K.t() * SCALE
                t = torch.tanh(raw / cap) if cap else torch.zeros_like(raw)
                z = cap * t if cap else raw
                if bias:
                    z = z - float(slopes[h]) * (at[:, None] - at[None]).abs()
                z = z.masked_fill(see == 0, -float("inf"))
                L = torch.logsumexp(z, 1)
                P = torch.exp(z - L[:, None])
                W = P @ V
                dS = P * (D @ V.t() - (D * W).sum(1, keepdim=True)) * (1 - t * t)
                A, aD = P @ V.abs(), D.abs()
                eo = (u + 2 * f) * A + u * W.abs() + floor * (see @ V.abs() + 1)
                within(o[at, at_h], W, eo, f"o of head {h}, document {int(i)}")
                within(lse[h, at], L, 2.0 ** -21 * (L.abs() + 2 * cap + 40) + 2 * f, f"lse of head {h}, document {int(i)}")
                E = (aD * eo).sum(1, keepdim=True) + f * (aD * A).sum(1, keepdim=True)
                flushed = 2.0 ** -126 * (aD @ V.abs().t() + (aD * A).sum(1, keepdim=True))
                eds = flushed + (u + 3 * f) * dS.abs() + P * (E + 2 * f * (aD @ V.abs().t()) + 2 * f * (aD * A).sum(1, keepdim=True)) + floor * see
                dQ = SCALE * dS @ K
                within(dq[at, at_h], dQ, 1.01 * SCALE * (eds @ K.abs()) + u * dQ.abs() + floor, f"dq of head {h}, document {int(i)}")
                sums[0] += SCALE * dS.t() @ Q
                sums[1] += P.t() @ D
                sums[2] += 1.01 * SCALE * (eds.t() @ Q.abs())
                sums[3] += ((u + 3 * f) * P + floor * see).t() @ aD
            c2 = slice(hk * 64, hk * 64 + 64)
            within(dk[at, c2], sums[0], sums[2] + u * sums[0].abs() + floor, f"dk of head {hk}, document {int(i)}")
            within(dv[at, c2], sums[1], sums[3] + u * sums[1].abs() + floor, f"dv of head {hk}, document {int(i)}")
