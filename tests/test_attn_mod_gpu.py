"""Attention with modified and masked scores against the 64-bit restatement (oracle/mod_oracle.py).

Bounds, per element, with u = finfo.eps / 2 of the 16-bit type: the weights P and the gradients dS are rounded to 16 bits as MFMA operands
(u relative; below the normal range an absolute 2^-25 in fp16, and in bf16, as in the fp32
arithmetic before it, numbers under 2^-126 are flushed) and every result is rounded once; o enters delta = rowsum(dO o O)
rounded.  fp32 sums and the score arithmetic add f = (n + 64) 2^-24 + 2^-18 (scores up to ~40: 40 log2(e) 2^-23 plus the exponential's 2^-22)
relative to the sums of magnitudes.  So with A = P |v|:  |do| <= (u + f) A + u |o| + floor;  E = |dO| . (u + f) (A + |o|) the error of delta:
|d dq| <= scale ((u + 2f) |dS| |k| + P (E + f |dO| |v|) |k|) + u |dq|, and likewise for dk and dv."""
import math

import pytest
import torch

from apla_amd import ops
from apla_amd._lib import AplaHipError
from oracle import mod_oracle as O

pytestmark = pytest.mark.gpu


def within(got, want, bound, what):
    """|got - want| <= bound everywhere; names the worst place."""
    off = (got - want).abs() / bound
    if not bool((off <= 1).all()):
        i = int(torch.nan_to_num(off, float("inf")).argmax())
        at = [int(x) for x in torch.unravel_index(torch.tensor(i), off.shape)]
        pytest.fail(f"{what} at {at}: {float(got.flatten()[i])!r}, expected {float(want.flatten()[i])!r} within {float(bound.flatten()[i]):.3e}; "
                    f"{int((~(off <= 1)).sum())} of {off.numel()} places are off")


DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
SCALE = 0.125


def rnd(shape, dt, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dt)


def documents(n, kind, seed=0):
    if kind == "sorted":         # lengths around 40, the last eighth padding
        r = torch.Generator().manual_seed(seed + n)
        d = torch.repeat_interleave(torch.arange(n), torch.randint(1, 80, (n,), generator=r))[:n]
        d[n - n // 8:] = -1
        return d.int()
    if kind == "mixed":          # ids in no order
        return (torch.arange(n) * 7 % 5).int() - (torch.arange(n) % 11 == 3).int() * 9
    return torch.zeros(n, dtype=torch.int32)


def run_case(dt, lq, lk, Hq, Hkv, *, cap=0.0, bias=0, causal=False, prefix=None, docs=None, packed=True, cap_k=None, train=True, poison=False, qscale=2.0):
    """Runs one configuration, compares every output with the oracle, returns the outputs."""
    S, Tq = len(lq), sum(lq)
    offs = lambda n: [sum(n[:i]) for i in range(len(n) + 1)]       # noqa: E731
    oq, ok = offs(lq), (offs(lk) if cap_k is None else [cap_k * s for s in range(S + 1)])
    Tk = ok[-1]
    q, k, v, do = rnd((Tq, Hq * 64), dt, 1, qscale), rnd((Tk, Hkv * 64), dt, 2), rnd((Tk, Hkv * 64), dt, 3), rnd((Tq, Hq * 64), dt, 4)
    slopes = (0.5 ** (torch.arange(Hq) % 5 + 1).float()) if bias else None
    pos_q = pos_k = None
    if bias == 2:                # coordinates on a grid; bias 3: one coordinate, not in order
        pos_k = torch.cat([torch.stack((torch.arange(n) // 9, torch.arange(n) % 9), 1) for n in [ok[s + 1] - ok[s] for s in range(S)]]).float()
    elif bias == 3:
        pos_k = torch.cat([(torch.arange(ok[s + 1] - ok[s]) * 13 % 101).float() * 0.5 for s in range(S)])
    if pos_k is not None:
        pos_q = pos_k if lq == lk and cap_k is None else torch.cat([pos_k[ok[s] + lk[s] - lq[s]:][:lq[s]] for s in range(S)])
    doc_k = torch.cat([documents(ok[s + 1] - ok[s], docs, s) for s in range(S)]) if docs else None
    doc_q = (doc_k if lq == lk and cap_k is None else torch.cat([doc_k[ok[s] + lk[s] - lq[s]:][:lq[s]] for s in range(S)])) if docs else None
    pre = None if prefix is None else torch.tensor([min(prefix, max(lk)) * (s + 1) // S for s in range(S)], dtype=torch.int32)
    see = [O.visible(lq[s], lk[s], causal, 0 if pre is None else int(pre[s]), None if doc_q is None else doc_q[oq[s]:oq[s + 1]],
                     None if doc_k is None else doc_k[ok[s]:ok[s] + lk[s]]) for s in range(S)]
    if poison:                   # whatever nobody sees, and the upstream gradient of rows that see nothing, is not finite
        seen, rows = torch.zeros(Tk, dtype=torch.bool), torch.zeros(Tq, dtype=torch.bool)
        for s in range(S):
            seen[ok[s]:ok[s] + lk[s]] = see[s].any(0)
            rows[oq[s]:oq[s + 1]] = see[s].any(1)
        k[~seen], v[~seen] = float("nan"), float("inf")
        do[~rows] = float("nan")
    cu = lambda n: torch.tensor(n, dtype=torch.int32, device="cuda")     # noqa: E731
    g = lambda t: None if t is None else t.cuda()                        # noqa: E731
    mod = ops.ScoreMod(softcap=cap, slopes=g(slopes), pos_q=g(pos_q), pos_k=g(pos_k), doc_q=g(doc_q), doc_k=g(doc_k), causal=causal, prefix=g(pre))
    if cap_k is not None:
        kw = dict(batch=S, len_k=cu(lk))
    elif packed:
        kw = dict(cu_q=cu(oq), cu_k=cu(ok), max_q=max(lq), max_k=max(lk))
    else:
        kw = dict(batch=S)
    qc, kc, vc, dc = q.cuda(), k.cuda(), v.cuda(), do.cuda()
    with ops.use_half(dt):
        o, lse = ops.attn_mod_fwd(qc, kc, vc, Hq, Hkv, SCALE, mod, **kw)
        o2, lse2 = ops.attn_mod_fwd(qc, kc, vc, Hq, Hkv, SCALE, mod, **kw)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
        grads = ops.attn_mod_bwd(qc, kc, vc, o, dc, lse, Hq, Hkv, SCALE, mod, **kw) if train else ()
        if train:
            assert all(torch.equal(a, b) for a, b in zip(grads, ops.attn_mod_bwd(qc, kc, vc, o, dc, lse, Hq, Hkv, SCALE, mod, **kw)))
    u, floor = torch.finfo(dt).eps / 2, (2.0 ** -24 if dt == torch.float16 else 2.0 ** -126)
    oc, lc, gc = o.cpu().double(), lse.cpu().double(), [x.cpu().double() for x in grads]
    if train:
        bk, bv = torch.zeros(Tk, Hkv * 64, dtype=torch.float64), torch.zeros(Tk, Hkv * 64, dtype=torch.float64)
        wk, wv = torch.zeros_like(bk), torch.zeros_like(bv)
    for s in range(S):
        f = (lk[s] + lq[s] * (Hq // Hkv) + 64) * 2.0 ** -24 + 2.0 ** -18
        rq, rk = slice(oq[s], oq[s + 1]), slice(ok[s], ok[s] + lk[s])
        dist = O.distance(lq[s], lk[s], None if pos_q is None else pos_q[rq], None if pos_k is None else pos_k[rk]) if bias else None
        for h in range(Hq):
            c, d = slice(h * 64, h * 64 + 64), slice(h // (Hq // Hkv) * 64, h // (Hq // Hkv) * 64 + 64)
            Q, K, V, D = q[rq, c].double(), k[rk, d].double(), v[rk, d].double(), do[rq, c].double()
            w = O.attend(Q, K, V, SCALE, see[s], cap, float(slopes[h]) if bias else 0.0, dist, D if train else None)
            nz = lambda t: torch.nan_to_num(t, 0.0, 0.0, 0.0)     # noqa: E731   (masked places may hold anything)
            V, K, D = nz(V).abs(), nz(K).abs(), nz(D).abs()
            A, seen = w["p"] @ V, see[s].double()
            within(oc[rq, c], w["o"], (u + 2 * f) * A + u * w["o"].abs() + floor * (seen @ V + 1), f"o of head {h}")
            empty = ~see[s].any(1)
            assert bool((lc[h, rq][empty] == -math.inf).all()) and bool((oc[rq, c][empty] == 0).all())
            L = w["lse"][~empty]
            within(lc[h, rq][~empty], L, 2.0 ** -21 * (L.abs() + (2 * cap if cap else 0) + 40) + 2 * f, f"lse of head {h}")
            if not train:
                continue
            E = (D * ((u + 2 * f) * A + u * w["o"].abs() + floor * (seen @ V + 1))).sum(1, keepdim=True) + f * (D * A).sum(1, keepdim=True)
            # (a weight under 2^-126 is flushed before it multiplies dP - delta, whose size is at most |dO||v| + |dO| A)
            flushed = 2.0 ** -126 * (D @ V.t() + (D * A).sum(1, keepdim=True))
            eds = flushed + (u + 3 * f) * w["ds"].abs() + w["p"] * (E + 2 * f * (D @ V.t()) + 2 * f * (D * A).sum(1, keepdim=True)) + floor * seen
            within(gc[0][rq, c], w["dq"], 1.01 * SCALE * (eds @ K) + u * w["dq"].abs() + floor, f"dq of head {h}")
            assert bool((gc[0][rq, c][empty] == 0).all())
            wk[rk, d] += w["dk"]
            wv[rk, d] += w["dv"]
            bk[rk, d] += 1.01 * SCALE * (eds.t() @ Q.abs())
            bv[rk, d] += ((u + 3 * f) * w["p"] + floor * seen).t() @ D
    if train:
        within(gc[1], wk, bk + u * wk.abs() + floor, "dk")
        within(gc[2], wv, bv + u * wv.abs() + floor, "dv")
    return o, lse, grads


LENGTHS = [[1], [2, 1, 3], [64], [65, 31], [127, 128, 129], [1, 300, 17], [197, 50]]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_packed_lengths(lens, dtype):
    run_case(DT[dtype], lens, lens, 2, 2)
    run_case(DT[dtype], lens, lens, 3, 1, causal=True, bias=1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("bias", [0, 1, 2, 3])
@pytest.mark.parametrize("mask", ["none", "causal", "prefix", "docs", "causal_docs", "mixed_docs"])
def test_every_modification(mask, bias, cap, dtype):
    kw = dict(causal="causal" in mask or mask == "prefix", prefix=70 if mask == "prefix" else None,
              docs="mixed" if "mixed" in mask else "sorted" if "docs" in mask else None)
    run_case(DT[dtype], [150, 33], [150, 33], 4, 2, cap=cap, bias=bias, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nq,nk,Hq,Hkv", [(1, 1, 1, 1), (1, 197, 3, 3), (1, 700, 8, 2), (4, 513, 8, 1), (3, 65, 6, 6), (40, 600, 4, 2), (20, 5, 2, 1)])
def test_queries_and_keys_of_different_lengths(nq, nk, Hq, Hkv, dtype):
    """Few queries against many keys (the forms split over the keys), and more queries than keys (causal rows that see nothing)."""
    for kw in (dict(), dict(causal=True, bias=1, cap=20.0), dict(causal=True, prefix=min(nk, 9))):
        run_case(DT[dtype], [nq, nq], [nk, nk], Hq, Hkv, packed=False, **kw)


@pytest.mark.parametrize("lens", [[0, 5, 0, 70, 0], [0, 0], [3, 0]])
def test_sequences_of_length_zero(lens):
    """Empty sequences between others, queries without keys, keys without queries."""
    if max(lens):
        run_case(torch.bfloat16, lens, lens, 2, 1, causal=True)
    run_case(torch.bfloat16, [4] * len(lens), [max(n, 1) if i == 1 else n for i, n in enumerate(lens)], 2, 2)
    run_case(torch.bfloat16, [max(n, 1) if i == 1 else n for i, n in enumerate(lens)], [66] * len(lens), 2, 2, docs=None)


@pytest.mark.parametrize("nq", [1, 3, 40])
@pytest.mark.parametrize("docs", [None, "sorted"])
def test_cache_with_used_lengths(nq, docs):
    """Keys past len_k are never looked at (they are NaN), their gradient rows stay 0, and caches may hold nothing yet."""
    lk = [1100, 70, 64, nq, 1]
    for train in (False, True):
        run_case(torch.bfloat16, [min(nq, 1)] * 5 if nq == 1 else [nq] * 5, [max(n, nq) for n in lk], 8, 2, cap=30.0, bias=1, causal=True, cap_k=1200, docs=docs,
                 train=train, poison=True)
    run_case(torch.bfloat16, [nq] * 3, [0, 70, 0], 4, 2, causal=True, cap_k=100, poison=True, train=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_non_finite_values_in_masked_places(dtype):
    """Padding documents hold NaN / inf in k, v and do; and a causal row does not notice an infinite value that only later rows see."""
    run_case(DT[dtype], [150, 200], [150, 200], 2, 1, docs="sorted", causal=True, poison=True)
    dt, n = DT[dtype], 100
    q, k, v, do = (rnd((n, 64), dt, s).cuda() for s in range(4))
    bad_k, bad_v, bad_q, bad_do = k.clone(), v.clone(), q.clone(), do.clone()
    bad_v[60, 3], bad_v[70, 9], bad_k[80] = float("inf"), float("nan"), float("-inf")
    mod = ops.ScoreMod(causal=True)
    with ops.use_half(dt):
        o, lse = ops.attn_mod_fwd(q, k, v, 1, 1, SCALE, mod, batch=1)
        ob, lb = ops.attn_mod_fwd(q, bad_k, bad_v, 1, 1, SCALE, mod, batch=1)
        assert torch.equal(o[:60], ob[:60]) and torch.equal(lse[:, :80], lb[:, :80])
        assert not torch.isfinite(ob[60:, 3]).any() and not torch.isfinite(ob[70:, 9]).any() and torch.equal(o[60:80, 20:], ob[60:80, 20:])
        # an early row's non-finite query or gradient reaches only the keys that this row sees
        bad_q[30, 5], bad_do[40, 7] = float("nan"), float("inf")
        ref = ops.attn_mod_bwd(q, k, v, o, do, lse, 1, 1, SCALE, mod, batch=1)
        got = ops.attn_mod_bwd(bad_q, k, v, o, bad_do, lse, 1, 1, SCALE, mod, batch=1)
        assert torch.equal(ref[0][41:], got[0][41:]) and torch.equal(ref[1][41:], got[1][41:]) and torch.equal(ref[2][41:], got[2][41:])
        assert not torch.isfinite(got[2][:41, 7]).any()


def test_strided_operands_and_outputs_and_rows_behind_the_last_sequence():
    """q, k, v as columns of fused rows, gradients into one fused buffer, class-token queries as strided rows; rows behind the last sequence stay."""
    dt, H, n = torch.bfloat16, 3, 90
    qkv, do = rnd((n + 10, 3 * H * 64), dt, 1).cuda(), rnd((n + 10, H * 64), dt, 2).cuda()
    cut = [qkv[:, i * H * 64:(i + 1) * H * 64] for i in range(3)]
    cu = torch.tensor([0, 30, n], dtype=torch.int32, device="cuda")
    kw = dict(cu_q=cu, cu_k=cu, max_q=60, max_k=60)
    o, lse = torch.full((n + 10, H * 64), 7.0, dtype=dt, device="cuda"), torch.full((H, n + 10), 7.0, device="cuda")
    ops.attn_mod_fwd(*cut, H, H, SCALE, None, o=o, lse=lse, **kw)
    assert bool((o[n:] == 7).all()) and bool((lse[:, n:] == 7).all())
    dense = [c[:n].contiguous() for c in cut]
    o1, l1 = ops.attn_mod_fwd(*dense, H, H, SCALE, None, **kw)
    assert torch.equal(o[:n], o1) and torch.equal(lse[:, :n], l1)
    o0, l0 = ops.attn_mod_fwd(*cut, H, H, SCALE, None, **kw)
    assert bool((o0[n:] == 0).all()) and bool((l0[:, n:] == float("-inf")).all())
    fused = torch.full_like(qkv, 7.0)
    parts = [fused[:, i * H * 64:(i + 1) * H * 64] for i in range(3)]
    ops.attn_mod_bwd(*cut, o, do, lse, H, H, SCALE, None, dq=parts[0], dk=parts[1], dv=parts[2], **kw)
    ref = ops.attn_mod_bwd(*dense, o1, do[:n].contiguous(), l1, H, H, SCALE, None, **kw)
    assert bool((fused[n:] == 7).all()) and all(torch.equal(p[:n], r) for p, r in zip(parts, ref))
    assert all(bool((g[n:] == 0).all()) for g in ops.attn_mod_bwd(*cut, o0, do, l0, H, H, SCALE, None, **kw))
    ops.attn_mod_bwd(*cut, o, do, lse, H, H, SCALE, None, dq=parts[0], dk=parts[1], dv=parts[2], zero_rest=True, **kw)
    assert bool((fused[n:] == 0).all()) and all(torch.equal(p[:n], r) for p, r in zip(parts, ref))
    two = qkv[:80].view(2, 40, -1)
    ocls, _ = ops.attn_mod_fwd(two[:, 0, :H * 64], cut[1][:80], cut[2][:80], H, H, SCALE, None, batch=2)
    full, _ = ops.attn_mod_fwd(cut[0][:80], cut[1][:80], cut[2][:80], H, H, SCALE, None, batch=2)
    assert bool(((ocls - full.view(2, 40, -1)[:, 0]).abs().float() <= 2.0 ** -7 * (full.view(2, 40, -1)[:, 0].abs().float() + 1)).all())


def test_equal_to_the_plain_attention_of_the_library():
    """Without modifications the operator is apla_attn_fwd / apla_attn_bwd up to the rounding of weights and results."""
    B, N, H, dt = 2, 197, 3, torch.bfloat16
    qkv, do = rnd((B * N, 3 * H * 64), dt, 1).cuda(), rnd((B * N, H * 64), dt, 2).cuda()
    cut = [qkv[:, i * H * 64:(i + 1) * H * 64] for i in range(3)]
    o, lse = ops.attn_fwd(qkv, B, N, H, SCALE)
    o2, lse2 = ops.attn_mod_fwd(*cut, H, H, SCALE, batch=B)
    assert bool(((o - o2).abs().float() <= 2.0 ** -7 * 4).all()) and bool(((lse.transpose(0, 1).reshape(H, -1) - lse2).abs() <= 1e-4).all())
    d = ops.attn_bwd(qkv, o, do, lse, B, N, H, SCALE).float()
    e = torch.cat(ops.attn_mod_bwd(*cut, o2, do, lse2, H, H, SCALE, batch=B), 1).float()
    assert float((d - e).norm() / d.norm()) <= 4 * 2.0 ** -8


def test_gradient_against_differences():
    """Directional derivatives of sum(w o) in 64 bits by central differences of the oracle, against the kernel's gradients."""
    dt, n, H = torch.float16, 70, 1
    q, k, v, w = (rnd((n, 64), dt, s) for s in range(4))
    see, dist = O.visible(n, n, True, 11), O.distance(n, n)
    mod = ops.ScoreMod(softcap=4.0, slopes=torch.tensor([0.125], device="cuda"), causal=True, prefix=torch.tensor([11], dtype=torch.int32, device="cuda"))
    with ops.use_half(dt):
        qc, kc, vc = q.cuda(), k.cuda(), v.cuda()
        o, lse = ops.attn_mod_fwd(qc, kc, vc, H, H, SCALE, mod, batch=1)
        g = [x.cpu().double() for x in ops.attn_mod_bwd(qc, kc, vc, o, w.cuda(), lse, H, H, SCALE, mod, batch=1)]
    val = lambda a, b, c: (O.attend(a, b, c, SCALE, see, 4.0, 0.125, dist)["o"] * w.double()).sum()      # noqa: E731
    base, h = [q.double(), k.double(), v.double()], 1e-4
    for i in range(3):
        d = rnd((n, 64), torch.float64, 10 + i)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        diff = (val(*up) - val(*down)) / (2 * h)
        assert abs(float(diff - (g[i] * d).sum())) <= 4 * 2.0 ** -11 * float(g[i].norm() * d.norm()) + 1e-6


def test_long_sequence_passes_the_tile_list_and_stays_deterministic():
    """More keys than one list of tiles holds (256 x 64), checked on rows against the oracle."""
    dt, n = torch.bfloat16, 16384 + 200
    q, k, v = rnd((3, 64), dt, 1, 2.0), rnd((n, 64), dt, 2), rnd((n, 64), dt, 3)
    big = rnd((n, 64), dt, 4, 2.0)
    big[[0, 9000, n - 1]] = q
    o, lse = ops.attn_mod_fwd(big.cuda(), k.cuda(), v.cuda(), 1, 1, SCALE, ops.ScoreMod(causal=True), batch=1)
    see = torch.zeros(3, n, dtype=torch.bool)
    for r, i in enumerate((0, 9000, n - 1)):
        see[r, :i + 1] = True
    w = O.attend(q.double(), k.double(), v.double(), SCALE, see)
    f = (n + 64) * 2.0 ** -24 + 2.0 ** -18
    got = o[[0, 9000, n - 1]].cpu().double()
    assert bool(((got - w["o"]).abs() <= (2.0 ** -8 + f) * (w["p"] @ v.double().abs()) + 2.0 ** -8 * w["o"].abs()).all())
    assert bool(((lse[0, [0, 9000, n - 1]].cpu().double() - w["lse"]).abs() <= 2.0 ** -21 * 60 + 2 * f).all())


def test_offsets_past_32_bits():
    """A cache of which the last keys lie more than 2^32 bytes (and 2^31 elements) behind its start: row stride of a wide fused buffer."""
    dt, n, wide = torch.bfloat16, 66000, 32832
    buf = torch.zeros(n, wide, dtype=dt, device="cuda")
    k, v, q = rnd((n, 64), dt, 1).cuda(), rnd((n, 64), dt, 2).cuda(), rnd((1, 64), dt, 3, 2.0).cuda()
    buf[:, wide - 128:wide - 64], buf[:, wide - 64:] = k, v
    a = ops.attn_mod_fwd(q, buf[:, wide - 128:wide - 64], buf[:, wide - 64:], 1, 1, SCALE, batch=1)
    b = ops.attn_mod_fwd(q, k, v, 1, 1, SCALE, batch=1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_offsets_that_do_not_fit_are_cut_to_the_tensors():
    """Device-side offsets and lengths outside the tensors (which the host cannot see) read and write nothing outside them."""
    dt = torch.bfloat16
    q, k, v = (rnd((64, 64), dt, s).cuda() for s in range(3))
    o = torch.full((64, 64), 7.0, dtype=dt, device="cuda")
    ops.attn_mod_fwd(q, k, v, 1, 1, SCALE, cu_q=torch.tensor([0, 30, 900], dtype=torch.int32, device="cuda"),
                     cu_k=torch.tensor([-5, 30, 20], dtype=torch.int32, device="cuda"), max_q=40, max_k=64, o=o)
    ref, _ = ops.attn_mod_fwd(q[:30], k[:30], v[:30], 1, 1, SCALE, batch=1)
    assert torch.equal(o[:30], ref) and bool((o[30:] == 0).all())
    full, _ = ops.attn_mod_fwd(q, k, v, 1, 1, SCALE, batch=2, len_k=torch.tensor([99, -3], dtype=torch.int32, device="cuda"))
    part, _ = ops.attn_mod_fwd(q[:32], k[:32], v[:32], 1, 1, SCALE, batch=1)
    assert torch.equal(full[:32], part) and bool((full[32:] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,Hq,Hkv,kw", [([900], 2, 1, dict(causal=True, bias=1)), ([700, 30, 520], 4, 1, dict(docs="sorted", cap=9.0)), ([1500], 1, 1, dict(docs="mixed", poison=True))], ids=str)
def test_few_blocks_are_split_over_their_tiles(lens, Hq, Hkv, kw, dtype):
    """Long sequences of few heads: the backward shares a block's tiles among workgroups and adds their partial sums, the forward runs in 16-row tiles."""
    run_case(DT[dtype], lens, lens, Hq, Hkv, **kw)


def test_many_blocks_of_long_sequences():
    """Enough blocks that nothing is split: the 128-row forward and single-pass backward on lengths around tile and block borders."""
    lens = [257, 256, 255, 193, 192, 129, 128, 127, 65, 64, 63, 1] * 3
    q, k, v, do = (rnd((sum(lens), 6 * 64), torch.bfloat16, s, 1.0 + (s == 0)).cuda() for s in range(4))
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    mod = ops.ScoreMod(softcap=20.0, causal=True)
    kw = dict(cu_q=cu, cu_k=cu, max_q=257, max_k=257)
    o, lse = ops.attn_mod_fwd(q, k, v, 6, 6, SCALE, mod, **kw)
    g = ops.attn_mod_bwd(q, k, v, o, do, lse, 6, 6, SCALE, mod, **kw)
    for s in (0, 1, 4, 11, 13, 29):        # the same sequences alone (other kernels run them): equal up to the rounding of weights and results
        a, b = int(cu[s]), int(cu[s + 1])
        one, l1 = ops.attn_mod_fwd(q[a:b], k[a:b], v[a:b], 6, 6, SCALE, mod, batch=1)
        assert bool(((o[a:b] - one).abs().float() <= 2.0 ** -7 * (one.abs().float() + 3)).all()) and bool(((lse[:, a:b] - l1).abs() <= 1e-4).all())
        for x, y in zip(g, ops.attn_mod_bwd(q[a:b], k[a:b], v[a:b], one, do[a:b], l1, 6, 6, SCALE, mod, batch=1)):
            assert float((x[a:b].float() - y.float()).norm()) <= 4 * 2.0 ** -8 * float(y.float().norm()) + 1e-6


def test_side_stream_and_two_captured_graphs():
    """Another stream, and two graphs over the same tensors (each with scratch of its own) replayed next to each other on new inputs."""
    dt, n = torch.bfloat16, 900
    q, k, v, do = rnd((2 * n, 128), dt, 1).cuda(), rnd((2 * n, 64), dt, 2).cuda(), rnd((2 * n, 64), dt, 3).cuda(), rnd((2 * n, 128), dt, 4).cuda()
    doc = documents(n, "sorted").repeat(2).cuda()
    mod = ops.ScoreMod(softcap=10.0, slopes=torch.tensor([0.5, 0.25], device="cuda"), doc_q=doc, doc_k=doc, causal=True)

    def both():
        o, lse = ops.attn_mod_fwd(q, k, v, 2, 1, SCALE, mod, batch=2)
        one = ops.attn_mod_fwd(q[::n].contiguous(), k, v, 2, 1, SCALE, batch=2)
        return (o, lse, *one, *ops.attn_mod_bwd(q, k, v, o, do, lse, 2, 1, SCALE, mod, batch=2))
    eager = both()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        side = both()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, side))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both())
        graphs.append(g)
    for r in range(3):
        q.copy_(rnd((2 * n, 128), dt, 30 + r))
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, b) for out in outs for a, b in zip(want, out))


def test_refusals():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")      # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")       # noqa: E731
    q, k = z(8, 128), z(8, 64)
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    F = lambda mod=None, q=q, k=k, v=k, Hq=2, Hkv=1, scale=SCALE, **kw: ops.attn_mod_fwd(q, k, v, Hq, Hkv, scale, mod, **(kw or dict(batch=2)))   # noqa: E731
    M = ops.ScoreMod
    f32 = lambda *s: torch.zeros(*s, device="cuda")      # noqa: E731
    bad = [lambda: F(Hq=3), lambda: F(q=z(8, 192), Hq=3, Hkv=2), lambda: F(scale=0.0), lambda: F(scale=-1.0), lambda: F(scale=float("nan")), lambda: F(batch=3),
           lambda: F(batch=0), lambda: F(batch=2, max_q=4), lambda: F(cu_q=cu), lambda: F(cu_q=cu, cu_k=cu), lambda: F(cu_q=cu, cu_k=cu, max_q=9, max_k=8),
           lambda: F(cu_q=cu, cu_k=i32(3), max_q=8, max_k=8), lambda: F(v=z(6, 64)), lambda: F(batch=2, len_k=i32(3)), lambda: F(q=z(8, 136)[:, 4:132]),
           lambda: F(q=q[:1].expand(8, 128)), lambda: F(M(slopes=f32(3))), lambda: F(M(slopes=f32(2), pos_q=f32(8), pos_k=f32(7))),
           lambda: F(M(slopes=f32(2), pos_q=f32(8, 3), pos_k=f32(8, 3))), lambda: F(M(slopes=f32(2), pos_q=f32(8, 2), pos_k=f32(8))), lambda: F(M(doc_q=i32(8), doc_k=i32(7))),
           lambda: F(M(causal=True, prefix=i32(3))), lambda: F(batch=2, o=z(8, 64)), lambda: F(batch=2, o=q), lambda: F(batch=2, lse=f32(8, 2)),
           lambda: M(softcap=-1.0), lambda: M(softcap=float("inf")), lambda: M(pos_q=f32(8)), lambda: M(pos_q=f32(8), pos_k=f32(8)), lambda: M(doc_q=i32(8)), lambda: M(prefix=i32(2)),
           lambda: ops.attn_mod_bwd(q, k, k, q, q, f32(2, 8), 2, 1, SCALE, batch=2, dq=q), lambda: ops.attn_mod_bwd(q, k, k, q, z(8, 64), f32(2, 8), 2, 1, SCALE, batch=2),
           lambda: ops.attn_mod_bwd(q, k, k, q, q, f32(2, 7), 2, 1, SCALE, batch=2)]
    for n, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {n} was accepted")
    for f in (lambda: F(q=q.float()), lambda: F(M(slopes=z(2))), lambda: F(M(doc_q=f32(8), doc_k=f32(8))), lambda: F(batch=2, len_k=f32(2)), lambda: F(batch=2, o=z(8, 128).half())):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(NotImplementedError):
        M(slopes=f32(2).requires_grad_(True))


@pytest.mark.parametrize("cap", [300.0, 9e5])
def test_caps_far_above_the_scores_change_nothing(cap):
    """cap tanh(s / cap) of scores |s| <= 12 is s to s^3 / (3 cap^2) = 6.4e-3 at 300 and 0 at 9e5; lse must keep to that plus fp32 rounding of the scores
    (2^-20: eight roundings of values up to 2^5 in log2 units, half a step each) however large the cap is."""
    T, H = 512, 2
    q, k, v = (rnd((T, H * 64), torch.bfloat16, 40 + i).cuda() for i in range(3))
    s = torch.stack([q[:, 64 * h:64 * h + 64].double() @ k[:, 64 * h:64 * h + 64].double().t() * 0.125 for h in range(H)])
    assert float(s.abs().max()) <= 12
    want = torch.logsumexp(cap * torch.tanh(s / cap), 2)
    for mod in (ops.ScoreMod(softcap=cap), ops.ScoreMod(softcap=cap, slopes=torch.zeros(H, device="cuda"))):
        for rows in (T, 3):      # whole tiles, and the few-row kernel
            _, lse = ops.attn_mod_fwd(q[:rows], k, v, H, H, 0.125, mod, batch=1)
            # per score: fp32 product and cap relative to the score (sum of 64 products: 2^-24 * 64 * 1 / 8 * |q||k| <= 2^-17), logarithm and its sum 2^-20
            assert float((lse.double() - want[:, :rows]).abs().max()) <= 2.0 ** -16


def test_row_strides_up_to_their_limit():
    """Rows 2^24 - 8 elements apart (a column of very wide rows), tiles that end inside the sequence: offsets within a tile pass 2^30 bytes."""
    T, ld = 70, (1 << 24) - 8
    buf = torch.empty(T * ld, dtype=torch.bfloat16, device="cuda")
    wide = torch.as_strided(buf, (T, 256), (ld, 1))
    wide.copy_(rnd((T, 256), torch.bfloat16, 50))
    flat, do = wide.contiguous(), rnd((T, 64), torch.bfloat16, 51).cuda()
    for rows in (T, 2):
        res = []
        for x in (wide, flat):
            q, k, v = x[:rows, :64], x[:, 64:128], x[:, 128:192]
            mod = ops.ScoreMod(causal=True)
            o, lse = ops.attn_mod_fwd(q, k, v, 1, 1, 0.125, mod, batch=1)
            res.append((o, lse, *ops.attn_mod_bwd(q, k, v, o, do[:rows], lse, 1, 1, 0.125, mod, batch=1)))
        assert all(torch.equal(a, b) for a, b in zip(*res))
    with pytest.raises(AplaHipError, match="stride"):
        ops.attn_mod_fwd(torch.as_strided(buf, (2, 64), (ld + 8, 1)), flat[:, :64], flat[:, :64], 1, 1, 0.125, batch=1)


def test_gradients_of_short_sequences_are_rounded_once():
    """Two keys of equal scores (q = 0, or k = 0): P = 1/2, o = (v1 + v2) / 2 and dS = +-(dO.v1 - dO.v2) / 4 in whole sixteenths, up to 13 bits.  With operands of
    small integers dq and dk are then off by the rounding of the result (2^-8, bf16) and 2^-16 of what is added, though dS itself has more bits than bf16."""
    S, g = 96, torch.Generator().manual_seed(60)
    ints = lambda rows, lo, hi, step=1: (torch.randint(lo, hi + 1, (rows, 64), generator=g) * step).double()      # noqa: E731
    a, v, do = ints(2 * S, -8, 8), ints(2 * S, -4, 4, 2), ints(2 * S, -8, 8)
    zero = torch.zeros_like(a)
    vs, ds_ = v.reshape(S, 2, 64), do.reshape(S, 2, 64)
    o = vs.mean(1, keepdim=True)
    dS = 0.5 * ((ds_ @ vs.transpose(1, 2)) - (ds_ * o).sum(-1, keepdim=True))          # [S, query, key]
    h = lambda t: t.bfloat16().cuda()      # noqa: E731
    for q, k in ((zero, a), (a, zero)):
        og, lse = ops.attn_mod_fwd(h(q), h(k), h(v), 1, 1, 0.125, batch=S)
        assert torch.equal(og.double().cpu().reshape(S, 2, 64), o.expand(S, 2, 64))
        dq, dk, _ = ops.attn_mod_bwd(h(q), h(k), h(v), og, h(do), lse, 1, 1, 0.125, batch=S)
        for got, x, w in ((dq, k, dS), (dk, q, dS.transpose(1, 2))):
            want, mag = 0.125 * (w @ x.reshape(S, 2, 64)), 0.125 * (w.abs() @ x.reshape(S, 2, 64).abs())
            assert ((got.double().cpu().reshape(S, 2, 64) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * mag).all()
