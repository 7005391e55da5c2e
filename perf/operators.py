"""What the rotary / normalised-query / modified-score attention operators are measured on.

``own`` False: elementary torch operations in 32 bits, rounded once at the end.  ``own`` True: the framework's entry points
(``apla_amd.ops``).  A case's ``op`` is ``rotary``, ``qk_norm`` or ``attn``; ``train`` adds the backward pass and its gradients to
the outputs.  Head dimension is 64 everywhere, as in the rest of the framework.
"""
import math

import numpy as np
import torch

own = False
HD = 64
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a serving step: one new token for each of 32 sequences at far positions of a stretched table
        dict(name="rotary_tokens", op="rotary", dtype="bf16", train=False, T=32, heads=32, rot=64, layout="half", far=131072, stretch=4.0, pos="random"),
        # queries and keys of a 518-px batch of 8 (1370 tokens, 24 heads each) out of the fused qkv rows, a quarter of the head turned, both directions
        dict(name="rotary_partial_train", op="rotary", dtype="bf16", train=True, T=8 * 1370, heads=48, rot=16, layout="interleaved", far=1370, stretch=1.0, pos="row"),
        # one 224-px image through a trained block: 197 tokens, 12 heads, LayerNorm of q and k, positions on the patch grid
        dict(name="qk_norm_image", op="qk_norm", dtype="bf16", train=False, T=197, hq=12, hkv=12, norm="layer", rot=64, layout="half", far=197, pos="row"),
        # the same block in training at batch 128, with the gradients of the four norm vectors
        dict(name="qk_norm_train", op="qk_norm", dtype="bf16", train=True, T=128 * 197, hq=12, hkv=12, norm="layer", rot=64, layout="half", far=197, pos="row"),
        # packed tokens of long sequences, three query heads to a key head, RMS norm, three quarters of the head turned, fp16
        dict(name="qk_norm_shared_fp16", op="qk_norm", dtype="fp16", train=True, T=32768 + 77, hq=24, hkv=8, norm="rms", rot=48, layout="interleaved", far=16384, pos="random"),
        # the class token of one image against its 197 tokens, bias by the distance on the patch grid: the smallest call
        dict(name="attn_class_token", op="attn", dtype="bf16", train=False, S=1, nq=1, nk=197, hq=12, hkv=12, cap=0.0, bias=2, causal=False, prefix=0, docs=0, ragged=False),
        # single-token serving: 32 sequences with caches of up to 8192 keys, of different used lengths, capped scores and distance bias
        dict(name="attn_decode", op="attn", dtype="bf16", train=False, S=32, nq=1, nk=8192, hq=24, hkv=8, cap=50.0, bias=1, causal=True, prefix=0, docs=0, ragged=True),
        # self-supervised images read in raster order with a prefix that all tokens see: 257 tokens, batch 64, both directions
        dict(name="attn_prefix_train", op="attn", dtype="bf16", train=True, S=64, nq=257, nk=257, hq=12, hkv=12, cap=0.0, bias=0, causal=True, prefix=257, docs=0, ragged=False),
        # 518-px images, capped scores, fp16, both directions
        dict(name="attn_cap_train_fp16", op="attn", dtype="fp16", train=True, S=8, nq=1370, nk=1370, hq=24, hkv=24, cap=30.0, bias=0, causal=False, prefix=0, docs=0, ragged=False),
        # documents packed into one long causal row, its end padded, shared key heads, distance bias, both directions
        dict(name="attn_docs_train", op="attn", dtype="bf16", train=True, S=1, nq=8192, nk=8192, hq=12, hkv=4, cap=0.0, bias=1, causal=True, prefix=0, docs=700, ragged=False),
        # crops of many sizes packed one behind the other, from one token up, evaluation with the patch-grid bias, fp16
        dict(name="attn_ragged_fp16", op="attn", dtype="fp16", train=False, S=48, nq=1370, nk=1370, hq=12, hkv=6, cap=0.0, bias=2, causal=False, prefix=0, docs=0, ragged=True),
        # one long causal sequence, evaluation
        dict(name="attn_long_causal", op="attn", dtype="bf16", train=False, S=1, nq=16384, nk=16384, hq=12, hkv=4, cap=0.0, bias=0, causal=True, prefix=0, docs=0, ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype, train, op = rng.choice(["bf16", "fp16"]), rng.random() < 0.6, rng.choice(["rotary", "qk_norm", "attn", "attn", "attn"])
    rot, layout = 2 * rng.randint(1, 32), rng.choice(["half", "interleaved"])
    if op == "rotary":
        return dict(op=op, dtype=dtype, train=train, T=_log(rng, 1, 20000), heads=rng.randint(1, 32), rot=rot, layout=layout,
                    far=_log(rng, 64, 131072), stretch=rng.choice([1.0, 2.0, 8.0]), pos=rng.choice(["random", "row"]))
    if op == "qk_norm":
        hkv = rng.randint(1, 8)
        return dict(op=op, dtype=dtype, train=train, T=_log(rng, 1, 30000), hq=hkv * rng.randint(1, 3), hkv=hkv, norm=rng.choice(["layer", "rms"]),
                    rot=rot, layout=layout, far=_log(rng, 64, 32768), pos=rng.choice(["random", "row"]))
    hkv = rng.choice([1, 2, 3, 4, 6])
    hq, cap, bias = hkv * rng.choice([1, 1, 2, 3, 4]), rng.choice([0.0, 0.0, 20.0, 50.0]), rng.choice([0, 1, 2])
    if rng.random() < 0.3:      # few queries against a cache
        return dict(op=op, dtype=dtype, train=False, S=_log(rng, 1, 24), nq=rng.randint(1, 4), nk=_log(rng, 1, 8192), hq=hq, hkv=hkv, cap=cap, bias=min(bias, 1),
                    causal=rng.random() < 0.5, prefix=0, docs=0, ragged=rng.random() < 0.7)
    n = _log(rng, 1, 4096)
    causal, S = rng.random() < 0.5, max(1, min(64, 16384 // n))
    return dict(op=op, dtype=dtype, train=train, S=rng.randint(1, max(1, S // 2)), nq=n, nk=n, hq=hq, hkv=hkv, cap=cap, bias=bias, causal=causal,
                prefix=rng.randint(1, n) if causal and rng.random() < 0.5 else 0, docs=_log(rng, 16, 1024) if rng.random() < 0.3 else 0, ragged=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------ what a case fixes: lengths, prefixes, documents
def _lengths(c):
    """(query lengths, used key lengths) of the sequences; ragged ones fall off from the longest, the last holds one token."""
    S = c["S"]
    if not c["ragged"]:
        return [c["nq"]] * S, [c["nk"]] * S
    f = [1.0 - s / S for s in range(S)]
    nk = [max(1, int(c["nk"] * x ** 2)) for x in f]
    if S > 1:
        nk[-1] = 1
    return ([c["nq"]] * S if c["nq"] != c["nk"] else nk), nk


def _is_cache(c):
    return c["nq"] != c["nk"]


def _prefixes(c):
    return [c["prefix"] * (s + 1) // c["S"] for s in range(c["S"])]


def _documents(c, n):
    """Document ids of n tokens: lengths around c["docs"], the last sixteenth padding (id -1)."""
    r = np.random.RandomState(n + c["docs"])
    ids = np.repeat(np.arange(n, dtype=np.int64), r.randint(1, 2 * c["docs"] + 1, n))[:n] if c["docs"] else np.zeros(n, np.int64)
    if c["docs"] and n >= 16:
        ids[n - n // 16:] = -1
    return ids


def _pairs(c):
    """Visible (query, key) pairs of one head."""
    total = 0
    for nq, nk, pre in zip(*_lengths(c), _prefixes(c)):
        i = np.arange(nq) + nk - nq
        if c["docs"]:
            ids = _documents(c, nk)
            lo, hi = np.searchsorted(np.where(ids < 0, 1 << 40, ids), ids, "left"), np.searchsorted(np.where(ids < 0, 1 << 40, ids), ids, "right")
            hi = np.where(ids < 0, lo, hi)
        else:
            lo, hi = np.zeros(nq, np.int64), np.full(nq, nk)
        if c["causal"]:
            hi = np.minimum(hi, np.maximum(i + 1, pre))
        total += int(np.maximum(0, hi - lo).sum())
    return total


# ------------------------------------------------------------------------------------------------ inputs
def _frequencies(rot, stretch, device):
    """Angles per position, 64 bits: base 10000, positions compressed by `stretch` (a table trained on a shorter range)."""
    return 10000.0 ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot) / stretch


def _angles(c, device):
    return torch.arange(c["far"], device=device, dtype=torch.float64)[:, None] * _frequencies(c["rot"], c.get("stretch", 1.0), device)


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dt = DT[c["dtype"]]

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dt)

    st = {"case": c}
    if c["op"] in ("rotary", "qk_norm"):
        T = c["T"]
        heads = c["heads"] if c["op"] == "rotary" else c["hq"] + c["hkv"]
        extra = heads // 2 if c["op"] == "rotary" else c["hkv"]      # the value columns of the same fused rows
        st["qkv"] = rand(T, (heads + extra) * HD, scale=2.0)
        a = _angles(c, dev)
        st["table"] = torch.cat((a.cos(), a.sin()), 1).float()
        st["pos"] = torch.randint(0, c["far"], (T,), device=dev, generator=g, dtype=torch.int32) if c["pos"] == "random" else None
        if c["op"] == "qk_norm":
            par = torch.randn(4, HD, device=dev, generator=g) * 0.2
            par[:2] += 1.0
            st["par"] = par
        if c["train"]:
            st["dy"] = rand(T, heads * HD)
        return st
    S, hq, hkv = c["S"], c["hq"], c["hkv"]
    lq, lk = _lengths(c)
    off = lambda n: torch.tensor([0] + list(np.cumsum(n)), device=dev, dtype=torch.int32)     # noqa: E731
    packed = c["ragged"] and not _is_cache(c)
    Tq, Tk = sum(lq), (sum(lk) if packed else S * c["nk"])
    st["q"], st["k"], st["v"] = rand(Tq, hq * HD, scale=2.0), rand(Tk, hkv * HD), rand(Tk, hkv * HD)
    st["cu_q"] = st["cu_k"] = off(lq) if packed else None
    st["len_k"] = torch.tensor(lk, device=dev, dtype=torch.int32) if _is_cache(c) and c["ragged"] else None
    st["slopes"] = 2.0 ** (-8.0 * (torch.arange(hq, device=dev, dtype=torch.float32) + 1) / hq) if c["bias"] else None
    st["pos_q"] = st["pos_k"] = None
    if c["bias"] == 2:          # coordinates on a patch grid of the sequence's own width
        grid = lambda n: np.stack(np.divmod(np.arange(n), max(1, math.isqrt(n))), 1).astype(np.float32)     # noqa: E731
        st["pos_k"] = torch.from_numpy(np.concatenate([grid(n) for n in (lk if packed else [c["nk"]] * S)])).to(dev)
        st["pos_q"] = st["pos_k"] if not _is_cache(c) else torch.from_numpy(np.concatenate([grid(nk)[nk - n:] for n, nk in zip(lq, lk)])).to(dev)
    st["doc"] = torch.from_numpy(np.concatenate([_documents(c, n) for n in lk])).to(dev, torch.int32) if c["docs"] else None
    st["prefix"] = torch.tensor(_prefixes(c), device=dev, dtype=torch.int32) if c["prefix"] else None
    if c["train"]:
        st["do"] = rand(Tq, hq * HD)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _turn(x, cos, sin, layout, sign):
    """x [T, heads, rot] turned by sign * angle, cos / sin [T, 1, rot/2]."""
    r = x.shape[-1] // 2
    a, b = (x[..., :r], x[..., r:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    u, w = a * cos - sign * b * sin, b * cos + sign * a * sin
    return torch.cat((u, w), -1) if layout == "half" else torch.stack((u, w), -1).flatten(-2)


def _rotate(x, c, cos, sin, sign):
    rot = c["rot"]
    return torch.cat((_turn(x[..., :rot], cos, sin, c["layout"], sign), x[..., rot:]), -1)


def _rows(st):
    c = st["case"]
    return st["pos"].long() if st["pos"] is not None else torch.arange(c["T"], device="cuda") % c["far"]


def _rotary_plain(st):
    c = st["case"]
    T, h, r = c["T"], c["heads"], c["rot"] // 2
    t = st["table"][_rows(st)]
    cos, sin = t[:, None, :r], t[:, None, r:]
    x = st["qkv"][:, :h * HD].float().view(T, h, HD)
    y = _rotate(x, c, cos, sin, 1.0).reshape(T, -1).to(st["qkv"].dtype)
    if not c["train"]:
        return {"y": y}
    dx = _rotate(st["dy"].float().view(T, h, HD), c, cos, sin, -1.0).reshape(T, -1).to(y.dtype)
    return {"y": y, "dx": dx}


def _qk_norm_math(x, par, eps, norm, hq):
    """x [T, heads, 64] -> (x^, 1/deviation, weights [heads, 64], biases)."""
    h = x.shape[1]
    xc = x - x.mean(-1, keepdim=True) if norm == "layer" else x
    rs = (xc.square().mean(-1, keepdim=True) + eps).rsqrt()
    w = torch.cat((par[0].expand(hq, HD), par[1].expand(h - hq, HD)))
    b = torch.cat((par[2].expand(hq, HD), par[3].expand(h - hq, HD)))
    return xc * rs, rs, w, b


def _qk_norm_formula(x, par, c, cos, sin, dy):
    hq = c["hq"]
    xh, rs, w, b = _qk_norm_math(x, par, 1e-6, c["norm"], hq)
    y = _rotate(xh * w + b, c, cos, sin, 1.0)
    if dy is None:
        return y, None, None
    g = _rotate(dy, c, cos, sin, -1.0)
    dpar = torch.stack(((g * xh)[:, :hq].sum((0, 1)), (g * xh)[:, hq:].sum((0, 1)), g[:, :hq].sum((0, 1)), g[:, hq:].sum((0, 1))))
    gw = g * w
    dx = gw - xh * (gw * xh).mean(-1, keepdim=True)
    if c["norm"] == "layer":
        dx = dx - gw.mean(-1, keepdim=True)
    return y, dx * rs, dpar


def _qk_norm_plain(st):
    c = st["case"]
    T, h, r = c["T"], c["hq"] + c["hkv"], c["rot"] // 2
    t = st["table"][_rows(st)]
    x = st["qkv"][:, :h * HD].float().view(T, h, HD)
    dy = st["dy"].float().view(T, h, HD) if c["train"] else None
    y, dx, dpar = _qk_norm_formula(x, st["par"], c, t[:, None, :r], t[:, None, r:], dy)
    out = {"qk": y.reshape(T, -1).to(st["qkv"].dtype)}
    if c["train"]:
        out |= {"dqk": dx.reshape(T, -1).to(st["qkv"].dtype), "dpar": dpar}
    return out


def _padded(c, n, T, cu, used):
    """Index [S, n] of every sequence's rows (clamped), which of them are rows, and the sequences' lengths."""
    i = torch.arange(n, device="cuda")
    start = cu[:-1].long() if cu is not None else torch.arange(c["S"], device="cuda") * n
    length = cu.diff().long() if cu is not None else used.long() if used is not None else torch.full((c["S"],), n, device="cuda")
    return (start[:, None] + i).clamp(max=T - 1), i < length[:, None], length


def _attn_plain(st):
    c = st["case"]
    S, hq, hkv, cap = c["S"], c["hq"], c["hkv"], c["cap"]
    scale, dt = HD ** -0.5, st["q"].dtype
    iq, okq, lq = _padded(c, c["nq"], st["q"].shape[0], st["cu_q"], None)
    ik, okk, lk = _padded(c, c["nk"], st["k"].shape[0], st["cu_k"], st["len_k"])
    nq, nk = iq.shape[1], ik.shape[1]
    pick = lambda x, i, h: x[i].float().view(S, i.shape[1], h, HD).transpose(1, 2)          # noqa: E731
    share = lambda x: x[:, :, None].expand(S, hkv, hq // hkv, nk, HD).reshape(S, hq, nk, HD)    # noqa: E731
    fold = lambda x: x.view(S, hkv, hq // hkv, nk, HD).sum(2)                               # noqa: E731

    def back(x, i, ok, T):
        out = torch.zeros(T, x.shape[1] * HD, device="cuda", dtype=dt)
        out[i[ok]] = x.transpose(1, 2)[ok].reshape(-1, x.shape[1] * HD).to(dt)
        return out

    q, k, v = pick(st["q"], iq, hq), share(pick(st["k"], ik, hkv)), share(pick(st["v"], ik, hkv))
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    if cap:
        s = torch.tanh(s / cap)
        slope_of_cap = 1 - s * s if c["train"] else None
        s = s * cap
    at_q = torch.arange(nq, device="cuda") + (lk - lq)[:, None]
    at_k = torch.arange(nk, device="cuda")
    if c["bias"] == 1:
        s = s - st["slopes"][:, None, None] * (at_q[:, :, None] - at_k).abs()[:, None]
    elif c["bias"] == 2:
        d = st["pos_q"][iq][:, :, None] - st["pos_k"][ik][:, None]
        s = s - st["slopes"][:, None, None] * d.square().sum(-1).sqrt()[:, None]
    see = okq[:, :, None] & okk[:, None]
    if c["causal"]:
        pre = st["prefix"].long()[:, None, None] if st["prefix"] is not None else 0
        see = see & ((at_k <= at_q[:, :, None]) | (at_k < pre))
    if c["docs"]:
        dq, dk = st["doc"][iq], st["doc"][ik]
        see = see & (dq[:, :, None] == dk[:, None]) & (dq >= 0)[:, :, None]
    s = s.masked_fill(~see[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    s = (s - m).exp_()
    total = s.sum(-1, keepdim=True)
    p = s / torch.where(total == 0, 1.0, total)
    lse = (m + total.log()).squeeze(-1)
    o32 = torch.matmul(p, v)
    o = back(o32, iq, okq, st["q"].shape[0])
    out = {"o": o, "lse": lse.transpose(1, 2)[okq].t().contiguous()}
    if not c["train"]:
        return out
    do = pick(st["do"], iq, hq) * okq[:, None, :, None]
    delta = (do * pick(o, iq, hq)).sum(-1, keepdim=True)
    dv = fold(torch.matmul(p.transpose(-1, -2), do))
    ds = p * (torch.matmul(do, v.transpose(-1, -2)) - delta)
    if cap:
        ds = ds * slope_of_cap
    ds = ds * scale
    dk, dq = fold(torch.matmul(ds.transpose(-1, -2), q)), torch.matmul(ds, k)
    return out | {"dq": back(dq, iq, okq, st["q"].shape[0]), "dk": back(dk, ik, okk, st["k"].shape[0]), "dv": back(dv, ik, okk, st["k"].shape[0])}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _rotary_own(st):
    from apla_amd import ops
    c = st["case"]
    kw = dict(layout=c["layout"], pos=st["pos"], seq_len=0 if st["pos"] is not None else c["far"])
    out = {"y": ops.rotary_fwd(st["qkv"][:, :c["heads"] * HD], st["table"], c["heads"], **kw)}
    if c["train"]:
        out["dx"] = ops.rotary_bwd(st["dy"], st["table"], c["heads"], **kw)
    return out


def _qk_norm_own(st):
    from apla_amd import ops
    c, par = st["case"], st["par"]
    kw = dict(norm=c["norm"], q_weight=par[0], k_weight=par[1], q_bias=par[2], k_bias=par[3], eps=1e-6, table=st["table"], layout=c["layout"],
              pos=st["pos"], seq_len=0 if st["pos"] is not None else c["far"])
    out = {"qk": ops.qk_norm_rotary_fwd(st["qkv"], c["hq"], c["hkv"], **kw)}
    if c["train"]:
        out["dqk"], out["dpar"] = ops.qk_norm_rotary_bwd(st["dy"], st["qkv"], c["hq"], c["hkv"], **kw)
    return out


def _attn_own(st):
    from apla_amd import ops
    c = st["case"]
    mod = ops.ScoreMod(softcap=c["cap"], slopes=st["slopes"], pos_q=st["pos_q"], pos_k=st["pos_k"], doc_q=st["doc"], doc_k=st["doc"],
                       causal=c["causal"], prefix=st["prefix"])
    kw = dict(cu_q=st["cu_q"], cu_k=st["cu_k"], max_q=c["nq"], max_k=c["nk"]) if st["cu_q"] is not None else dict(batch=c["S"], len_k=st["len_k"])
    o, lse = ops.attn_mod_fwd(st["q"], st["k"], st["v"], c["hq"], c["hkv"], HD ** -0.5, mod, **kw)
    if not c["train"]:
        return {"o": o, "lse": lse}
    dq, dk, dv = ops.attn_mod_bwd(st["q"], st["k"], st["v"], o, st["do"], lse, c["hq"], c["hkv"], HD ** -0.5, mod, **kw)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def run(state):
    op = state["case"]["op"]
    if own:
        from apla_amd import ops
        call = {"rotary": _rotary_own, "qk_norm": _qk_norm_own, "attn": _attn_own}[op]
        if state["case"]["dtype"] == "fp16":
            with ops.use_half(torch.float16):
                return call(state)
        return call(state)
    with torch.no_grad():
        return {"rotary": _rotary_plain, "qk_norm": _qk_norm_plain, "attn": _attn_plain}[op](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "rotary":
        n = c["T"] * c["heads"] * HD
        table = min(c["far"], c["T"]) * c["rot"] * 4 + (c["T"] * 4 if c["pos"] == "random" else 0)
        return {"bytes": (2 if c["train"] else 1) * n * 4 + table, "flops": (2 if c["train"] else 1) * 3 * c["T"] * c["heads"] * c["rot"]}
    if c["op"] == "qk_norm":
        n = c["T"] * (c["hq"] + c["hkv"]) * HD
        table = min(c["far"], c["T"]) * c["rot"] * 4 + (c["T"] * 4 if c["pos"] == "random" else 0)
        return {"bytes": n * (4 + (4 if c["train"] else 0)) + table + (4 * HD * 8 if c["train"] else 4 * HD * 4), "flops": n * (30 if c["train"] else 10)}
    lq, lk = _lengths(c)
    q, kv = sum(lq) * c["hq"] * HD * 2, sum(lk) * c["hkv"] * HD * 2
    pairs = _pairs(c) * c["hq"]
    extra = (sum(lk) * 8 if c["bias"] == 2 else 0) + (sum(lk) * 4 if c["docs"] else 0) + sum(lq) * c["hq"] * 4
    # the forward reads q, k, v and writes o; the backward's inputs beyond them are do (q's size), its outputs dq, dk, dv
    return {"bytes": 2 * q + 2 * kv + extra + (2 * q + 2 * kv if c["train"] else 0), "flops": pairs * HD * (14 if c["train"] else 4)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_turn(x, angle, rot, layout, sign):
    """Complex multiplication of the pairs; x [T, heads, 64], angle [T, rot/2]."""
    z = x.clone()
    turn = torch.polar(torch.ones_like(angle), sign * angle)[:, None]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    w = torch.complex(x[..., first], x[..., second]) * turn
    z[..., first], z[..., second] = w.real, w.imag
    return z


def _exact_rows(c, st):
    rows = st["pos"].long() if st["pos"] is not None else torch.arange(c["T"], device="cuda") % c["far"]
    return rows.double()[:, None] * _frequencies(c["rot"], c.get("stretch", 1.0), "cuda")


def _exact_attn(c, st):
    lq, lk = _lengths(c)
    hq, group, scale = c["hq"], c["hq"] // c["hkv"], HD ** -0.5
    packed = st["cu_q"] is not None
    col = lambda x, h: x[:, h * HD:(h + 1) * HD].double()       # noqa: E731
    o, lse = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(hq, st["q"].shape[0], dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(st["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    a = 0
    for s, (n, m, pre) in enumerate(zip(lq, lk, _prefixes(c))):
        b = a if packed else s * c["nk"]
        rows, keys = slice(a, a + n), slice(b, b + m)
        i, j = torch.arange(n, device="cuda")[:, None] + (m - n), torch.arange(m, device="cuda")[None]
        hide = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hide = (j > i) & (j >= pre)
        if c["docs"]:
            x, y = st["doc"][rows][:, None], st["doc"][keys][None]
            hide = hide | (x != y) | (x < 0)
        far = (i - j).abs().double() if c["bias"] == 1 else torch.cdist(st["pos_q"][rows].double(), st["pos_k"][keys].double(), compute_mode="donot_use_mm_for_euclid_dist") if c["bias"] == 2 else None
        for h in range(hq):
            Q, K, V = col(st["q"][rows], h), col(st["k"][keys], h // group), col(st["v"][keys], h // group)
            z = Q @ K.t() * scale
            t = torch.tanh(z / c["cap"]) if c["cap"] else None
            z = c["cap"] * t if t is not None else z
            z = z - st["slopes"][h].double() * far if far is not None else z
            z[hide] = -math.inf
            L = torch.logsumexp(z, 1)
            P = torch.exp(z - torch.where(L == -math.inf, 0.0, L)[:, None])
            C = slice(h * HD, (h + 1) * HD)
            G = slice(h // group * HD, (h // group + 1) * HD)
            O = P @ V
            o[rows, C], lse[h, rows] = O, L
            if c["train"]:
                D = col(st["do"][rows], h)
                E = P * (D @ V.t() - (D * O).sum(1, keepdim=True)) * scale
                E = E * (1 - t * t) if t is not None else E
                dq[rows, C] = E @ K
                dk[keys, G] += E.t() @ Q
                dv[keys, G] += P.t() @ D
        a += n
    return {"o": o, "lse": lse} | ({"dq": dq, "dk": dk, "dv": dv} if c["train"] else {})


def exact(case, seed):
    c = case
    if c["op"] == "attn" and sum(n * m for n, m in zip(*_lengths(c))) * c["hq"] > 6_000_000_000:
        return None
    st = prepare(c, seed)
    if c["op"] == "attn":
        return _exact_attn(c, st)
    T, angle = c["T"], _exact_rows(c, st)
    heads = c["heads"] if c["op"] == "rotary" else c["hq"] + c["hkv"]
    x = st["qkv"][:, :heads * HD].double().view(T, heads, HD)
    dy = st["dy"].double().view(T, heads, HD) if c["train"] else None
    if c["op"] == "rotary":
        out = {"y": _exact_turn(x, angle, c["rot"], c["layout"], 1).reshape(T, -1)}
        return out | ({"dx": _exact_turn(dy, angle, c["rot"], c["layout"], -1).reshape(T, -1)} if c["train"] else {})
    par, hq = st["par"].double(), c["hq"]
    mean = x.mean(-1, keepdim=True) if c["norm"] == "layer" else torch.zeros_like(x[..., :1])
    dev = torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + 1e-6)
    hat = (x - mean) / dev
    side = torch.tensor([0] * hq + [1] * (heads - hq), device="cuda")
    out = {"qk": _exact_turn(hat * par[side] + par[2 + side], angle, c["rot"], c["layout"], 1).reshape(T, -1)}
    if c["train"]:
        g = _exact_turn(dy, angle, c["rot"], c["layout"], -1)
        u = g * par[side]
        back = (u - (u.mean(-1, keepdim=True) if c["norm"] == "layer" else 0) - hat * (u * hat).mean(-1, keepdim=True)) / dev
        rows = [(g * hat)[:, side == 0].sum((0, 1)), (g * hat)[:, side == 1].sum((0, 1)), g[:, side == 0].sum((0, 1)), g[:, side == 1].sum((0, 1))]
        out |= {"dqk": back.reshape(T, -1), "dpar": torch.stack(rows)}
    return out
