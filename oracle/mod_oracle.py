"""Rotary positions, query / key norm and attention with modified scores, restated in 64 bits on the CPU from their formulas (test
infrastructure; the product never imports it).  Every function also returns what the error bounds of the tests are made of."""
import torch


def rotate(x, table, positions, layout, sign=1.0):
    """x [T, heads, 64] fp64; table [P, rot] (cos | sin); positions int64 [T]."""
    r = table.shape[1] // 2
    out = x.clone()
    for t in range(x.shape[0]):
        p = int(positions[t])
        if p < 0 or p >= table.shape[0]:
            out[t, :, :2 * r] = float("nan")
            continue
        c, s = table[p, :r].double(), sign * table[p, r:].double()
        a, b = (x[t, :, :r], x[t, :, r:2 * r]) if layout == "half" else (x[t, :, 0:2 * r:2], x[t, :, 1:2 * r:2])
        u, w = a * c - b * s, b * c + a * s
        if layout == "half":
            out[t, :, :r], out[t, :, r:2 * r] = u, w
        else:
            out[t, :, 0:2 * r:2], out[t, :, 1:2 * r:2] = u, w
    return out


def qk_norm(x, w, b, eps, kind):
    """x [T, heads, 64] fp64, w / b [heads, 64]; LayerNorm or RMS norm of every head."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w + b


def visible(nq, nk, causal=False, prefix=0, doc_q=None, doc_k=None):
    """[nq, nk] bool: which keys the rows of one sequence see."""
    i, j = torch.arange(nq)[:, None] + (nk - nq), torch.arange(nk)[None]
    see = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        see &= (j <= i) | (j < prefix)
    if doc_q is not None:
        see &= (doc_q[:, None] == doc_k[None]) & (doc_q[:, None] >= 0)
    return see


def distance(nq, nk, pos_q=None, pos_k=None):
    if pos_q is None:
        return ((torch.arange(nq)[:, None] + (nk - nq)) - torch.arange(nk)[None]).abs().double()
    d = pos_q.double().reshape(nq, 1, -1) - pos_k.double().reshape(1, nk, -1)
    return d.square().sum(-1).sqrt()


def attend(q, k, v, scale, see, softcap=0.0, slope=0.0, dist=None, do=None):
    """One head of one sequence, fp64: q [nq, 64], k / v [nk, 64].  Values in masked places are not used at all.  Returns a dict with o, lse
    (and dq, dk, dv), the weights p, and the absolute sums the bounds are made of."""
    nq, nk = see.shape
    out = {"o": torch.zeros(nq, 64, dtype=torch.float64), "lse": torch.full((nq,), -float("inf"), dtype=torch.float64),
           "p": torch.zeros(nq, nk, dtype=torch.float64), "ds": torch.zeros(nq, nk, dtype=torch.float64)}
    raw = torch.zeros(nq, nk, dtype=torch.float64)
    for i in range(nq):
        js = see[i].nonzero().flatten()
        if js.numel() == 0:
            continue
        s = k[js] @ q[i] * scale
        raw[i, js] = s
        z = softcap * torch.tanh(s / softcap) if softcap else s
        if dist is not None:
            z = z - slope * dist[i, js]
        L = torch.logsumexp(z, 0)
        p = torch.exp(z - L)
        out["p"][i, js], out["lse"][i], out["o"][i] = p, L, p @ v[js]
    if do is None:
        return out
    out["dq"] = torch.zeros(nq, 64, dtype=torch.float64)
    out["dk"], out["dv"] = torch.zeros(nk, 64, dtype=torch.float64), torch.zeros(nk, 64, dtype=torch.float64)
    for i in range(nq):
        js = see[i].nonzero().flatten()
        if js.numel() == 0:
            continue
        p = out["p"][i, js]
        ds = p * (v[js] @ do[i] - (do[i] * out["o"][i]).sum())
        if softcap:
            ds = ds * (1 - torch.tanh(raw[i, js] / softcap) ** 2)
        out["ds"][i, js] = ds
        out["dq"][i] = scale * (ds @ k[js])
        out["dk"][js] += scale * ds[:, None] * q[i]
        out["dv"][js] += p[:, None] * do[i]
    return out
