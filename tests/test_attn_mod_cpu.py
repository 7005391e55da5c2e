"""Host side of the rotary / query-key norm / modified-score attention operators: refusals of the C entry points (which come before any
launch, so they answer without a GPU), workspace sizes, rotary tables, and the oracle against automatic differentiation."""
import ctypes
import math

import pytest
import torch

from apla_amd import _lib, ops
from apla_amd import rotary as R
from apla_amd._lib import AplaHipError
from oracle import mod_oracle as O

EINVAL = -22
P16 = ctypes.c_void_p(1 << 20)      # an aligned address that is never used: every call below is refused before a launch


def attn_args(**kw):
    a = _lib.AttnMod()
    for n in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "delta"):
        setattr(a, n, 1 << 20)
    a.S, a.Tq, a.Tk, a.max_q, a.max_k, a.Hq, a.Hkv, a.scale = 2, 8, 8, 4, 4, 2, 1, 0.125
    a.ldq = a.ldo = a.lddo = a.lddq = 128
    a.ldk = a.ldv = a.lddk = a.lddv = 64
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad", [dict(S=0), dict(S=70000), dict(Hq=3, Hkv=2), dict(Hkv=0), dict(Tq=0), dict(max_q=9), dict(max_k=0), dict(Tq=9), dict(scale=0.0),
                                 dict(scale=-1.0), dict(scale=math.nan), dict(softcap=-1.0), dict(softcap=math.inf), dict(softcap=1e-9), dict(q=0), dict(lse=0), dict(k=(1 << 20) + 8), dict(ldq=64),
                                 dict(ldk=68), dict(doc_q=1 << 20), dict(pos_dim=1), dict(pos_dim=3, pos_q=1 << 20, pos_k=1 << 20, slopes=1 << 20),
                                 dict(pos_dim=1, pos_q=1 << 20, pos_k=1 << 20), dict(prefix=1 << 20), dict(doc_q=1 << 20, doc_k=1 << 20),
                                 dict(Tq=1 << 25, Tk=1 << 25, S=1, max_q=1 << 25, max_k=4, cu_q=1 << 20, cu_k=1 << 20)], ids=str)
def test_attention_entry_points_refuse(bad):
    for fn in (_lib.lib().apla_attn_mod_fwd, _lib.lib().apla_attn_mod_bwd):
        assert fn(attn_args(**bad), None) == EINVAL and _lib.lib().apla_last_error()


@pytest.mark.parametrize("bad", [dict(d_o=0), dict(delta=0), dict(dq=(1 << 20) + 2), dict(lddv=32), dict(lddq=132)], ids=str)
def test_attention_backward_refuses(bad):
    assert _lib.lib().apla_attn_mod_bwd(attn_args(**bad), None) == EINVAL
    assert _lib.lib().apla_attn_mod_fwd(None, None) == EINVAL and _lib.lib().apla_attn_mod_bwd(None, None) == EINVAL


def test_attention_workspace_sizes():
    size = _lib.lib().apla_attn_mod_workspace_bytes
    assert size(attn_args(), 0) == 0 and size(attn_args(), 1) == 0 and size(None, 0) == -1 and size(attn_args(Hq=3, Hkv=2), 0) == -1
    docs = attn_args(doc_q=1 << 20, doc_k=1 << 20, S=2, Tq=400, Tk=600, max_q=200, max_k=300)
    assert size(docs, 1) >= 2 * (5 + 4) * 8 and size(docs, 1) > size(docs, 0) > 0
    cache = attn_args(S=1, Tq=1, Tk=65536, max_q=1, max_k=65536, Hq=8, Hkv=1)       # one token against a long cache: split over the keys
    assert size(cache, 0) > 0 and size(cache, 1) == 8 * 8 * 256                     # backward: eight partial sums of dQ [1, 8, 64], fp32


def test_rotary_entry_points_refuse():
    h = _lib.lib()
    ok = dict(x=P16, ldx=128, y=P16, ldy=128, T=4, heads=2, table=P16, P=8, rot=32, layout=0, pos=None, seq_len=0, inverse=0)
    for bad in (dict(x=None), dict(y=ctypes.c_void_p((1 << 20) + 8)), dict(ldx=64), dict(ldy=130), dict(T=0), dict(heads=0), dict(heads=5000), dict(table=None), dict(P=0),
                dict(rot=31), dict(rot=66), dict(rot=-2), dict(layout=2), dict(P=3), dict(seq_len=9), dict(seq_len=-1)):
        assert h.apla_rotary(*(ok | bad).values(), None) == EINVAL, bad
    ok = dict(x=P16, ldx=192, y=P16, ldy=192, T=4, Hq=2, Hkv=1, norm=1, eps=1e-6, qw=None, kw=None, qb=None, kb=None, table=None, P=0, rot=0, layout=0, pos=None, seq_len=0)
    for bad in (dict(norm=0), dict(norm=3), dict(eps=-1.0), dict(Hq=-1), dict(ldx=128), dict(rot=64)):
        assert h.apla_qk_norm_rotary_fwd(*(ok | bad).values(), None) == EINVAL, bad
    ok = dict(dy=P16, lddy=192, x=P16, ldx=192, dx=P16, lddx=192, T=4, Hq=2, Hkv=1, norm=1, eps=1e-6, qw=None, kw=None, table=None, P=0, rot=0, layout=0, pos=None, seq_len=0,
              dparams=P16, workspace=P16, bytes=h.apla_qk_norm_rotary_workspace_bytes())
    for bad in (dict(workspace=None), dict(bytes=16), dict(dy=None), dict(lddx=64), dict(norm=7)):
        assert h.apla_qk_norm_rotary_bwd(*(ok | bad).values(), None) == EINVAL, bad


def test_no_cpu_path():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for f in (lambda: ops.rotary_fwd(x, torch.zeros(4, 64), 1), lambda: ops.qk_norm_rotary_fwd(torch.zeros(4, 128, dtype=torch.bfloat16), 1, 1),
              lambda: ops.attn_mod_fwd(x, x, x, 1, 1, 0.125, batch=1)):
        with pytest.raises(AplaHipError):
            f()


def test_score_mod_refuses():
    t = torch.zeros(2)
    for kw in (dict(softcap=-1.0), dict(softcap=math.nan), dict(softcap=1e-9), dict(pos_q=t, slopes=t), dict(pos_q=t, pos_k=t), dict(doc_k=t), dict(prefix=t)):
        with pytest.raises(ValueError):
            ops.ScoreMod(**kw)
    with pytest.raises(NotImplementedError):
        ops.ScoreMod(slopes=torch.zeros(2, requires_grad=True))


def test_rotary_tables():
    t = R.rotary_table(200_000, 64)
    p, i = 199_999, 3
    assert t.shape == (200_000, 64) and abs(float(t[p, i]) - math.cos(p * 10000.0 ** (-2 * i / 64))) < 1e-7 and abs(float(t[p, 32 + i]) - math.sin(p * 10000.0 ** (-2 * i / 64))) < 1e-7
    f = R.rotary_frequencies(64)
    assert torch.allclose(R.rotary_frequencies(64, scaling="linear", factor=4.0), f / 4)
    n = R.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert float(n[0]) == 1.0 and abs(float(n[-1] * 4 / f[-1]) - 1) < 1e-9
    y = R.rotary_frequencies(64, scaling="yarn", factor=4.0, trained=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns > 40], f[turns > 40]) and torch.allclose(y[turns < 0.8], f[turns < 0.8] / 4) and bool((y <= f).all()) and bool((y >= f / 4 - 1e-18).all())
    g = R.rotary_table_2d((3, 5), 32, prefix=2)
    assert g.shape == (17, 32) and bool((g[:2, :16] == 1).all()) and bool((g[:2, 16:] == 0).all())
    assert torch.equal(g[2 + 5:2 + 10, :8], g[2 + 5, :8].expand(5, 8)) and torch.equal(g[2::5, 8:16], g[2, 8:16].expand(3, 8))
    for bad in (lambda: R.rotary_frequencies(63), lambda: R.rotary_frequencies(64, scaling="cubic"), lambda: R.rotary_frequencies(64, factor=0.5), lambda: R.rotary_frequencies(2, scaling="ntk"),
                lambda: R.rotary_frequencies(64, scaling="yarn", factor=2.0), lambda: R.rotary_table_2d((3, 5), 30), lambda: R.rotary_table_2d((0, 5))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_oracle_gradients_are_those_of_automatic_differentiation(cap):
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(n, 64, generator=g, dtype=torch.float64) for n in (9, 12, 12, 9))
    doc = torch.tensor([0, 0, 0, 1, 1, 1, 1, 2, 2, 2, -1, -1])
    see, dist = O.visible(9, 12, True, 2, doc[3:], doc), O.distance(9, 12)
    w = O.attend(q, k, v, 0.125, see, cap, 0.25, dist, do)
    a, b, c = (t.clone().requires_grad_(True) for t in (q, k, v))
    s = a @ b.t() * 0.125
    s = (cap * torch.tanh(s / cap) if cap else s) - 0.25 * dist
    p = torch.softmax(s.masked_fill(~see, -1e300), 1) * see.any(1, keepdim=True)
    ref = torch.autograd.grad(p @ c, (a, b, c), do)
    assert all(float((x - y).abs().max()) < 1e-12 for x, y in zip(ref, (w["dq"], w["dk"], w["dv"])))
    assert bool((w["lse"][~see.any(1)] == -math.inf).all()) and bool((~see.any(1)).any())


def test_overlap_of_row_strided_views():
    b = torch.zeros(6, 64, dtype=torch.bfloat16)
    row = lambda off, stride: torch.as_strided(b, (1, 8), (stride, 1), off)      # noqa: E731
    assert ops._overlap(row(0, 0), row(0, 0)) and ops._overlap(row(0, 0), row(4, 7)) and not ops._overlap(row(0, 0), row(8, 0))
    assert not ops._overlap(b[:, :32], b[:, 32:]) and ops._overlap(b[:, :40], b[:, 32:]) and not ops._overlap(b[:3], b[3:])
    assert not ops._overlap(b[:, :32], row(64 + 32, 0)) and ops._overlap(b[:, :32], row(64 + 24, 0)) and not ops._overlap(row(64 + 32, 5), b[:, :32])
    assert not ops._overlap(b[:0], b)


def test_rows_set_where_one_side_is_empty_are_those_of_the_sequences():
    t = lambda: torch.full((12, 2), 7.0)      # noqa: E731
    rows = lambda x: [i for i in range(12) if float(x[i, 0]) == 0.0 and float(x[i, 1]) == 0.0]      # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)      # noqa: E731
    for args, want in (((None, 6, None), list(range(12))), ((None, 6, i32(2, 9)), [0, 1, 6, 7, 8, 9, 10, 11]), ((None, 6, i32(0, -1)), []),
                       ((i32(1, 4, 4, 9), 5, None), [1, 2, 3, 4, 5, 6, 7, 8]), ((i32(1, 4, 4, 9), 2, None), [1, 2, 4, 5]), ((i32(1, 4, 4, 9), 5, i32(1, 3, 2)), [1, 4, 5]),
                       ((i32(0, 0), 0, None), [])):
        x = t()
        ops._zero_rows(x, *args, 0.0, False)
        assert rows(x) == want and float(x.sum()) == 14.0 * (12 - len(want)), args
    x = t()
    ops._zero_rows(x, i32(1, 4, 4, 9), 5, None, 0.0, True)
    assert rows(x) == list(range(12))


def test_plans_that_a_captured_graph_reads_are_kept(monkeypatch):
    from apla_amd.attn_features import AttnFeatures
    f, dev = AttnFeatures(dict(causal=True), 2), torch.device("cuda")
    capturing = [True]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    first = f.plan([5], dev)
    capturing[0] = False
    for n in range(10, 60):
        f.plan([n], dev)
    assert f.plan([5], dev) is first and len(f._plans) <= 17
