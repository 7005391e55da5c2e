"""Which kernel the forward of attention with modified scores takes (a host query, answered without a GPU)."""
import pytest

from apla_amd import _lib


def few(S=1, Hq=1, Hkv=1, max_q=1, max_k=64):
    a = _lib.AttnMod()
    a.S, a.Hq, a.Hkv, a.max_q, a.max_k = S, Hq, Hkv, max_q, max_k
    return _lib.lib().apla_attn_mod_few_rows(a)


@pytest.mark.parametrize("kw,want", [(dict(), 1), (dict(S=1000, Hq=8, Hkv=1, max_q=4), 1), (dict(S=1000, Hq=8, Hkv=1, max_q=5), 0), (dict(Hq=64, Hkv=64, max_q=128), 1), (dict(Hq=65, Hkv=65, max_q=128), 0),
                                     (dict(max_q=8192), 1), (dict(max_q=8193), 0), (dict(S=0), -1), (dict(Hq=3, Hkv=2), -1), (dict(max_k=0), -1)], ids=str)
def test_few_rows_or_few_blocks_take_the_form_for_few_rows(kw, want):
    assert few(**kw) == want


def test_no_arguments():
    assert _lib.lib().apla_attn_mod_few_rows(None) == -1


@pytest.mark.parametrize("kw", [dict(S=65535, Tq=65535, Tk=65535, max_q=1, max_k=1, Hq=300, Hkv=300), dict(S=60000, Tq=1 << 20, Tk=1 << 20, max_q=4096, max_k=4096, Hq=12, Hkv=12, cu_q=1 << 20, cu_k=1 << 20)], ids=str)
def test_more_workgroups_than_a_launch_takes_are_refused(kw):
    a = _lib.AttnMod()
    for n in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "delta", "workspace"):
        setattr(a, n, 1 << 20)
    a.scale, a.workspace_bytes = 0.125, 1 << 60
    for n, v in kw.items():
        setattr(a, n, v)
    a.ldq = a.ldo = a.lddo = a.lddq = a.Hq * 64
    a.ldk = a.ldv = a.lddk = a.lddv = a.Hkv * 64
    for f in (_lib.lib().apla_attn_mod_fwd, _lib.lib().apla_attn_mod_bwd):
        assert f(a, None) == -22 and b"workgroups" in _lib.lib().apla_last_error()
