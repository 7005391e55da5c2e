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
