"""Configuration of attention features (block_conf["attention"]) without a GPU."""
import pytest

from apla_amd.attn_features import AttnFeatures


@pytest.mark.parametrize("conf,on", [({}, False), (dict(rope=None), False), (dict(rope=False), False), (dict(rope=True), True), (dict(rope={}), True), (dict(rope=dict(rot=32)), True)], ids=str)
def test_rope_is_on_unless_it_is_left_out_or_switched_off(conf, on):
    """`rope: {}` in a YAML file asks for rotary positions with every default."""
    f = AttnFeatures(conf, 2)
    assert (f.rope is not None) == on
    assert ("table" in f.plan([10], "cpu")) == on
    if on:
        assert f.plan([10], "cpu")["table"].shape == (10, conf["rope"].get("rot", 64) if isinstance(conf["rope"], dict) else 64)
