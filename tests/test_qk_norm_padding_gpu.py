"""Query / key norm next to masked places: a head whose incoming gradient is all zero (a row that sees nothing, a key that nobody sees) gives zero gradients,
whatever the row holds."""
import pytest
import torch
from torch import nn

from apla_amd import functional as AF
from apla_amd import ops
from apla_amd import rotary as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("rot,layout", [(0, "half"), (64, "half"), (34, "half"), (48, "interleaved")])
@pytest.mark.parametrize("T,Hq,Hkv", [(70, 6, 2), (33, 3, 1), (257, 8, 8)])
def test_heads_without_a_gradient(T, Hq, Hkv, rot, layout, norm, dtype):
    H, g = Hq + Hkv, torch.Generator().manual_seed(1)
    x, dy = (torch.randn(T, H, 64, generator=g).to(dtype) for _ in range(2))
    dead = torch.rand(T, H, generator=g) < 0.4
    dy[dead] = 0
    dy[3, 0], dy[4, 1, :63], dead[3, 0], dead[4, 1] = -0.0, 0, True, False       # a head of which one value has a gradient is an ordinary one
    dy[4, 1, 63] = 1
    bad = x.clone()
    bad[dead] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0]).repeat(16).to(dtype)
    w = [torch.randn(64, generator=g).cuda() for _ in range(2)]
    kw = dict(norm=norm, q_weight=w[0], k_weight=w[1], **(dict(table=R.rotary_table(T, rot, device="cuda"), layout=layout) if rot else {}))
    flat = lambda t: t.reshape(T, H * 64).cuda()      # noqa: E731
    with ops.use_half(dtype):
        ref, dref = ops.qk_norm_rotary_bwd(flat(dy), flat(x), Hq, Hkv, **kw)
        got, dpar = ops.qk_norm_rotary_bwd(flat(dy), flat(bad), Hq, Hkv, **kw)
        alone, _ = ops.qk_norm_rotary_bwd(flat(dy), flat(bad), Hq, Hkv, want_params=False, **kw)
    assert torch.equal(got, ref) and torch.equal(dpar, dref) and torch.equal(alone, ref)
    assert bool((got.view(T, H, 64)[dead.cuda()] == 0).all()) and bool((got.view(T, H, 64)[4, 1] != 0).any())


def test_padding_of_the_fused_node_may_hold_anything():
    """Padding tokens (document -1) of NaN: their gradient is 0, the norm's gradients are those of finite padding."""
    T, H = 90, 2
    g = torch.Generator().manual_seed(2)
    x, do = torch.randn(T, 3 * H * 64, generator=g).bfloat16().cuda(), torch.randn(T, H * 64, generator=g).bfloat16().cuda()
    doc = torch.arange(T, dtype=torch.int32) // 31
    doc[60:70] = doc[85:] = -1
    doc = doc.cuda()
    mod = ops.ScoreMod(doc_q=doc, doc_k=doc)
    norms = [nn.LayerNorm(64).cuda() for _ in range(2)]
    par = [p for n in norms for p in n.parameters()]
    res = []
    for fill in (0.5, float("nan")):
        a = x.clone()
        a[doc < 0] = fill
        a.requires_grad_(True)
        o = AF.attention_mod_qkv(a, H, 0.125, mod=mod, q_norm=norms[0], k_norm=norms[1], table=R.rotary_table(T, 64, device="cuda"), batch=1)
        res.append((o, *torch.autograd.grad(o, [a] + par, do)))
    assert all(torch.equal(u, v) for u, v in zip(*res)) and bool((res[0][1][doc < 0] == 0).all())


@pytest.mark.parametrize("norm", [False, True])
def test_padding_may_stand_outside_the_table(norm):
    """Padding tokens of position -1: NaN in their q and k, which the mask hides, and a gradient of 0."""
    T, H = 90, 2
    g = torch.Generator().manual_seed(3)
    x, do = torch.randn(T, 3 * H * 64, generator=g).bfloat16().cuda(), torch.randn(T, H * 64, generator=g).bfloat16().cuda()
    doc = torch.arange(T, dtype=torch.int32) // 31
    doc[60:70] = doc[85:] = -1
    doc, pos = doc.cuda(), torch.arange(T, dtype=torch.int32).cuda()
    norms = [nn.RMSNorm(64).cuda() for _ in range(2)] if norm else [None, None]
    par = [p for n in norms if norm for p in n.parameters()]
    res = []
    for p in (pos, torch.where(doc < 0, -1, pos).int()):
        a = x.clone().requires_grad_(True)
        o = AF.attention_mod_qkv(a, H, 0.125, mod=ops.ScoreMod(doc_q=doc, doc_k=doc), q_norm=norms[0], k_norm=norms[1], table=R.rotary_table(T, 64, device="cuda"), pos=p, batch=1)
        res.append((o, *torch.autograd.grad(o, [a] + par, do)))
    assert all(torch.equal(u, v) for u, v in zip(*res)) and bool((res[0][1][doc < 0] == 0).all())


def test_a_position_outside_the_table_is_nan_in_gradients_that_arrive():
    dy, pos = torch.randn(4, 128).bfloat16().cuda(), torch.tensor([0, 9, -1, 3], dtype=torch.int32, device="cuda")
    dy[2, 64:] = 0
    dx = ops.rotary_bwd(dy, R.rotary_table(8, 32, device="cuda"), 2, pos=pos).view(4, 2, 64)
    assert bool(torch.isnan(dx[1, :, :32]).all()) and bool(torch.isnan(dx[2, 0, :32]).all()) and bool((dx[2, 1] == 0).all()) and bool(torch.isfinite(dx[[0, 3]]).all())
