"""Gradients of whole models with attention features against the same model in 64 bits on the CPU under automatic differentiation.

fp16, u = 2^-11: a value and a gradient pass about 15 roundings each per block, independent of one another; one of q or k weighs up to the score's size, at most 8 here
(the cap, or scores of normalised rows), in the gradient.  sqrt(30 blocks) * 8 u is 3 % for two blocks, 7.5 % for twelve."""
import math

import pytest
import torch
import torch.nn.functional as F

from apla_amd import ops
from apla_amd import rotary as R
from apla_amd.apla import build_apla
from apla_amd.vit import VisionTransformer

pytestmark = pytest.mark.gpu
FULL = dict(qk_norm="layer", rope=dict(rot=32, base=50.0), softcap=8.0, distance_bias=True, causal=True, prefix=5)


class Cfg:
    partial_size = 64


def tolerance(blocks):
    return math.sqrt(30 * blocks) * 8 * 2.0 ** -11


def cpu64(t):
    return t.detach().double().cpu()


def norm(x, m, kind="layer"):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + m.eps) * cpu64(m.weight)
    return x if getattr(m, "bias", None) is None else x + cpu64(m.bias)


def turned(x, rope, side):
    """x [B, H, n, 64] turned by its place on the patch grid, pairs (i, i + rot / 2)."""
    rot = rope.get("rot", 64)
    t = R.rotary_table_2d((side, side), rot, rope.get("base", 100.0)).double()
    c, s, a, b = t[:, :rot // 2], t[:, rot // 2:], x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., rot:]), -1)


def attention(attn, h, conf):
    B, n, D = h.shape
    H, side = D // 64, math.isqrt(n - 1)
    q, k, v = (h @ cpu64(attn.qkv.weight).t() + cpu64(attn.qkv.bias)).view(B, n, 3, H, 64).permute(2, 0, 3, 1, 4)
    if conf.get("qk_norm"):
        q, k = norm(q, attn.q_norm, conf["qk_norm"]), norm(k, attn.k_norm, conf["qk_norm"])
    if conf.get("rope"):
        rope = {} if conf["rope"] is True else conf["rope"]
        q, k = turned(q, rope, side), turned(k, rope, side)
    s = q @ k.transpose(-1, -2) * 0.125
    if conf.get("softcap"):
        s = conf["softcap"] * torch.tanh(s / conf["softcap"])
    if conf.get("distance_bias"):
        y, x = torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij")
        at = torch.cat((torch.full((1, 2), (side - 1) / 2.0), torch.stack((y, x), -1).reshape(-1, 2))).double()
        slopes = 2.0 ** (-8.0 * (torch.arange(H).double() + 1) / H)
        s = s - slopes[:, None, None] * (at[:, None] - at[None]).square().sum(-1).sqrt()
    if conf.get("causal"):
        i = torch.arange(n)
        s = s.masked_fill((i[None] > i[:, None]) & (i[None] >= conf.get("prefix", 0)), -math.inf)
    return (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, n, D)


def model64(vit, x, conf):
    """(normalised tokens, [projection rows of every block that ask for a gradient])"""
    x, params = cpu64(x), []
    for blk in vit.blocks:
        a = blk.attn
        w = cpu64(a.proj_weight1).requires_grad_(True)
        params.append(w)
        order = torch.argsort(cpu64(a.inds).long())
        full, bias = torch.cat((w, cpu64(a.proj_weight2)))[order], torch.cat((cpu64(a.proj_bias1), cpu64(a.proj_bias2)))[order]
        x = x + attention(a, norm(x, blk.norm1), conf) @ full.t() + bias
        h = F.gelu(norm(x, blk.norm2) @ cpu64(blk.mlp.fc1.weight).t() + cpu64(blk.mlp.fc1.bias))
        x = x + h @ cpu64(blk.mlp.fc2.weight).t() + cpu64(blk.mlp.fc2.bias)
    return norm(x, vit.norm), params


def test_gradient_and_step_along_it():
    """Two blocks with every feature: the gradient itself, and the 64-bit model's change along it, which is its length."""
    torch.manual_seed(0)
    m = VisionTransformer(img_size=[64], patch_size=16, embed_dim=128, depth=2, num_heads=2, mlp_ratio=4, qkv_bias=True, block_conf=dict(attention=FULL))
    g = torch.Generator().manual_seed(0)
    with torch.no_grad():
        for name, p in m.named_parameters():
            p.copy_(torch.randn(p.shape, generator=g) * (0.1 if "norm" in name else 0.06) + (1.0 if "norm" in name and name.endswith("weight") else 0.0))
    build_apla(Cfg(), m, "apla_attn")
    m = m.cuda()
    x, w = torch.randn(2, 17, 128, generator=g), torch.randn(2, 17, 128, generator=g)
    with ops.use_half(torch.float16):
        params = [blk.attn.proj_weight1 for blk in m.blocks]
        got = [cpu64(t) for t in torch.autograd.grad((m.run_blocks(x.cuda())[1].float() * w.cuda()).sum(), params)]
    out, p64 = model64(m, x, FULL)
    want = torch.autograd.grad((out * w).sum(), p64)
    for a, b in zip(got, want):
        assert float((a - b).norm()) <= tolerance(2) * float(b.norm())
    g0 = params[0].detach().clone()
    value = lambda: float((model64(m, x, FULL)[0].detach() * w).sum())      # noqa: E731
    d, h = got[0] / got[0].norm(), 1e-4
    params[0].data = (g0.double() + (h * d).cuda())
    up = value()
    params[0].data = (g0.double() - (h * d).cuda())
    down = value()
    params[0].data = g0
    assert abs((up - down) / (2 * h) - float(got[0].norm())) <= tolerance(2) * float(got[0].norm())


@pytest.mark.parametrize("conf", [FULL, dict(rope=True), dict(qk_norm="rms"), dict(causal=True)], ids=["full", "rope", "rms", "causal"])
def test_gradients_of_a_training_step(conf):
    """The loss of a classifier on the module path: its gradients in the projection rows of every block are those of the 64-bit model."""
    from apla_amd.models import Classifier
    from apla_amd.module_trainer import ModulePathTrainer
    torch.manual_seed(0)
    tp = dict(img_size=[64], patch_size=16, block_conf=dict(attention=dict(conf)))
    model = Classifier(dict(backbone_type="vit_tiny", n_classes=10, transformers_params=tp, adaptation=dict(mode="apla", params=dict(partial_size=64))), dict(which_GPUs="0"))
    tr = ModulePathTrainer(model, lr=0.0, weight_decay=0.0, compute_dtype=torch.float16, loss_scale=256.0)
    tokens, run = [], model.backbone.run_blocks
    model.backbone.run_blocks = lambda x, *a, **k: (tokens.append(x), run(x, *a, **k))[1]
    x, y = torch.randn(4, 3, 64, 64, generator=torch.Generator().manual_seed(1)).cuda(), torch.tensor([1, 2, 3, 4])
    loss = float(tr.train_step(x, y.cuda()))
    out, params = model64(model.backbone, tokens[0], conf)
    logits = out[:, 0] @ cpu64(model.fc.weight).t() + cpu64(model.fc.bias)
    want_loss = F.cross_entropy(logits, y)
    assert abs(loss - float(want_loss.detach())) <= tolerance(12) * float(want_loss.detach())
    for blk, want in zip(model.backbone.blocks, torch.autograd.grad(want_loss, params)):
        got = cpu64(blk.attn.proj_weight1.grad)       # (the optimizer has taken the loss scale out)
        assert float((got - want).norm()) <= tolerance(12) * float(want.norm())
