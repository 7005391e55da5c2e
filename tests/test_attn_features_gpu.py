"""q / k norm, rotary positions and modified scores as modules use them: the fused node against its parts, the modules against a 64-bit
restatement, the plugin, packed crops, and training steps."""
import math

import pytest
import torch
from torch import nn

from apla_amd import functional as AF
from apla_amd import ops
from apla_amd import rotary as R
from apla_amd.apla import build_apla
from apla_amd.attn_features import AttnFeatures
from apla_amd.nested import BlockDiagonalMask
from apla_amd.vit import Attention, VisionTransformer
from oracle import mod_oracle as O

pytestmark = pytest.mark.gpu
FULL = dict(qk_norm="layer", rope=dict(rot=32, base=50.0), softcap=8.0, distance_bias=True, causal=True, prefix=5)


class Cfg:
    partial_size = 64


def randomise(m, seed=0):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "norm" in n:
                p.copy_(torch.randn(p.shape, generator=g) * 0.1 + (1.0 if n.endswith("weight") else 0.0))
            else:
                p.copy_(torch.randn(p.shape, generator=g) * 0.06)
    return m


def dense_reference(qkv, attn, n, H):
    """o of one image's qkv rows [n, 3 * H * 64] (fp64) with every feature of FULL, and the largest score error that 16-bit q / k would cause
    per unit of rounding."""
    side = math.isqrt(n - 1)
    q, k, v = qkv.reshape(n, 3, H, 64).unbind(1)
    table = R.rotary_table_2d((side, side), 32, 50.0)
    rot = lambda x, m: O.rotate(O.qk_norm(x, m.weight.detach().double().cpu(), m.bias.detach().double().cpu(), 1e-6, "layer"), table, torch.arange(n), "half")   # noqa: E731
    q, k = rot(q, attn.q_norm), rot(k, attn.k_norm)
    y, x = torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij")
    pos = torch.cat((torch.full((1, 2), (side - 1) / 2), torch.stack((y, x), -1).reshape(-1, 2)))
    see, dist = O.visible(n, n, True, 5), O.distance(n, n, pos, pos)
    out, ds, mag = [], 0.0, []
    for h in range(H):
        w = O.attend(q[:, h], k[:, h], v[:, h], 0.125, see, 8.0, 2.0 ** (-8 * (h + 1) / H), dist)
        out.append(w["o"])
        mag.append(w["p"] @ v[:, h].abs())
        ds = max(ds, float((q[:, h].abs() @ k[:, h].abs().t()).max()) * 0.125)
    return torch.cat(out, 1), torch.cat(mag, 1), ds


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fused_node_is_its_parts_and_the_formula(dtype):
    B, n, H = 2, 50, 3
    attn = randomise(Attention(H * 64, H, features=FULL)).cuda()
    with ops.use_half(dtype):
        x = (torch.randn(B, n, 3 * H * 64, generator=torch.Generator().manual_seed(1)) * 2).to(dtype).cuda().requires_grad_(True)
        do = torch.randn(B, n, H * 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
        par = [attn.q_norm.weight, attn.k_norm.weight, attn.q_norm.bias, attn.k_norm.bias]
        o = AF.attention_features(attn, x)
        g = torch.autograd.grad(o, [x] + par, do)
        kw = attn.features.plan([n] * B, x.device)
        qk = AF.qk_norm_rotary(x, H, H, norm="layer", q_weight=par[0], k_weight=par[1], q_bias=par[2], k_bias=par[3], eps=1e-6, table=kw["table"], seq_len=n)
        c = H * 64
        o2, lse = AF.attention_mod(qk[..., :c], qk[..., c:], x[..., 2 * c:], H, H, 0.125, kw["mod"], batch=B)
        g2 = torch.autograd.grad(o2, [x] + par, do)
        assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(g, g2)) and lse.shape == (H, B * n)
    u = torch.finfo(dtype).eps / 2
    for b in range(B):      # q and k are rounded after the rotation (2 u of the score's magnitudes), then the bounds of the attention itself
        want, mag, ds = dense_reference(x[b].detach().double().cpu(), attn, n, H)
        assert bool(((o[b].detach().double().cpu() - want).abs() <= (2 * (2.1 * u * ds) + u + 2.0 ** -15) * mag + u * want.abs() + 1e-6).all())


def test_rotary_function_and_its_gradient():
    x = torch.randn(2, 17, 128, generator=torch.Generator().manual_seed(3)).bfloat16().cuda().requires_grad_(True)
    t = R.rotary_table(17, 64, device="cuda")
    y = AF.rotary(x, t, 2, seq_len=17)
    (g,) = torch.autograd.grad(y, x, y.detach())
    assert float((g.float() - x.detach().float()).abs().max()) <= 3 * 2.0 ** -8 * float(x.detach().abs().max())     # R^T R = 1 up to three roundings of a pair


class TimmAttention(nn.Module):
    """A timm-style host module: qkv, q_norm, k_norm, proj."""

    def __init__(self, dim, heads, q_norm, k_norm):
        super().__init__()
        self.num_heads, self.scale = heads, (dim // heads) ** -0.5
        self.qkv, self.proj = nn.Linear(dim, 3 * dim), nn.Linear(dim, dim)
        self.q_norm, self.k_norm = q_norm, k_norm
        self.attn_drop, self.proj_drop = nn.Dropout(0.0), nn.Dropout(0.0)


class Host(nn.Module):
    def __init__(self, make, n=1):
        super().__init__()
        self.blocks = nn.ModuleList([nn.Module() for _ in range(n)])
        for b in self.blocks:
            b.attn = make()


@pytest.mark.parametrize("norm", [nn.LayerNorm, nn.RMSNorm])
def test_plugin_keeps_the_norms_of_the_module_it_replaces(norm):
    n, H, D = 30, 2, 128
    host = Host(lambda: randomise(TimmAttention(D, H, norm(64, eps=1e-5), norm(64, eps=1e-5))))
    src = host.blocks[0].attn
    ref = [p.detach().double().clone() for p in (src.qkv.weight, src.qkv.bias, src.proj.weight, src.proj.bias)]
    qn, kn = src.q_norm, src.k_norm
    build_apla(Cfg(), host, "apla_attn")
    new = host.blocks[0].attn.cuda()
    assert new.q_norm is qn and new.k_norm is kn and not any(p.requires_grad for p in qn.parameters())
    x = torch.randn(1, n, D, generator=torch.Generator().manual_seed(4)) * 2
    with ops.use_half(torch.float16):
        y, _ = new(x.cuda())
    X = x[0].double()
    q, k, v = (X @ ref[0].t() + ref[1]).reshape(n, 3, H, 64).unbind(1)
    kind = "layer" if norm is nn.LayerNorm else "rms"
    wb = lambda m: (m.weight.detach().double().cpu(), 0.0 if getattr(m, "bias", None) is None else m.bias.detach().double().cpu())     # noqa: E731
    q, k = O.qk_norm(q, *wb(qn), 1e-5, kind), O.qk_norm(k, *wb(kn), 1e-5, kind)
    o = torch.cat([O.attend(q[:, h], k[:, h], v[:, h], 0.125, O.visible(n, n))["o"] for h in range(H)], 1)
    want = o @ ref[2].t() + ref[3]
    plain = torch.cat([O.attend(*(t[:, h] for t in (X @ ref[0].t() + ref[1]).reshape(n, 3, H, 64).unbind(1)), 0.125, O.visible(n, n))["o"] for h in range(H)], 1) @ ref[2].t() + ref[3]
    err = float((y[0].detach().double().cpu() - want.detach()).norm() / want.detach().norm())
    # ten roundings of 2^-11 on the way, q and k twice with scores up to ~8: (10 + 2 * 2 * 8) 2^-11
    assert err <= 42 * 2.0 ** -11 and float((plain - want).norm() / want.norm()) > 0.1


def test_plugin_refuses_what_it_cannot_keep():
    for bad in ((nn.LayerNorm(64), nn.Identity()), (nn.LayerNorm(64), nn.RMSNorm(64)), (nn.LayerNorm(32), nn.LayerNorm(32)), (nn.BatchNorm1d(64), nn.BatchNorm1d(64)),
                (nn.LayerNorm(64, eps=1e-5), nn.LayerNorm(64, eps=1e-6))):
        with pytest.raises(NotImplementedError):
            build_apla(Cfg(), Host(lambda: TimmAttention(128, 2, *bad)), "apla_attn")
    host = build_apla(Cfg(), Host(lambda: TimmAttention(128, 2, nn.Identity(), nn.Identity())), "apla_attn")
    assert not hasattr(host.blocks[0].attn, "q_norm")
    attn = Attention(128, 2, attn_drop=0.1, features=dict(softcap=5.0)).cuda().train()
    x = torch.zeros(1, 10, 128, device="cuda")
    with pytest.raises(NotImplementedError):
        attn(x)
    attn.eval()(x)
    attn.return_attn_matrix = True
    with pytest.raises(NotImplementedError):
        attn(x)
    for conf in (dict(qk_norm="batch"), dict(prefix=3), dict(ropes={}), dict(rope=dict(theta=1))):
        with pytest.raises(ValueError):
            AttnFeatures(conf, 2)
    with pytest.raises(ValueError):
        Attention(128, 2, features=dict(rope=True)).cuda()(torch.zeros(1, 12, 128, device="cuda"))     # 11 patches are no square grid


def test_packed_crops_are_the_crops_one_by_one():
    H, D = 2, 128
    attn = randomise(Attention(D, H, features=FULL)).cuda()
    qkv = [torch.randn(b, n, 3 * D, generator=torch.Generator().manual_seed(n)).bfloat16().cuda().requires_grad_(True) for b, n in ((2, 26), (3, 10))]
    mask, packed = BlockDiagonalMask.from_tensor_list(qkv)
    o = AF.attention_features(attn, packed, mask)
    do = torch.randn(o.shape, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    g = torch.autograd.grad(o, qkv, do)
    for x, part, dpart, got in zip(qkv, mask.split(o), mask.split(do), g):
        one = AF.attention_features(attn, x)
        assert torch.equal(one, part)
        assert torch.equal(torch.autograd.grad(one, x, dpart.contiguous())[0], got)


@pytest.mark.parametrize("conf", [FULL, dict(rope=True), dict(qk_norm="rms"), dict(causal=True)], ids=["full", "rope", "rms", "causal"])
def test_training_steps_on_the_module_path(conf):
    """A classifier whose blocks have the features: the fused engine refuses it, the module-path trainer runs forward, backward and optimizer steps, and the
    gradient of the loss agrees with a difference along a direction in one projection row block."""
    from apla_amd.engine import AplaTrainEngine
    from apla_amd.models import Classifier
    from apla_amd.module_trainer import ModulePathTrainer
    torch.manual_seed(0)
    tp = dict(img_size=[64], patch_size=16, block_conf=dict(attention=dict(conf)))
    model = Classifier(dict(backbone_type="vit_tiny", n_classes=10, transformers_params=tp, adaptation=dict(mode="apla", params=dict(partial_size=64))), dict(which_GPUs="0"))
    with pytest.raises(NotImplementedError):
        AplaTrainEngine(model, 4, 64)
    tr = ModulePathTrainer(model, lr=1e-3)
    x, y = torch.randn(4, 3, 64, 64, generator=torch.Generator().manual_seed(1)).cuda(), torch.tensor([1, 2, 3, 4]).cuda()
    losses = [float(tr.train_step(x, y)) for _ in range(2)]
    grads = [p.grad for p in model.parameters() if p.requires_grad]
    assert all(math.isfinite(v) for v in losses) and math.isfinite(float(tr.grad_norm)) and all(g is None or bool(torch.isfinite(g).all()) for g in grads)
    _, emb, _ = tr.forward_only(x)
    plain = VisionTransformer(img_size=[64], patch_size=16, embed_dim=192, depth=12, num_heads=3, mlp_ratio=4, qkv_bias=True)
    assert emb.shape == (4, 192) and set(plain.state_dict()) <= set(VisionTransformer(img_size=[64], patch_size=16, embed_dim=192, depth=12, num_heads=3, mlp_ratio=4, qkv_bias=True,
                                                                                      block_conf=dict(attention=dict(conf))).state_dict())


def test_gradient_of_the_loss_through_a_model_against_differences():
    """fp16, full features, two blocks: the directional derivative along the trainable projection rows by central differences (the forward's
    rounding noise of 2^-11 of the output over a step of 2^-3 of the weights bounds the agreement)."""
    torch.manual_seed(0)
    m = VisionTransformer(img_size=[64], patch_size=16, embed_dim=128, depth=2, num_heads=2, mlp_ratio=4, qkv_bias=True, block_conf=dict(attention=FULL))
    randomise(m)
    build_apla(Cfg(), m, "apla_attn")
    m = m.cuda()
    x, w = torch.randn(2, 17, 128, generator=torch.Generator().manual_seed(1)).cuda(), torch.randn(2, 17, 128, generator=torch.Generator().manual_seed(2)).cuda()
    with ops.use_half(torch.float16):
        val = lambda: (m.run_blocks(x)[1].float() * w).sum()      # noqa: E731
        p = m.blocks[0].attn.proj_weight1
        (g,) = torch.autograd.grad(val(), p)
        d = torch.randn(p.shape, generator=torch.Generator().manual_seed(3)).cuda()
        h = 2.0 ** -3 * float(p.detach().norm() / d.norm())
        with torch.no_grad():
            p.add_(h * d)
            up = float(val())
            p.sub_(2 * h * d)
            down = float(val())
    diff, an = (up - down) / (2 * h), float((g * d).sum())
    # noise: 2 * 34 * 128 output values with errors of ~8 roundings each, independent; curvature: h^2 (a step of 1/8 changes the gradient by O(1/64))
    noise = 8 * 2.0 ** -11 * float((2 * 17 * 128) ** 0.5) * 2 / (2 * h)
    assert abs(diff - an) <= noise + 0.05 * float(g.norm() * d.norm()) / 4, (diff, an, noise)


def test_broadcast_and_unaligned_inputs():
    """One key / value row for all tokens (stride 0) and rows at an odd address: copied, and the gradient of a broadcast input is summed."""
    T, H = 40, 2
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(T * 128 + 1, generator=g).bfloat16().cuda()
    q = flat[1:].reshape(T, 128)
    k1 = torch.randn(1, 128, generator=g).bfloat16().cuda().requires_grad_(True)
    kc = k1.detach().expand(T, 128).contiguous().requires_grad_(True)
    table = R.rotary_table(T, 64, device="cuda")
    do = torch.randn(T, 128, generator=g).bfloat16().cuda()
    o, _ = AF.attention_mod(q, AF.rotary(k1.expand(T, 128), table, H), k1.expand(T, 128), H, H, 0.125, ops.ScoreMod(causal=True), batch=1)
    oc, _ = AF.attention_mod(q.clone(), AF.rotary(kc, table, H), kc, H, H, 0.125, ops.ScoreMod(causal=True), batch=1)
    assert torch.equal(o, oc)
    (a,), (b,) = torch.autograd.grad(o, k1, do), torch.autograd.grad(oc, kc, do)
    # a: 16-bit sums over 40 rows of what b holds row by row; each of a sum's partial results may be rounded to 16 bits
    want = b.double().sum(0)
    assert ((a[0].double() - want).abs() <= 2 * T * 2.0 ** -8 * b.double().abs().sum(0)).all()


def test_arguments_changed_between_forward_and_backward_are_refused():
    T, H = 16, 1
    z = lambda: torch.randn(T, 64, device="cuda").bfloat16().requires_grad_(True)      # noqa: E731
    slopes, used, table = torch.ones(H, device="cuda"), torch.full((1,), T, dtype=torch.int32, device="cuda"), R.rotary_table(T, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for t, make in ((slopes, lambda: AF.attention_mod(z(), z(), z(), H, H, 0.125, ops.ScoreMod(slopes=slopes), batch=1)[0]),
                    (used, lambda: AF.attention_mod(z(), z(), z(), H, H, 0.125, batch=1, len_k=used)[0]),
                    (table, lambda: AF.rotary(z(), table, H)), (w, lambda: AF.qk_norm_rotary(z(), H, 0, q_weight=w))):
        make().sum().backward()
        o = make()
        t.add_(0)
        with pytest.raises(RuntimeError, match="in place"):
            o.sum().backward()
