"""Rotary positions, q / k norm and attention with modified scores as autograd nodes: what they save, and what they refuse."""
import pytest
import torch
from torch import nn

from apla_amd import functional as AF
from apla_amd import ops
from apla_amd import rotary as R

pytestmark = pytest.mark.gpu
T, H = 48, 2


def rows(seed, cols=H * 64):
    return torch.randn(T, cols, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda().requires_grad_(True)


def nodes():
    """name -> (function of its differentiable inputs, those inputs, the other tensors that its backward reads)"""
    table, pos = R.rotary_table(T, 64, device="cuda"), torch.arange(T, dtype=torch.int32).flip(0).cuda()
    slopes, doc, prefix = torch.full((H,), 0.25, device="cuda"), (torch.arange(T, dtype=torch.int32) // 20).cuda(), torch.tensor([5], dtype=torch.int32).cuda()
    mod = ops.ScoreMod(softcap=9.0, slopes=slopes, doc_q=doc, doc_k=doc, causal=True, prefix=prefix)
    used = torch.tensor([T - 3], dtype=torch.int32).cuda()
    w = [(torch.rand(64, generator=torch.Generator().manual_seed(9 + i)) + 0.5).cuda().requires_grad_(True) for i in range(2)]
    w16 = [p.detach().bfloat16().requires_grad_(True) for p in w]
    norms = [nn.LayerNorm(64).cuda() for _ in range(2)]
    return {
        "rotary": (lambda x: AF.rotary(x, table, H, pos=pos), [rows(1)], [table, pos]),
        "norm": (lambda x, a, b: AF.qk_norm_rotary(x, 1, 1, q_weight=a, k_weight=b, table=table, pos=pos), [rows(2), *w], [table, pos]),
        "norm16": (lambda x, a, b: AF.qk_norm_rotary(x, 1, 1, norm="rms", q_weight=a, k_weight=b, table=table, pos=pos), [rows(2), *w16], [table, pos]),
        "attention": (lambda q, k, v: AF.attention_mod(q, k, v, H, H, 0.125, mod, batch=1, len_k=used)[0], [rows(3), rows(4), rows(5)], [slopes, doc, prefix, used]),
        "qkv": (lambda x, *_: AF.attention_mod_qkv(x, H, 0.125, mod=mod, q_norm=norms[0], k_norm=norms[1], table=table, pos=pos, batch=1),
                [rows(6, 3 * H * 64), norms[0].weight, norms[1].weight], [table, pos, slopes, doc, prefix]),
    }


NAMES = ["rotary", "norm", "norm16", "attention", "qkv"]


def gradients(f, inputs):
    o = f(*inputs)
    return torch.autograd.grad(o, inputs, torch.ones_like(o))


@pytest.mark.parametrize("name", NAMES)
def test_what_the_backward_reads_passes_saved_tensor_hooks(name):
    """Kept on the host between the passes: every tensor that the backward reads is handed out, and the gradients are the same bits."""
    f, inputs, side = nodes()[name]
    seen = []

    def out(t):
        seen.append(t.data_ptr())
        return t.cpu()
    want = gradients(f, inputs)
    with torch.autograd.graph.saved_tensors_hooks(out, lambda t: t.cuda()):
        got = gradients(f, inputs)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert {t.data_ptr() for t in side} <= set(seen)


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(name):
    f, inputs, _ = nodes()[name]
    o = f(*inputs)
    (g, *_) = torch.autograd.grad(o.float().square().sum(), inputs, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):      # (not the part of it that other nodes know)
        (g.float().square().sum() + o.float().sum()).backward()


@pytest.mark.parametrize("name", NAMES)
def test_arguments_changed_in_place_are_refused(name):
    f, inputs, side = nodes()[name]
    for t in side + inputs[1:]:
        o = f(*inputs)
        with torch.no_grad():
            t.add_(0)
        with pytest.raises(RuntimeError, match="in place"):
            torch.autograd.grad(o, inputs, torch.ones_like(o))


def test_a_score_modification_changed_after_the_forward_does_not_matter():
    q, k, v = rows(1), rows(2), rows(3)
    mod = ops.ScoreMod(softcap=5.0, slopes=torch.full((H,), 0.5, device="cuda"), causal=True)
    o, _ = AF.attention_mod(q, k, v, H, H, 0.125, mod, batch=1)
    want = torch.autograd.grad(o, (q, k, v), torch.ones_like(o), retain_graph=True)
    mod.softcap, mod.slopes, mod.causal = 0.0, None, False
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(o, (q, k, v), torch.ones_like(o))))


def test_tensors_made_in_inference_mode_may_be_arguments():
    """A plan or table that an evaluation built first is used in training."""
    with torch.inference_mode():
        table, slopes = R.rotary_table(T, 64, device="cuda"), torch.full((H,), 0.5, device="cuda")
    q, k, v = rows(1), rows(2), rows(3)
    f = lambda a, b, c: AF.attention_mod(AF.rotary(a, table, H), b, c, H, H, 0.125, ops.ScoreMod(slopes=slopes), batch=1)[0]      # noqa: E731
    got = gradients(f, [q, k, v])
    table, slopes = table.clone(), slopes.clone()
    assert all(torch.equal(a, b) for a, b in zip(got, gradients(f, [q, k, v])))


def test_a_learned_table_is_refused():
    table, x = R.rotary_table(T, 64, device="cuda").requires_grad_(True), rows(1, 3 * H * 64)
    for f in (lambda: AF.rotary(x, table, 3 * H), lambda: AF.qk_norm_rotary(x, H, H, table=table), lambda: AF.attention_mod_qkv(x, H, 0.125, table=table, batch=1)):
        with pytest.raises(NotImplementedError, match="table"):
            f()
        with torch.no_grad():
            assert torch.isfinite(f().float()).all()


def test_a_captured_backward_refuses_leaves_of_a_living_eager_graph():
    """The gradient of such a leaf is added on the eager graph's stream, which a capture must not touch.  Without the eager graph the backward is captured."""
    w, x = torch.rand(64, device="cuda").add_(0.5).requires_grad_(True), rows(1)
    step = lambda: torch.autograd.grad(AF.qk_norm_rotary(x, H, 0, q_weight=w), [x, w], torch.ones_like(x))      # noqa: E731
    eager = AF.qk_norm_rotary(x, H, 0, q_weight=w)
    refused, g = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(refused):
            step()
    del eager
    with torch.cuda.graph(g):
        got = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(rows(20 + i))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
