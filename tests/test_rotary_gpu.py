"""Rotary positions and the norm of queries and keys against the 64-bit restatement (oracle/mod_oracle.py).

Bounds: the result is rounded once (half a step, u = finfo.eps / 2, relative); before that fp32 arithmetic on values of size m (the pair's
sum of magnitudes) adds a few 2^-24 m, bounded here by 2^-20 m.  Sums over n rows in fp32 add (n / 8 + 64) 2^-24 of the sum of magnitudes."""
import pytest
import torch

from apla_amd import ops
from apla_amd import rotary as R
from oracle import mod_oracle as O

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
CASES = [(1, 1, 64, "half"), (7, 3, 64, "interleaved"), (33, 12, 32, "half"), (130, 5, 34, "half"), (65, 8, 2, "interleaved"), (19, 16, 62, "half"),
         (300, 6, 48, "interleaved"), (257, 24, 64, "half")]


def u_of(dt):
    return torch.finfo(dt).eps / 2


def make(shape, dt, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dt)


def table_of(P, rot):
    return R.rotary_table(P, rot, base=1000.0)


def pair_size(x, rot, layout):
    """Sum of magnitudes of an element's pair (itself past rot)."""
    r, m = rot // 2, x.abs().clone()
    if layout == "half":
        m[..., :r] = m[..., r:rot] = x[..., :r].abs() + x[..., r:rot].abs()
    else:
        m[..., 0:rot:2] = m[..., 1:rot:2] = x[..., 0:rot:2].abs() + x[..., 1:rot:2].abs()
    return m


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,heads,rot,layout", CASES)
def test_rotary_both_directions(T, heads, rot, layout, dtype):
    dt, P = DT[dtype], 97
    wide = make((T, (heads + 2) * 64), dt, 1)                 # the rows of a fused activation: columns behind the heads are not touched
    pos = torch.randint(0, P, (T,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    table = table_of(P, rot)
    with ops.use_half(dt):
        xg = wide.cuda()
        for kw, positions in ((dict(pos=pos.cuda()), pos), (dict(seq_len=50), torch.arange(T) % 50)):
            x = wide[:, :heads * 64].double().reshape(T, heads, 64)
            m = pair_size(x, rot, layout)
            for fn, sign in ((ops.rotary_fwd, 1.0), (ops.rotary_bwd, -1.0)):
                got = fn(xg[:, :heads * 64], table.cuda(), heads, layout=layout, **kw).cpu().double().reshape(T, heads, 64)
                want = O.rotate(x, table, positions, layout, sign)
                assert bool(((got - want).abs() <= u_of(dt) * want.abs() + 2.0 ** -20 * m + 1e-7).all())
                assert torch.equal(got[..., rot:], x[..., rot:])
        inplace = wide.cuda()
        ops.rotary_fwd(inplace[:, :heads * 64], table.cuda(), heads, layout=layout, seq_len=50, out=inplace[:, :heads * 64])
        assert torch.equal(inplace[:, heads * 64:].cpu(), wide[:, heads * 64:])
        assert torch.equal(inplace[:, :heads * 64], ops.rotary_fwd(xg[:, :heads * 64], table.cuda(), heads, layout=layout, seq_len=50))


def test_rotary_position_outside_the_table_is_nan_in_its_row_only():
    x, table = make((5, 128), torch.bfloat16, 3), table_of(8, 32)
    pos = torch.tensor([0, 8, 7, -1, 3], dtype=torch.int32)
    y = ops.rotary_fwd(x.cuda(), table.cuda(), 2, pos=pos.cuda()).cpu().float().reshape(5, 2, 64)
    assert bool(torch.isnan(y[[1, 3], :, :32]).all()) and bool(torch.isfinite(y[[0, 2, 4]]).all()) and bool(torch.isfinite(y[..., 32:]).all())


def test_rotary_far_positions_keep_the_angle():
    """Position 1 000 003 at the highest frequency: the angle's own error is that of the 64-bit table rounded to fp32."""
    P = 1_000_004
    pos = torch.tensor([P - 1, 500_001], dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    rows = pos.double()[:, None] * inv
    x = make((2, 64), torch.float16, 4)
    with ops.use_half(torch.float16):
        y = ops.rotary_fwd(x.cuda(), R.rotary_table(P, 64, device="cuda"), 1, pos=pos.cuda()).cpu().double()
    want = O.rotate(x.double().reshape(2, 1, 64), torch.cat((rows.cos(), rows.sin()), 1), torch.arange(2), "half").reshape(2, 64)
    assert bool(((y - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -20 * 4).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("T,Hq,Hkv,rot,layout", [(1, 1, 1, 64, "half"), (5, 3, 1, 0, "half"), (70, 6, 2, 30, "half"), (197, 12, 12, 64, "half"),
                                                 (129, 8, 4, 48, "interleaved"), (1500, 2, 2, 64, "interleaved")])
def test_qk_norm_rotary_both_directions(T, Hq, Hkv, rot, layout, norm, dtype):
    dt, H, eps = DT[dtype], Hq + Hkv, 1e-6
    wide, dy = make((T, (H + Hkv) * 64), dt, 5, 2.0), make((T, H * 64), dt, 6)
    par = torch.randn(4, 64, generator=torch.Generator().manual_seed(7)) * 0.3
    par[:2] += 1.0
    P = 61
    table = table_of(P, rot) if rot else None
    positions = torch.arange(T) % P
    side = torch.tensor([0] * Hq + [1] * Hkv)
    x = wide[:, :H * 64].double().reshape(T, H, 64).requires_grad_(True)
    w = par.double()[:2].clone().requires_grad_(True)
    b = par.double()[2:].clone().requires_grad_(True)
    yn = O.qk_norm(x, w[side], b[side], eps, norm)
    want = O.rotate(yn.detach(), table, positions, layout) if rot else yn.detach()
    g = O.rotate(dy.double().reshape(T, H, 64), table, positions, layout, -1.0) if rot else dy.double().reshape(T, H, 64)
    gx, gw, gb = torch.autograd.grad(yn, (x, w, b), g)
    with ops.use_half(dt):
        kw = dict(norm=norm, q_weight=par[0].cuda(), k_weight=par[1].cuda(), q_bias=par[2].cuda(), k_bias=par[3].cuda(), eps=eps)
        if rot:
            kw.update(table=table.cuda(), layout=layout, seq_len=P)
        y = ops.qk_norm_rotary_fwd(wide.cuda(), Hq, Hkv, **kw)
        fused = torch.full((T, (H + Hkv) * 64), 7.0, dtype=dt, device="cuda")
        dx, dpar = ops.qk_norm_rotary_bwd(dy.cuda(), wide.cuda(), Hq, Hkv, out=fused[:, :H * 64], **kw)
        again, dpar2 = ops.qk_norm_rotary_bwd(dy.cuda(), wide.cuda(), Hq, Hkv, **kw)
        assert torch.equal(dpar, dpar2) and torch.equal(again, dx) and bool((fused[:, H * 64:] == 7.0).all())
        assert torch.equal(ops.qk_norm_rotary_bwd(dy.cuda(), wide.cuda(), Hq, Hkv, want_params=False, **kw)[0], dx)
    u = u_of(dt)
    m = pair_size(yn.detach(), rot, layout) if rot else yn.detach().abs()
    # x^ carries up to 64 additions of values <= 8 standard deviations: 2^-18 of the row's size
    assert bool(((y.cpu().double().reshape(T, H, 64) - want).abs() <= u * want.abs() + 2.0 ** -18 * (m + 8)).all())
    row = gx.abs().amax(-1, keepdim=True) + (g.abs().amax(-1, keepdim=True) * 2 / x.detach().std(-1, keepdim=True).clamp(min=1e-3))
    assert bool(((dx.cpu().double().reshape(T, H, 64) - gx).abs() <= u * gx.abs() + 2.0 ** -17 * row).all())
    xh = (yn.detach() - b.detach()[side]) / w.detach()[side]
    n = (T * max(Hq, Hkv) / 8 + 64) * 2.0 ** -24 + 2.0 ** -18
    for k in range(2):
        size = (g * xh)[:, side == k].abs().sum((0, 1)), g[:, side == k].abs().sum((0, 1))
        assert bool(((dpar[k].cpu().double() - gw[k]).abs() <= n * (size[0] + size[1])).all())
        assert bool(((dpar[2 + k].cpu().double() - gb[k]).abs() <= n * size[1]).all())


@pytest.mark.parametrize("T,Hq,Hkv", [(2, 769, 1), (3, 401, 399), (1, 1, 1021)])
def test_qk_norm_rotary_of_hundreds_of_odd_heads(T, Hq, Hkv):
    """Few tokens of many heads that no block size divides: the blocks are spread over as many workgroups as the sums' workspace has rows, not more."""
    test_qk_norm_rotary_both_directions(T, Hq, Hkv, 32, "half", "layer", "bf16")


def test_qk_norm_rotary_constant_row_and_defaults():
    """A head of equal values: variance 0, LayerNorm gives the bias; no weights means 1 / 0, no table means no rotation."""
    x = torch.full((3, 192), 2.5, dtype=torch.bfloat16)
    y = ops.qk_norm_rotary_fwd(x.cuda(), 2, 1, norm="layer").cpu()
    assert bool((y == 0).all())
    y = ops.qk_norm_rotary_fwd(x.cuda(), 2, 1, norm="rms").cpu().float()
    assert bool(((y - 1).abs() <= 2.0 ** -8).all())
    empty = torch.empty(0, 192, dtype=torch.bfloat16, device="cuda")
    assert ops.qk_norm_rotary_fwd(empty, 2, 1).shape == (0, 192)
    assert bool((ops.qk_norm_rotary_bwd(empty, empty, 2, 1)[1] == 0).all()) and ops.rotary_fwd(empty, table_of(4, 8).cuda(), 3).shape == (0, 192)


def test_refusals():
    x, tab = torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda"), table_of(8, 16).cuda()
    bad = [lambda: ops.rotary_fwd(x, tab, 3), lambda: ops.rotary_fwd(x, tab[:2].contiguous(), 2), lambda: ops.rotary_fwd(x, tab, 2, layout="thirds"),
           lambda: ops.rotary_fwd(x, table_of(8, 64).repeat(1, 2).cuda(), 2), lambda: ops.rotary_fwd(x, tab, 2, seq_len=9), lambda: ops.rotary_fwd(x, tab, 2, seq_len=-1),
           lambda: ops.rotary_fwd(x, tab, 2, pos=torch.zeros(3, dtype=torch.int32, device="cuda")), lambda: ops.rotary_fwd(x, None, 2),
           lambda: ops.rotary_fwd(x[:1].expand(4, 128), tab, 2), lambda: ops.rotary_fwd(torch.zeros(4, 132, dtype=torch.bfloat16, device="cuda")[:, 4:], tab, 2),
           lambda: ops.rotary_fwd(x, tab, 2, out=x.view(-1)[:384].view(3, 128)), lambda: ops.rotary_fwd(x[:3], tab, 2, out=x[1:]),
           lambda: ops.qk_norm_rotary_fwd(x, 2, 1), lambda: ops.qk_norm_rotary_fwd(x, 0, 1), lambda: ops.qk_norm_rotary_fwd(x, 1, 1, norm="batch"),
           lambda: ops.qk_norm_rotary_fwd(x, 1, 1, eps=-1.0), lambda: ops.qk_norm_rotary_fwd(x, 1, 1, q_weight=torch.ones(32, device="cuda")),
           lambda: ops.qk_norm_rotary_fwd(x, 1, 1, seq_len=4), lambda: ops.qk_norm_rotary_bwd(x[:3], x, 1, 1),
           lambda: ops.qk_norm_rotary_bwd(x[:3], torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda"), 1, 1, out=x[1:])]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {k} was accepted")
    for f in (lambda: ops.rotary_fwd(x.float(), tab, 2), lambda: ops.rotary_fwd(x, tab.double(), 2), lambda: ops.rotary_fwd(x, tab, 2, pos=torch.zeros(4, device="cuda")),
              lambda: ops.qk_norm_rotary_fwd(x, 1, 1, q_weight=torch.ones(64, device="cuda", dtype=torch.bfloat16))):
        with pytest.raises(TypeError):
            f()


def test_side_stream_and_graph():
    """Another stream than the tensors' own, and a captured forward + backward replayed on new inputs with eager work between."""
    dt = torch.bfloat16
    x, dy = make((257, 8 * 64), dt, 8).cuda(), make((257, 6 * 64), dt, 9).cuda()
    w = torch.rand(64, device="cuda") + 0.5
    kw = dict(norm="rms", q_weight=w, k_weight=w, table=table_of(257, 64).cuda())
    f = lambda: (ops.qk_norm_rotary_fwd(x, 4, 2, **kw), *ops.qk_norm_rotary_bwd(dy, x, 4, 2, **kw))     # noqa: E731
    eager = f()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        side = f()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, side))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    for k in range(3):
        x.copy_(make((257, 8 * 64), dt, 20 + k))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(f(), out))
