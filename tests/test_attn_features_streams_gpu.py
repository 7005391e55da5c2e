"""Plans of attention features (attn_features.py) that several streams and captured graphs share."""
import copy
import io

import pytest
import torch

from apla_amd import functional as AF
from apla_amd import ops
from apla_amd.vit import Attention

pytestmark = pytest.mark.gpu
N, H, D, PREFIX = 64, 2, 128, 40


def setup():
    attn = Attention(D, H, features=dict(causal=True, prefix=PREFIX)).cuda().eval()
    qkv = torch.randn(2, N, 3 * D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    rows = qkv.reshape(2 * N, 3 * D)
    mod = ops.ScoreMod(causal=True, prefix=torch.full((2,), PREFIX, dtype=torch.int32).cuda())
    want, _ = ops.attn_mod_fwd(rows[:, :D], rows[:, D:2 * D], rows[:, 2 * D:], H, H, attn.scale, mod, batch=2)
    torch.cuda.synchronize()
    return attn, qkv, want.reshape(2, N, D)


def keep_busy(stream):
    """Some tens of milliseconds of products in the stream's queue."""
    with torch.cuda.stream(stream):
        a = torch.ones(4096, 4096, device="cuda", dtype=torch.bfloat16)
        for _ in range(400):
            a @ a


def small_blocks(value):
    """Small integer tensors on the current stream: what freed memory of a prefix would be used for next."""
    return [torch.full((2,), value, dtype=torch.int32, device="cuda") for _ in range(64)]


@torch.no_grad()
def test_a_plan_first_built_in_a_capture_is_that_graph_s_alone():
    attn, qkv, want = setup()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = AF.attention_features(attn, qkv)
    assert torch.equal(AF.attention_features(attn, qkv), want)      # before the first replay
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(AF.attention_features(attn, qkv), want)


@torch.no_grad()
def test_a_plan_built_on_one_stream_is_complete_on_another():
    attn, qkv, want = setup()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        small_blocks(0)
    torch.cuda.synchronize()
    keep_busy(a)
    with torch.cuda.stream(a):
        attn.features.plan([N] * 2, qkv.device)
    with torch.cuda.stream(b):
        got = AF.attention_features(attn, qkv)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@torch.no_grad()
def test_memory_of_a_plan_given_up_waits_for_the_streams_that_read_it():
    attn, qkv, want = setup()
    side = torch.cuda.Stream()
    attn.features.plan([N] * 2, qkv.device)
    torch.cuda.synchronize()
    keep_busy(side)
    with torch.cuda.stream(side):
        got = AF.attention_features(attn, qkv)
    attn.features.prefix = 1        # what later plans write into memory that comes free
    for n in range(100, 120):
        attn.features.plan([n] * 2, qkv.device)
    held = small_blocks(0)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and len(held) == 64


@torch.no_grad()
def test_modules_with_plans_are_copied_and_stored():
    attn, qkv, want = setup()
    AF.attention_features(attn, qkv)
    assert torch.equal(AF.attention_features(copy.deepcopy(attn), qkv), want)
    torch.save(attn, io.BytesIO())
