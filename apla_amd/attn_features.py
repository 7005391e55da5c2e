"""What an attention module may do beyond softmax(q k^T) v, as configured by ``block_conf["attention"]`` of the backbones (YAML:
``model_params.transformers_params.block_conf.attention``; self-supervised: ``student.attention``):

    qk_norm: layer | rms        norm of every query and key head before the scores (modules ``q_norm`` / ``k_norm``, as in timm)
    rope: {rot: 64, base: 100.0, layout: half}     rotary positions on the patch grid (class token not turned)
    softcap: 30.0               scores capped to softcap * tanh(s / softcap)
    distance_bias: true         minus 2^(-8 (h + 1) / H) times the distance on the patch grid (class token at its centre)
    causal: true, prefix: 17    raster-order autoregression over a prefix that every token sees

``AttnFeatures`` turns a batch geometry (equal sequences, or a BlockDiagonalMask) into the tables, positions and ScoreMod of
functional.attention_mod_qkv, built once per geometry and kept by the module."""
import math
from typing import Optional, Sequence

import torch

from . import ops
from .rotary import rotary_table_2d

_KEYS = {"qk_norm", "rope", "softcap", "distance_bias", "causal", "prefix"}
_ROPE_KEYS = {"rot", "base", "layout"}


def grid_side(n: int) -> int:
    """Side of the square patch grid behind one class token."""
    side = math.isqrt(n - 1)
    if n < 2 or side * side != n - 1:
        raise ValueError(f"rope / distance_bias need a class token and a square patch grid; got {n} tokens")
    return side


class AttnFeatures:
    def __init__(self, conf, num_heads: int):
        conf = dict(conf)
        unknown = set(conf) - _KEYS
        if unknown:
            raise ValueError(f"block_conf['attention']: unknown keys {sorted(unknown)}; known: {sorted(_KEYS)}")
        self.qk_norm = conf.get("qk_norm") or None
        if self.qk_norm not in (None, "layer", "rms"):
            raise ValueError(f"qk_norm must be layer or rms, got {self.qk_norm!r}")
        rope = conf.get("rope")
        rope = None if rope is False else rope      # ({}: all defaults)
        if rope is not None:
            rope = {} if rope is True else dict(rope)
            if set(rope) - _ROPE_KEYS:
                raise ValueError(f"rope: unknown keys {sorted(set(rope) - _ROPE_KEYS)}; known: {sorted(_ROPE_KEYS)}")
        self.rope = rope
        self.softcap = float(conf.get("softcap") or 0.0)
        self.distance_bias, self.causal = bool(conf.get("distance_bias", False)), bool(conf.get("causal", False))
        self.prefix = int(conf.get("prefix") or 0)
        if self.prefix and not self.causal:
            raise ValueError("a prefix needs causal: true")
        self.num_heads = num_heads
        self._plans, self._captured = {}, set()

    def plan(self, seqlens: Sequence[int], device, packed_mask=None) -> dict:
        """Keyword arguments of functional.attention_mod_qkv for these sequences (equal ones: [n] * batch)."""
        key, cuda = (tuple(seqlens), packed_mask is not None, str(device)), torch.device(device).type == "cuda"
        capturing = cuda and torch.cuda.is_current_stream_capturing()
        p, home = self._plans.get(key, (None, None))
        if p is None:
            p = self._build(list(seqlens), device, packed_mask, capturing)
            if capturing and self.prefix:      # a node of this graph fills the prefix at every replay: a plan for this graph alone
                return p
            if len(self._plans) - len(self._captured) >= 16:      # layouts seen lately, not every one ever seen; a captured graph keeps reading its own
                self._plans = {k: v for k, v in self._plans.items() if k in self._captured}
            home = torch.cuda.current_stream(device).cuda_stream if cuda and torch.cuda.is_available() else None      # (a number: modules are copied and stored)
            self._plans[key] = (p, home)
        if capturing:
            self._captured.add(key)
        elif home is not None and torch.cuda.current_stream(device).cuda_stream != home:
            # what a plan holds was copied from the host and is complete on every stream; given up, its memory waits for this one too
            mod = p["mod"]
            for t in (mod.slopes, mod.pos_q, mod.prefix, *(p.get(n) for n in ("table", "pos", "cu_q"))):
                if t is not None:
                    t.record_stream(torch.cuda.current_stream(device))
        return p

    def _build(self, seqlens, device, packed_mask, capturing: bool) -> dict:
        out = {}
        kinds = sorted(set(seqlens))
        if self.rope is not None:
            rot, base = int(self.rope.get("rot", 64)), float(self.rope.get("base", 100.0))
            tables = {n: rotary_table_2d((grid_side(n),) * 2, rot, base) for n in kinds}
            first = {n: sum(k for k in kinds if k < n) for n in kinds}
            out.update(table=torch.cat([tables[n] for n in kinds]).to(device), layout=self.rope.get("layout", "half"))
            if len(kinds) == 1:
                out["seq_len"] = kinds[0]
            else:
                out["pos"] = torch.cat([first[n] + torch.arange(n) for n in seqlens]).int().to(device)
        slopes = pos = prefix = None
        if self.distance_bias:
            slopes = (2.0 ** (-8.0 * (torch.arange(self.num_heads, dtype=torch.float64) + 1) / self.num_heads)).float().to(device)
            places = {n: _places(grid_side(n)) for n in kinds}
            pos = torch.cat([places[n] for n in seqlens]).contiguous().to(device)
        if self.prefix:
            prefix = torch.full((len(seqlens),), self.prefix, dtype=torch.int32, device=device if capturing else None).to(device)
        out["mod"] = ops.ScoreMod(softcap=self.softcap, slopes=slopes, pos_q=pos, pos_k=pos, causal=self.causal, prefix=prefix)
        if packed_mask is None:
            out["batch"] = len(seqlens)
        else:
            cu = packed_mask.cu_seqlens(device)
            out.update(cu_q=cu, cu_k=cu, max_q=packed_mask.max_seqlen, max_k=packed_mask.max_seqlen)
        return out


def _places(side: int) -> torch.Tensor:
    y, x = torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij")
    centre = torch.full((1, 2), (side - 1) / 2.0)
    return torch.cat((centre, torch.stack((y, x), -1).reshape(-1, 2).float()))


def make_norms(kind: Optional[str]):
    """(q_norm, k_norm) modules over a head of 64 values."""
    if kind is None:
        return None, None
    cls = torch.nn.LayerNorm if kind == "layer" else torch.nn.RMSNorm
    return cls(64, eps=1e-6), cls(64, eps=1e-6)


def has_features(attn) -> bool:
    """Does this attention module do anything that the plain kernels do not?"""
    return isinstance(getattr(attn, "features", None), AttnFeatures) or real_norm(getattr(attn, "q_norm", None)) or real_norm(getattr(attn, "k_norm", None))


def real_norm(m) -> bool:
    return m is not None and not isinstance(m, torch.nn.Identity)
