"""Tables of rotary positions for ops.rotary_* / ops.qk_norm_rotary_* (cosines, then sines, of rot / 2 angles per position).

The angles are formed in 64 bits and rounded once: fp32 arithmetic on position * frequency would lose 2^-24 * position of the angle, half a
turn at position 10^7 and 2^-7 at 131072.  A caller builds a table once and passes it to every call; modules with attention features build one
each per geometry (1370 positions x 64: 350 KB)."""
import math
from typing import Optional, Sequence

import torch


def rotary_frequencies(rot: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0, trained: int = 0,
                       beta_fast: float = 32.0, beta_slow: float = 1.0) -> torch.Tensor:
    """fp64 [rot / 2] angles per position, base^(-2 i / rot), for ranges ``factor`` times the trained one:
    "linear"  every angle divided by factor (positions squeezed into the trained range);
    "ntk"     the base raised by factor^(rot / (rot - 2)): the slowest pair is squeezed by factor, the fastest not at all;
    "yarn"    per pair: those that turn more than beta_fast times over the ``trained`` range stay, those below beta_slow turns are divided by
              factor, a linear ramp over the pair index between.  The ramp's ends are rounded outwards to whole indices and cut to
              0 .. rot - 1, as published: its upper end may lie past the last pair, rot / 2 - 1, which then is divided in part."""
    if rot % 2 or not 2 <= rot <= 64:
        raise ValueError(f"rot must be even, 2..64, got {rot}")
    if base <= 1.0 or factor < 1.0:
        raise ValueError("need base > 1 and factor >= 1")
    if scaling == "ntk":
        if rot < 4:
            raise ValueError("ntk scaling needs rot >= 4")
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        if trained <= 0 or not beta_fast > beta_slow > 0:
            raise ValueError("yarn scaling needs the trained range and beta_fast > beta_slow > 0")
        pair = lambda turns: rot / 2 * math.log(trained / (2 * math.pi * turns)) / math.log(base)      # noqa: E731  (index of the pair with that many turns)
        lo, hi = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot - 1)
        i = torch.arange(rot // 2, dtype=torch.float64)
        ramp = torch.where(i >= hi, 1.0, ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1))      # (hi <= lo: no pair turns even beta_slow times)
        return f * (1 - ramp) + f / factor * ramp
    if scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return f


def rotary_table(positions, rot: int = 64, base: float = 10000.0, *, device=None, amplitude: float = 1.0, **scaling) -> torch.Tensor:
    """fp32 [P, rot].  ``positions``: how many (0 .. P-1), or a tensor of P places.  ``amplitude`` multiplies cosines and sines (the attention
    temperature of stretched ranges); ``scaling``: see rotary_frequencies."""
    p = torch.arange(positions, dtype=torch.float64) if isinstance(positions, int) else torch.as_tensor(positions).double().reshape(-1)
    dev = device or p.device
    a = p.to(dev)[:, None] * rotary_frequencies(rot, base, **scaling).to(dev)
    return torch.cat((a.cos() * amplitude, a.sin() * amplitude), 1).float()


def rotary_table_2d(grid: Sequence[int], rot: int = 64, base: float = 100.0, *, prefix: int = 1, device=None) -> torch.Tensor:
    """fp32 [prefix + h * w, rot] for the tokens of a vision transformer: ``prefix`` tokens that do not turn (class / register tokens: angle 0), then
    the patches of a (h, w) grid in raster order.  The first half of the pairs turns with the row, the second half with the column,
    each with the frequencies base^(-2 i / (rot / 2))."""
    h, w = (int(n) for n in grid)
    if rot % 4 or not 4 <= rot <= 64 or h < 1 or w < 1 or prefix < 0:
        raise ValueError(f"need rot a multiple of 4, 4..64, and a grid (got rot={rot}, grid={tuple(grid)}, prefix={prefix})")
    f = rotary_frequencies(rot // 2, base)
    y, x = torch.meshgrid(torch.arange(h, dtype=torch.float64), torch.arange(w, dtype=torch.float64), indexing="ij")
    a = torch.cat((y.reshape(-1, 1) * f, x.reshape(-1, 1) * f), 1)
    a = torch.cat((torch.zeros(prefix, rot // 2, dtype=torch.float64), a))
    return torch.cat((a.cos(), a.sin()), 1).float().to(device or "cpu")
