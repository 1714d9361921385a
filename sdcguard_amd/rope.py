"""Rotary positions: the heads of queries or keys rotated by their tokens' positions (no counterpart in the reference).

Pair i of a head at position p is turned by the angle 2 pi p turns[i]: (a, b) becomes (a c - b s, b c + a s) with
c = mscale cos, s = mscale sin.  A pair is (i, i + rot / 2) of the first rot = 2 len(turns) elements, or (2 i, 2 i + 1)
with `interleaved`; elements past rot are copied.  Angles are taken in 64 bits, so positions of a million lose nothing.
The work is one launch of sdc_rope (csrc/rope.hip; checks and gradient in csrc/bind.cpp); there is no CPU implementation.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

SCALINGS = ("linear", "base", "ramp", "bands")


def frequencies(rot: int, base: float = 10000.0, scaling: Optional[dict] = None, device="cuda"):
    """(turns, mscale): the turns each of the rot / 2 pairs makes per position (float64, on `device`), base ** (-2 i / rot)
    / 2 pi, and the factor on the rotated elements.  `scaling` (a dict with "kind" and "factor") stretches them for
    contexts longer than the trained one:

      linear   every pair slower by factor (positions interpolated)
      base     the base raised by factor ** (rot / (rot - 2)): the fastest pair kept, the slowest slower by factor
      ramp     pairs that turn over "fast" (32) times within "trained" positions kept, those under "slow" (1) times slower
               by factor, a linear ramp over the pair number between; mscale = 1 + 0.1 ln factor
      bands    by wavelength: shorter than trained / "high" (4) kept, longer than trained / "low" (1) slower by factor,
               between them blended linearly in trained / wavelength"""
    rot = int(rot)
    if rot < 2 or rot % 2:
        raise ValueError(f"an even number of rotated elements is needed, not {rot}")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"the base must be a number over 1, not {base!r}")
    i = torch.arange(rot // 2, dtype=torch.float64)
    inv, mscale = float(base) ** (-2.0 * i / rot), 1.0
    if scaling is not None:
        kind, factor = scaling.get("kind"), float(scaling.get("factor", 1.0))
        if kind not in SCALINGS:
            raise ValueError(f"scaling {kind!r}: one of {', '.join(SCALINGS)}")
        if not (math.isfinite(factor) and factor >= 1.0):
            raise ValueError(f"a scaling factor is a number of at least 1, not {factor!r}")
        if kind in ("ramp", "bands") and not float(scaling.get("trained", 0)) > 0:
            raise ValueError(f"scaling {kind!r} needs the trained length (\"trained\")")
        if kind == "linear":
            inv = inv / factor
        elif kind == "base":
            if rot == 2:
                raise ValueError("scaling the base needs more than one pair")
            inv = (float(base) * factor ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
        elif kind == "ramp":
            trained, fast, slow = (float(scaling[k]) if k in scaling else d
                                   for k, d in (("trained", 0.0), ("fast", 32.0), ("slow", 1.0)))
            # the pair number that turns n times in `trained` positions
            at = lambda n: rot * math.log(trained / (n * 2.0 * math.pi)) / (2.0 * math.log(base))      # noqa: E731
            lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
            keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            inv = inv / factor * (1.0 - keep) + inv * keep
            mscale = 1.0 + 0.1 * math.log(factor)
        else:
            trained, low, high = (float(scaling[k]) if k in scaling else d
                                  for k, d in (("trained", 0.0), ("low", 1.0), ("high", 4.0)))
            if not high > low:
                raise ValueError("bands need high over low")
            turns = trained * inv / (2.0 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
            inv = inv / factor * (1.0 - keep) + inv * keep
    return (inv / (2.0 * math.pi)).to(device), mscale


def rotate(x: torch.Tensor, positions: torch.Tensor, turns: torch.Tensor, *, interleaved: bool = False,
           mscale: float = 1.0, inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (tokens, heads, head size), or with more leading dimensions, rotated by `positions` (one per token: a tensor of
    the leading dimensions' shape, of the last of them, or one row for all tokens in their order).  bf16, fp16 or fp32, any strides.  Differentiable in x; with
    `out` (x itself to rotate in place) it writes there and takes no gradient.  `inverse` rotates by the negative
    angles.  Queued on the current stream of x's device."""
    return _lib.bound().rotate(x, positions, turns, interleaved, mscale, inverse, out)
