"""Rotary positions: the heads of queries or keys rotated by their tokens' positions (no counterpart in the reference).

Pair i of a head at position p is turned by the angle 2 pi p turns[i]: (a, b) becomes (a c - b s, b c + a s) with
c = mscale cos, s = mscale sin.  A pair is (i, i + rot / 2) of the first rot = 2 len(turns) elements, or (2 i, 2 i + 1)
with `interleaved`; elements past rot are copied.  Angles are taken in 64 bits, so positions of a million lose nothing.
The work is one launch of sdc_rope (csrc/rope.hip); there is no CPU implementation.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

DT_F32 = 4
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


def dtype_code(dt: torch.dtype) -> int:
    return DT_F32 if dt == torch.float32 else _lib.dtype_code(dt)


def check_turns(turns: torch.Tensor, head_size: int, device) -> int:
    """The number of rotated elements; raises where turns is not a table of frequencies for this head size."""
    if turns.dim() != 1 or turns.dtype != torch.float64 or not turns.is_contiguous() or turns.device != device:
        raise ValueError("turns must be a contiguous float64 vector on the tensors' device (frequencies())")
    rot = 2 * turns.shape[0]
    if rot > head_size:
        raise ValueError(f"{rot} rotated elements in heads of {head_size}")
    return rot


def check_positions(positions: torch.Tensor, tokens: int, device) -> torch.Tensor:
    if positions.dtype not in (torch.int64, torch.int32) or positions.device != device:
        raise ValueError("positions must be int64 or int32 on the tensors' device")
    if positions.numel() != tokens:
        raise ValueError(f"{positions.numel()} positions for {tokens} tokens")
    return positions.reshape(-1).contiguous()


def _rotate(x, pos, turns, interleaved, mscale, inverse, out):
    T, H, D = x.shape
    rc = _lib.lib().sdc_rope(dtype_code(x.dtype), x.data_ptr(), x.stride(0), x.stride(1), x.stride(2), out.data_ptr(),
                             out.stride(0), out.stride(1), out.stride(2), T, H, D, pos.data_ptr(), pos.element_size(),
                             turns.data_ptr(), 2 * turns.shape[0], int(interleaved), float(mscale), int(inverse),
                             _lib.stream_of(x))
    _lib.check(rc, "sdc_rope")
    return out


class _Rotation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, turns, interleaved, mscale, inverse):
        ctx.save_for_backward(pos, turns)
        ctx.how = interleaved, mscale, inverse
        return _rotate(x, pos, turns, interleaved, mscale, inverse, torch.empty(x.shape, dtype=x.dtype, device=x.device))

    @staticmethod
    def backward(ctx, dy):
        pos, turns = ctx.saved_tensors
        interleaved, mscale, inverse = ctx.how
        # the transposed rotation is the one by the negative angle, the factor on the result the same
        return _Rotation.apply(dy, pos, turns, interleaved, mscale, not inverse), None, None, None, None, None


def rotate(x: torch.Tensor, positions: torch.Tensor, turns: torch.Tensor, *, interleaved: bool = False,
           mscale: float = 1.0, inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (tokens, heads, head size), or with more leading dimensions, rotated by `positions` (one per token; a tensor of
    the leading dimensions' shape, or of the last of them).  bf16, fp16 or fp32, any strides.  Differentiable; with
    `out` (x itself to rotate in place) it writes there and takes no gradient.  `inverse` rotates by the negative
    angles.  Queued on the current stream of x's device."""
    _lib.require_gpu(x, positions, turns, out)
    if x.dim() < 3:
        raise ValueError("x must be (..., tokens, heads, head size)")
    lead, dev = x.shape[:-2], x.device
    check_turns(turns, x.shape[-1], dev)
    if positions.shape != lead and positions.dim() < len(lead) and positions.shape == lead[len(lead) - positions.dim():]:
        positions = positions.expand(lead)
    x3 = x.flatten(0, -3) if x.dim() > 3 else x
    pos = check_positions(positions, x3.shape[0], dev)
    with torch.cuda.device(dev):
        if out is not None:
            if out.shape != x.shape or out.dtype != x.dtype or out.device != dev:
                raise ValueError("out must have x's shape, type and device")
            if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
                raise ValueError("out takes no gradient: rotate without it")
            o3 = out.view(x3.shape) if x.dim() > 3 else out
            _rotate(x3, pos, turns, interleaved, mscale, inverse, o3)
            return out
        if torch.is_grad_enabled() and x.requires_grad:
            y = _Rotation.apply(x3, pos, turns, interleaved, mscale, inverse)
        else:
            y = _rotate(x3, pos, turns, interleaved, mscale, inverse,
                        torch.empty(x3.shape, dtype=x.dtype, device=dev))
    return y.view(x.shape) if x.dim() > 3 else y
