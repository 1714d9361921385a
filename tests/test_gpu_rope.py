"""Rotary positions on the GPU (sdc_rope through rope.rotate) against the float64 oracle and, bit for bit, against the
same three fp32 operations in torch; gradients against the formula and against differences; strides, layouts, parts of
a head, lengths from zero, far positions, graph capture, other streams, refusals."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _turns(rot, base=10000.0):
    from sdcguard_amd.rope import frequencies
    return frequencies(rot, base, device=DEV)[0]


def _bits(x, pos, turns, interleaved, mscale):
    """The rotation as fp32 operations on 64-bit angles rounded once, in torch."""
    rot = 2 * turns.numel()
    t = pos.double()[:, None] * turns
    a = (t - t.round()) * (2 * math.pi)
    c, s = (torch.cos(a) * mscale).float()[:, None], (torch.sin(a) * mscale).float()[:, None]
    y = x.float().clone()
    xf = x.float()
    ia, ib = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., ia] = xf[..., ia] * c - xf[..., ib] * s
    y[..., ib] = xf[..., ib] * c + xf[..., ia] * s
    return y.to(x.dtype)


def _check(y, x, pos, turns, interleaved, mscale=1.0, inverse=False):
    ref = paged.rotate(x.double().cpu().numpy(), pos.cpu().numpy(), turns.cpu().numpy(), interleaved, mscale, inverse)
    err = np.abs(y.double().cpu().numpy() - ref)
    # one rounding to the output's type, and fp32 products of rounded cosines: 3 roundings of terms up to |a| + |b|;
    # an angle in turns is off by its product's rounding, 2^-53 of the turns made
    far = float(pos.abs().max()) * float(turns.max()) * 2 * math.pi * 2.0 ** -52 if pos.numel() else 0.0
    size = float(x.abs().max()) if x.numel() else 0.0
    tol = torch.finfo(x.dtype).eps / 2 * np.abs(ref) + (3 * 2.0 ** -23 + 2 * far) * size * 2 * mscale
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 2, 2), (1, 32, 128, 128), (5, 3, 80, 48), (7, 2, 64, 20), (33, 4, 96, 96),
                                       (1030, 2, 64, 32), (3, 1, 7, 6), (9, 2, 256, 256), (4, 1, 1024, 1024)])
def test_matches_the_oracle_and_torch_bit_for_bit(T, H, D, rot, interleaved, dt):
    from sdcguard_amd.rope import rotate
    g = torch.Generator(device=DEV).manual_seed(T + D)
    x = torch.randn(T, H, D, device=DEV, generator=g).to(DTYPES[dt])
    pos = torch.randint(0, 1 << 20, (T,), device=DEV, generator=g)
    turns = _turns(rot, 500000.0)
    y = rotate(x, pos, turns, interleaved=interleaved, mscale=1.25)
    _check(y, x, pos, turns, interleaved, 1.25)
    assert torch.equal(y, _bits(x, pos, turns, interleaved, 1.25))
    assert torch.equal(y[..., rot:], x[..., rot:])
    back = rotate(x, pos, turns, interleaved=interleaved, inverse=True)
    _check(back, x, pos, turns, interleaved, 1.0, True)


def test_strides_positions_and_leading_dimensions():
    from sdcguard_amd.rope import rotate
    g = torch.Generator(device=DEV).manual_seed(3)
    wide = torch.randn(6, 5, 4 * 64 + 8, device=DEV, generator=g).bfloat16()
    x = wide[..., 8:].unflatten(-1, (4, 64))                      # (batch, tokens, heads, head size), rows 16 bytes on
    turns = _turns(64)
    pos = torch.randint(0, 9000, (5,), device=DEV, generator=g, dtype=torch.int32)
    want = rotate(x.reshape(30, 4, 64).contiguous(), pos.expand(6, 5).reshape(-1), turns)
    assert torch.equal(rotate(x, pos, turns), want.view(6, 5, 4, 64))
    assert torch.equal(rotate(x, pos.expand(6, 5).long(), turns), want.view(6, 5, 4, 64))
    odd = wide[..., 3:3 + 256].unflatten(-1, (4, 64))[0]          # rows that start at any 2 bytes
    assert torch.equal(rotate(odd, pos, turns), rotate(odd.contiguous(), pos, turns))
    tr = torch.randn(64, 4, 5, device=DEV, generator=g).permute(2, 1, 0)              # elements far apart
    assert torch.equal(rotate(tr, pos, turns), rotate(tr.contiguous(), pos, turns))
    y = x[0].clone()
    assert rotate(y, pos, turns, out=y) is y and torch.equal(y, want.view(6, 5, 4, 64)[0])
    exp = x[0, :, :1].expand(5, 4, 64)                             # one head broadcast over four
    assert torch.equal(rotate(exp, pos, turns), rotate(exp.contiguous(), pos, turns))
    assert rotate(x[:0], pos, turns).shape == (0, 5, 4, 64)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_the_formula_and_differences(interleaved):
    from sdcguard_amd.rope import rotate
    g = torch.Generator(device=DEV).manual_seed(5)
    turns, pos = _turns(24), torch.tensor([0, 3, 70001], device=DEV)
    x = torch.randn(3, 2, 32, device=DEV, generator=g).requires_grad_()
    dy = torch.randn(3, 2, 32, device=DEV, generator=g)
    y = rotate(x, pos, turns, interleaved=interleaved, mscale=1.1)
    dx, = torch.autograd.grad(y, x, dy)
    _check(dx, dy, pos, turns, interleaved, 1.1, True)
    f = lambda z: (rotate(z, pos, turns, interleaved=interleaved, mscale=1.1).double() * dy.double()).sum()   # noqa: E731
    for i in range(8):                              # the map is linear: differences over a step of 1 are its gradient
        d = torch.randn(3, 2, 32, device=DEV, generator=g)
        with torch.no_grad():
            got = float(f(x + d) - f(x - d)) / 2
        want = float((dx.double() * d.double()).sum())
        # each of 2 x 192 outputs is off by 3 x 2^-24 of terms up to 10, times |dy| up to 5
        assert abs(got - want) <= 384 * 3 * 2.0 ** -24 * 50, (i, got, want)
    shared = torch.randn(3, 1, 32, device=DEV, generator=g).requires_grad_()           # one head shared by four
    ys = rotate(shared.expand(3, 4, 32), pos, turns, interleaved=interleaved)
    dys = torch.randn(3, 4, 32, device=DEV, generator=g)
    ds, = torch.autograd.grad(ys, shared, dys)
    each = rotate(dys, pos, turns, interleaved=interleaved, inverse=True)
    assert torch.allclose(ds, each.sum(1, keepdim=True), rtol=0, atol=8 * 2.0 ** -24 * 20)
    w, dy2 = torch.randn(3, 2, 32, device=DEV, generator=g), dy.clone().requires_grad_()
    dx2, = torch.autograd.grad(rotate(x, pos, turns, interleaved=interleaved), x, dy2, create_graph=True)
    ddy, = torch.autograd.grad((dx2 * w).sum(), dy2)                 # the gradient's gradient rotates forward again
    assert torch.equal(ddy, rotate(w, pos, turns, interleaved=interleaved))


def test_in_a_graph_and_on_another_stream():
    from sdcguard_amd.rope import rotate
    turns, pos = _turns(64), torch.arange(40, device=DEV)
    x = torch.randn(40, 2, 64, device=DEV).bfloat16()
    y = torch.empty_like(x)
    rotate(x, pos, turns, out=y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotate(x, pos, turns, out=y)
    for i in range(3):
        x.copy_(torch.randn(40, 2, 64, device=DEV))
        pos += i
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, rotate(x, pos, turns))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = rotate(x, pos, turns)
    s.synchronize()
    assert torch.equal(z, y)


def test_refusals():
    from sdcguard_amd import _lib
    from sdcguard_amd.rope import rotate
    x, turns, pos = torch.zeros(3, 2, 64, device=DEV, dtype=torch.bfloat16), _turns(64), torch.arange(3, device=DEV)
    for bad in (lambda: rotate(x[0], pos, turns), lambda: rotate(x, pos[:2], turns), lambda: rotate(x, pos.float(), turns),
                lambda: rotate(x, pos, turns.float()), lambda: rotate(x, pos, _turns(66)),
                lambda: rotate(x, pos, turns[::2]), lambda: rotate(x, pos, turns, out=x.float()),
                lambda: rotate(x, pos, turns, out=x[:2]),
                lambda: rotate(x.float().requires_grad_(), pos, turns, out=torch.empty(3, 2, 64, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.HipLibraryError):
        rotate(x.double(), pos, turns)
    with pytest.raises(_lib.HipLibraryError):
        rotate(x, pos.cpu(), turns)
