"""The paged operators at the ends of what their arguments and values may be: windows wider than any length, magnitudes and
scales at both ends of their types, steps and tables of nothing, and what autograd has to know of their calls."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged
from tests.test_gpu_kv_attn import DEV, append_checked, attend_checked, make, step, stood_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [(1 << 63) - 1, 1 << 62, 1 << 40])
@pytest.mark.parametrize("lens,N", [(((40, 3), (17, 1)), 16), (((3000, 1), (9, 1)), 1), (((20000, 1),), 16), (((18000, 70),), 16)])
def test_a_window_wider_than_any_length_is_none(lens, N, window):
    from sdcguard_amd.kv_attn import kv_attend
    c = make(lens, N=N, D=64, Hq=4, Hkv=2, seed=N)
    want = kv_attend(c["q"], c["kv"], c["scales"], *step(c), return_lse=True)
    got = kv_attend(c["q"], c["kv"], c["scales"], *step(c), window=window, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if lens[0][0] < 10000:
        attend_checked(c, window=window)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("layout,N", [("pages", 16), ("pages", 64), ("odd", 16), ("odd", 64)])
def test_append_of_the_largest_finite_values(layout, N, kind):
    """Magnitudes up to bf16's largest, in the one-pass and the two-pass kernels, in runs of 16 bytes and by single elements:
    no code changes its sign, and none is further off than half a step."""
    for big in (2.0 ** 127, 127.5 * 2.0 ** 120, 2e38, float(torch.finfo(torch.bfloat16).max)):
        c = make(((40, 40), (17, 1)), D=64, kind=kind, N=N, layout=layout, seed=N, garbage=False)
        c["k"].copy_(torch.randn(c["k"].shape, device=DEV).clamp(-3, 3) / 3 * 1e38)
        c["v"][::2].mul_(2.0 ** 100)
        c["k"][3, 0, 5], c["k"][3, 1, 6], c["v"][7, 0, 1], c["v"][40, 1, 2] = big, -big, -big, big
        append_checked(c)
        codes = c["kv"].view(torch.uint8).view(c["kv"].dtype).float()
        for x, page, h, slot, d in ((c["k"][3, 0, 5], 0, 0, 3, 5), (c["k"][3, 1, 6], 0, 1, 3, 6), (c["v"][7, 0, 1], 0, 0, 7, 65)):
            at = int(c["bt"][0, page])
            scale = float(c["scales"][at, h, d // 64])
            assert scale == paged.smallest_scale(abs(float(x)), kind)
            assert math.copysign(1.0, float(x)) == math.copysign(1.0, float(codes[at, h, slot, d]))


def attend_tight(c, **kw):
    """attend_checked with a bound that only the keys which a row sees, at their weights, have a part in."""
    from sdcguard_amd.kv_attn import kv_attend
    o, lse = kv_attend(c["q"], c["kv"], c["scales"], *step(c), return_lse=True, **kw)
    D, T, kv = c["D"], c["T"], stood_for(c["kv"], c["scales"])
    case = (c["qsl"].tolist(), c["lens"].tolist(), c["bt"].cpu().numpy(), c["N"], D ** -0.5)
    q = c["q"][:T].double().cpu().numpy()
    ro, rl, mass, terms = paged.attend(q, kv, *case)
    kv[..., D:] = c["scales"].double().abs().cpu().numpy()[:, :, None, 1:] * paged.TOP[c["kind"]]
    top = paged.attend(q, kv, *case)[0]
    n = int(c["lens"].max())
    ds = (D + 16) * 2.0 ** -24 * terms + 2.0 ** -20
    # a probability's product with its scale is rounded to 11 bits, or by a fp16 step of 2^-24 where the row's largest product
    # is 2^4 or more; a maximum of up to 2^8 that carries the scales' exponent is rounded to 2^-16
    got, gl = o[:T].double().cpu().numpy(), lse[:T].double().cpu().numpy()
    tol = torch.finfo(c["dt"]).eps / 2 * abs(ro) + (2.0 ** -11 + 2.0 ** -15 + 2 * ds[..., None] + (n + 16) * 2.0 ** -23) * mass \
        + n * 2.0 ** -29 * top
    err = abs(got - ro)
    assert (err <= tol).all(), (np.argwhere(~(err <= tol))[:5], err[~(err <= tol)][:5], tol[~(err <= tol)][:5])
    assert (abs(gl - rl) <= ds + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * abs(rl) + 2.0 ** -16).all(), abs(gl - rl).max()


STEPS = (((700, 1), (40, 1)), ((700, 50), (90, 90)), ((9000, 1), (300, 1)))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("lens", STEPS, ids=["decode", "chunk", "split"])
@pytest.mark.parametrize("D", [64, 40])
def test_attention_of_value_scales_at_both_ends(D, lens, kind):
    """Values of all magnitudes that bf16 has: neither the weights' sum nor their products leave their types."""
    c = make(lens, D=D, Hq=8, Hkv=1, seed=21, kind=kind, garbage=False)
    for e in (-126, -110, -60, -24, 24, 60, 100, 110, 118):
        c["scales"][..., 1] = 2.0 ** e
        attend_tight(c)


@pytest.mark.parametrize("N", [16, 6])
@pytest.mark.parametrize("lens", STEPS, ids=["decode", "chunk", "split"])
def test_attention_of_value_scales_far_from_each_other(lens, N):
    """Pages whose value scales lie up to 2^160 under another's of the same part, which a row may not see or hardly weigh:
    pages of zeros (2^-126) among ordinary ones, and small scales before a large one."""
    c = make(lens, D=64, Hq=8, Hkv=1, N=N, seed=22, garbage=False)
    pages = c["bt"][0, :lens[0][0] // N].long()
    c["scales"][pages[::2], :, 1] = 2.0 ** -126
    c["kv"].view(torch.uint8)[pages[::2], :, :, 64:] = 0
    attend_tight(c)
    c["q"].abs_()
    ks, at = c["scales"][..., 0].clone(), pages[-2:]
    for last in (0, 20, 60, 100):
        c["scales"][pages, :, 1] = 2.0 ** -30
        c["scales"][at, :, 1] = 2.0 ** last
        attend_tight(c)                                # (a chunk's first rows do not see these pages)
        c["kv"].view(torch.uint8)[at, :, :, :64], c["scales"][at, :, 0] = 0xF0, 1.0
        attend_tight(c)                                # (scores of -1000 there: no weight at all)
        c["scales"][..., 0] = ks
    c["scales"][pages, :, 1] = (2.0 ** torch.linspace(-80, 80, pages.numel(), device=DEV))[:, None]
    attend_tight(c)
    c["scales"][pages, :, 1] = c["scales"][pages.flip(0), :, 1].clone()
    attend_tight(c)
