"""The paged operators at the ends of what their arguments and values may be: windows wider than any length, magnitudes and
scales at both ends of their types, steps and tables of nothing, and what autograd has to know of their calls."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import paged
from tests.test_gpu_kv_attn import DEV, append_checked, attend_checked, make, step

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
