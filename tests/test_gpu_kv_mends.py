"""The paged operators at the ends of what their arguments and values may be: windows wider than any length, magnitudes and
scales at both ends of their types, steps and tables of nothing, and what autograd has to know of their calls."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv_attn import DEV, attend_checked, make, step

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
