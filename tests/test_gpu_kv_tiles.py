"""The attention of chunks in tiles of 256 query rows, which a call takes where there is enough work: the cases of the other
attention tests again, with tables so wide that the work a call has to expect reaches that limit (the keys there are stay
the same, so the results do too)."""
from __future__ import annotations

import pytest
import torch

from tests import test_gpu_kv_attn as base
from tests import test_gpu_kv_edges as edges

pytestmark = pytest.mark.gpu
WORK = 640000000                                       # small tiles x keys x head size


@pytest.fixture(autouse=True)
def wide_tables(monkeypatch):
    def step(c):
        T, Hq, D = c["q"].shape
        Hkv, N, R = c["kv"].shape[1], c["N"], c["lens"].shape[0]
        G = Hq // Hkv
        small = (T // max(1, 16 // min(G, 16)) + R) * Hkv * -(-G // 16)
        W = max(c["bt"].shape[1], -(-(WORK // (small * D) + 1) // N))
        wide = torch.full((R, W), -7, dtype=torch.int32, device=base.DEV)
        wide[:, :c["bt"].shape[1]] = c["bt"][:R]
        return c["qsl"], c["lens"], wide

    monkeypatch.setattr(base, "step", step)
    monkeypatch.setattr(edges, "step", step)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_types(dt, kind):
    base.test_attention_types(base.MIXED, dt, kind)


@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (3, 3)])
def test_head_sizes(D, Hq, Hkv):
    base.attend_checked(base.make(((3, 3), (40, 1), (150, 60), (17, 2), (333, 300)), D=D, Hq=Hq, Hkv=Hkv, seed=D))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 1), (16, 1), (16, 8), (40, 2), (48, 1), (14, 2), (260, 1), (300, 1)])
def test_shared_heads(Hq, Hkv):
    base.attend_checked(base.make(((70, 1), (133, 104), (20, 17)), D=32, Hq=Hq, Hkv=Hkv, seed=Hq))


@pytest.mark.parametrize("N", [1, 3, 4, 8, 12, 16, 20, 24, 32, 48, 64, 100, 256])
@pytest.mark.parametrize("D", [32, 96, 128, 256])
def test_page_sizes(N, D):
    base.attend_checked(base.make(base.MIXED, D=D, N=N, seed=N, kind="int8" if N % 2 else "e4m3"))


@pytest.mark.parametrize("layout", ["slots", "odd"])
def test_cache_layouts(layout):
    base.test_attention_cache_layouts(layout)


def test_long_chunks_in_parts():
    base.attend_checked(base.make(((9000, 70), (200, 1), (4000, 3)), D=64, Hq=4, Hkv=1, seed=2))
    base.attend_checked(base.make(((3000, 70), (2500, 1), (9, 1), (4000, 35), (1, 1)), D=96, Hq=4, Hkv=1, seed=3))


def test_scores_scales_nan_and_bad_pages():
    base.test_attention_scores_that_rise_and_scales_that_differ()
    base.test_attention_non_finite_keys_and_values_reach_only_the_queries_that_see_them()
    base.test_attention_pages_outside_the_cache_are_nan_and_unused_entries_are_not_read()
    base.test_attention_of_nothing_and_of_extreme_scores()


@pytest.mark.parametrize("N", [16, 8, 6])
def test_scales_of_every_kind(N):
    edges.test_scales_of_every_kind(((150, 100), (60, 1)), N)


@pytest.mark.parametrize("D", [80, 96, 160, 256])
def test_values_that_are_nan(D):
    edges.test_values_that_are_nan_under_a_chunk(D)


@pytest.mark.parametrize("D", [64, 80, 256])
def test_strides(D):
    edges.test_outputs_and_queries_of_any_stride(D)


@pytest.mark.parametrize("R", [62, 63, 64, 65, 126, 127, 128, 129, 255, 256, 300])
def test_many_requests(R):
    lens = [(1 + (7 * i) % 40, 1) if i % 9 else (0, 0) for i in range(R)]
    lens[R // 2], lens[R - 1] = (90, 70), (33, 33)
    base.attend_checked(base.make(lens, D=32, Hq=2, Hkv=1, N=8, seed=R + 1, garbage=False, pad=2))


@pytest.mark.parametrize("Hq", [1, 4, 16])
def test_chunks_on_both_sides_of_the_limit_between_the_kernels(Hq):
    edges.test_chunks_on_both_sides_of_the_limit_between_the_kernels(Hq)


@pytest.mark.parametrize("window", [90, 200, 500])
@pytest.mark.parametrize("N", [16, 8])
def test_windows(window, N):
    """Under a window the expected work is the window's: enough padding for it."""
    pad = WORK // (128 * (window + 16)) * 16
    base.attend_checked(base.make(((700, 300), (40, 1), (90, 90), (800, 1), (5, 5)), D=128, Hq=1, Hkv=1, N=N, seed=window,
                                  pad=pad), window=window)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_far_pages(kind):
    base.test_attention_far_pages(kind, 40)


def test_same_bits():
    from sdcguard_amd.kv_attn import kv_attend
    c = base.make(((3000, 200), (64, 1), (700, 90)), seed=17, D=128, Hq=8, Hkv=2)
    s = base.step(c)
    first = kv_attend(c["q"], c["kv"], c["scales"], *s)
    for _ in range(3):
        assert torch.equal(first, kv_attend(c["q"], c["kv"], c["scales"], *s))


def test_the_two_kernels_agree():
    from sdcguard_amd.kv_attn import kv_attend
    c = base.make(((1500, 400), (700, 1)), seed=18, D=128, Hq=8, Hkv=2)
    wide = kv_attend(c["q"], c["kv"], c["scales"], *base.step(c), return_lse=True)
    own = kv_attend(c["q"], c["kv"], c["scales"], c["qsl"], c["lens"], c["bt"], return_lse=True)
    torch.testing.assert_close(wide[0], own[0], rtol=2 ** -7, atol=2e-3)
    torch.testing.assert_close(wide[1], own[1], rtol=1e-5, atol=1e-5)
    assert not torch.equal(wide[0], own[0])            # (different roundings: both were run)
