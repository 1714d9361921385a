"""The paged append and attention where their tiles, parts and searches end: steps of more requests than a wave has lanes,
groups of heads that do not divide a tile, chunks on both sides of the limit between the two attention kernels, parts of
a long context beside windows, scales of every kind under a chunk, odd page sizes, strided outputs, large heads; and the
operators together as a serving step uses them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_kv_attn import DEV, _turns, append_checked, attend_checked, make, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [62, 63, 64, 65, 126, 127, 128, 129, 255, 256, 300])
def test_many_requests(R):
    lens = [(1 + (7 * i) % 40, 1) if i % 9 else (0, 0) for i in range(R)]
    c = make(lens, D=32, Hq=2, Hkv=1, N=8, seed=R, garbage=False, pad=R % 3)
    append_checked(c, _turns(32))
    attend_checked(c)
    lens[R // 2] = (90, 70)                            # one chunk among them: more tokens than requests
    lens[R - 1] = (33, 33)
    c = make(lens, D=32, Hq=2, Hkv=1, N=8, seed=R + 1, garbage=False, pad=2)
    append_checked(c, _turns(32))
    attend_checked(c)


@pytest.mark.parametrize("Hq,Hkv", [(5, 1), (7, 1), (17, 1), (36, 4), (100, 1), (260, 1), (300, 1), (9, 3)])
@pytest.mark.parametrize("D", [16, 96])
def test_groups_that_do_not_divide_a_tile(Hq, Hkv, D):
    attend_checked(make(((70, 40), (33, 1), (20, 3), (5, 5)), D=D, Hq=Hq, Hkv=Hkv, seed=Hq))


@pytest.mark.parametrize("Hq", [1, 4, 16])
def test_chunks_on_both_sides_of_the_limit_between_the_kernels(Hq):
    TB = 16 // Hq
    for n in (2 * TB - 1, 2 * TB, 2 * TB + 1, 256 // Hq - 1, 256 // Hq, 256 // Hq + 1):
        attend_checked(make(((n + 50, n), (40, 1), (n, n), (9, 2)), D=64, Hq=Hq, Hkv=1, seed=n))


@pytest.mark.parametrize("N", [1, 4, 12, 16, 20, 48])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_chunks_page_sizes_and_heads(N, kind, D):
    attend_checked(make(((200, 150), (77, 77), (130, 1)), D=D, Hq=2, Hkv=1, N=N, kind=kind, seed=N + D))


@pytest.mark.parametrize("window", [0, 600, 1500])
def test_parts_of_chunks_and_of_single_tokens(window):
    """Contexts that are cut into parts for chunks and for single tokens, joined together."""
    c = make(((3000, 70), (2500, 1), (9, 1), (4000, 35), (1, 1)), D=96, Hq=4, Hkv=1, seed=window)
    attend_checked(c, window=window)
    c = make(((3000, 300), (2500, 1), (700, 9)), D=128, Hq=2, Hkv=1, N=1, seed=window, kind="int8")
    attend_checked(c, window=window)


@pytest.mark.parametrize("N", [16, 8, 6])
@pytest.mark.parametrize("lens", [((150, 100), (60, 1)), ((90, 1), (300, 1))], ids=["chunk", "decode"])
def test_scales_of_every_kind(lens, N):
    c = make(lens, D=64, Hq=4, Hkv=2, N=N, seed=N, garbage=False)
    pages = c["bt"][0, :lens[0][0] // N].long()
    sc = c["scales"]
    sc[pages[::4], 0, 0] *= -1.0                        # negative, zero, tiny and huge factors
    sc[pages[1::4], 0, 1] *= -1.0
    sc[pages[2::4], 1, 1] = 0.0
    sc[pages[3::4], 1, 0] = 0.0
    sc[pages[::3], 0, 1] *= 2.0 ** -40
    attend_checked(c)
    sc[pages[1], 1, 1] = float("nan")
    sc[pages[-1], 0, 0] = float("nan")
    o, lse = attend_checked(c)
    assert o[lens[0][1] - 1].isnan().all()
    assert torch.isnan(lse[lens[0][1] - 1, :2]).all() and not torch.isnan(lse[lens[0][1] - 1, 2:]).any()


@pytest.mark.parametrize("D", [80, 96, 160, 256])
def test_values_that_are_nan_under_a_chunk(D):
    c = make(((120, 90),), D=D, Hq=2, Hkv=1, seed=D)
    raw = c["kv"].view(torch.uint8)
    for p, d in ((40, 0), (77, D - 1), (100, 5), (10, 3)):
        raw[c["bt"][0, p // 16].long(), 0, p % 16, D + d] = 0x7F
    o, _ = attend_checked(c)
    assert o[:, :, 3].isnan().all() and not o[:, :, 1].isnan().any()
    assert not o[:70, :, 5].isnan().any() and o[70:, :, 5].isnan().all()


@pytest.mark.parametrize("D", [64, 80, 256])
def test_outputs_and_queries_of_any_stride(D):
    from sdcguard_amd.kv_attn import kv_attend
    for lens in (((100, 60), (30, 1)), ((70, 1), (1100, 1))):
        c = make(lens, D=D, Hq=4, Hkv=2, seed=D)
        want = kv_attend(c["q"], c["kv"], c["scales"], *step(c))
        T = c["q"].shape[0]
        far = torch.empty(D, 4, T, dtype=c["dt"], device=DEV).permute(2, 1, 0)
        odd = torch.empty(T, 4, D + 3, dtype=c["dt"], device=DEV)[..., 3:]
        for out in (far, odd):
            q = torch.empty_strided(c["q"].shape, out.stride(), dtype=c["dt"], device=DEV) if out is far else odd.clone()
            q = q.copy_(c["q"])
            assert kv_attend(q, c["kv"], c["scales"], *step(c), out=out) is out and torch.equal(out, want)


def test_tables_and_lengths_of_64_bits_and_sliced():
    from sdcguard_amd.kv_attn import kv_attend
    c = make(((100, 60), (30, 1)), seed=31)
    want = kv_attend(c["q"], c["kv"], c["scales"], *step(c))
    wide = torch.full((5, 2 * c["bt"].shape[1]), -1, dtype=torch.int32, device=DEV)
    wide[:2, ::2] = c["bt"]
    got = kv_attend(c["q"], c["kv"], c["scales"], c["qsl"].long(), c["lens"].long(), wide[:, ::2].long())
    assert torch.equal(got, want)


@pytest.mark.parametrize("D,rot", [(512, 512), (1024, 1024), (1024, 64)])
def test_append_of_large_heads(D, rot):
    append_checked(make(((3, 3), (40, 1), (50, 20)), D=D, Hq=2, Hkv=1, seed=D, garbage=False), _turns(rot))


def test_a_wider_table_changes_nothing():
    """Parts follow the lengths: a table with room for far more gives the same keys the same weight."""
    from sdcguard_amd.kv_attn import kv_attend
    for lens in (((900, 1), (2000, 1)), ((900, 200), (2000, 1))):
        c = make(lens, D=64, seed=33)
        want, lse = kv_attend(c["q"], c["kv"], c["scales"], *step(c), return_lse=True)
        wide = torch.zeros(2, 4000, dtype=torch.int32, device=DEV)
        wide[:, :c["bt"].shape[1]] = c["bt"]
        c["bt"] = wide
        o, l2 = attend_checked(c)
        torch.testing.assert_close(o, want, rtol=2 ** -7, atol=1e-3)
        torch.testing.assert_close(l2, lse, rtol=1e-5, atol=1e-5)


def test_two_streams_at_once():
    """Calls on two streams keep workspaces of their own."""
    from sdcguard_amd.kv_attn import kv_attend
    cs = [make(((6000, 1), (300, 1)), D=128, Hq=8, Hkv=1, seed=s) for s in (40, 41)]
    want = [kv_attend(c["q"], c["kv"], c["scales"], *step(c)) for c in cs]
    torch.cuda.synchronize()
    ss = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cs, ss)):
            with torch.cuda.stream(s):
                got[i].append(kv_attend(c["q"], c["kv"], c["scales"], *step(c)))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("N,D", [(64, 128), (256, 128), (200, 96), (256, 40)])
def test_append_of_chunks_into_large_pages(N, D, kind):
    """Pages that several waves share, in one pass and in two, new and grown."""
    c = make(((300, 300), (500, 200), (257, 1)), D=D, Hq=2, Hkv=3, N=N, kind=kind, seed=N + D, garbage=False)
    append_checked(c, _turns(D))
    c["k"].mul_(64.0)                                  # the same step again, its scales grown over the older codes
    c["lens"].add_(1)
    c["bt"][c["bt"] < 0] = c["kv"].shape[0] - 1
    append_checked(c, _turns(D))
