"""The append to a paged 8-bit cache and the attention over it on the GPU (sdc_kv_append, sdc_kv_attend through
sdcguard_amd.kv_attn) against the float64 oracle: scales exactly, every code within half a step of its value, outputs
within a bound derived from the roundings; lengths from zero, pages that end inside a tile, odd page and head sizes,
shared heads, windows, rows without keys, NaN in places that are masked and in places that are not, pages outside the
cache, far pages, strided caches, captured padding, graphs, streams, refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def stood_for(kv, scales):
    """The cache's values, (pages, heads, slots, 2 D) float64."""
    D = kv.shape[3] // 2
    c = kv.view(torch.uint8).cpu().view(kv.dtype).float().double().numpy().copy()
    s = scales.double().cpu().numpy()
    c[..., :D] *= s[:, :, None, :1]
    c[..., D:] *= s[:, :, None, 1:]
    return c


def make(lens, *, D=64, Hq=4, Hkv=2, N=16, kind="e4m3", dt="bf16", seed=0, pad=0, garbage=True, layout="pages", extra=2):
    """A step: (seq_len, query_len) per request, a cache with random codes and scales, queries, keys and values as views
    of one projection's output.  garbage: unused pages hold NaN codes and scales, and so do the slots past each
    sequence."""
    g = torch.Generator().manual_seed(seed)
    R = len(lens)
    W = max(1, max(-(-n // N) for n, _ in lens)) + 1
    need = [-(-n // N) for n, _ in lens]
    NB = sum(need) + extra
    order = torch.randperm(NB, generator=g)
    bt = torch.full((R, W), -7, dtype=torch.int32)
    at = 0
    for r, k in enumerate(need):
        bt[r, :k] = order[at:at + k].to(torch.int32)
        at += k
    x = torch.randn(NB, Hkv, N, 2 * D, generator=g) * 2.0 ** torch.randint(-2, 3, (NB, Hkv, 1, 1), generator=g)
    scales = torch.rand(NB, Hkv, 2, generator=g) * 0.02 + 0.001
    top = paged.TOP[kind]
    code = (x / x.abs().amax((2, 3), keepdim=True) * top)
    code = code.round().to(torch.int8) if kind == "int8" else code.to(torch.float8_e4m3fn)
    code = code.view(torch.uint8)
    if garbage:
        live = torch.zeros(NB, N, dtype=torch.bool)
        for r, (n, _) in enumerate(lens):
            for p in range(n):
                live[bt[r, p // N], p % N] = True
        code[~live[:, None].expand(NB, Hkv, N)] = 0x7F
        scales[~live.any(1)] = float("nan")
    qlens = [q for _, q in lens]
    T = sum(qlens) + pad
    wide = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(DTYPES[dt]).to(DEV)
    q, k, v = (t.view(T, -1, D) for t in wide.split([Hq * D, Hkv * D, Hkv * D], 1))
    qsl = torch.tensor([0] + qlens).cumsum(0).to(torch.int32)
    if layout == "slots":                            # (pages, slots, heads, 2 D) in memory
        mem = torch.empty(NB, N, Hkv, 2 * D, dtype=torch.uint8, device=DEV)
        kv = mem.permute(0, 2, 1, 3)
        kv.copy_(code)
    elif layout == "odd":                            # rows 2 D + 3 bytes apart
        mem = torch.empty(NB, Hkv, N, 2 * D + 3, dtype=torch.uint8, device=DEV)
        kv = mem[..., 3:]
        kv.copy_(code)
    else:
        kv = code.to(DEV)
    return {"q": q, "k": k, "v": v, "kv": kv.view(CODES[kind]), "scales": scales.to(DEV), "qsl": qsl.to(DEV),
            "lens": torch.tensor([n for n, _ in lens], dtype=torch.int32, device=DEV), "bt": bt.to(DEV), "N": N, "D": D,
            "kind": kind, "dt": DTYPES[dt], "T": sum(qlens)}


def step(c):
    return c["qsl"], c["lens"], c["bt"]


def attend_checked(c, window=0, scale=None, **kw):
    from sdcguard_amd.kv_attn import kv_attend
    o, lse = kv_attend(c["q"], c["kv"], c["scales"], *step(c), window=window, scale=scale, return_lse=True, **kw)
    torch.cuda.synchronize()
    D, T = c["D"], c["T"]
    kv = stood_for(c["kv"], c["scales"])
    q = c["q"][:T].double().cpu().numpy()
    sc = D ** -0.5 if scale is None else scale
    ro, rl, mass, terms = paged.attend(q, kv, c["qsl"].tolist(), c["lens"].tolist(), c["bt"].cpu().numpy(), c["N"], sc,
                                       window)
    got, gl = o.double().cpu().numpy(), lse.double().cpu().numpy()
    assert not got[T:].any() and np.isneginf(gl[T:]).all()
    got, gl = got[:T], gl[:T]
    assert np.array_equal(np.isnan(got), np.isnan(ro)), (np.argwhere(np.isnan(got) != np.isnan(ro))[:5])
    assert np.array_equal(np.isneginf(gl), np.isneginf(rl))
    n = max(1, int(c["lens"].max()))
    # a score is a sum of D products in fp32, its factors and the exponent's argument rounded; a query in 16 bits may
    # lose 2^-24 of its row's largest element
    ds = (D + 16) * 2.0 ** -24 * terms + 2.0 ** -20
    # probabilities rounded to 11 bits (small ones to 2^-38 of the largest value's scale), sums in fp32
    with np.errstate(invalid="ignore"):
        big = np.nanmax(np.abs(np.where(np.isfinite(kv), kv, 0.0)))
        tol = torch.finfo(c["dt"]).eps / 2 * np.abs(ro) + (2.0 ** -11 + 2 * ds[..., None] + (n + 16) * 2.0 ** -23) * mass \
            + n * 2.0 ** -38 * big
        if c["dt"] == torch.float16:
            tol = tol + 2.0 ** -25                                   # its smallest step
        err = np.abs(got - ro)
        bad = ~(err <= tol) & np.isfinite(ro)
        assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])
        fin = np.isfinite(rl)
        assert (np.abs(gl - rl)[fin] <= (ds + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * np.abs(rl))[fin]).all()
    return o, lse


MIXED = ((1, 1), (0, 0), (5, 5), (17, 1), (33, 9), (130, 1), (300, 40), (64, 64), (2, 5))
DECODE = ((1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (0, 0), (31, 1), (63, 1), (64, 1), (65, 1), (127, 1), (129, 1), (600, 1),
          (1023, 1), (1025, 1))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("lens", [MIXED, DECODE], ids=["mixed", "decode"])
def test_attention_types(lens, dt, kind):
    attend_checked(make(lens, kind=kind, dt=dt, pad=3))


@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 128, 192, 256, 7, 100])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (3, 3)])
def test_attention_head_sizes(D, Hq, Hkv):
    attend_checked(make(((3, 3), (40, 1), (150, 20), (17, 2)), D=D, Hq=Hq, Hkv=Hkv, seed=D))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 1), (16, 1), (16, 8), (40, 2), (48, 1), (14, 2)])
def test_attention_shared_heads(Hq, Hkv):
    attend_checked(make(((70, 1), (33, 4), (20, 17)), D=32, Hq=Hq, Hkv=Hkv, seed=Hq))


@pytest.mark.parametrize("N", [1, 3, 8, 16, 24, 32, 64, 100, 256])
def test_attention_page_sizes(N):
    attend_checked(make(MIXED, D=32, N=N, seed=N, kind="int8" if N % 2 else "e4m3"))


@pytest.mark.parametrize("window", [1, 2, 16, 33, 64, 100, 1000])
def test_attention_windows(window):
    attend_checked(make(MIXED, D=32, seed=window), window=window)
    attend_checked(make(DECODE, D=32, seed=window), window=window)


@pytest.mark.parametrize("layout", ["slots", "odd"])
def test_attention_cache_layouts(layout):
    for lens in (MIXED, DECODE):
        attend_checked(make(lens, layout=layout, pad=2))


def test_attention_long_and_split():
    """Sequences long enough to be split over many workgroups, beside short ones; a bound on the lengths."""
    c = make(((9000, 1), (3, 1), (5000, 1), (257, 1)), D=128, Hq=8, Hkv=1, seed=1)
    o, lse = attend_checked(c)
    o2, lse2 = attend_checked(c, max_seq_len=9000)
    torch.testing.assert_close(o2, o, rtol=2 ** -7, atol=1e-3)
    attend_checked(make(((9000, 70), (200, 1), (4000, 3)), D=64, Hq=4, Hkv=1, seed=2))


def test_attention_scores_that_rise_and_scales_that_differ():
    """Keys whose scores grow along the sequence, so that every tile rescales what came before; pages whose value scales
    differ by 2^20 in both directions."""
    for lens in (((700, 1),), ((700, 50),)):
        c = make(lens, D=64, Hq=2, Hkv=1, seed=3, garbage=False)
        ramp = torch.linspace(0.2, 4.0, c["bt"].shape[1] - 1, device=DEV)
        pages = c["bt"][0, :-1].long()
        c["scales"][pages, :, 0] = ramp[:, None] * 0.01
        attend_checked(c)
        c["scales"][pages, :, 1] = (2.0 ** torch.linspace(-20, 0, pages.numel(), device=DEV))[:, None]
        attend_checked(c)
        c["scales"][pages, :, 1] = c["scales"][pages.flip(0), :, 1].clone()
        attend_checked(c)


def test_attention_non_finite_keys_and_values_reach_only_the_queries_that_see_them():
    for D, lens in ((64, ((100, 60),)), (64, ((100, 1),)), (128, ((70, 9),))):
        for part in ("key", "value"):
            c = make(lens, D=D, seed=4)
            n, ql = lens[0]
            for p in (n - ql + ql // 2, max(0, n - ql - 3)):
                raw = c["kv"].view(torch.uint8)
                raw[c["bt"][0, p // 16].long(), 1, p % 16, (5 if part == "key" else D + 5)] = 0xFF       # -NaN
                o, _ = attend_checked(c)
                nan = o.isnan()
                assert not nan[:, :2].any() and nan[-1, 2:].any()
                assert part == "key" or int(nan[-1, 2].sum()) == 1
    c = make(((100, 60),), seed=5, kind="int8")
    for i in (0, 1):                                                   # a page's scale that is NaN, mid-sequence
        c["scales"][c["bt"][0, 4].long(), 0, i] = float("nan")
        o, _ = attend_checked(c)
        assert not o[:24, :2].isnan().any() and o[24:, :2].isnan().all() and not o[:, 2:].isnan().any()
    c = make(((100, 60), (50, 1)), seed=6)
    c["q"][3, 1, 2] = float("inf")
    c["q"][60, 0, 0] = float("nan")
    o, _ = attend_checked(c)
    assert o[3, 1].isnan().all() and o[60, 0].isnan().all() and int(o.isnan().any(-1).sum()) == 2


def test_attention_pages_outside_the_cache_are_nan_and_unused_entries_are_not_read():
    for bad in (-1, 1 << 30, -(1 << 31)):
        c = make(((100, 30), (40, 1), (90, 1)), seed=7)
        c["bt"][0, 5] = bad                                            # positions 80 .. 95
        c["bt"][2, 0] = bad
        o, _ = attend_checked(c)
        assert not o[:10].isnan().any() and o[10:30].isnan().all() and not o[30].isnan().any() and o[31].isnan().all()


def test_attention_of_nothing_and_of_extreme_scores():
    c = make(((0, 0), (0, 0)), pad=5)
    attend_checked(c)
    c = make(((40, 3), (0, 0)), seed=8)
    c["lens"][0] = 0                                                   # three queries without a position
    attend_checked(c)
    c = make(((200, 30), (77, 1)), seed=9, garbage=False)
    attend_checked(c, scale=0.0)
    attend_checked(c, scale=-0.3)
    c["scales"][..., 1] = 0.0
    o, _ = attend_checked(c)
    assert not o.any()
    c["q"].zero_()
    attend_checked(c)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("ql", [1, 40])
def test_attention_far_pages(kind, ql):
    """A cache of more than 2^32 bytes: pages at both ends."""
    N, D, Hkv = 64, 128, 2
    NB = (1 << 32) // (Hkv * N * 2 * D) + 40
    c = make(((1000, ql),), N=N, D=D, Hkv=Hkv, Hq=4, kind=kind, seed=10, extra=0)
    small, sc, n = c["kv"].view(torch.uint8), c["scales"], c["kv"].shape[0]
    kv = torch.empty(NB, Hkv, N, 2 * D, dtype=torch.uint8, device=DEV)
    scales = torch.full((NB, Hkv, 2), float("nan"), device=DEV)
    o, lse = attend_checked(c)
    ids = torch.tensor([i if i % 2 else NB - 1 - i for i in range(n)], device=DEV)
    kv[ids], scales[ids] = small, sc
    far = {**c, "kv": kv.view(CODES[kind]), "scales": scales}
    far["bt"] = torch.where(c["bt"] >= 0, ids[c["bt"].clamp(min=0).long()].to(torch.int32), c["bt"])
    from sdcguard_amd.kv_attn import kv_attend
    o2, lse2 = kv_attend(far["q"], far["kv"], far["scales"], *step(far), return_lse=True)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


# ---------------------------------------------------------------------------------------------------- the append
def append_checked(c, turns=None, interleaved=False, mscale=1.0, positions=None, query=True):
    from sdcguard_amd.kv_attn import kv_append
    before = stood_for(c["kv"], torch.nan_to_num(c["scales"]))
    raw0 = c["kv"].view(torch.uint8).cpu().clone()
    sc0 = c["scales"].cpu().clone()
    q = kv_append(c["k"], c["v"], c["kv"], c["scales"], *step(c), turns=turns, interleaved=interleaved, mscale=mscale,
                  positions=positions, query=c["q"] if query else None)
    torch.cuda.synchronize()
    T = c["T"]
    own = [p for _, p in paged.tokens(c["qsl"].tolist(), c["lens"].tolist())]
    pos = np.maximum(np.array(own, np.float64), 0) if positions is None else positions[:T].double().cpu().numpy()
    key = c["k"][:T].double().cpu().numpy()
    if turns is not None:
        key = paged.rotate(key, pos, turns.cpu().numpy(), interleaved, mscale)
    val = c["v"][:T].double().cpu().numpy()
    want, scales, tol = paged.append(key, val, before, np.nan_to_num(sc0.double().numpy()), c["qsl"].tolist(),
                                     c["lens"].tolist(), c["bt"].cpu().numpy(), c["kind"], c["N"])
    got_s = c["scales"].cpu()
    touched = torch.zeros(c["kv"].shape[0], dtype=torch.bool)
    bt = c["bt"].cpu()
    for r, p in paged.tokens(c["qsl"].tolist(), c["lens"].tolist()):
        if p >= 0 and p // c["N"] < bt.shape[1] and 0 <= bt[r, p // c["N"]] < touched.numel():
            touched[bt[r, p // c["N"]]] = True
    assert np.array_equal(got_s.double().numpy()[touched.numpy()], scales[touched.numpy()])
    assert torch.equal(c["kv"].view(torch.uint8).cpu()[~touched], raw0[~touched])
    assert torch.equal(got_s[~touched].view(torch.int32), sc0[~touched].view(torch.int32))
    got = stood_for(c["kv"], torch.nan_to_num(c["scales"]))
    # a nearest code, of a value that is itself a few fp32 roundings off
    most = np.repeat([np.abs(key).max(initial=0.0), np.abs(val).max(initial=0.0)], c["D"])
    slack = tol * 2.0 ** -16 + 8 * 2.0 ** -24 * most
    ok = (np.abs(got - want) <= tol + (tol > 0) * slack) | (np.isnan(got) & np.isnan(want))
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5], tol[~ok][:5])
    if query:
        from sdcguard_amd.rope import rotate
        p = torch.tensor(pos, device=DEV).long()
        ref = rotate(c["q"][:T], p, turns, interleaved=interleaved, mscale=mscale) if turns is not None else c["q"][:T]
        assert torch.equal(q[:T], ref) and not q[T:].any()
    return c


def _turns(rot):
    from sdcguard_amd.rope import frequencies
    return frequencies(rot, device=DEV)[0]


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("lens", [MIXED, DECODE], ids=["mixed", "decode"])
def test_append_types(lens, dt, kind):
    append_checked(make(lens, kind=kind, dt=dt, pad=3, garbage=False), _turns(64))


@pytest.mark.parametrize("D,rot,interleaved", [(16, 16, False), (80, 48, True), (128, 128, False), (128, 64, True), (96, 96, True),
                                               (256, 256, False), (7, 6, False), (100, 20, True), (64, 0, False)])
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (6, 6)])
def test_append_head_sizes(D, rot, interleaved, Hq, Hkv):
    append_checked(make(((3, 3), (40, 1), (150, 20), (17, 2)), D=D, Hq=Hq, Hkv=Hkv, seed=D, garbage=False),
                   _turns(rot) if rot else None, interleaved, 1.2)


@pytest.mark.parametrize("N", [1, 3, 8, 24, 64, 256])
@pytest.mark.parametrize("layout", ["pages", "slots", "odd"])
def test_append_pages_and_layouts(N, layout):
    append_checked(make(MIXED, D=32, N=N, seed=N, layout=layout, garbage=False, kind="int8" if N % 2 else "e4m3"), _turns(32))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_growing_and_shrinking_magnitudes(kind):
    """Token by token into the same pages, magnitudes over 2^40: scales grow, old codes follow, new pages start anew."""
    c = make(((40, 1), (17, 1)), kind=kind, seed=11, garbage=False)
    for i in range(9, 41):
        c["lens"] = torch.tensor([i, i - 8], dtype=torch.int32, device=DEV)
        c["k"].copy_(torch.randn(2, 2, 64, device=DEV) * 2.0 ** ((i * 7) % 40 - 20))
        c["v"].copy_(torch.randn(2, 2, 64, device=DEV) * 2.0 ** ((i * 3) % 13 - 6))
        if i == 30:
            c["k"].zero_()
        append_checked(c, _turns(64))


def test_append_values_that_are_not_finite():
    for kind in ("e4m3", "int8"):
        c = make(((5, 5), (20, 1)), kind=kind, seed=12, garbage=False)
        c["k"][1, 0, 3], c["k"][2, 0, 4], c["v"][5, 1, 0] = float("inf"), float("nan"), float("-inf")
        from sdcguard_amd.kv_attn import kv_append
        want = c["k"][:5, 0].double().cpu()
        kv_append(c["k"], c["v"], c["kv"], c["scales"], *step(c))
        got = stood_for(c["kv"], c["scales"])
        p0, p1 = int(c["bt"][0, 0]), int(c["bt"][1, 1])
        if kind == "int8":
            assert np.isnan(got[p0, 0, :, :64]).all() and np.isnan(got[p1, 1, :, 64:]).all()
            assert not np.isnan(got[p0, 1]).any() and not np.isnan(got[p0, 0, :, 64:]).any()
        else:
            assert np.array_equal(np.isnan(got[p0, 0, :5, :64]), ~np.isfinite(want.numpy()))
            assert np.isnan(got[p1, 1, 3, 64]) and int(np.isnan(got[p1]).sum()) == 1
            fin = want[torch.isfinite(want)].abs().max().item()
            assert float(c["scales"][p0, 0, 0]) == paged.smallest_scale(fin, kind)


def test_append_outside_the_table_or_the_cache_is_not_written():
    c = make(((40, 20), (30, 1), (200, 1)), seed=13, garbage=False)
    c["bt"][0, 1], c["bt"][1, 1] = -1, 1 << 30
    c["lens"][2] = 1 << 20                                             # past the table
    append_checked(c, _turns(64))


def test_append_positions_given_and_sixteen_bit_caches():
    from sdcguard_amd.kv_attn import kv_append, make_cache
    from sdcguard_amd.rope import rotate
    c = make(MIXED, seed=14, garbage=False, pad=2)
    pos = torch.randint(0, 100000, (c["T"] + 2,), device=DEV, dtype=torch.int32)
    append_checked(c, _turns(64), positions=pos)
    append_checked(c, _turns(64), positions=pos.long(), query=False)
    for D in (64, 20):
        for dt in (torch.bfloat16, torch.float16):
            c = make(MIXED, seed=15, D=D, garbage=False)
            kv, scales = make_cache(c["kv"].shape[0], 2, 16, D, dt, DEV)
            assert scales is None
            k, v = c["k"].to(dt), c["v"].to(dt)
            kv_append(k, v, kv, None, *step(c), turns=_turns(D))
            toks = paged.tokens(c["qsl"].tolist(), c["lens"].tolist())
            own = torch.tensor([max(p, 0) for _, p in toks], device=DEV)
            rk = rotate(k, own, _turns(D))
            want = torch.zeros_like(kv)
            for t, (r, p) in enumerate(toks):
                if p >= 0:
                    want[int(c["bt"][r, p // 16]), :, p % 16] = torch.cat([rk[t], v[t]], -1)
            assert torch.equal(kv, want)


def test_append_then_attend_in_a_graph_and_on_another_stream():
    from sdcguard_amd.kv_attn import kv_append, kv_attend, make_cache
    lens = ((26, 1), (5, 1), (60, 1))                                  # four more tokens stay in the last pages
    turns = _turns(64)
    c = make(lens, seed=16, garbage=False)
    kv, scales = make_cache(c["kv"].shape[0] + 4, 2, 16, 64, device=DEV)
    c["kv"], c["scales"] = kv, scales

    def both(c):
        q = kv_append(c["k"], c["v"], c["kv"], c["scales"], *step(c), turns=turns, query=c["q"])
        return kv_attend(q, c["kv"], c["scales"], *step(c))

    both(c)
    e = {**c, "kv": kv.view(torch.uint8).clone().view(kv.dtype), "scales": scales.clone()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(c)
    kv.view(torch.uint8).copy_(e["kv"].view(torch.uint8))
    scales.copy_(e["scales"])
    for i in range(4):
        c["k"].copy_(torch.randn(3, 2, 64, device=DEV) * (i + 1))
        c["lens"].add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, both(e)) and torch.equal(scales, e["scales"])
        assert torch.equal(kv.view(torch.uint8), e["kv"].view(torch.uint8))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o = kv_attend(c["q"], kv, scales, *step(c))
    s.synchronize()
    assert torch.equal(o, kv_attend(c["q"], kv, scales, *step(c)))


def test_same_call_same_bits():
    from sdcguard_amd.kv_attn import kv_attend
    for lens in (((9000, 1), (300, 1)), ((3000, 200), (64, 1))):
        c = make(lens, seed=17, D=128, Hq=8, Hkv=2)
        first = kv_attend(c["q"], c["kv"], c["scales"], *step(c))
        for _ in range(3):
            assert torch.equal(first, kv_attend(c["q"], c["kv"], c["scales"], *step(c)))


def test_refusals():
    from sdcguard_amd import _lib
    from sdcguard_amd.kv_attn import kv_append, kv_attend
    c = make(((20, 2), (5, 1)), seed=18)
    k, v, q, kv, sc, (qsl, lens, bt) = c["k"], c["v"], c["q"], c["kv"], c["scales"], step(c)
    for bad in (lambda: kv_append(k[0], v[0], kv, sc, qsl, lens, bt), lambda: kv_append(k, v[:2], kv, sc, qsl, lens, bt),
                lambda: kv_append(k, v, kv[..., :100], sc, qsl, lens, bt), lambda: kv_append(k, v, kv, None, qsl, lens, bt),
                lambda: kv_append(k, v, kv, sc[:1], qsl, lens, bt), lambda: kv_append(k, v, kv, sc.half(), qsl, lens, bt),
                lambda: kv_append(k, v, kv[:, :1], sc, qsl, lens, bt), lambda: kv_append(k, v, kv, sc, qsl[:1], lens, bt),
                lambda: kv_append(k, v, kv, sc, qsl.float(), lens, bt), lambda: kv_append(k, v, kv, sc, qsl, lens, bt[:1]),
                lambda: kv_append(k, v, kv, sc, qsl, lens, bt, turns=_turns(66)),
                lambda: kv_append(k, v, kv, sc, qsl, lens, bt, turns=_turns(64), positions=qsl[:2]),
                lambda: kv_append(k, v, kv, sc, qsl, lens, bt, query=q[:1]),
                lambda: kv_append(k, v, kv, sc, qsl, lens, bt, query_out=q),
                lambda: kv_append(k, v, kv.view(torch.uint8), sc, qsl, lens, bt),
                lambda: kv_attend(q[0], kv, sc, qsl, lens, bt), lambda: kv_attend(q[:, :3], kv, sc, qsl, lens, bt),
                lambda: kv_attend(q, kv.view(torch.bfloat16), sc, qsl, lens, bt),
                lambda: kv_attend(q, kv, None, qsl, lens, bt), lambda: kv_attend(q, kv, sc, qsl, lens, bt, window=-1),
                lambda: kv_attend(q, kv, sc, qsl, lens, bt, max_seq_len=-1),
                lambda: kv_attend(q, kv, sc, qsl, lens, bt, out=q[:1]), lambda: kv_attend(q, kv, sc, lens, lens, bt)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.HipLibraryError):
        kv_attend(q.float(), kv, sc, qsl, lens, bt)
    with pytest.raises(_lib.HipLibraryError):
        kv_attend(q, kv, sc, qsl.cpu(), lens, bt)
