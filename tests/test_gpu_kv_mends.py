"""The paged operators at the ends of what their arguments and values may be: windows wider than any length, magnitudes and
scales at both ends of their types, steps and tables of nothing, and what autograd has to know of their calls."""
from __future__ import annotations

import importlib.util
import math

import pytest
import torch

from oracle import paged
from sdcguard_amd import _lib
from tests.test_gpu_kv_attn import DEV, _turns, append_checked, attend_checked, make, step

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


def plain64(c):
    """(o, lse, mass, top, terms) of the step's queries in float64 on the device: the outputs, sum p |v| / sum p, the same with
    each value its scale's largest, and the largest |q| . |k| scale of a row.  (Finite caches, no window.)"""
    D, N, Hkv = c["D"], c["N"], c["kv"].shape[1]
    code = c["kv"].view(torch.uint8).view(c["kv"].dtype).float().double()
    sc = c["scales"].double()
    outs = []
    for r, n in enumerate(c["lens"].tolist()):
        a, b = int(c["qsl"][r]), int(c["qsl"][r + 1])
        pages = c["bt"][r, :-(-n // N)].long()
        x = code[pages].transpose(1, 2).reshape(-1, Hkv, 2 * D)[:n]              # (keys, kv heads, 2 D)
        ks, vs = sc[pages].repeat_interleave(N, 0)[:n].unbind(-1)
        q = c["q"][a:b].double().view(b - a, Hkv, -1, D)
        k, v = x[..., :D] * ks[..., None], x[..., D:] * vs[..., None]
        s = torch.einsum("thgd,khd->thgk", q, k) * D ** -0.5
        terms = torch.einsum("thgd,khd->thgk", q.abs(), k.abs()).amax(-1) * D ** -0.5
        seen = torch.arange(n, device=DEV) <= torch.arange(n - (b - a), n, device=DEV)[:, None]
        s = s.masked_fill(~seen[:, None, None], float("-inf"))
        p = torch.softmax(s, -1)
        flat = [torch.einsum("thgk,khd->thgd", p, y) for y in (v, v.abs(), vs[..., None].abs() * paged.TOP[c["kind"]])]
        outs.append([y.flatten(1, 2) for y in (flat[0], torch.logsumexp(s, -1), flat[1], flat[2], terms)])
    return [torch.cat(y) for y in zip(*outs)]


def attend_tight(c, **kw):
    """attend_checked with a bound that only the keys which a row sees, at their weights, have a part in."""
    from sdcguard_amd.kv_attn import kv_attend
    o, lse = kv_attend(c["q"], c["kv"], c["scales"], *step(c), return_lse=True, **kw)
    D, T, n, info = c["D"], c["T"], int(c["lens"].max()), torch.finfo(c["dt"])
    ro, rl, mass, top, terms = plain64(c)
    ds = (D + 16) * 2.0 ** -24 * terms + 2.0 ** -20
    # the output's rounding, of a subnormal one by half the type's smallest step; a probability's product with its scale is
    # rounded to 11 bits, or by a fp16 step of 2^-24 where the row's largest product is 2^4 or more; a maximum of up to 2^8
    # that carries the scales' exponent is rounded to 2^-16
    tol = info.eps / 2 * ro.abs() + info.smallest_normal * info.eps / 2 \
        + (2.0 ** -11 + 2.0 ** -15 + 2 * ds[..., None] + (n + 16) * 2.0 ** -23) * mass + n * 2.0 ** -29 * top
    err = (o[:T].double() - ro).abs()
    assert (err <= tol).all(), (int((~(err <= tol)).sum()), (~(err <= tol)).nonzero()[:5], err[~(err <= tol)][:5], tol[~(err <= tol)][:5])
    bad = ~((lse[:T].double() - rl).abs() <= ds + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * rl.abs() + 2.0 ** -16)
    assert not bad.any(), (bad.nonzero()[:5], lse[:T][bad][:5], rl[bad][:5])


def tall(c):
    """The step with so wide a table that its chunks are taken in tiles of 256 rows, and whether they were."""
    R, W = c["bt"].shape
    wide = torch.full((R, max(W, 2000000 // c["N"])), -7, dtype=torch.int32, device=DEV)
    wide[:, :W] = c["bt"]
    return {**c, "bt": wide}


class launches:
    """How often a kernel was launched, by name."""
    def __enter__(self):
        _lib.lib().sdc_profile_reset()
        _lib.lib().sdc_profile_enable(1)
        return lambda name: _lib.profile_read(name)[1]

    def __exit__(self, *a):
        _lib.lib().sdc_profile_enable(0)
        _lib.lib().sdc_profile_reset()


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


TALL = (((700, 200), (90, 90)), ((9000, 70), (300, 1)))


@pytest.mark.parametrize("lens", TALL, ids=["chunk", "split"])
@pytest.mark.parametrize("D,N", [(64, 16), (128, 8), (256, 16)])
def test_chunks_weigh_keys_whose_values_are_zeros(D, N, lens):
    """Pages of zeros have the smallest scale, 2^-126: their keys take their part of the weights all the same, beside values of
    ordinary and of large scales."""
    c = tall(make(lens, D=D, Hq=4, Hkv=1, N=N, seed=23, garbage=False))
    pages = c["bt"][0, :lens[0][0] // N].long()
    c["kv"].view(torch.uint8)[pages[1::2], :, :, D:] = 0
    with launches() as count:
        for ordinary in (2.0 ** -7, 1.0, 2.0 ** 20, 2.0 ** 39):
            c["scales"][pages, :, 1] = ordinary
            c["scales"][pages[1::2], :, 1] = 2.0 ** -126
            attend_tight(c)
            c["scales"][pages[1::2], :, 0] *= 0.5      # (weights mostly under 2^-13 of the largest, of many keys)
            attend_tight(c)
            c["scales"][pages[1::2], :, 0] *= 2.0
        assert count("kv_attend_tiles") == 8


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("lens", TALL, ids=["chunk", "split"])
def test_chunks_of_value_scales_at_both_ends_and_far_from_each_other(lens, kind):
    c = tall(make(lens, D=64, Hq=4, Hkv=1, seed=24, kind=kind, garbage=False))
    pages = c["bt"][0, :lens[0][0] // 16].long()
    for e in (-126, -110, -60, -24, 24, 60, 100, 118):
        c["scales"][..., 1] = 2.0 ** e
        attend_tight(c)
    for last in (0, 20, 60, 100):
        c["scales"][pages, :, 1] = 2.0 ** -30
        c["scales"][pages[-2:], :, 1] = 2.0 ** last
        attend_tight(c)
    c["scales"][pages, :, 1] = (2.0 ** torch.linspace(-80, 80, pages.numel(), device=DEV))[:, None]
    attend_tight(c)
    c["scales"][pages, :, 1] = c["scales"][pages.flip(0), :, 1].clone()
    attend_tight(c)


@pytest.mark.parametrize("N", [16, 8, 6])
@pytest.mark.parametrize("large", [False, True])
def test_keys_that_are_nan_reach_lse_too(large, N):
    """A page outside the cache, and one whose key scale is NaN: where the other keys score hundreds more as well."""
    c = make(((300, 200), (90, 1)), D=64, Hq=4, Hkv=2, N=N, seed=25, garbage=False)
    c["bt"][0, 150 // N] = -1
    c["scales"][c["bt"][1, 1].long(), 1, 0] = float("nan")
    for scale in (None, 10.0, 300.0):
        with launches() as count:
            o, lse = attend_checked(tall(c) if large else c, scale=scale)
            assert count("kv_attend_tiles") == int(large)
        first = 150 // N * N - 100                     # the first row that sees the page
        assert lse[first:200].isnan().all() and not lse[:first].isnan().any()
        assert lse[200, 2:].isnan().all() and not lse[200, :2].isnan().any()


@pytest.mark.parametrize("large", [False, True])
def test_queries_up_to_the_largest_number(large):
    """bf16's largest numbers are queries like others."""
    c = make(((300, 200), (90, 1)), D=64, Hq=4, Hkv=1, seed=26, garbage=False)
    c["scales"][..., 0] = 2.0 ** -132                  # (scores of a few units)
    c["q"][:, :, 5] = torch.finfo(torch.bfloat16).max
    c["q"][1::2, :, 5] *= -1.0
    attend_tight(tall(c) if large else c)


def test_calls_that_would_drop_a_gradient_are_refused():
    from sdcguard_amd.kv_attn import kv_append, kv_attend
    from sdcguard_amd.rope import rotate
    c = make(((20, 2), (5, 1)), seed=27, garbage=False)
    k, v, q, kv, sc, st = c["k"], c["v"], c["q"], c["kv"], c["scales"], step(c)
    turns, pos = _turns(64), torch.arange(3, device=DEV)
    leaf = lambda t: t.clone().requires_grad_()                                                   # noqa: E731
    calls = (lambda: kv_append(leaf(k), v, kv, sc, *st), lambda: kv_append(k, leaf(v), kv, sc, *st),
             lambda: kv_append(k, v, kv, leaf(sc), *st), lambda: kv_append(k, v, kv, sc, *st, turns=leaf(turns)),
             lambda: kv_append(k, v, kv, sc, *st, query=leaf(q)),
             lambda: kv_append(k, v, kv, sc, *st, query=q, query_out=leaf(q)),
             lambda: kv_attend(leaf(q), kv, sc, *st), lambda: kv_attend(q, kv, leaf(sc), *st),
             lambda: kv_attend(q, kv, sc, *st, out=leaf(q)), lambda: rotate(q, pos, leaf(turns)))
    codes, before = kv.view(torch.uint8).clone(), sc.clone()
    for call in calls:
        with pytest.raises(ValueError, match="takes? no gradient"):
            call()
    assert torch.equal(codes, kv.view(torch.uint8)) and torch.equal(before, sc)
    with torch.no_grad():
        for call in calls:
            call()
        assert torch.equal(kv_attend(leaf(q), kv, sc, *st), kv_attend(q, kv, sc, *st))
    with torch.inference_mode():
        kv_attend(q, kv, sc, *st)


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad
    from sdcguard_amd.kv_attn import kv_append, kv_attend
    from sdcguard_amd.rope import rotate
    c = make(((20, 2), (5, 1)), seed=28, garbage=False)
    k, v, q, kv, sc, st = c["k"], c["v"], c["q"], c["kv"], c["scales"], step(c)
    turns, pos = _turns(64), torch.arange(3, device=DEV)
    codes = kv.view(torch.uint8).clone()
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))                              # noqa: E731
        for call in (lambda: rotate(dual(q), pos, turns), lambda: rotate(q, pos, dual(turns)),
                     lambda: rotate(q, pos, turns, out=dual(q.clone())),
                     lambda: rotate(dual(q.float()).requires_grad_(), pos, turns),
                     lambda: kv_append(dual(k), v, kv, sc, *st), lambda: kv_append(k, v, kv, sc, *st, query=dual(q)),
                     lambda: kv_attend(dual(q), kv, sc, *st)):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(ValueError, match="forward-mode"):
                    call()
    assert torch.equal(codes, kv.view(torch.uint8))


def test_autograd_knows_what_was_written_in_place():
    from sdcguard_amd.kv_attn import kv_append, kv_attend, make_cache
    from sdcguard_amd.rope import rotate
    c = make(((20, 2), (5, 1)), seed=29, garbage=False)
    k, v, q, kv, sc, st = c["k"], c["v"], c["q"].contiguous(), c["kv"], c["scales"], step(c)
    turns, pos = _turns(64), torch.arange(3, device=DEV)
    x = q.float().requires_grad_()
    y = x * 2.0
    z = (y * y).sum()                                  # y is kept for the gradient
    with torch.no_grad():
        rotate(y, pos, turns, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    full, _ = make_cache(4, 2, 16, 64, torch.bfloat16, DEV)
    for call, wrote, kept in ((lambda: kv_append(k, v, kv, sc, *st), (kv, sc), (k, v)),
                              (lambda: kv_append(k, v, kv, sc, *st, query=q), (kv, sc), (k, v, q)),
                              (lambda: kv_append(k, v, kv, sc, *st, query=q, query_out=q), (kv, sc, q), (k, v)),
                              (lambda: kv_append(k, v, full, None, *st), (full,), (k, v)),
                              (lambda: kv_attend(q, kv, sc, *st, out=c["q"]), (c["q"],), (q, kv, sc)),
                              (lambda: kv_attend(q, kv, sc, *st), (), (q, kv, sc)),
                              (lambda: rotate(q, pos, turns), (), (q, pos, turns))):
        before = [t._version for t in wrote + kept]
        call()
        after = [t._version for t in wrote + kept]
        assert all(b > a for a, b in zip(before, after[:len(wrote)])) and after[len(wrote):] == before[len(wrote):]
    with torch.inference_mode():
        held, hs = make_cache(4, 2, 16, 64, device=DEV)
        kv_append(k, v, held, hs, *st)
    kv_append(k, v, held, hs, *st)                     # (tensors of inference mode have no version to raise)


def test_outputs_that_overlap_are_refused():
    from sdcguard_amd.kv_attn import kv_append, kv_attend
    from sdcguard_amd.rope import rotate
    c = make(((20, 2), (5, 1)), seed=30, garbage=False)
    k, v, kv, sc, st = c["k"], c["v"], c["kv"], c["scales"], step(c)
    q = c["q"].contiguous()
    turns, pos = _turns(64), torch.arange(3, device=DEV)
    long = torch.randn(4, 4, 64, device=DEV).bfloat16()
    once = torch.empty(1, 4, 64, device=DEV, dtype=torch.bfloat16).expand(3, 4, 64)
    flat = torch.randn(3 * 4 * 64, device=DEV).bfloat16()
    kk = flat[:3 * 2 * 64].view(3, 2, 64)
    for call in (lambda: rotate(long[1:], pos, turns, out=long[:3]), lambda: rotate(long[:3], pos, turns, out=once),
                 lambda: kv_append(k, v, kv, sc, *st, query=long[1:], query_out=long[:3]),
                 lambda: kv_append(k, v, kv, sc, *st, query=q, query_out=once),
                 lambda: kv_append(kk, v, kv, sc, *st, query=q, query_out=flat.view(3, 4, 64)),
                 lambda: kv_append(k, v, kv[:1].expand_as(kv), sc, *st),
                 lambda: kv_append(k, v, kv, sc[:1].expand_as(sc), *st),
                 lambda: kv_attend(long[1:], kv, sc, *st, out=long[:3]), lambda: kv_attend(q, kv, sc, *st, out=once)):
        with pytest.raises(ValueError, match="memory|twice"):
            call()
    want = kv_attend(q, kv, sc, *st)
    assert torch.equal(kv_attend(q, kv, sc, *st, out=q), want) and torch.equal(q, want)           # (in place)


def test_positions_of_another_shape_are_refused():
    """As many positions as tokens, but not the tokens' shape: they would go to the wrong ones."""
    from sdcguard_amd.rope import rotate
    x, turns = torch.randn(6, 5, 4, 64, device=DEV), _turns(64)
    pos = torch.randint(0, 9000, (6, 5), device=DEV)
    want = rotate(x, pos, turns)
    assert torch.equal(rotate(x, pos.reshape(-1), turns), want)
    for bad in (pos.t().contiguous(), pos.t(), pos.view(3, 10), pos.view(1, 30), pos.view(6, 5, 1), pos[:, :1], pos[:1]):
        with pytest.raises(ValueError, match="positions"):
            rotate(x, bad, turns)
    assert torch.equal(rotate(x[0], pos[:1], turns), rotate(x[0], pos[0], turns))


@pytest.mark.parametrize("T", [1, 40, 3000])
def test_steps_without_requests_and_tables_without_pages(T):
    """A captured step that is all padding, and requests that have no page: nothing is written, zeros and -inf come out."""
    from sdcguard_amd.kv_attn import kv_append, kv_attend
    for D in (64, 40):
        for R, W in ((0, 5), (0, 0), (2, 0), (0, 200000)):
            c = make(((20, 2),), D=D, Hq=8, Hkv=2, seed=31, garbage=False)
            k, v = (torch.randn(T, 2, D, device=DEV).bfloat16() for _ in range(2))
            q = torch.randn(T, 8, D, device=DEV).bfloat16()
            st = (torch.full((R + 1,), min(R, 1) * T, device=DEV, dtype=torch.int32),
                  torch.full((R,), T, device=DEV, dtype=torch.int32), torch.zeros(R, W, device=DEV, dtype=torch.int32))
            st[0][0] = 0
            codes, sc = c["kv"].view(torch.uint8).clone(), c["scales"].clone()
            rotated = kv_append(k, v, c["kv"], c["scales"], *st, turns=_turns(D), query=q)
            o, lse = kv_attend(q, c["kv"], c["scales"], *st, return_lse=True)
            assert not o.any() and torch.isneginf(lse).all() and bool(rotated.any()) == (R > 0)
            assert torch.equal(codes, c["kv"].view(torch.uint8)) and torch.equal(sc, c["scales"])


def test_scales_that_are_no_numbers_are_refused():
    from sdcguard_amd.kv_attn import kv_attend
    c = make(((20, 2), (5, 1)), seed=32)
    for scale in (float("nan"), float("inf"), -1e300):
        with pytest.raises(ValueError, match="finite"):
            kv_attend(c["q"], c["kv"], c["scales"], *step(c), scale=scale)


@pytest.mark.parametrize("cache", ["e4m3", "int8"])
def test_the_example_guards_the_scales_too(cache):
    from tests.test_gpu_guarded_decode import PATH
    spec = importlib.util.spec_from_file_location("guarded_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    _, _, bad, found = m.main(48, cache, quiet=True)
    assert bad == 0 and found["entries"] == [(1, 0)] and found["scale_entries"] == [(0, 0)]


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("N", [16, 6])
def test_value_scales_on_both_sides_of_each_limit(N, large):
    """Pages of two scales, within what a part takes as they are, within what it takes relative to one, and past both; beside
    pages of scale 0, of zeros, and of a subnormal scale."""
    c = make(((300, 200), (90, 1), (1, 1)), D=64, Hq=4, Hkv=1, N=N, seed=33, garbage=False)
    c = tall(c) if large else c
    for hi, lo in ((39, -60), (40, -61), (41, -60), (42, -59), (80, -19), (80, -20), (80, -21), (-60, -70), (-61, -125), (-100, -126),
                   (-125, -126), (-126, -126), (118, 19), (118, 17), (60, -60)):
        for other in (2.0 ** lo, 0.0, 2.0 ** -126, 2.0 ** -135):
            c["scales"][:, :, 1] = 2.0 ** hi
            c["scales"][::3, :, 1] = 2.0 ** lo
            c["scales"][::7, :, 1] = other
            attend_tight(c)


@pytest.mark.parametrize("D,apart", [(40, False), (64, True)])
@pytest.mark.parametrize("size", [-110, 0, 127])
def test_plain_rows_take_queries_of_any_size(size, D, apart):
    """Head sizes that no tile takes, and parts that are left to plain rows, with queries up to bf16's largest and down to small
    ones: scores of a few units."""
    c = make(((300, 40), (90, 1)), D=D, Hq=4, Hkv=1, seed=34, garbage=False)
    c["q"].mul_(2.0 ** (size - 2)).clamp_(-torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).max)
    c["scales"][..., 0] = 2.0 ** (-size - 6) if size >= 0 else 2.0 ** 104
    if apart:
        c["scales"][:, :, 1] = 2.0 ** -70
        c["scales"][::2, :, 1] = 2.0 ** 40
    attend_tight(c)
