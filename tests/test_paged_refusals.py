"""What the rotation, the append and the attention over a paged cache refuse, without a GPU: the C entry points' status
for arguments out of range (nothing is launched or read then), the Python entry points' errors for CPU tensors, and
the frequencies of scaled rotations."""
from __future__ import annotations

import math

import pytest
import torch

from sdcguard_amd import _lib, kv_attn, rope

X = 4096            # an address that is never read: every call below is refused, or has nothing to do


def _rope(**kw):
    a = dict(dtype=0, x=X, sxt=128, sxh=64, sxd=1, y=X, syt=128, syh=64, syd=1, T=4, H=2, D=64, pos=X, pb=8, turns=X,
             rot=64, inter=0, m=1.0, inv=0, stream=0)
    a.update(kw)
    return _lib.lib().sdc_rope(*a.values())


def _append(**kw):
    a = dict(dtype=0, cache=0, key=X, skt=128, skh=64, skd=1, val=X, svt=128, svh=64, svd=1, T=4, Hkv=2, D=64, kv=X,
             cb=4096, ch=2048, cn=128, NB=4, N=16, scales=X, sb=4, sh=2, qsl=X, lens=X, R=1, bt=X, sbt=1, W=1, pos=0,
             pb=0, turns=X, rot=64, inter=0, m=1.0, q=0, sqt=0, sqh=0, sqd=0, qo=0, sot=0, soh=0, sod=0, Hq=0, stream=0)
    a.update(kw)
    return _lib.lib().sdc_kv_append(*a.values())


def _attend(**kw):
    a = dict(dtype=0, cache=0, q=X, sqt=128, sqh=64, sqd=1, o=X, sot=128, soh=64, sod=1, lse=0, slt=2, T=4, Hq=2, D=64,
             kv=X, cb=4096, ch=2048, cn=128, NB=4, Hkv=2, N=16, scales=X, sb=4, sh=2, qsl=X, lens=X, R=1, bt=X, sbt=1,
             W=1, scale=1.0, window=0, max_len=16, ws=0, wsb=0, stream=0)
    a.update(kw)
    return _lib.lib().sdc_kv_attend(*a.values())


@pytest.mark.parametrize("kw", [{"dtype": 2}, {"T": -1}, {"D": 0}, {"rot": 3}, {"rot": 66}, {"rot": 4096, "D": 8192},
                                {"pb": 2}, {"x": 0}, {"y": 0}, {"pos": 0}, {"turns": 0}, {"H": -1}])
def test_rotation_refuses(kw):
    assert _rope(**kw) == _lib.SDC_EINVAL


@pytest.mark.parametrize("kw", [{"dtype": 4}, {"cache": 3}, {"cache": -1}, {"T": -1}, {"Hkv": 0}, {"D": 0}, {"D": 2048},
                                {"NB": 0}, {"N": 0}, {"N": 1 << 17}, {"R": -1}, {"W": -1}, {"rot": 65}, {"rot": 128},
                                {"pos": X, "pb": 3}, {"q": X, "Hq": 0, "qo": X}, {"q": X, "Hq": 2}, {"key": 0},
                                {"val": 0}, {"kv": 0}, {"scales": 0}, {"qsl": 0}, {"lens": 0}, {"bt": 0}, {"turns": 0}])
def test_append_refuses(kw):
    assert _append(**kw) == _lib.SDC_EINVAL


@pytest.mark.parametrize("kw", [{"dtype": 4}, {"cache": 2}, {"T": -1}, {"Hq": 3}, {"Hq": 0}, {"Hkv": 0}, {"D": 0},
                                {"D": 257}, {"NB": 0}, {"N": 0}, {"R": -1}, {"W": -1}, {"window": -1}, {"max_len": -1},
                                {"max_len": 17}, {"q": 0}, {"o": 0}, {"kv": 0}, {"scales": 0}, {"qsl": 0}, {"bt": 0}])
def test_attention_refuses(kw):
    assert _attend(**kw) == _lib.SDC_EINVAL


def test_nothing_to_do_is_done():
    assert _rope(T=0, x=0, y=0) == 0 and _rope(H=0) == 0 and _append(T=0, key=0) == 0 and _attend(T=0, q=0) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    kv, sc = kv_attn.make_cache(2, 2, 16, 64, device="cpu")
    turns, _ = rope.frequencies(64, device="cpu")
    with pytest.raises(_lib.HipLibraryError):
        rope.rotate(x, i, turns)
    with pytest.raises(_lib.HipLibraryError):
        kv_attn.kv_append(x, x, kv, sc, i, i[:1], i.view(1, 2))
    with pytest.raises(_lib.HipLibraryError):
        kv_attn.kv_attend(x, kv, sc, i, i[:1], i.view(1, 2))


@pytest.mark.parametrize("bad", [{"rot": 0}, {"rot": 7}, {"base": 1.0}, {"base": float("nan")},
                                 {"scaling": {"kind": "no"}}, {"scaling": {"kind": "linear", "factor": 0.5}},
                                 {"scaling": {"kind": "ramp", "factor": 4.0}},
                                 {"scaling": {"kind": "bands", "factor": 4.0, "trained": 8192, "low": 4, "high": 1}},
                                 {"rot": 2, "scaling": {"kind": "base", "factor": 2.0}}])
def test_frequencies_refuse(bad):
    with pytest.raises(ValueError):
        rope.frequencies(**{"rot": 64, "device": "cpu", **bad})


def test_frequencies_of_scaled_rotations():
    plain, m = rope.frequencies(64, 500000.0, device="cpu")
    assert m == 1.0 and plain[0].item() == 1 / (2 * math.pi)
    assert torch.allclose(plain * 2 * math.pi, 500000.0 ** (-torch.arange(32).double() / 32), rtol=1e-14)
    lin, _ = rope.frequencies(64, 500000.0, {"kind": "linear", "factor": 8.0}, device="cpu")
    assert torch.allclose(lin, plain / 8, rtol=1e-14)
    base, _ = rope.frequencies(64, 500000.0, {"kind": "base", "factor": 8.0}, device="cpu")
    assert base[0] == plain[0] and math.isclose(base[-1].item(), plain[-1].item() / 8, rel_tol=1e-12)
    for kind in ("ramp", "bands"):
        t, m = rope.frequencies(64, 500000.0, {"kind": kind, "factor": 8.0, "trained": 8192}, device="cpu")
        assert t[0] == plain[0] and math.isclose(t[-1].item(), plain[-1].item() / 8, rel_tol=1e-12)
        assert ((t <= plain) & (t >= plain / 8 * (1 - 1e-12))).all() and (t[:-1] > t[1:]).all()
        assert m == (1.0 + 0.1 * math.log(8.0) if kind == "ramp" else 1.0)


@pytest.mark.parametrize("window", [(1 << 63) - 1, (1 << 63) - 16, 1 << 62, 1 << 40, 1 << 31])
def test_a_window_wider_than_any_length_is_none(window):
    """The parts that a call's keys are cut into, by the workspace that they need."""
    need = _lib.lib().sdc_kv_attend_workspace
    for T, R, N, most in ((1, 1, 16, 200000), (1, 1, 1, 5000), (64, 64, 16, 131072), (4096, 2, 16, 131072), (3, 0, 8, 70000)):
        assert need(T, R, 32, 8, 128, N, most, window) == need(T, R, 32, 8, 128, N, most, 0)
    assert need(1, 1, 32, 8, 128, 16, 200000, window) > 0


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_attention_refuses_scales_that_are_no_numbers(scale):
    assert _attend(scale=scale) == _lib.SDC_EINVAL
