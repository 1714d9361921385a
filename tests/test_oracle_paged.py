"""The float64 oracle of rotary positions and the paged 8-bit cache against independent statements: the rotation as
complex products and its gradient by differences, the scales by trying powers of two, attention by a softmax per row."""
from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import paged


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [2, 6, 10])
def test_rotation_is_a_complex_product_and_its_gradient_the_inverse(rot, interleaved):
    rng = np.random.default_rng(rot)
    x, pos = rng.standard_normal((3, 2, 10)), np.array([0, 7, 100003])
    turns = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot) / (2 * math.pi)
    y = paged.rotate(x, pos, turns, interleaved, 1.3)
    ia, ib = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2), np.arange(rot // 2, rot))
    z = (x[..., ia] + 1j * x[..., ib]) * 1.3 * np.exp(2j * math.pi * pos[:, None] * turns)[:, None]
    assert np.allclose(y[..., ia], z.real, atol=1e-9) and np.allclose(y[..., ib], z.imag, atol=1e-9)
    assert np.array_equal(y[..., rot:], x[..., rot:])
    dy = rng.standard_normal(x.shape)
    dx = paged.rotate(dy, pos, turns, interleaved, 1.3, inverse=True)
    for _ in range(5):                                      # the map is linear: its differences are exact
        d = rng.standard_normal(x.shape)
        lhs = ((paged.rotate(x + d, pos, turns, interleaved, 1.3) - y) * dy).sum()
        # elements past rot pass their gradient unchanged: dx there is dy
        assert abs(lhs - (dx * d).sum()) < 1e-9 * (1 + abs(lhs))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_scales_are_the_smallest_powers_of_two(kind):
    rng = np.random.default_rng(1)
    for amax in list(np.exp(rng.uniform(-60, 60, 200))) + [paged.TOP[kind], np.nextafter(paged.TOP[kind], 1e9), 1e-45]:
        s = paged.smallest_scale(float(amax), kind)
        assert s * paged.TOP[kind] >= amax and math.frexp(s)[0] == 0.5
        assert s == 2.0 ** -126 or s / 2 * paged.TOP[kind] < amax
    assert paged.smallest_scale(0.0, kind) == 2.0 ** -126


def test_append_grows_scales_and_starts_pages_anew():
    D, N = 2, 4
    stored, scales = np.ones((3, 1, N, 2 * D)), np.full((3, 1, 2), 2.0 ** -9)
    key, val = np.full((3, 1, D), 900.0), np.full((3, 1, D), 1e-3)
    # request 0 appends position 3 of page 0 and 4, 5 of page 2
    v, s, tol = paged.append(key, val, stored, scales, [0, 3], [6], np.array([[0, 2]]), "e4m3", N)
    assert s[0, 0, 0] == 4.0 and s[0, 0, 1] == 2.0 ** -9 and s[2, 0, 0] == 4.0 and s[2, 0, 1] < 2.0 ** -17
    assert np.array_equal(v[0, 0, 3], [900, 900, 1e-3, 1e-3]) and np.array_equal(v[2, 0, 1], v[0, 0, 3])
    assert (tol[0, 0, :3, :D] > 0).all() and not tol[0, 0, :3, D:].any() and not tol[1].any() and np.isinf(tol[2, 0, 2:]).all()


def test_attention_is_a_softmax_per_row():
    rng = np.random.default_rng(2)
    N, D = 4, 3
    kv, q = rng.standard_normal((5, 2, N, 2 * D)), rng.standard_normal((4, 4, D))
    bt = np.array([[3, 1, 0], [2, 4, 9]])
    o, lse, mass, _ = paged.attend(q, kv, [0, 3, 4], [6, 1], bt, N, 0.7, window=5)
    for t, p in ((0, 3), (1, 4), (2, 5)):
        for h in range(4):
            keys = [j for j in range(p + 1) if j > p - 5]
            rows = np.array([kv[bt[0, j // N], h // 2, j % N] for j in keys])
            w = np.exp(rows[:, :D] @ q[t, h] * 0.7)
            assert np.allclose(o[t, h], (w[:, None] * rows[:, D:]).sum(0) / w.sum()) and np.isclose(lse[t, h], np.log(w.sum()))
    assert np.allclose(o[3, 0], kv[2, 0, 0, D:]) and (mass >= np.abs(o) - 1e-12).all()
    o, lse, _, _ = paged.attend(q, kv, [0, 4], [2], bt, N, 1.0)                     # two rows without a position
    assert not o[:2].any() and np.isneginf(lse[:2]).all() and o[2:].any()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_scales_hold_the_largest_values_of_32_bits(kind):
    for amax in (2.0 ** 127, 127.0 * 2.0 ** 120, 127.5 * 2.0 ** 120, 2e38, 255.0 * 2.0 ** 120, 2.0 ** 128 * (1 - 2.0 ** -24)):
        s = paged.smallest_scale(amax, kind)
        assert s * paged.TOP[kind] >= amax > s / 2 * paged.TOP[kind]
        assert s <= 2.0 ** (120 if kind == "e4m3" else 122)
