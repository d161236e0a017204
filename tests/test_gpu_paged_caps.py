"""Caps of the paged cache's scores (softcap) over their whole range: errors go with the score, not with the cap."""
from __future__ import annotations

import numpy as np
import pytest

from paged import HALF, Cache, attention, attention_tolerance, bits16, from_bits
from test_gpu_paged import attend, types  # noqa: F401

pytestmark = pytest.mark.gpu

ROOM = 140000   # of tables by which long keys are dealt and rows' keys shared

# (call, tokens of room, new rows, lengths, heads, kv-heads)
WAYS = {"decode": ("decode", 0, [1, 1, 1], [300, 40, 7], 4, 2), "dealt": ("decode", ROOM, [1, 1, 1], [300, 40, 7], 4, 2),
        "few rows": ("prefill", 0, [30, 3], [90, 40], 4, 2), "shared": ("prefill", ROOM, [50, 20], [100, 90], 4, 2),
        "shared by eight": ("prefill", ROOM, [200], [230], 4, 4)}


@pytest.fixture(params=WAYS)
def way(request):
    return request.param


def capped_tolerance(cache, ref, absv, mag, seen, cap):
    """attention_tolerance of scores without a cap (a cap shrinks their errors), and the cap's own: at most 14 half steps of fp32 of the
    capped score (a quotient below 1 with 3 half steps times 2 cap, a sum with the cap, where the score is at least 0.46 of it; a polynomial
    within 2^-25 and 6 roundings below), with caps up to 64 also 2^-22 of the cap; weights move by as much."""
    err = 2.0 ** -20 * np.minimum(mag, cap) + (2.0 ** -22 * cap if cap <= 64 else 0.0)
    return attention_tolerance(cache, ref, absv, mag, seen) + 2 * err * absv


def check(ti, types, monkeypatch, way, dim, cap, q_amp, scale, slopes=None, seed=70, k_amp=None):  # noqa: F811
    fn, room, new, lens, heads, kv_heads = WAYS[way]
    monkeypatch.setattr(Cache, "wide", room)
    rng = np.random.RandomState(seed)
    cache = Cache(ti, rng, lens, kv_heads, dim, 16, *types)
    rows = sum(new)
    x = rng.standard_normal((rows, heads, dim)) * np.resize(q_amp, heads)[None, :, None]
    bits = bits16(x.reshape(rows, -1), types[0])
    x = from_bits(bits, types[0])
    assert np.isfinite(x).all()
    cache.upload()
    got = from_bits(attend(ti, cache, bits, heads, new, fn=fn, scale=scale, cap=cap, slopes=slopes), types[0])
    ref, absv, mag, seen = attention(cache, x, new, heads, scale, cap=cap, slopes=slopes)
    tol = capped_tolerance(cache, ref, absv, mag, seen, cap)
    bad = ~(np.abs(got - ref) <= tol)
    at = np.argwhere(bad)[:1].ravel()
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first {at}: {got[tuple(at)]!r} for {ref[tuple(at)]!r}, may be {tol[tuple(at)]:.3g} off"


@pytest.mark.parametrize("cap,slopes", [(1e3, True), (1e5, False), (1e8, True), (1e30, False)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_caps_far_above_the_scores(ti, types, monkeypatch, way, dim, cap, slopes):  # noqa: F811
    check(ti, types, monkeypatch, way, dim, cap, 2.0, dim ** -0.5, np.array([0.0, 0.25, 0.01, 1.0]) if slopes else None)


@pytest.mark.parametrize("cap", [0.5, 20.0, 65.0, 1e3, 1e5])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_scores_on_both_sides_of_the_cap(ti, types, monkeypatch, way, dim, cap):  # noqa: F811
    """Heads of a group, which share their steps: scores of about 1.5, of half the cap, and of many times the cap."""
    q = np.array([0.1, 0.1 * max(cap, 2.0) / 3, 0.1, 0.1 * min(2 * cap, 3e4)])
    check(ti, types, monkeypatch, way, dim, cap, q, 15.0 * dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 256])
def test_scale_and_cap_at_the_ends(ti, types, monkeypatch, way, dim):  # noqa: F811
    """Keys of zeros score 0 whatever the quotient of scale and cap."""
    fn, room, new, lens, heads, kv_heads = WAYS[way]
    monkeypatch.setattr(Cache, "wide", room)
    rng = np.random.RandomState(71)
    cache = Cache(ti, rng, lens, kv_heads, dim, 16, *types)
    for b, n in enumerate(lens):
        for j in range(0, n, 2):
            cache.k[cache.table[b, j // 16], :, j % 16] = 0
    bits = bits16(rng.standard_normal((sum(new), heads * dim)), types[0])
    cache.upload()
    for scale, cap in ((1e20, 1e-20), (-1e30, 1e-20), (1e-20, 1e20), (1e-30, 1e30), (-0.1, 1e6), (1e-45, 5.0)):
        got = from_bits(attend(ti, cache, bits, heads, new, fn=fn, scale=scale, cap=cap), types[0])
        ref, absv, mag, seen = attention(cache, from_bits(bits, types[0]), new, heads, scale, cap=cap)
        # (errors of a product, however large, move a capped score by the cap at most twice)
        assert (np.abs(got - ref) <= capped_tolerance(cache, ref, absv, np.minimum(mag, cap), seen, cap)).all(), (scale, cap)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinite_and_undefined_scores(ti, monkeypatch, way, dim):
    """An infinite score is the cap's; one that is no number reaches the rows that see it, in the key's head."""
    fn, room, new, lens, heads, kv_heads = WAYS[way]
    monkeypatch.setattr(Cache, "wide", room)
    for cap in (4.0, 1e4):
        for value in (np.inf, np.nan):
            rng = np.random.RandomState(72)
            cache = Cache(ti, rng, lens, kv_heads, dim, 16, "bf16", "same")
            cache.k[cache.table[0, 0], 0, 3, 5] = value
            bits = bits16(np.abs(rng.standard_normal((sum(new), heads * dim))) + 0.5, "bf16")
            cache.upload()
            got = from_bits(attend(ti, cache, bits, heads, new, fn=fn, cap=cap), "bf16").reshape(sum(new), kv_heads, -1)
            hit = got[: new[0], 0]
            assert np.isnan(hit).all() if np.isnan(value) else np.isfinite(hit).all()
            assert np.isfinite(got[: new[0], 1:]).all() and np.isfinite(got[new[0]:]).all()
            if value == np.inf and cap == 1e4:   # all the weight; it and the output are rounded
                want = cache.values("v", 0, 3)[0]
                assert (np.abs(hit.reshape(-1, dim) - want) <= 2.02 * HALF["bf16"] * np.abs(want)).all()
