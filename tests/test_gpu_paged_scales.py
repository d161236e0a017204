"""Scales of the paged cache's scores at the ends of their range, with products that suit them."""
from __future__ import annotations

import numpy as np
import pytest

from paged import Cache, attention, attention_tolerance, bits16, from_bits, round16
from test_gpu_paged import attend
from test_gpu_paged_caps import WAYS

pytestmark = pytest.mark.gpu


class Zero(float):
    """A scale of 0 that the call is given as it is."""

    def __bool__(self):
        return True


@pytest.mark.parametrize("shaped", [False, True])
@pytest.mark.parametrize("scale", [2e-37, -2e-37, 1e-45, Zero(0.0), 1e30], ids=str)
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_small_scales_of_large_products(ti, monkeypatch, dim, way, scale, shaped):
    """bf16 queries and keys whose products are up to about 1e37 (or 1e-31): scores of about 1, or (scales of next to nothing) none."""
    fn, room, new, lens, heads, kv_heads = WAYS[way]
    monkeypatch.setattr(Cache, "wide", room)
    rng = np.random.RandomState(81)
    cache = Cache(ti, rng, lens, kv_heads, dim, 16, "bf16", "same")
    amp = 5e17 if abs(scale) < 1 else 3e-16
    cache.k = round16(cache.k * amp, "bf16")
    bits = bits16(rng.standard_normal((sum(new), heads * dim)) * amp, "bf16")
    cache.upload()
    slopes = 2.0 ** -rng.uniform(2, 8, heads) if shaped else None
    got = from_bits(attend(ti, cache, bits, heads, new, fn=fn, scale=scale, slopes=slopes), "bf16")
    ref, absv, mag, seen = attention(cache, from_bits(bits, "bf16"), new, heads, float(np.float32(scale)), slopes=slopes)
    assert (np.abs(got - ref) <= attention_tolerance(cache, ref, absv, mag, seen)).all()
