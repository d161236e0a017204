"""Every kernel of the paged cache's attention in every form, by sizes of which it is asserted that they choose it."""
from __future__ import annotations

import numpy as np
import pytest

from paged import TINY, Cache, attention, attention_tolerance, bits16, from_bits
from test_gpu_paged import attend, types  # noqa: F401
from test_gpu_paged_caps import capped_tolerance

pytestmark = pytest.mark.gpu

FORM = {"plain": "plain", "cap": "shaped", "both": "shaped", "far cap, slopes": "far cap"}


@pytest.fixture
def launched(ti, monkeypatch):
    """Names of what the calls launched."""
    got = []
    for fn in ("ti_paged_decode", "ti_paged_prefill"):
        def call(cache, args, stream, real=getattr(ti.lib(), fn)):
            got.append(ti.paged_kernel_name(cache._obj, args._obj))
            return real(cache, args, stream)
        monkeypatch.setattr(ti.lib(), fn, call)
    return got


def shape_of(shape, heads, rng):
    kw = {} if shape == "plain" else dict(cap=3e3 if "far" in shape else 6.0)
    if shape == "both" or "slopes" in shape:
        kw["slopes"] = 2.0 ** -rng.uniform(2, 8, heads)
    return kw


def check(ti, cache, rng, heads, new, fn="prefill", amp=2.0, **kw):
    """check_attention by a tolerance that a cap does not widen beyond its own error."""
    x = rng.standard_normal((sum(new), heads * cache.dim)) * amp
    bits = bits16(x, cache.dtype)
    x = from_bits(bits, cache.dtype)
    cache.upload()
    got = from_bits(attend(ti, cache, bits, heads, new, fn=fn, **kw), cache.dtype)
    kw = {k: v for k, v in kw.items() if k != "max_len"}
    ref, absv, mag, seen = attention(cache, x, new, heads, cache.dim ** -0.5, **kw)
    tol = capped_tolerance(cache, ref, absv, mag, seen, kw["cap"]) if "cap" in kw else attention_tolerance(cache, ref, absv, mag, seen)
    bad = ~(np.abs(got - ref) <= tol)
    at = np.argwhere(bad)[:1].ravel()
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first {at}: {got[tuple(at)]!r} for {ref[tuple(at)]!r}, may be {tol[tuple(at)]:.3g} off"


def label(types):  # noqa: F811
    return "int8" if types[1] == "i8" else "16 bits"


@pytest.mark.parametrize("shape", FORM)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_single_tokens(ti, types, dim, shape, launched, monkeypatch):  # noqa: F811
    """In one split, in some, and dealt; a window that begins inside a run, a row that sees nothing."""
    rng = np.random.RandomState(90)
    for wide, lens, window, name in ((0, [80, 1, 33], 60, "stream"), (0, [1500, 700, 30], 1400, "stream"), (140000, [7400, 30, 700], 6300, "deal")):
        monkeypatch.setattr(Cache, "wide", wide)
        check(ti, Cache(ti, rng, lens, 2, dim, 16, *types), rng, 6, [1] * 3, "decode", window=window, first=[3, 30, 0], **shape_of(shape, 6, rng))
        last = launched[-1]
        assert last.startswith(f"paged_{name}_kernel<{dim},{label(types)},{FORM[shape]}>") and (wide or last.endswith("splits 1") == (lens[0] < 100)), last


@pytest.mark.parametrize("shape", FORM)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_of_four_waves_or_pairs(ti, types, dim, shape, launched, monkeypatch):  # noqa: F811
    """Keys shared in LDS (heads of 256: by pairs of waves), in one split and in many, of which most are empty."""
    rng = np.random.RandomState(91)
    waves = 8 if dim == 256 else 4
    new = [7 * i % 38 for i in range(32)]   # (18 a sequence)
    lens = [n + int(x) for n, x in zip(new, rng.randint(0, 30, 32))]
    check(ti, Cache(ti, rng, lens, 8, dim, 16, *types), rng, 16, new, window=20, **shape_of(shape, 16, rng))
    assert launched[-1] == f"paged_block_kernel<{dim},{waves},{label(types)},{FORM[shape]}>, splits 1"
    monkeypatch.setattr(Cache, "wide", 20000)
    check(ti, Cache(ti, rng, [300, 90], 2, dim, 32, *types, holes=[(0, 3)]), rng, 4, [120, 50], first=[11 * (i % 7) for i in range(170)], **shape_of(shape, 4, rng))
    assert launched[-1].startswith(f"paged_block_kernel<{dim},{waves},{label(types)},{FORM[shape]}>, splits ") and not launched[-1].endswith("splits 1")


@pytest.mark.parametrize("shape", FORM)
def test_rows_of_eight_waves(ti, types, shape, launched, monkeypatch):  # noqa: F811
    """Heads of 128: one split (24 prompts of 49 rows) and many, by tables with room for long prompts."""
    rng = np.random.RandomState(92)
    monkeypatch.setattr(Cache, "wide", 2048)
    lens = [49 + 3 * i for i in range(24)]
    check(ti, Cache(ti, rng, lens, 8, 128, 16, *types), rng, 32, [49] * 24, **shape_of(shape, 32, rng))
    assert launched[-1] == f"paged_block_kernel<128,8,{label(types)},{FORM[shape]}>, splits 1"
    monkeypatch.setattr(Cache, "wide", 40000)
    check(ti, Cache(ti, rng, [230, 260], 4, 128, 64, *types, holes=[(1, 1)]), rng, 8, [200, 30], window=150, prefix=[220, 0], **shape_of(shape, 8, rng))
    assert launched[-1].startswith(f"paged_block_kernel<128,8,{label(types)},{FORM[shape]}>, splits ") and not launched[-1].endswith("splits 1")


@pytest.mark.parametrize("dim,waves,hint", [(64, 4, 1), (128, 4, 1), (128, 8, 0), (256, 8, 1)])
def test_long_runs_of_zero_values_of_many_rows(ti, dim, waves, hint, launched):
    """int8: 20160 tokens whose values are 0 (the least scale) before 64 that are not, summed by the kernel of many rows (in one split by the hint);
    their scores 8 octaves above the first tokens'.  A prefix shows every row all tokens, so all rows are alike."""
    rng = np.random.RandomState(93)
    n, rows, heads = 20224, 512, 8
    cache = Cache(ti, rng, [n], 1, dim, 256, "f16", "i8")
    cache.vs[:] = np.float32(TINY)
    cache.v[:] = 0
    cache.k[:] = 127
    cache.ks[:] = 1.0
    e = cache.table[0]
    cache.k[e[0], 0, :64] = 0
    last, at = (n - 64) // 256, (n - 64) % 256
    cache.v[e[last], 0, at: at + 64] = rng.randint(-127, 128, (64, dim))
    cache.vs[e[last], 0, at // 16: at // 16 + 4] = 0.01
    x = np.ones((rows, heads * dim))
    cache.upload()
    scale = 7.9 * np.log(2) / (127 * dim)
    got = from_bits(attend(ti, cache, bits16(x, "f16"), heads, [rows], scale=scale, max_len=hint, prefix=[n]), "f16")
    assert launched[-1].startswith(f"paged_block_kernel<{dim},{waves},int8,plain>") and launched[-1].endswith("splits 1") == (hint == 1), launched
    ref, absv, mag, seen = attention(cache, x[:1, :dim], [1], 1, scale)
    assert np.abs(ref).max() > 0 and seen[0][0] == n
    assert (np.abs(got.reshape(-1, dim) - ref) <= attention_tolerance(cache, ref, absv, mag, seen)).all()


def test_results_repeat(ti, types, launched, monkeypatch):  # noqa: F811
    """The same call gives the same bits, whatever a call in between left in caches."""
    rng = np.random.RandomState(94)
    for fn, wide, new, lens in (("decode", 0, [1] * 3, [900, 40, 300]), ("decode", 140000, [1] * 3, [900, 40, 300]), ("prefill", 0, [20, 3], [90, 300]),
                                ("prefill", 20000, [120, 50], [300, 90])):
        monkeypatch.setattr(Cache, "wide", wide)
        cache = Cache(ti, rng, lens, 2, 128, 32, *types)
        bits = bits16(rng.standard_normal((sum(new), 4 * 128)), types[0])
        cache.upload()
        first = attend(ti, cache, bits, 4, new, fn=fn)
        for _ in range(3):
            assert np.array_equal(attend(ti, cache, bits, 4, new, fn=fn), first)
    assert {n.split("_kernel")[0] for n in launched} == {"paged_stream", "paged_deal", "paged_block"}
