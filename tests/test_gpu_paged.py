"""The paged key/value cache (ti_paged_append, ti_paged_read, ti_paged_decode, ti_paged_prefill) against 64-bit numpy (paged.py).

Places of the cache that hold no token are NaN (int8: under NaN scales), and so is everything outside its rows: none of it may reach
an output, and outputs behind the rows stay as they were."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from paged import HALF, TINY, Cache, attention, attention_tolerance, bits16, from_bits, rotate, starts

pytestmark = pytest.mark.gpu
MARK = 0x7BCD   # bits of rows that no call writes


def upload(ti, a):
    return ti.DeviceBuffer.from_array(np.ascontiguousarray(a))


def rows16(rng, rows, width, dtype, amp=1.0, pitch=None):
    """(values float64, bits [rows][pitch]) with NaN between the rows."""
    bits = np.full((rows, pitch or width), 0x7FFF, np.uint16)
    bits[:, :width] = bits16(rng.standard_normal((rows, width)) * amp, dtype)
    return from_bits(bits[:, :width], dtype), bits


def attend(ti, cache, q_bits, heads, new, fn=None, extra=3, scale=None, cap=0.0, slopes=None, first=None, prefix=None, window=0, max_len=0, stream=None):
    """The call's rows as values [rows][heads * dim]; checks the rows and columns that it has to leave."""
    L, w = ti.lib(), heads * cache.dim
    rows, ldq = q_bits.shape
    ldo = w + 8
    ref = C.byref(cache.c)
    up = lambda x, t: None if x is None else upload(ti, np.asarray(x, t))  # noqa: E731
    keep = dict(q=upload(ti, q_bits), out=upload(ti, np.full((rows + extra, ldo), MARK, np.uint16)), start=up(starts(new), np.int32),
                slopes=up(slopes, np.float32), first=up(first, np.int32), prefix=up(prefix, np.int32))
    p = lambda n: None if keep[n] is None else keep[n].ptr  # noqa: E731
    a = ti.PagedAttnArgs(q=p("q"), out=p("out"), row_start=None if fn == "decode" else p("start"), slopes=p("slopes"), first=p("first"), prefix=p("prefix"),
                         rows=rows, heads=heads, ldq=ldq, ldo=ldo, max_len=max_len, window=window, scale=scale or cache.dim ** -0.5, softcap=cap)
    n = L.ti_paged_workspace_bytes(ref, C.byref(a))
    ws = upload(ti, np.full(max(n, 16), 0xFF, np.uint8))   # (NaN)
    a.workspace, a.workspace_bytes = ws.ptr, n
    ti.check((L.ti_paged_decode if fn == "decode" else L.ti_paged_prefill)(ref, C.byref(a), stream))
    ti.sync()
    got = keep["out"].download(np.uint16, (rows + extra, ldo))
    assert (got[rows:] == MARK).all() and (got[:, w:] == MARK).all()
    return got[:rows, :w]


def check_attention(ti, cache, rng, heads, new, fn="prefill", amp=1.0, q=None, ref_cache=None, **kw):
    rows = sum(new)
    x, bits = rows16(rng, rows, heads * cache.dim, cache.dtype, amp, pitch=heads * cache.dim + 16) if q is None else q
    cache.upload()
    got_bits = attend(ti, cache, bits, heads, new, fn=fn, **kw)
    kw = {k: v for k, v in kw.items() if k in ("cap", "slopes", "first", "prefix", "window")}
    ref, absv, mag, seen = attention(ref_cache or cache, x, new, heads, cache.dim ** -0.5, **kw)
    gone = np.isnan(ref).all(1) & (seen[0] == 0)      # tokens outside the table
    assert (got_bits[gone] == MARK).all()
    got = from_bits(got_bits, cache.dtype)[~gone]
    ref, tol = ref[~gone], attention_tolerance(cache, ref, absv, mag, seen, kw.get("cap", 0.0))[~gone]
    assert np.isfinite(ref).all()
    bad = ~(np.abs(got - ref) <= tol)
    at = np.argwhere(bad)[:1].ravel()
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first {at}: {got[tuple(at)]!r} for {ref[tuple(at)]!r}, may be {tol[tuple(at)]:.3g} off"


TYPES = [("f16", "same"), ("bf16", "same"), ("f16", "i8"), ("bf16", "i8")]


@pytest.fixture(params=TYPES, ids=["-".join(t) for t in TYPES])
def types(request):
    return request.param


# ---------------------------------------------------------------- single tokens
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (6, 2), (20, 1)])
def test_decode(ti, types, dim, heads, kv_heads):
    rng = np.random.RandomState(dim + heads)
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 64, 200]
    check_attention(ti, Cache(ti, rng, lens, kv_heads, dim, 32, *types), rng, heads, [1] * len(lens), "decode")


@pytest.mark.parametrize("page", [16, 64, 128, 256])
@pytest.mark.parametrize("length", [129, 700, 2049])
def test_decode_long(ti, types, page, length):
    """Keys cut over workgroups; the hint of the length right, too small, missing."""
    rng = np.random.RandomState(page + length)
    cache = Cache(ti, rng, [length, 5, length // 2], 2, 64, page, *types, room=length + 3 * page)
    q = rows16(rng, 3, 4 * 64, types[0], 1.5)
    for hint in (length, 40, 0):
        check_attention(ti, cache, rng, 4, [1] * 3, "decode", q=q, max_len=hint)


@pytest.mark.parametrize("kw", [dict(cap=5.0), dict(window=50), dict(window=1), dict(cap=30.0, window=100), "slopes", "first", "all"], ids=str)
def test_decode_scores_and_masks(ti, types, kw):
    rng = np.random.RandomState(5)
    lens = [1, 40, 333, 160, 99]
    more = dict(slopes=2.0 ** -rng.uniform(1, 8, 8)) if kw in ("slopes", "all") else {}
    if kw in ("first", "all"):
        more |= dict(first=[0, 39, 100, 160, 1000])    # the third documents' rows, one key, none
    if kw == "all":
        more |= dict(cap=10.0, window=120, prefix=[0, 3, 500, 2, 50])
    check_attention(ti, Cache(ti, rng, lens, 2, 128, 16, *types), rng, 8, [1] * len(lens), "decode", amp=3.0, **(more or kw))


def test_decode_sharp_and_flat_rows(ti, types):
    """Scores up to about 100 and all equal."""
    rng = np.random.RandomState(6)
    cache = Cache(ti, rng, [500, 500], 2, 64, 64, *types)
    for amp in (20.0, 0.0):
        check_attention(ti, cache, rng, 4, [1, 1], "decode", amp=amp)


def test_decode_queries_of_any_size(ti, types):
    """Queries from subnormal numbers to the type's largest (int8 caches multiply them in fp16), with a scale that suits."""
    rng = np.random.RandomState(7)
    tiny, big = (1e-6, 3e4) if types[0] == "f16" else (1e-30, 1e30)
    cache = Cache(ti, rng, [100], 1, 64, 32, *types)
    for amp in (tiny, big):
        x, bits = rows16(rng, 1, 2 * 64, types[0], 1.0)
        bits = bits16(np.clip(x * amp, -6e4 if types[0] == "f16" else -1e38, 6e4 if types[0] == "f16" else 1e38), types[0])
        x = from_bits(bits, types[0])
        cache.upload()
        got = from_bits(attend(ti, cache, bits, 2, [1], fn="decode", scale=0.125 / amp), types[0])
        ref, absv, mag, seen = attention(cache, x, [1], 2, 0.125 / amp)
        assert (np.abs(got - ref) <= attention_tolerance(cache, ref, absv, mag, seen)).all(), amp


def test_values_of_many_sizes(ti):
    """int8: blocks whose value scales lie 2^30 apart; the small ones' tokens have most of the weight."""
    rng = np.random.RandomState(8)
    cache = Cache(ti, rng, [64], 1, 64, 16, "f16", "i8")
    for blk, s in enumerate((2e-9, 1.0, 2e-9, 2.0)):
        cache.vs[cache.table[0, blk], 0, 0] = s
    x, bits = rows16(rng, 1, 64, "f16")
    q = x.reshape(64)
    q32 = q / np.abs(q).max()
    for blk in range(4):   # keys along the query in blocks 0 and 2, against it in the others: scores about 40 apart
        k = np.rint(q32 * 127) * (1 if blk % 2 == 0 else -1)
        cache.k[cache.table[0, blk], 0] = k
        cache.ks[cache.table[0, blk], 0, 0] = 1.0
    s = float(np.abs(np.rint(q32 * 127) @ q))
    cache.upload()
    got = from_bits(attend(ti, cache, bits, 1, [1], fn="decode", scale=20.0 / s), "f16")
    ref, absv, mag, seen = attention(cache, x, [1], 1, 20.0 / s)
    assert (np.abs(got - ref) <= attention_tolerance(cache, ref, absv, mag, seen)).all()


# ---------------------------------------------------------------- rows of several tokens
RAGGED = [([1], [1]), ([5], [5]), ([17, 0, 3], [17, 9, 40]), ([1, 1, 33, 1, 64], [200, 7, 33, 90, 65]), ([130, 70], [130, 300])]


@pytest.mark.parametrize("new,lens", RAGGED, ids=[str(r[0]) for r in RAGGED])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prefill(ti, types, new, lens, dim):
    rng = np.random.RandomState(len(new) + dim)
    check_attention(ti, Cache(ti, rng, lens, 2, dim, 32, *types), rng, 6 if dim == 64 else 4, new)


@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 1), (17, 1), (40, 2)])
def test_prefill_groups(ti, types, heads, kv_heads):
    rng = np.random.RandomState(heads)
    check_attention(ti, Cache(ti, rng, [70, 33], kv_heads, 64, 16, *types), rng, heads, [35, 20])


MASKS = [dict(cap=4.0), dict(window=20), dict(window=1), "slopes", "first", "prefix", "all"]


@pytest.mark.parametrize("kw", MASKS, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prefill_scores_and_masks(ti, types, kw, dim):
    """Documents inside a sequence, prefixes, windows; rows that see nothing."""
    rng = np.random.RandomState(11)
    new, lens = [150, 1, 40], [150, 70, 200]
    more = {}
    if kw in ("slopes", "all"):
        more |= dict(slopes=2.0 ** -rng.uniform(1, 8, 4))
    if kw in ("first", "all"):
        pos = [p for n, l in zip(new, lens) for p in range(l - n, l)]
        more |= dict(first=[p // 37 * 37 if i % 11 else p + 1 + i % 2 * 500 for i, p in enumerate(pos)])
    if kw in ("prefix", "all"):
        more |= dict(prefix=[60, 1000, 0])
    if kw == "all":
        more |= dict(cap=8.0, window=90)
    check_attention(ti, Cache(ti, rng, lens, 2, dim, 64, *types), rng, 4, new, amp=3.0, **(more or kw))


def test_prefill_behind_a_long_cache(ti, types):
    rng = np.random.RandomState(12)
    cache = Cache(ti, rng, [1500, 900], 1, 64, 64, *types)
    q = rows16(rng, 37, 2 * 64, types[0], 1.5)
    for hint in (1500, 0, 10):
        check_attention(ti, cache, rng, 2, [30, 7], q=q, max_len=hint)


@pytest.mark.parametrize("dim", [64, 128])
def test_prefill_many_rows(ti, types, dim):
    """Rows and keys past several blocks of the kernel of many rows."""
    rng = np.random.RandomState(13)
    check_attention(ti, Cache(ti, rng, [700, 300], 1, dim, 32, *types), rng, 2, [600, 299])


@pytest.mark.parametrize("fn", ["decode", "prefill"])
@pytest.mark.parametrize("entry", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
def test_holes(ti, types, fn, entry):
    """Tokens in pages that the table does not have are not seen, wherever its entry points."""
    rng = np.random.RandomState(14)
    lens = [200, 40, 33]
    cache = Cache(ti, rng, lens, 2, 64, 16, *types, holes=[(0, 0), (0, 1), (0, 5), (0, 12), (1, 0), (1, 1), (1, 2), (2, 2)], bad_entry=entry)
    check_attention(ti, cache, rng, 4, [1] * 3 if fn == "decode" else [100, 5, 33], fn)


def test_lengths_past_the_table(ti, types):
    """Tokens past the table are not there; their rows are left."""
    rng = np.random.RandomState(15)
    for lens, new in (([70, 64, -5], [10, 64, 3]), ([2 ** 31 - 1, 66, -2 ** 31], [3, 4, 5]), ([2, 1, 0], [5, 1, 2]), ([65, 64, 0], [1, 1, 1])):
        full = Cache(ti, np.random.RandomState(16), [64, 64, 64], 1, 64, 16, *types)   # (every place holds a token)
        full.lens = np.asarray(lens, np.int32)
        check_attention(ti, full, rng, 2, new, "decode" if new == [1, 1, 1] else "prefill")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fn", ["decode", "prefill", "prefill many"])
@pytest.mark.parametrize("what", ["nan", "inf", "both"])
def test_what_a_row_does_not_see_does_not_reach_it(ti, dtype, fn, what):
    """NaN and infinities in keys and values of tokens behind a row, in front of its window and of its document; a row that sees an
    infinite value has it."""
    rng = np.random.RandomState(18)
    many = fn == "prefill many"
    lens, new = ([271], [1]) if fn == "decode" else ([300], [300 if many else 40])
    clean = Cache(ti, rng, lens, 2, 64, 16, dtype, "same", room=304)
    bad = Cache.__new__(Cache)
    bad.__dict__.update(clean.__dict__)
    bad.k, bad.v = clean.k.copy(), clean.v.copy()
    v = {"nan": np.nan, "inf": np.inf, "both": np.nan}[what]
    for j in (150, 271, 290):
        e = clean.table[0, j // 16]
        bad.k[e, 0, j % 16, 3] = v
        bad.v[e, 1, j % 16, 5] = -np.inf if what == "both" else v
    pos = list(range(lens[0] - new[0], lens[0]))
    first = [p // 30 * 30 for p in pos]
    heads = 4
    x, bits = rows16(rng, new[0], heads * 64, dtype)
    out = []
    for c in (clean, bad):
        c.upload()
        out.append(from_bits(attend(ti, c, bits, heads, new, fn="decode" if fn == "decode" else "prefill", first=first, window=25), dtype).reshape(-1, heads, 64))
    sees = np.array([[lo <= j <= p and j > p - 25 for j in (150, 271, 290)] for p, lo in zip(pos, first)])
    hit = sees.any(1)
    assert (~hit).any() and (hit.any() or fn == "decode")
    # a key that is no number spoils what sees it in kv-head 0 (an infinite one with scores of +inf, or has no weight with -inf), a value only its column in kv-head 1
    assert np.array_equal(out[0][~hit], out[1][~hit])
    keep = [d for d in range(64) if d != 5]
    assert np.isfinite(out[1][:, 2:, keep]).all()
    assert not np.isfinite(out[1][hit][:, 2:, 5]).any()
    if what == "both":
        assert (out[1][hit][:, 2:, 5] == -np.inf).all()


def test_int8_blocks_that_are_no_numbers(ti):
    """NaN scales reach the rows that see their tokens, and no others."""
    rng = np.random.RandomState(19)
    cache = Cache(ti, rng, [100, 100], 1, 64, 16, "bf16", "i8")
    cache.vs[cache.table[0, 2], 0, 0] = np.nan
    cache.ks[cache.table[1, 2], 0, 0] = np.nan
    for fn, new in (("decode", [1, 1]), ("prefill", [80, 80])):
        x, bits = rows16(rng, sum(new), 2 * 64, "bf16")
        cache.upload()
        got = from_bits(attend(ti, cache, bits, 2, new, fn=fn, window=30), "bf16")
        pos = [p for n in new for p in range(100 - n, 100)]
        hit = np.array([p >= 32 and p - 30 < 47 for p in pos])
        assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()


# ---------------------------------------------------------------- writing and reading
def append(ti, cache, x, new, heads, x_f32, rope=None, rot=0, halves=False, extra=2, use_start=True, stream=None):
    """The call's q rows as bits; x [rows][(heads + 2 kv_heads) dim] as the device holds it."""
    L, w = ti.lib(), heads * cache.dim
    rows = x.shape[0]
    keep = dict(x=upload(ti, x), q=upload(ti, np.full((rows + extra, w + 8), MARK, np.uint16)), start=upload(ti, starts(new)),
                rope=None if rope is None else upload(ti, rope.astype(np.float32)))
    a = ti.PagedAppendArgs(x=keep["x"].ptr, q=keep["q"].ptr if heads else None, row_start=keep["start"].ptr if use_start else None,
                           rope_cs=None if rope is None else keep["rope"].ptr, rows=rows, heads=heads, ldx=x.shape[1], ldq=w + 8, x_f32=int(x_f32),
                           rope_len=0 if rope is None else rope.shape[0], rot_dim=rot, rope_kind=ti.ROPE_HALVES if halves else ti.ROPE_PAIRS)
    ti.check(L.ti_paged_append(C.byref(cache.c), C.byref(a), stream))
    ti.sync()
    got = keep["q"].download(np.uint16, (rows + extra, w + 8))
    assert (got[rows:] == MARK).all() and (got[:, w:] == MARK).all()
    return got[:rows, :w]


def check_append(ti, cache, rng, new, heads, x_f32, rot=0, halves=False, amp=1.0, rope_len=None, use_start=True):
    """One append against the definition, the whole cache compared; cache's lens count the new tokens."""
    D, kvh, rows = cache.dim, cache.kvh, sum(new)
    width = (heads + 2 * kvh) * D
    x = rng.standard_normal((rows, width)) * amp
    x = x.astype(np.float32).astype(np.float64) if x_f32 else from_bits(bits16(x, cache.dtype), cache.dtype)
    pitch = width + 8
    raw = np.full((rows, pitch), np.nan, np.float32) if x_f32 else np.full((rows, pitch), 0x7FFF, np.uint16)
    raw[:, :width] = x if x_f32 else bits16(x, cache.dtype)
    n_pos = rope_len if rope_len is not None else int(max(cache.lens)) + 1
    ang = np.arange(n_pos)[:, None] * 10000.0 ** (-np.arange(0, max(rot, 2), 2) / max(rot, 2))
    rope = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32) if rot else None
    cache.upload()
    before = cache.download()
    q_bits = append(ti, cache, raw, new, heads, x_f32, rope, rot, halves, use_start=use_start)
    after = cache.download()
    # rotation: two products and a sum of fp32, 2^-22 of their magnitudes
    slack = lambda t, y: HALF[cache.dtype] * np.abs(y) * 1.01 + 2.0 ** -22 * amp * 8 + 2.0 ** -25  # noqa: E731
    turn = lambda y, p: rotate(y.reshape(-1, D), rope[p], rot, halves) if rot else y.reshape(-1, D)  # noqa: E731
    want = [after[0].copy(), after[1].copy()]
    touched = np.zeros((2,) + after[0].shape[:3], bool)
    blocks = {}
    m = 0
    room = cache.table.shape[1] * cache.page
    for b, n in enumerate(new):
        p0 = int(cache.lens[b]) - n
        for i in range(n):
            p = p0 + i
            if not 0 <= p < room or (rot and p >= n_pos):
                assert (q_bits[m] == MARK).all()
                m += 1
                continue
            q = turn(x[m, : heads * D], p).ravel()
            assert (np.abs(from_bits(q_bits[m], cache.dtype) - q) <= slack("q", q)).all()
            e = cache.table[b, p // cache.page]
            if 0 <= e < cache.pages:
                kv = (turn(x[m, heads * D:(heads + kvh) * D], p), x[m, (heads + kvh) * D:].reshape(kvh, D))
                for w in range(2):
                    touched[w, e, :, p % cache.page] = True
                    if cache.kv == "same":
                        got = after[w][e, :, p % cache.page]
                        assert (np.abs(got - kv[w]) <= slack("kv", kv[w])).all()
                    else:
                        blocks.setdefault((w, e, p % cache.page // 16), []).append((p % 16, kv[w], p0 > p - p % 16, p0 - (p - p % 16)))
            m += 1
    if cache.kv == "i8":
        for (w, e, blk), toks in blocks.items():
            for h in range(kvh):
                old_s, new_s = float(before[2 + w][e, h, blk]), float(after[2 + w][e, h, blk])
                most = max(max(np.abs(t[1][h]).max() for t in toks) / 127, TINY)
                has_old, n_old = toks[0][2], toks[0][3]
                want_s = max(most, old_s) if has_old else most
                assert abs(new_s - want_s) <= 2.0 ** -20 * want_s
                for at, v, _, _ in toks:   # half a step of the scale, the fp32 scale's and quotient's own errors
                    got = after[w][e, h, 16 * blk + at]
                    assert (np.abs(got) <= 127).all() and (np.abs(got * new_s - v[h]) <= 0.5 * new_s * (1 + 2.0 ** -12) + 2.0 ** -22 * 8 * amp * (rot > 0)).all()
                if has_old:
                    o = before[w][e, h, 16 * blk: 16 * blk + n_old]
                    got = after[w][e, h, 16 * blk: 16 * blk + n_old]
                    assert (np.abs(got - o * (old_s / new_s)) <= 0.5 + 2.0 ** -12).all()
                    if new_s == old_s:
                        assert np.array_equal(got, o)
                    touched[w, e, h, 16 * blk: 16 * blk + n_old] = True
    for w in range(2):   # nothing else moved
        same = (after[w] == before[w]) | (np.isnan(after[w]) & np.isnan(before[w]))
        assert same[~touched[w]].all()
    if cache.kv == "i8":
        for w in range(2):
            s0, s1 = before[2 + w], after[2 + w]
            for e in range(cache.pages):
                for blk in range(cache.page // 16):
                    if (w, e, blk) not in blocks:
                        assert np.array_equal(s0[e, :, blk], s1[e, :, blk], equal_nan=True)
    return x


APPENDS = [([1], [1]), ([1, 1, 1], [5, 17, 32]), ([3, 0, 20, 1], [3, 8, 41, 16]), ([100, 33], [140, 33])]


@pytest.mark.parametrize("new,lens", APPENDS, ids=[str(a[0]) for a in APPENDS])
@pytest.mark.parametrize("dim,rot,halves", [(64, 64, False), (64, 32, True), (128, 128, True), (128, 48, False), (256, 256, False), (256, 0, False)])
@pytest.mark.parametrize("x_f32", [True, False])
def test_append(ti, types, new, lens, dim, rot, halves, x_f32):
    rng = np.random.RandomState(dim + rot)
    cache = Cache(ti, rng, [l - n for l, n in zip(lens, new)], 2, dim, 32, *types, room=max(lens) + 20)
    cache.lens = np.asarray(lens, np.int32)
    check_append(ti, cache, rng, new, 4, x_f32, rot, halves)


def test_append_one_row_a_sequence(ti, types):
    rng = np.random.RandomState(21)
    lens = list(range(1, 40))
    cache = Cache(ti, rng, [l - 1 for l in lens], 3, 64, 16, *types, room=48)
    cache.lens = np.asarray(lens, np.int32)
    check_append(ti, cache, rng, [1] * len(lens), 6, True, 64, use_start=False)


def test_append_without_queries(ti, types):
    rng = np.random.RandomState(22)
    cache = Cache(ti, rng, [0, 20], 2, 64, 16, *types, room=64)
    cache.lens = np.asarray([30, 25], np.int32)
    check_append(ti, cache, rng, [30, 5], 0, False)


def test_append_into_holes_and_past_the_tables(ti, types):
    """Rows of holes are left out; rows past the pages' table or the rotation's are left, q among them."""
    rng = np.random.RandomState(23)
    cache = Cache(ti, rng, [0, 16, 60, 0], 1, 64, 16, *types, room=64, holes=[(0, 1), (1, 1)])
    cache.lens = np.asarray([40, 30, 70, 2], np.int32)
    check_append(ti, cache, rng, [40, 14, 10, 5], 2, True, 64, rope_len=64)


def test_append_grows_scales(ti):
    """A block's tokens one by one, each larger than those before: old tokens keep their values to half a step of every scale they
    were moved to."""
    rng = np.random.RandomState(24)
    cache = Cache(ti, rng, [0], 1, 64, 16, "f16", "i8", room=32)
    cache.upload()
    amps, x = 1.3 ** np.arange(20), None
    rows = np.zeros((20, 128), np.float32)
    for p in range(20):
        rows[p] = (rng.uniform(-1, 1, 128) * amps[p]).astype(np.float32)
        cache.set_lens([p + 1])
        append(ti, cache, rows[p:p + 1], [1], 0, True)
    k, v, ks, vs = cache.download()
    e = cache.table[0]
    for p in range(20):
        blk = p // 16
        for w, (c, s) in enumerate(((k, ks), (v, vs))):
            want = rows[p, 64 * w: 64 * w + 64]
            scales = [max(np.abs(rows[16 * blk: i + 1, 64 * w: 64 * w + 64]).max(), 0) / 127 for i in range(p, min(20, 16 * blk + 16))]
            err = 0.5 * sum(sorted(set(scales))) * 1.001
            assert (np.abs(c[e[blk], 0, p % 16] * s[e[blk], 0, 0] - want) <= err).all()


@pytest.mark.parametrize("value", [0.0, 1e-35, np.nan, np.inf, -np.inf])
def test_append_of_zeros_and_no_numbers(ti, value):
    """Zeros and what is below the least scale are held as zeros; a value that is no number makes its block NaN, and it stays so."""
    rng = np.random.RandomState(25)
    cache = Cache(ti, rng, [0], 2, 64, 16, "bf16", "i8", room=48)
    cache.upload()
    x = np.zeros((20, 256), np.float32)
    x[:, :] = 0.0 if value == value and abs(value) < 1 else rng.standard_normal(x.shape)
    x[3, 5] = value          # kv-head 0's k
    cache.set_lens([20])
    append(ti, cache, x, [20], 0, True)
    x2 = rng.standard_normal((5, 256)).astype(np.float32)
    cache.set_lens([25])
    append(ti, cache, x2, [5], 0, True)
    k, v, ks, vs = cache.download()
    e = cache.table[0]
    bad = not np.isfinite(value)
    assert np.isnan(ks[e[0], 0, 0]) == bad
    if not bad:
        assert ks[e[0], 0, 0] == np.float32(TINY) and (k[e[0], 0] == 0).all()
    assert np.isfinite(ks[e[0], 1, 0]) and np.isfinite(vs[e[0], :, 0]).all() and np.isfinite(ks[e[1], :, 0]).all()


@pytest.mark.parametrize("new,lens", APPENDS, ids=[str(a[0]) for a in APPENDS])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_read(ti, types, new, lens, dim):
    rng = np.random.RandomState(26)
    cache = Cache(ti, rng, lens, 3, dim, 32, *types, holes=[(0, 0)] if lens[0] > 100 else [])
    ref = cache.upload()
    rows, w = sum(new), 3 * dim
    out = [upload(ti, np.full((rows + 2, w + 8 * (i + 1)), MARK, np.uint16)) for i in range(2)]
    start = upload(ti, starts(new))
    ti.check(ti.lib().ti_paged_read(ref, start.ptr, rows, out[0].ptr, w + 8, out[1].ptr, w + 16, None))
    ti.sync()
    for i, name in enumerate("kv"):
        got = out[i].download(np.uint16, (rows + 2, w + 8 * (i + 1)))
        assert (got[rows:] == MARK).all() and (got[:, w:] == MARK).all()
        m = 0
        for b, n in enumerate(new):
            for p in range(lens[b] - n, lens[b]):
                want = cache.values(name, b, p)
                want = np.zeros(w) if want is None else want.ravel()
                have = from_bits(got[m, :w], cache.dtype)
                assert np.array_equal(have, want) if cache.kv == "same" else (np.abs(have - want) <= HALF[cache.dtype] * np.abs(want) * 1.01).all()
                m += 1


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("kv", ["same", "i8"])
def test_prompts_then_steps(ti, kv):
    """Two ragged prompts and 40 tokens each, as a server runs a layer: append and attention of the prompts' chunks, then append and
    decode token by token on a stream of its own, then the tokens read into a cache of the other kind, which attends alike."""
    rng = np.random.RandomState(30)
    heads, kvh, D, room = 4, 2, 64, 160
    cache = Cache(ti, rng, [0, 0], kvh, D, 16, "bf16", kv, room=room)
    cache.upload()
    w = (heads + 2 * kvh) * D
    ang = np.arange(room)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    rope = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    stream = C.c_void_p()
    ti.lib().ti_stream_create.argtypes = [C.POINTER(C.c_void_p)]
    ti.check(ti.lib().ti_stream_create(C.byref(stream)))
    lens = np.zeros(2, int)
    chunks = [[50, 17], [33, 40]] + [[1, 1]] * 40
    for i, new in enumerate(chunks):
        lens = lens + new
        rows = sum(new)
        x = rng.standard_normal((rows, w)).astype(np.float32)
        cache.set_lens(lens)
        q_bits = append(ti, cache, x, new, heads, True, rope, D, stream=stream)
        k, v, ks, vs = cache.download()
        cache.k, cache.v = k, v
        if kv == "i8":
            cache.ks, cache.vs = ks, vs
        if i < 2 or i % 8 == 0 or i == len(chunks) - 1:
            got = from_bits(attend(ti, cache, q_bits, heads, new, fn="decode" if new == [1, 1] else "prefill", stream=stream), "bf16")
            ref, absv, mag, seen = attention(cache, from_bits(q_bits, "bf16"), new, heads, D ** -0.5)
            assert (np.abs(got - ref) <= attention_tolerance(cache, ref, absv, mag, seen)).all(), i
    ti.check(ti.lib().ti_stream_destroy(stream))
    # all tokens to a cache of the other kind: rows k | v
    rows = int(lens.sum())
    kv_rows = upload(ti, np.zeros((rows, 2 * kvh * D), np.uint16))
    start = upload(ti, starts(lens))
    ti.check(ti.lib().ti_paged_read(C.byref(cache.c), start.ptr, rows, kv_rows.ptr, 2 * kvh * D, kv_rows.ptr + 2 * kvh * D, 2 * kvh * D, None))
    ti.sync()
    other = Cache(ti, rng, [0, 0], kvh, D, 32, "bf16", "i8" if kv == "same" else "same", room=room)
    other.upload()
    other.set_lens(lens)
    append(ti, other, kv_rows.download(np.uint16, (rows, 2 * kvh * D)), list(lens), 0, False)
    other.k, other.v, other.ks, other.vs = other.download()
    got = from_bits(attend(ti, other, q_bits, heads, [1, 1], fn="decode"), "bf16")
    ref, absv, mag, seen = attention(other, from_bits(q_bits, "bf16"), [1, 1], heads, D ** -0.5)
    assert (np.abs(got - ref) <= attention_tolerance(other, ref, absv, mag, seen)).all()


@pytest.mark.parametrize("kv", ["same", "i8"])
def test_captured_steps(ti, kv):
    """A step (append, decode) captured once and replayed as the sequences grow, eager work between; two graphs share a workspace."""
    import torch
    rng = np.random.RandomState(31)
    heads, kvh, D, room, B = 4, 2, 64, 1024, 3
    cache = Cache(ti, rng, [500, 3, 77], kvh, D, 16, "f16", kv, room=room)
    cache.upload()
    L, w = ti.lib(), (heads + 2 * kvh) * D
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    x, q, out = dev(np.zeros((B, w), np.float32)), dev(np.zeros((B, heads * D), np.int16)), dev(np.zeros((B, heads * D), np.int16))
    lens = dev(np.array([500, 3, 77], np.int32))
    cache.c.len = lens.data_ptr()
    a = ti.PagedAppendArgs(x=x.data_ptr(), q=q.data_ptr(), rows=B, heads=heads, ldx=w, ldq=heads * D, x_f32=1)
    t = ti.PagedAttnArgs(q=q.data_ptr(), out=out.data_ptr(), rows=B, heads=heads, ldq=heads * D, ldo=heads * D, max_len=600, scale=D ** -0.5)
    n = L.ti_paged_workspace_bytes(C.byref(cache.c), C.byref(t))
    ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    t.workspace, t.workspace_bytes = ws.data_ptr(), n
    assert n > 0

    def step():
        s = torch.cuda.current_stream().cuda_stream
        ti.check(L.ti_paged_append(C.byref(cache.c), C.byref(a), s))
        ti.check(L.ti_paged_decode(C.byref(cache.c), C.byref(t), s))

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i in range(6):
        lens += 1 + i
        x.copy_(dev(rng.standard_normal((B, w)).astype(np.float32)))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        replayed = out.clone(), cache.download()
        out.zero_()
        step()   # the same tokens again, eagerly
        torch.cuda.synchronize()
        assert torch.equal(out, replayed[0]) and (out != 0).any()
        assert all(y is z or np.array_equal(y, z, equal_nan=True) for y, z in zip(cache.download(), replayed[1]))


def test_no_rows(ti, types):
    """Sequences without rows, and a batch without any, change nothing."""
    rng = np.random.RandomState(32)
    cache = Cache(ti, rng, [20, 0, 5], 1, 64, 16, *types)
    cache.upload()
    before = cache.download()
    x = np.zeros((4, 3 * 64), np.float32)
    assert (append(ti, cache, x, [0, 0, 0], 1, True) == MARK).all()     # 4 rows behind the last sequence
    q = np.zeros((4, 64), np.uint16)
    assert (attend(ti, cache, q, 1, [0, 0, 0]) == MARK).all()
    assert all(y is z or np.array_equal(y, z, equal_nan=True) for y, z in zip(cache.download(), before))


def test_offsets_past_32_bits(ti):
    """Pages behind the first 4 GiB of a cache's keys and values."""
    import torch
    kvh, D, page = 8, 128, 256
    pages = 2 ** 32 // (kvh * D * page * 2) + 3
    rng = np.random.RandomState(33)
    L = ti.lib()
    k, v = (torch.full((pages, kvh, page, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    small = Cache(ti, rng, [300], kvh, D, page, "f16", "same", spare=0)
    table = np.array([[pages - 1, pages - 2]], np.int32)
    for c, e in enumerate(table[0]):
        for big, src in ((k, small.k), (v, small.v)):
            big[int(e)] = torch.from_numpy(src[small.table[0, c]]).half().cuda()
    small.upload()
    tb = upload(ti, table)
    far = ti.PagedCache()
    C.memmove(C.byref(far), C.byref(small.c), C.sizeof(far))
    far.k, far.v, far.table, far.pages = k.data_ptr(), v.data_ptr(), tb.ptr, pages
    x, bits = rows16(rng, 40, 8 * D, "f16")
    outs, ones = [], upload(ti, np.ones((1, 16 * D), np.float32))
    for c in (small.c, far):
        small.c = c
        outs.append([attend(ti, small, bits[:1], 8, [1], fn="decode"), attend(ti, small, bits, 8, [40])])
        ti.check(L.ti_paged_append(C.byref(c), C.byref(ti.PagedAppendArgs(x=ones.ptr, rows=1, heads=0, ldx=16 * D, x_f32=1)), None))
        ti.sync()
    assert all(np.array_equal(a, b) for a, b in zip(*outs))
    assert (k[pages - 2, :, 299 - 256] == 1).all() and torch.isnan(k[pages - 2, :, 300 - 256:]).all()


# ---------------------------------------------------------------- sizes of the other kernels
def test_decode_of_many_sequences(ti, types):
    """More than two waves of sequences, empty ones among them, keys dealt over the workgroups."""
    rng = np.random.RandomState(40)
    lens = [int(x) for x in rng.randint(0, 500, 150)]
    lens[0] = lens[64] = lens[149] = 0
    lens[100] = 1300
    check_attention(ti, Cache(ti, rng, lens, 1, 64, 64, *types), rng, 2, [1] * 150, "decode")


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_long_of_wide_groups(ti, types, dim):
    rng = np.random.RandomState(41)
    check_attention(ti, Cache(ti, rng, [900, 10, 300], 2, dim, 16, *types), rng, 34, [1] * 3, "decode")


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_long_masks(ti, types, dim):
    """Windows and first keys in front of which runs begin; a row that sees nothing between two that do."""
    rng = np.random.RandomState(42)
    lens = [1500, 700, 30, 600]
    check_attention(ti, Cache(ti, rng, lens, 2, dim, 32, *types, holes=[(0, 40)]), rng, 4, [1] * 4, "decode", amp=2.0, window=500, first=[5, 650, 30, 0], cap=20.0,
                    slopes=2.0 ** -rng.uniform(2, 8, 4))


@pytest.mark.parametrize("shaped", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prefill_of_wide_workgroups(ti, types, dim, shaped):
    """Eight waves, keys in 32 splits of which most are empty."""
    rng = np.random.RandomState(43)
    cache = Cache(ti, rng, [330], 8, dim, 16, *types, room=2064)
    more = dict(cap=6.0, slopes=2.0 ** -rng.uniform(2, 8, 8), window=150) if shaped else {}
    check_attention(ti, cache, rng, 8, [256], amp=2.0, max_len=8192, **more)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("hint", [0, 8192])
def test_values_that_are_no_numbers_in_shared_blocks(ti, dtype, dim, hint):
    """An infinite and a NaN value reach the rows that see them, in their dimensions."""
    rng = np.random.RandomState(44)
    n = 256
    cache = Cache(ti, rng, [n + 30], 8, dim, 32, dtype, "same", room=2080)
    x, bits = rows16(rng, n, 8 * dim, dtype)
    cache.upload()
    clean = from_bits(attend(ti, cache, bits, 8, [n], max_len=hint), dtype).reshape(n, 8, dim)
    for j, d, v in ((100, 7, np.inf), (200, dim - 3, np.nan), (220, 70, -np.inf)):
        cache.v[cache.table[0, j // 32], 3, j % 32, d] = v
    cache.upload()
    got = from_bits(attend(ti, cache, bits, 8, [n], max_len=hint), dtype).reshape(n, 8, dim)
    pos = np.arange(30, n + 30)
    same = np.ones(got.shape, bool)
    for j, d in ((100, 7), (200, dim - 3), (220, 70)):
        same[pos >= j, 3, d] = False
    assert np.array_equal(got[same], clean[same])
    assert (got[pos >= 100, 3, 7] == np.inf).all() and np.isnan(got[pos >= 200, 3, dim - 3]).all() and (got[pos >= 220, 3, 70] == -np.inf).all()


def test_append_and_read_of_many_rows(ti, types):
    rng = np.random.RandomState(45)
    new, lens = [700, 0, 433], [705, 3, 440]
    cache = Cache(ti, rng, [l - n for l, n in zip(lens, new)], 2, 64, 128, *types, room=720)
    cache.lens = np.asarray(lens, np.int32)
    check_append(ti, cache, rng, new, 4, True, 64)


def test_append_of_many_sequences(ti, types):
    rng = np.random.RandomState(46)
    new = [int(x) for x in rng.randint(0, 4, 150)]
    lens = [n + int(x) for n, x in zip(new, rng.randint(0, 40, 150))]
    cache = Cache(ti, rng, [l - n for l, n in zip(lens, new)], 1, 64, 16, *types, room=48)
    cache.lens = np.asarray(lens, np.int32)
    check_append(ti, cache, rng, new, 2, False, 32, True)


def test_pages_that_sequences_share(ti, types):
    """A common prefix in the same pages, read by three sequences."""
    rng = np.random.RandomState(47)
    cache = Cache(ti, rng, [400, 300, 270], 2, 64, 64, *types)
    cache.table[1:, :4] = cache.table[0, :4]
    check_attention(ti, cache, rng, 4, [1] * 3, "decode")
    check_attention(ti, cache, rng, 4, [100, 20, 14])


@pytest.mark.parametrize("fn", ["decode", "prefill"])
def test_extreme_bounds(ti, types, fn):
    """First keys, prefixes and windows at the ends of their type."""
    rng = np.random.RandomState(48)
    lo, hi = -2 ** 31, 2 ** 31 - 1
    new = [1] * 4 if fn == "decode" else [40, 1, 30, 9]
    cache = Cache(ti, rng, [50, 60, 30, 9], 1, 64, 16, *types)
    rows = sum(new)
    check_attention(ti, cache, rng, 2, new, fn, first=[(lo, hi, 0)[i % 3] for i in range(rows)], prefix=[lo, hi, 0, -1], window=hi)
    check_attention(ti, cache, rng, 2, new, fn, prefix=[hi, lo, 1, 2])


def test_two_streams_at_once(ti, types):
    """Calls on two streams, each with its own workspace, as one after the other."""
    import torch
    rng = np.random.RandomState(49)
    L, heads, D = ti.lib(), 8, 64
    caches = [Cache(ti, rng, [n, 700], 2, D, 32, *types, room=1024) for n in (1000, 900)]
    jobs = []
    for cache in caches:
        ref = cache.upload()
        x, bits = rows16(rng, 62, heads * D, types[0])
        q = upload(ti, bits)
        start = upload(ti, starts([60, 2]))
        for fn, rows in (("decode", 2), ("prefill", 62)):
            out = torch.zeros(rows, heads * D, dtype=torch.int16, device="cuda")
            a = ti.PagedAttnArgs(q=q.ptr, out=out.data_ptr(), row_start=start.ptr if fn == "prefill" else None, rows=rows, heads=heads, ldq=heads * D, ldo=heads * D, scale=D ** -0.5)
            n = L.ti_paged_workspace_bytes(ref, C.byref(a))
            assert n > 0
            ws = torch.empty(n, dtype=torch.uint8, device="cuda")
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
            jobs.append((cache, a, out, ws, q, start, L.ti_paged_decode if fn == "decode" else L.ti_paged_prefill))
    torch.cuda.synchronize()
    alone = []
    for cache, a, out, _, _, _, fn in jobs:
        ti.check(fn(C.byref(cache.c), C.byref(a), None))
        ti.sync()
        alone.append(out.clone())
        out.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for i, (cache, a, *_, fn) in enumerate(jobs):
            ti.check(fn(C.byref(cache.c), C.byref(a), streams[i // 2].cuda_stream))
    torch.cuda.synchronize()
    for (_, _, out, *_), want in zip(jobs, alone):
        assert torch.equal(out, want) and (out != 0).any()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_captured_prompts(ti, types, dim):
    """Append and prompt attention of a chunk captured once and replayed for the chunks that follow, with eager calls between."""
    import torch
    rng = np.random.RandomState(50)
    heads, kvh, B, n = 8, 2, 2, 70
    cache = Cache(ti, rng, [0, 0], kvh, dim, 32, *types, room=512)
    cache.upload()
    L, w = ti.lib(), (heads + 2 * kvh) * dim
    x = torch.zeros(B * n, w, device="cuda")
    q, out = (torch.zeros(B * n, heads * dim, dtype=torch.int16, device="cuda") for _ in range(2))
    lens, start = torch.tensor([n, n], dtype=torch.int32, device="cuda"), torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
    cache.c.len = lens.data_ptr()
    a = ti.PagedAppendArgs(x=x.data_ptr(), q=q.data_ptr(), row_start=start.data_ptr(), rows=B * n, heads=heads, ldx=w, ldq=heads * dim, x_f32=1)
    t = ti.PagedAttnArgs(q=q.data_ptr(), out=out.data_ptr(), row_start=start.data_ptr(), rows=B * n, heads=heads, ldq=heads * dim, ldo=heads * dim, scale=dim ** -0.5)
    size = L.ti_paged_workspace_bytes(C.byref(cache.c), C.byref(t))
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    t.workspace, t.workspace_bytes = ws.data_ptr(), size

    def step():
        s = torch.cuda.current_stream().cuda_stream
        ti.check(L.ti_paged_append(C.byref(cache.c), C.byref(a), s))
        ti.check(L.ti_paged_prefill(C.byref(cache.c), C.byref(t), s))

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):   # (the first call of its kind may be a captured one)
        step()
    for i in range(5):
        x.copy_(torch.from_numpy(rng.standard_normal((B * n, w)).astype(np.float32)))
        g.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed) and (out != 0).any()
        lens += torch.tensor([n, n - 3], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kv", ["same", "i8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("fn", ["decode", "prefill"])
def test_values_near_the_largest(ti, kv, dim, fn):
    """Values up to 2e38: sums of weights times them stay inside fp32 where the result does."""
    rng = np.random.RandomState(51)
    new = [1] if fn == "decode" else [90]
    cache = Cache(ti, rng, [700], 1, dim, 32, "bf16", kv)
    if kv == "same":
        cache.v = from_bits(bits16(np.where(np.isnan(cache.v), np.nan, np.sign(cache.v) * 2e38), "bf16"), "bf16")
    else:
        cache.vs = np.where(np.isnan(cache.vs), np.nan, 1.5e36).astype(np.float32)
    check_attention(ti, cache, rng, 1, new, fn, amp=0.3)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_runs_of_zero_values(ti, dim):
    """int8: 20160 tokens whose values are 0 (the least scale) before some that are not, in one workgroup's sum; their scores 8 octaves above the first ones'."""
    rng = np.random.RandomState(52)
    n, rows = 20224, 40
    cache = Cache(ti, rng, [n], 1, dim, 256, "f16", "i8")
    cache.vs[:] = np.float32(TINY)
    cache.v[:] = 0
    cache.k[:] = 127
    cache.ks[:] = 1.0
    e = cache.table[0]
    cache.k[e[0], 0, :64] = 0
    last = (n - 64) // 256
    cache.v[e[last], 0, (n - 64) % 256: (n - 64) % 256 + 64] = rng.randint(-127, 128, (64, dim))
    cache.vs[e[last], 0, (n - 64) % 256 // 16: (n - 64) % 256 // 16 + 4] = 0.01
    x = np.full((rows, dim), 1.0)
    bits = bits16(x, "f16")
    cache.upload()
    scale = 7.9 * np.log(2) / (127 * dim)
    got = from_bits(attend(ti, cache, bits, 1, [rows], scale=scale, max_len=1), "f16")
    ref, absv, mag, seen = attention(cache, x, [rows], 1, scale)
    assert np.abs(ref).max() > 0
    assert (np.abs(got - ref) <= attention_tolerance(cache, ref, absv, mag, seen)).all()
