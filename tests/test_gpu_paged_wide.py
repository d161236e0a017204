"""The paged cache's attention by tables that have room for much longer sequences: kernels and splits are chosen by the room, so that
short sequences meet the ways of long ones too -- single tokens' keys dealt over the workgroups, rows' keys shared and in many splits."""
from __future__ import annotations

import numpy as np
import pytest

from paged import HALF, Cache, from_bits, starts
from test_gpu_paged import (MARK, check_append, check_attention, test_decode, test_decode_long, test_decode_long_masks, test_decode_long_of_wide_groups,  # noqa: F401
                            test_decode_of_many_sequences, test_decode_queries_of_any_size, test_decode_scores_and_masks, test_decode_sharp_and_flat_rows,
                            test_extreme_bounds, test_holes, test_int8_blocks_that_are_no_numbers, test_long_runs_of_zero_values, test_pages_that_sequences_share,
                            test_prefill, test_prefill_behind_a_long_cache, test_prefill_groups, test_prefill_many_rows, test_prefill_scores_and_masks,
                            test_prompts_then_steps, test_captured_prompts, test_captured_steps, test_two_streams_at_once, test_values_near_the_largest,
                            test_values_of_many_sizes, test_values_that_are_no_numbers_in_shared_blocks, test_what_a_row_does_not_see_does_not_reach_it, types, upload)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def wide_tables(monkeypatch):
    monkeypatch.setattr(Cache, "wide", 140000)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_dealt_windows(ti, types, dim):
    """Windows and first keys in front of which runs begin; a row that sees nothing between two that do."""
    rng = np.random.RandomState(60)
    lens = [7400, 30, 6600, 900]
    check_attention(ti, Cache(ti, rng, lens, 1, dim, 64, *types, holes=[(0, 40)]), rng, 3, [1] * 4, "decode", amp=2.0, window=6300, first=[2000, 30, 0, 850], cap=20.0,
                    slopes=2.0 ** -rng.uniform(8, 12, 3))


@pytest.mark.parametrize("shaped", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_shared_keys_in_one_split(ti, types, dim, shaped, monkeypatch):
    """Many prompts of few rows, one workgroup a tile."""
    monkeypatch.setattr(Cache, "wide", 0)
    rng = np.random.RandomState(61)
    new = [7 * i % 38 for i in range(32)]   # (18 a sequence)
    lens = [n + int(x) for n, x in zip(new, rng.randint(0, 30, 32))]
    more = dict(cap=6.0, slopes=2.0 ** -rng.uniform(2, 8, 16), window=20) if shaped else {}
    check_attention(ti, Cache(ti, rng, lens, 8, dim, 16, *types), rng, 16, new, amp=2.0, **more)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_shared_keys_and_windows(ti, types, dim):
    """Windows and slopes of rows whose keys are shared, in two splits."""
    rng = np.random.RandomState(64)
    check_attention(ti, Cache(ti, rng, [700], 8, dim, 32, *types, holes=[(0, 9)]), rng, 16, [330], amp=2.0, window=300, slopes=2.0 ** -rng.uniform(2, 8, 16))


@pytest.mark.parametrize("seqs", [65, 66, 4225, 4300])
def test_rows_of_very_many_sequences(ti, seqs, monkeypatch):
    """Sequences of 0 to 2 rows, found in one, two and three steps; empty ones first, last and in long runs."""
    monkeypatch.setattr(Cache, "wide", 0)
    rng = np.random.RandomState(62)
    new = rng.randint(0, 3, seqs)
    new[[0, 63, 64, seqs - 1]] = 0
    new[seqs // 3: seqs // 2] = 0
    new = [int(x) for x in new]
    lens = [n + int(x) for n, x in zip(new, rng.randint(0, 15, seqs))]
    cache = Cache(ti, rng, [l - n for l, n in zip(lens, new)], 1, 64, 16, "f16", "i8", room=17)
    cache.lens = np.asarray(lens, np.int32)
    check_append(ti, cache, rng, new, 2, False, 32, True)
    check_attention(ti, Cache(ti, rng, lens, 1, 64, 16, "f16", "same", room=17), rng, 2, new)


@pytest.mark.parametrize("seqs", [57, 64, 90])
def test_read_of_narrow_rows(ti, types, seqs):
    """Rows of 16 threads' work, of many sequences."""
    rng = np.random.RandomState(63)
    new = [int(x) for x in rng.randint(0, 3, seqs)]
    lens = [n + int(x) for n, x in zip(new, rng.randint(0, 30, seqs))]
    cache = Cache(ti, rng, lens, 1, 64, 16, *types)
    ref, rows = cache.upload(), sum(new)
    k, v = (upload(ti, np.full((rows + 1, 64), MARK, np.uint16)) for _ in range(2))
    start = upload(ti, starts(new))
    ti.check(ti.lib().ti_paged_read(ref, start.ptr, rows, k.ptr, 64, v.ptr, 64, None))
    ti.sync()
    for buf, name in ((k, "k"), (v, "v")):
        got = buf.download(np.uint16, (rows + 1, 64))
        want = np.array([cache.values(name, b, p)[0] for b, n in enumerate(new) for p in range(lens[b] - n, lens[b])])
        assert (got[rows:] == MARK).all()
        assert (np.abs(from_bits(got[:rows], cache.dtype) - want) <= HALF[cache.dtype] * np.abs(want) * 1.01).all()
