"""Rows that ti_paged_append leaves: what their places held stays as it was."""
from __future__ import annotations

import numpy as np
import pytest

from paged import Cache
from test_gpu_paged import check_append, types  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x_f32", [True, False])
@pytest.mark.parametrize("rope_len", [16, 25, 32, 48])
def test_rotation_tables_that_end_inside_the_cache(ti, types, rope_len, x_f32):  # noqa: F811
    """Rows past the rotation table: blocks of them alone keep their bytes and scales, with older tokens in front or without; in a block
    that rotated rows reach too, theirs decide the scale.  All places hold tokens from before."""
    rng = np.random.RandomState(80)
    cache = Cache(ti, rng, [64] * 5, 2, 64, 16, *types)
    cache.lens = np.asarray([60, 40, 64, 26, 33], np.int32)   # from 0, 20, 48, 25 (the table's end, or past it), 32 on
    check_append(ti, cache, rng, [60, 20, 16, 1, 1], 2, x_f32, 64, rope_len=rope_len)
