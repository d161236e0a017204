"""What the paged cache's attention launches for a call's sizes (host only: refused for the workspace, nothing runs)."""
from __future__ import annotations

import re

import pytest

import turboinfer_amd as T


@pytest.fixture(scope="module")
def L(ti_host):
    return ti_host.lib()


def needed(L, cache, args):
    """Bytes of workspace that the call itself asks for."""
    args.workspace, args.workspace_bytes = None, 0
    assert L.ti_paged_decode(cache, args, None) == 1
    m = re.search(rb"(\d+) needed", L.ti_last_error())
    return int(m.group(1)) if m else 0


@pytest.mark.parametrize("room,dealt", [(2 ** 31 - 16, False), (2 ** 31 - 32, True), (2 ** 20, True)])
def test_steps_of_dealt_sequences_fit_32_bits(L, room, dealt):
    """64 sequences at the end of the largest tables are 2^32 steps of 32 keys, which the dealt keys' 32-bit sums do not hold: equal splits."""
    heads, dim, seqs = 4, 64, 66
    cache = T.PagedCache(k=4096, v=4096, table=4096, len=4096, table_ld=room // 16, pages=8, page=16, kv_heads=1, head_dim=dim, seqs=seqs, dtype=T.PAGED_F16,
                         kv_type=T.KV_SAME)
    args = T.PagedAttnArgs(q=4096, out=4096, rows=seqs, heads=heads, ldq=heads * dim, ldo=heads * dim, scale=1.0)
    parts = needed(L, cache, args) // ((dim + 2) * 4)
    assert parts % (seqs * heads) != 0 if dealt else parts % (seqs * heads) == 0   # parts a head: 256 + 66 runs, or splits of every row
    most = room - 1   # the last token: the sum of 64 sequences' steps
    assert not dealt or 64 * (most // 32 + 1) < 2 ** 32
