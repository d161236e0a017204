"""What the paged cache's attention launches for a call's sizes (host only: refused for the workspace, nothing runs)."""
from __future__ import annotations

import ctypes as C
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


def name(L, cache, args):
    buf = C.create_string_buffer(96)
    assert L.ti_paged_kernel_name(cache, args, buf, 96) == 0
    return buf.value.decode()


@pytest.mark.parametrize("kv,label", [(T.KV_SAME, "16 bits"), (T.KV_I8, "int8")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_kernel_names(L, dim, kv, label):
    def call(rows=1, heads=8, kv_heads=8, seqs=1, room=2048, ragged=True, **kw):
        cache = T.PagedCache(k=4096, v=4096, k_scale=4096, v_scale=4096, table=4096, len=4096, table_ld=room // 16, pages=8, page=16, kv_heads=kv_heads, head_dim=dim,
                             seqs=seqs, dtype=T.PAGED_F16, kv_type=kv)
        return name(L, cache, T.PagedAttnArgs(rows=rows, heads=heads, scale=1.0, row_start=4096 if ragged else None, **kw))

    assert call(ragged=False, room=256, max_len=100) == f"paged_stream_kernel<{dim},{label},plain>, splits 1"
    assert call(ragged=False, room=200000).startswith(f"paged_deal_kernel<{dim},{label},plain>, runs ")
    assert call(ragged=False, room=200000, softcap=1e4).startswith(f"paged_deal_kernel<{dim},{label},far cap>, runs ")
    assert call(rows=8).startswith(f"paged_stream_kernel<{dim},{label},plain>, splits ")
    for shape, kw in (("plain", {}), ("shaped", dict(softcap=30.0)), ("shaped", dict(slopes=4096)), ("far cap", dict(softcap=1e-3))):
        assert call(rows=4000, heads=32, room=4000, **kw) == f"paged_block_kernel<{dim},{4 if dim == 64 else 8},{label},{shape}>, splits 1"
    assert call(rows=500, heads=16, room=512) in (f"paged_block_kernel<{dim},{8 if dim == 256 else 4},{label},plain>, splits {n}" for n in (1, 2, 3, 4))


def test_kernel_names_are_refused(L):
    cache, args = T.PagedCache(), T.PagedAttnArgs()
    buf = C.create_string_buffer(8)
    assert L.ti_paged_kernel_name(cache, args, buf, 8) == 1 and L.ti_paged_kernel_name(cache, args, None, 8) == 1
    assert L.ti_paged_kernel_name(cache, args, buf, 0) == 1 and L.ti_paged_kernel_name(None, args, buf, 8) == 1
