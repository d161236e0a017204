"""The paged cache on the CPU: places of blocks and tiles (paged.hpp), the bindings' structures, and what the calls refuse before
anything is launched."""
from __future__ import annotations

import ctypes as C
import os
import random
import subprocess

import pytest

import turboinfer_amd as T

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L(ti_host):
    return ti_host.lib()


def _cpp(tmp_path, body):
    (tmp_path / "t.cpp").write_text('#include <stdio.h>\n#include "paged.hpp"\nusing namespace ti;\nint main() {\n' + body + "}\n")
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-std=c++20", "-O1", "-I" + os.path.join(ROOT, "turboinfer_amd", "csrc", "kernels"), str(tmp_path / "t.cpp"), "-o", exe], check=True)
    return [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]


def test_blocks_lie_inside_the_cache(tmp_path):
    """Every block number of good and bad table entries and block numbers is -1 or inside the cache; good ones are all different."""
    got = _cpp(tmp_path, """
  const int bad[] = {-2147483647 - 1, -1, 7, 8, 2147483647};
  for (int lb = 0; lb < 5; ++lb) {
    const PagedShape s = {7, 3, lb, 5 << lb};
    for (int e = 0; e < 7; ++e)
      for (int h = 0; h < 3; ++h)
        for (int blk = 0; blk < 1 << lb; ++blk) printf("%d\\n", paged_block(s, e, h, blk));
    for (int e : bad) printf("%d\\n", paged_block(s, e, 2, 0) + 1);
    printf("%d\\n%d\\n", paged_block(s, 0, 0, 5 << lb) + 1, paged_block(s, 0, 0, -1) + 1);
  }
""")
    at = 0
    for lb in range(5):
        n = 21 << lb
        assert sorted(got[at:at + n]) == list(range(n))
        assert got[at + n:at + n + 7] == [0] * 7
        at += n + 7
    assert at == len(got)


@pytest.mark.parametrize("tile", [1, 16, 64, 256])
def test_tiles_of_ragged_rows(tile, tmp_path):
    """The numbers of a sequence's tiles lie in front of the next one's, and all below the number launched."""
    rng = random.Random(tile)
    for case in range(3):
        new = [rng.choice([0, 0, 1, 15, 16, 17, 255, 256, 257, rng.randrange(1000)]) for _ in range(40)]
        starts = [sum(new[:b]) for b in range(len(new) + 1)]
        got = _cpp(tmp_path, f"const int s[] = {{{', '.join(map(str, starts))}}};\n  for (int b = 0; b <= {len(new)}; ++b) "
                             f'printf("%ld %ld\\n", paged_tile0(s[b], b, {tile}), paged_touch0(s[b], b));\n'
                             f'  printf("%ld %ld\\n", paged_tiles(s[{len(new)}], {len(new)}, {tile}), paged_touches(s[{len(new)}], {len(new)}));\n')
        t0, c0 = got[0::2], got[1::2]
        for b, n in enumerate(new):
            assert t0[b] + -(-n // tile) <= t0[b + 1] <= t0[-1]
            for off in range(16):
                touched = (off + n - 1) // 16 - off // 16 + 1 if n else 0
                assert c0[b] + touched <= c0[b + 1] <= c0[-1]


def test_mirrors_of_the_structures(L):
    for i, s in enumerate((T.PagedCache, T.PagedAppendArgs, T.PagedAttnArgs)):
        assert L.ti_paged_struct_bytes(i) == C.sizeof(s)


def _cache(**kw):
    d = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, table=4096, len=4096, table_ld=4, pages=8, page=16, kv_heads=2, head_dim=64, seqs=3, dtype=T.PAGED_F16,
             kv_type=T.KV_SAME)
    return T.PagedCache(**(d | kw))


BAD_CACHES = [(dict(k=None), 1), (dict(v=None), 1), (dict(table=None), 1), (dict(len=None), 1), (dict(dtype=2), 1), (dict(kv_type=2), 1), (dict(kv_type=-1), 1),
              (dict(kv_type=T.KV_I8, k_scale=None), 1), (dict(kv_type=T.KV_I8, v_scale=None), 1), (dict(head_dim=96), 3), (dict(head_dim=0), 3), (dict(page=8), 3),
              (dict(page=48), 3), (dict(page=512), 3), (dict(page=0), 3), (dict(page=-16), 3), (dict(seqs=0), 1), (dict(kv_heads=0), 1), (dict(pages=0), 1),
              (dict(pages=2 ** 30, kv_heads=2), 1), (dict(table_ld=0), 1), (dict(table_ld=2 ** 28), 1), (dict(k=4104), 1), (dict(table=4098), 1)]


@pytest.mark.parametrize("change,code", BAD_CACHES, ids=[str(c[0]) for c in BAD_CACHES])
def test_refused_caches(L, change, code):
    c = _cache(**change)
    a = T.PagedAppendArgs(x=4096, q=4096, rows=3, heads=4, ldx=512, ldq=256, x_f32=1)
    t = T.PagedAttnArgs(q=4096, out=4096, rows=3, heads=4, ldq=256, ldo=256, scale=0.125)
    for rc in (L.ti_paged_append(c, a, None), L.ti_paged_read(c, None, 3, 4096, 128, 4096, 128, None), L.ti_paged_decode(c, t, None),
               L.ti_paged_prefill(c, t, None)):
        assert rc == code and b"ti_paged_" in L.ti_last_error()
    assert L.ti_paged_workspace_bytes(c, t) == 0
    assert L.ti_paged_append(None, a, None) == 1 and L.ti_paged_decode(None, t, None) == 1


def test_refused_appends(L):
    c = _cache()
    good = dict(x=4096, q=4096, rows=3, heads=4, ldx=512, ldq=256, x_f32=1, rope_cs=4096, rope_len=10, rot_dim=64, rope_kind=T.ROPE_PAIRS)
    for bad in (dict(x=None), dict(q=None), dict(rows=4), dict(rows=-1), dict(heads=-1), dict(ldx=504), dict(ldx=514), dict(ldq=248), dict(ldq=260), dict(x=4100),
                dict(q=4104), dict(rot_dim=8), dict(rot_dim=24), dict(rot_dim=80), dict(rope_len=0), dict(rope_kind=2), dict(rope_cs=4100),
                dict(row_start=4098), dict(x_f32=0, ldx=516)):
        assert L.ti_paged_append(c, T.PagedAppendArgs(**(good | bad)), None) == 1, bad
    assert L.ti_paged_append(c, None, None) == 1
    assert L.ti_paged_append(c, T.PagedAppendArgs(**(good | dict(rows=0, row_start=4096))), None) == 0   # nothing to do


def test_refused_reads(L):
    c = _cache()
    for args in ((None, 4, 4096, 128, 4096, 128), (None, 3, None, 128, 4096, 128), (None, 3, 4096, 120, 4096, 128), (None, 3, 4096, 128, 4096, 132),
                 (None, 3, 4104, 128, 4096, 128), (None, -1, 4096, 128, 4096, 128)):
        assert L.ti_paged_read(c, *args, None) == 1, args
    assert L.ti_paged_read(c, 4096, 0, 4096, 128, 4096, 128, None) == 0


def test_refused_attention(L):
    c = _cache()
    good = dict(q=4096, out=4096, rows=3, heads=4, ldq=256, ldo=256, scale=0.125)
    for bad in (dict(q=None), dict(out=None), dict(rows=4), dict(rows=-1), dict(heads=0), dict(heads=5), dict(ldq=248), dict(ldo=260), dict(q=4104), dict(out=4104),
                dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=2e30), dict(softcap=1e-30), dict(softcap=1e31), dict(rows=2 ** 23 + 1), dict(window=-1),
                dict(max_len=-1), dict(slopes=4098), dict(first=4098), dict(prefix=4098), dict(workspace=4104)):
        for fn in (L.ti_paged_decode, L.ti_paged_prefill):
            assert fn(c, T.PagedAttnArgs(**(good | bad)), None) == 1, bad
    assert L.ti_paged_decode(c, T.PagedAttnArgs(**(good | dict(row_start=4096))), None) == 1
    assert L.ti_paged_prefill(c, T.PagedAttnArgs(**(good | dict(row_start=4096, rows=0))), None) == 0
    # long keys of few rows need a workspace
    c = _cache(table_ld=4096)
    a = T.PagedAttnArgs(**good)
    need = L.ti_paged_workspace_bytes(c, a)
    assert need > 0
    assert L.ti_paged_decode(c, a, None) == 1 and b"workspace" in L.ti_last_error()
    a.workspace, a.workspace_bytes = 4096, 64
    assert L.ti_paged_decode(c, a, None) == 1 and b"workspace" in L.ti_last_error()


def test_workspace_of_any_length_serves(L):
    """ti_paged_workspace_bytes holds for every length that a call of the same arguments names (refused for its null rows, not for its workspace)."""
    rng = random.Random(5)
    for i in range(3000):
        kv_heads, G, dim = rng.choice([1, 2, 4, 8, 10, 32]), rng.choice([1, 2, 4, 5, 8, 20]), rng.choice([64, 128, 256])
        seqs = rng.choice([1, 2, 5, 12, 50, 300])
        c = _cache(kv_heads=kv_heads, head_dim=dim, seqs=seqs, table_ld=rng.choice([1, 16, 200, 3000]), pages=100, kv_type=rng.choice([T.KV_SAME, T.KV_I8]))
        rows = seqs if i % 3 == 0 else rng.randrange(1, 5000)
        a = T.PagedAttnArgs(rows=rows, heads=kv_heads * G, ldq=kv_heads * G * dim, ldo=kv_heads * G * dim, scale=1.0, row_start=None if i % 3 == 0 else 4096,
                            prefix=rng.choice([None, 4096]), window=rng.choice([0, 100, 3000]))
        n = L.ti_paged_workspace_bytes(c, a)
        a.workspace, a.workspace_bytes = 4096, n
        for max_len in (0, 1, 200, 300, 1000, 1536, 2047, 2048, 5000, 48000, 10 ** 6):
            a.max_len = max_len
            assert L.ti_paged_prefill(c, a, None) == 1 and b"null pointer" in L.ti_last_error(), (L.ti_last_error(), rows, seqs, kv_heads, G, dim, c.table_ld, max_len)
