"""A paged key/value cache in numpy, and the operators on it in 64 bits (oracle of tests/test_gpu_paged.py)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

BLOCK, TINY = 16, 2.0 ** -100
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}


def round16(x, dtype):
    """x as values of the 16-bit type, in float64."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float64)).to(TORCH[dtype]).double().numpy()


def bits16(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype]).view(torch.int16).numpy().view(np.uint16)


def from_bits(u, dtype):
    return torch.from_numpy(u.view(np.int16).copy()).view(TORCH[dtype]).double().numpy()


class Cache:
    """lens: tokens of every sequence; room: tokens that its table has places for.  Places that hold no token are `garbage`
    (16-bit: NaN; int8: any values under NaN scales).  holes: {(sequence, table column)}."""

    wide = 0   # tokens that tables have columns for: those behind the sequence's own name no page

    def __init__(self, ti, rng, lens, kv_heads, dim, page, dtype="f16", kv="same", room=None, holes=(), spare=2, amp=1.0, bad_entry=-1):
        self.ti, self.dtype, self.kv, self.page, self.kvh, self.dim = ti, dtype, kv, page, kv_heads, dim
        self.lens = np.asarray(lens, np.int32)
        cols = max(1, -(-int(room if room is not None else max(lens)) // page))
        n = len(lens)
        pages = n * cols + spare
        self.table = rng.permutation(pages)[: n * cols].reshape(n, cols).astype(np.int32)
        for at in holes:
            self.table[at] = bad_entry
        self.pages = pages
        nb = page // BLOCK
        if kv == "same":
            self.k, self.v = (np.full((pages, kv_heads, page, dim), np.nan) for _ in range(2))
            self.ks = self.vs = None
        else:
            self.k, self.v = (rng.randint(-127, 128, (pages, kv_heads, page, dim)).astype(np.float64) for _ in range(2))
            self.ks, self.vs = (np.full((pages, kv_heads, nb), np.nan, np.float32) for _ in range(2))
        for b, l in enumerate(lens):
            for t in range(min(int(l), cols * page)):
                e = self.table[b, t // page]
                if not 0 <= e < pages:
                    continue
                if kv == "same":
                    for x in (self.k, self.v):
                        x[e, :, t % page] = round16(rng.standard_normal((kv_heads, dim)) * amp, dtype)
                elif t % BLOCK == 0:
                    for x in (self.ks, self.vs):
                        x[e, :, t % page // BLOCK] = amp * rng.uniform(0.3, 3.0, kv_heads) / 50

    def values(self, name, b, t):
        """[kv_heads][dim] of token t of sequence b; None in a hole or past the table."""
        if t // self.page >= self.table.shape[1]:
            return None
        e = self.table[b, t // self.page]
        if not 0 <= e < self.pages:
            return None
        x = getattr(self, name)[e, :, t % self.page]
        return x if self.kv == "same" else x * getattr(self, name + "s")[e, :, t % self.page // BLOCK].astype(np.float64)[:, None]

    def upload(self):
        T = self.ti
        dev = T.DeviceBuffer.from_array
        raw = (lambda x: bits16(x, self.dtype)) if self.kv == "same" else (lambda x: x.astype(np.int8))
        more = max(0, -(-self.wide // self.page) - self.table.shape[1])
        table = np.ascontiguousarray(np.pad(self.table, ((0, 0), (0, more)), constant_values=-1))
        self.buf = {"k": dev(raw(self.k)), "v": dev(raw(self.v)), "table": dev(table), "len": dev(self.lens)}
        if self.kv == "i8":
            self.buf |= {"ks": dev(self.ks), "vs": dev(self.vs)}
        p = lambda n: self.buf[n].ptr if n in self.buf else None  # noqa: E731
        self.c = T.PagedCache(k=p("k"), v=p("v"), k_scale=p("ks"), v_scale=p("vs"), table=p("table"), len=p("len"), table_ld=table.shape[1],
                              pages=self.pages, page=self.page, kv_heads=self.kvh, head_dim=self.dim, seqs=len(self.lens),
                              dtype=T.PAGED_F16 if self.dtype == "f16" else T.PAGED_BF16, kv_type=T.KV_SAME if self.kv == "same" else T.KV_I8)
        return C.byref(self.c)

    def set_lens(self, lens):
        self.lens = np.asarray(lens, np.int32)
        self.buf["len"].upload(self.lens)

    def download(self):
        """The device's cache as values: (k, v) [pages][kv_heads][page][dim], and its scales."""
        shape = (self.pages, self.kvh, self.page, self.dim)
        if self.kv == "same":
            return tuple(from_bits(self.buf[n].download(np.uint16, shape), self.dtype) for n in "kv") + (None, None)
        s = (self.pages, self.kvh, self.page // BLOCK)
        return tuple(self.buf[n].download(np.int8, shape).astype(np.float64) for n in "kv") + tuple(self.buf[n].download(np.float32, s) for n in ("ks", "vs"))


def starts(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def rotate(x, cs, rot, halves):
    """x [heads][dim] float64 by cs [rot / 2][2]."""
    y = x.copy()
    a, b = (x[:, : rot // 2], x[:, rot // 2: rot]) if halves else (x[:, 0:rot:2], x[:, 1:rot:2])
    c, s = cs[:, 0].astype(np.float64), cs[:, 1].astype(np.float64)
    lo, hi = a * c - b * s, a * s + b * c
    if halves:
        y[:, : rot // 2], y[:, rot // 2: rot] = lo, hi
    else:
        y[:, 0:rot:2], y[:, 1:rot:2] = lo, hi
    return y


def attention(cache, q, new, heads, scale, cap=0.0, slopes=None, first=None, prefix=None, window=0):
    """(out, sum of w |v|, most |score| terms, (keys, largest |v| that its type could hold)) of rows q [rows][heads * dim] float64; NaN rows: not written."""
    G, D = heads // cache.kvh, cache.dim
    rows = q.shape[0]
    out, absv, mag = (np.full((rows, heads, D), np.nan) for _ in range(3))
    seen_n, top = np.zeros(rows, int), np.zeros((rows, heads, 1))
    room, m = cache.table.shape[1] * cache.page, 0
    for b, n in enumerate(new):
        L = min(max(int(cache.lens[b]), 0), room)
        have = [j for j in range(L) if cache.values("k", b, j) is not None]
        K = np.array([cache.values("k", b, j) for j in have]).reshape(len(have), cache.kvh, D)
        V = np.array([cache.values("v", b, j) for j in have]).reshape(len(have), cache.kvh, D)
        have = np.array(have, int)
        for i in range(n):
            p = int(cache.lens[b]) - n + i
            if not 0 <= p < room:
                m += 1
                continue
            see = have <= p
            if prefix is not None:
                see |= have < prefix[b]
            if first is not None:
                see &= have >= first[m]
            if window:
                see &= have > p - window
            seen_n[m] = see.sum()
            for h in range(heads):
                if not see.any():
                    out[m, h], absv[m, h], mag[m, h] = 0.0, 0.0, 0.0
                    continue
                k, v, x = K[see, h // G], V[see, h // G], q[m, h * D: (h + 1) * D]
                top[m, h] = np.abs(v).max() if cache.kv == "same" else 127 * max(float(cache.vs[cache.table[b, j // cache.page], h // G, j % cache.page // BLOCK]) for j in have[see])
                s = scale * (k @ x)
                mag[m, h] = abs(scale) * (np.abs(k) @ np.abs(x)).max()
                if cap:
                    s = cap * np.tanh(s / cap)
                if slopes is not None:
                    s = s + float(slopes[h]) * (have[see] - p)
                    mag[m, h] += np.abs(float(slopes[h]) * (have[see] - p)).max() / D   # (rounded once or twice, not D times)
                with np.errstate(all="ignore"):
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[m, h], absv[m, h] = w @ v, w @ np.abs(v)
            m += 1
    return out.reshape(rows, -1), absv.reshape(rows, -1), mag.reshape(rows, -1), (seen_n, np.broadcast_to(top, out.shape).reshape(rows, -1))


HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative to the value


def attention_tolerance(cache, ref, absv, mag, seen_n, cap=0.0):
    """How far an output may be: its own rounding; the weights' (int8 caches: fp16); scores' errors, which move weights by as much:
    products of D terms in fp32 and a few roundings more, with a cap also 2^-22 of it; sums of `seen` terms in fp32.
    Weights in fp16 also come to 0 where they are small: they are taken relative to 2^(m - 7), m at most the largest exponent and at
    least 8 below, so the largest is >= 2^7, the denominator too (int8: w = 2^(s + log2 vs - ..), the denominator sums w / vs, >= 2^7 /
    vs of that key), and a weight's rounding is at most 2^-25 of 1 there: 2^-32 of a value (int8: 2^-32 * 127 vs) for every key."""
    seen_n, top = seen_n
    p = HALF["f16" if cache.kv == "i8" else cache.dtype]
    score = (cache.dim + 16) * 2.0 ** -24 * mag + (2.0 ** -21 * cap) + 2.0 ** -21
    rel = p + 2 * score + (seen_n[:, None] + 64) * 2.0 ** -24
    small = 2.0 ** -24 if cache.dtype == "f16" else 0.0
    flush = seen_n[:, None] * top * 2.0 ** -32 if p == HALF["f16"] else 0.0
    return HALF[cache.dtype] * np.abs(ref) * 1.01 + rel * absv * (1 + p) + flush + small + 1e-30
