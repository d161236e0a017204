"""Operators of the paged key/value cache, measured through the framework's public entry points.

A cache layer is [pages][kv_heads][page][dim] keys and values in 16 bits, or in int8 with one fp32 scale
per block of 16 tokens and head; a table says which page holds a sequence's tokens.  Rows of a batch are
ragged: row i of sequence b is its token len[b] - n_b + i, the lengths counting the call's own rows.

* "append": rows q | k | v of a projection are rotated by their positions and written: q as rows, k and v
  into the cache (int8: a block whose scale grows is rescaled).  With an int8 cache the pass ends with
  "read" of the tokens in the blocks that it touched: a program that hands new tokens on.
* "read": the last tokens of the sequences back as rows (a sequence that leaves the card or moves to a
  cache of another type).
* "decode": one query row per sequence over its whole cache.
* "prefill": the rows of prompts, or of chunks behind what is cached.

Scores of both are scale * q.k, capped by cap * tanh(s / cap), plus slope_h * (key - row) (ALiBi); row p
sees key j where first <= j < len, j <= p or j < prefix, and j > p - window.
"""
import ctypes
import math

import torch

own = False

BLOCK = 16            # tokens that share a scale
TINY = 2.0 ** -100    # the least scale
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of 32 llama3-8b streams writes its layer's rows: latency
        dict(name="append f16 step x32", kind="append", dtype="f16", kv="same", heads=32, kv_heads=8, dim=128, page=64, seqs=32, new=1, dnew=0,
             length=2048, spread=1024, rot=128, halves=False, wide=True),
        # the same of 24 tinyllama streams into int8: blocks are rescaled, and read back for another process
        dict(name="append i8 step x24", kind="append", dtype="f16", kv="i8", heads=32, kv_heads=4, dim=64, page=32, seqs=24, new=1, dnew=0,
             length=700, spread=500, rot=64, halves=False, wide=True),
        # prompts of several requests in one batch, partly rotated heads, odd lengths
        dict(name="append i8 prompts 8k", kind="append", dtype="bf16", kv="i8", heads=32, kv_heads=8, dim=128, page=64, seqs=5, new=2500, dnew=1801,
             length=3100, spread=2011, rot=64, halves=True, wide=False),
        # one request is moved away
        dict(name="read i8 1k", kind="read", dtype="f16", kv="i8", heads=8, kv_heads=4, dim=64, page=32, seqs=1, new=1023, dnew=0, length=1400, spread=0),
        # a server drains: 16 requests to another machine
        dict(name="read bf16 x16 2k", kind="read", dtype="bf16", kv="same", heads=32, kv_heads=8, dim=128, page=64, seqs=16, new=2048, dnew=900,
             length=2048, spread=900),
        # one 7B user with 2048 tokens of context: every head has its own keys, latency
        dict(name="decode f16 x1 2k", kind="decode", dtype="f16", kv="same", heads=32, kv_heads=32, dim=128, page=64, seqs=1, length=2048, spread=0,
             cap=0.0, alibi=False, window=0),
        # llama3-8b streams of 4096 to 8192 tokens, 8-bit cache: the server's ordinary step
        dict(name="decode i8 x32 8k", kind="decode", dtype="f16", kv="i8", heads=32, kv_heads=8, dim=128, page=64, seqs=32, length=8192, spread=4096,
             cap=0.0, alibi=False, window=0),
        # capped scores and a window over heads of 256, ragged
        dict(name="decode bf16 x48 capped", kind="decode", dtype="bf16", kv="same", heads=16, kv_heads=8, dim=256, page=32, seqs=48, length=3001,
             spread=2900, cap=50.0, alibi=False, window=1024),
        # one long document in 8 bits: few rows, a long axis
        dict(name="decode i8 x1 128k", kind="decode", dtype="bf16", kv="i8", heads=32, kv_heads=8, dim=128, page=256, seqs=1, length=131072, spread=0,
             cap=0.0, alibi=False, window=0),
        # prompts of the test sizes' kind with distance biases, prefixes and several documents each
        dict(name="prefill f16 x12 alibi", kind="prefill", dtype="f16", kv="same", heads=32, kv_heads=4, dim=64, page=32, seqs=12, new=640, dnew=601,
             length=640, spread=601, cap=0.0, alibi=True, window=0, prefix=True, docs=True),
        # a 512-token chunk of two requests behind what they have cached in 8 bits
        dict(name="prefill i8 x2 512@8k", kind="prefill", dtype="bf16", kv="i8", heads=32, kv_heads=8, dim=128, page=64, seqs=2, new=512, dnew=0,
             length=8192, spread=1000, cap=0.0, alibi=False, window=0, prefix=False, docs=False),
        # one whole prompt, capped scores
        dict(name="prefill bf16 4k capped", kind="prefill", dtype="bf16", kv="same", heads=32, kv_heads=8, dim=128, page=64, seqs=1, new=4000, dnew=0,
             length=4000, spread=0, cap=30.0, alibi=False, window=0, prefix=False, docs=False),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    kind = rng.choice(["append", "append", "read", "decode", "decode", "decode", "prefill", "prefill"])
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 4), (16, 4), (8, 8), (12, 2), (8, 1), (20, 4)])
    c = dict(kind=kind, dtype=rng.choice(["f16", "bf16"]), kv=rng.choice(["same", "i8"]), heads=heads, kv_heads=kv_heads,
             dim=rng.choice([64, 128, 128, 256]), page=rng.choice([16, 32, 64, 128, 256]))
    if kind in ("append", "read"):
        seqs = log(1, 64)
        new = 1 if kind == "append" and rng.random() < 0.4 else log(1, 8000 // seqs)
        length = new + log(1, 1000)
        c |= dict(seqs=seqs, new=new, dnew=rng.randrange(new), length=length, spread=rng.randrange(length - new + 1))
        if kind == "append":
            c |= dict(rot=c["dim"] // rng.choice([1, 1, 2]), halves=rng.random() < 0.5, wide=rng.random() < 0.5)
        return c
    mask = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3, window=rng.choice([0, 0, 0, 300, 1024]))
    if kind == "decode":
        seqs = log(1, 64)
        length = log(1, 220000 // (seqs * kv_heads) * 4)
        return c | dict(seqs=seqs, length=length, spread=rng.randrange(length)) | mask
    heavy = (heads * c["dim"]) / 4096.0
    seqs = log(1, 12)
    new = log(1, max(2, int(2000 / math.sqrt(seqs * heavy))))
    length = new + (log(1, 3000) if rng.random() < 0.5 else 0)
    dnew = rng.randrange(new)
    return c | dict(seqs=seqs, new=new, dnew=dnew, length=length, spread=dnew) | mask | dict(prefix=rng.random() < 0.3, docs=rng.random() < 0.3)


def _lengths(c):
    """(new rows, length with them) of every sequence."""
    d = max(c["seqs"] - 1, 1)
    at = [(b * 7) % c["seqs"] for b in range(c["seqs"])] if c["seqs"] % 7 else list(range(c["seqs"]))
    ln = [c["length"] - c["spread"] * a // d for a in at]
    new = [1] * c["seqs"] if c["kind"] == "decode" else [min(c["new"] - c["dnew"] * a // d, n) for a, n in zip(at, ln)]
    return new, ln


def _read_lengths(c):
    """Tokens of every sequence in the blocks that an append touched."""
    return [n + (l - n) % BLOCK for n, l in zip(*_lengths(c))]


def _starts(n):
    s = [0]
    for v in n:
        s.append(s[-1] + v)
    return s


def _masks(c):
    """(first, prefix) as host lists; None where the case has none."""
    new, ln = _lengths(c)
    first = prefix = None
    if c.get("docs"):   # documents of 200 tokens, counted from the sequence's start
        first = [p // 200 * 200 for n, l in zip(new, ln) for p in range(l - n, l)]
    if c.get("prefix"):
        prefix = [l // (2 + b % 3) for b, l in enumerate(ln)]
    return first, prefix


def work(case):
    c = case
    new, ln = _lengths(c)
    rows, kvd, e = sum(new), c["kv_heads"] * c["dim"], 2 if c["kv"] == "same" else 1
    token = 2 * kvd * e + (2 * c["kv_heads"] * 4 / BLOCK if e == 1 else 0)   # bytes of a token's keys and values
    if c["kind"] == "append":
        x = rows * (c["heads"] * c["dim"] + 2 * kvd) * (4 if c["wide"] else 2)
        n = x + rows * c["heads"] * c["dim"] * 2 + rows * token + rows * c["rot"] * 4
        if e == 1:   # the touched blocks' older tokens, and the rows handed on
            r = sum(_read_lengths(c))
            n += (r - rows) * 2 * token + r * 2 * kvd * 2
        return {"bytes": n, "flops": rows * (c["heads"] + c["kv_heads"]) * c["dim"] * 3}
    if c["kind"] == "read":
        return {"bytes": rows * (token + 2 * kvd * 2), "flops": rows * 2 * kvd}
    first, prefix = _masks(c)
    pairs, seen, m = 0, 0, 0
    for b, (n, l) in enumerate(zip(new, ln)):
        low, high = l, 0
        for p in range(l - n, l):
            lo = max(first[m] if first else 0, p - c["window"] + 1 if c["window"] else 0)
            hi = max(p + 1, prefix[b] if prefix else 0)
            pairs, low, high, m = pairs + hi - lo, min(low, lo), max(high, hi), m + 1
        seen += max(0, high - low)
    return {"bytes": 2 * rows * c["heads"] * c["dim"] * 2 + seen * token, "flops": 4 * pairs * c["heads"] * c["dim"]}


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    hg = torch.Generator().manual_seed(seed + 1)
    dt = TYPES[c["dtype"]]
    new, ln = _lengths(c)
    rows, kvh, dim, page = sum(new), c["kv_heads"], c["dim"], c["page"]
    cols = max(-(-n // page) for n in ln)
    used = [-(-n // page) for n in ln]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=hg).to(torch.int32)   # pages as an allocator hands them out after a while
    table, at = torch.zeros(len(ln), cols, dtype=torch.int32), 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = dict(c=c, dt=dt, table=table.to(dev), len=i32(ln), start=i32(_starts(new)), rows=rows, longest=max(ln), most=max(new))
    shape = (pages, kvh, page, dim)
    if c["kv"] == "same":
        s["k"], s["v"] = (torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt) for _ in range(2))
        s["ks"] = s["vs"] = None
    else:   # int8 of normal values: the largest of a block of 16 tokens at about 3 deviations
        s["k"], s["v"] = (torch.randn(shape, generator=g, device=dev).mul_(42.0).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2))
        s["ks"], s["vs"] = ((torch.rand(pages, kvh, page // BLOCK, generator=g, device=dev) * 0.6 + 0.7) / 42.0 for _ in range(2))
    qd = c["heads"] * dim
    if c["kind"] == "append":
        x = torch.randn(rows, qd + 2 * kvh * dim, generator=g, device=dev)
        s["x"] = x if c["wide"] else x.to(dt)
        s["q"] = torch.empty(rows, qd, dtype=dt, device=dev)
        ang = torch.arange(max(ln), dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=dev) / c["rot"])
        s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        if c["kv"] == "i8":
            back = _read_lengths(c)
            s["back"], s["back_rows"] = i32(_starts(back)), sum(back)
            s["kr"], s["vr"] = (torch.empty(sum(back), kvh * dim, dtype=dt, device=dev) for _ in range(2))
    elif c["kind"] == "read":
        s["kr"], s["vr"] = (torch.empty(rows, kvh * dim, dtype=dt, device=dev) for _ in range(2))
    else:
        s["q"] = torch.randn(rows, qd, generator=g, device=dev).mul_(1.5).to(dt)   # scores of about 1.5 deviations
        s["out"] = torch.empty(rows, qd, dtype=dt, device=dev)
        first, prefix = _masks(c)
        s["first"] = None if first is None else i32(first)
        s["prefix"] = None if prefix is None else i32(prefix)
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, c["heads"] + 1, device=dev) / c["heads"]).float() if c["alibi"] else None
    return s


def run(state):
    if own:
        return _own(state)
    kind = state["c"]["kind"]
    if kind == "append":
        return _append(state)
    if kind == "read":
        return _read(state, state["start"], state["rows"])
    return _attend(state)


# ---------------------------------------------------------------- the framework's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _handles(s):
    """The argument structures that a program keeps beside its buffers."""
    import turboinfer_amd as T
    c = s["c"]
    cache = T.PagedCache(k=_ptr(s["k"]), v=_ptr(s["v"]), k_scale=_ptr(s["ks"]), v_scale=_ptr(s["vs"]), table=_ptr(s["table"]), len=_ptr(s["len"]),
                         table_ld=s["table"].shape[1], pages=s["k"].shape[0], page=c["page"], kv_heads=c["kv_heads"], head_dim=c["dim"],
                         seqs=c["seqs"], dtype=T.PAGED_F16 if c["dtype"] == "f16" else T.PAGED_BF16, kv_type=T.KV_SAME if c["kv"] == "same" else T.KV_I8)
    L, args, extra = T.lib(), None, None
    ref = ctypes.byref(cache)
    if c["kind"] == "append":
        args = T.PagedAppendArgs(x=_ptr(s["x"]), q=_ptr(s["q"]), row_start=_ptr(s["start"]), rope_cs=_ptr(s["rope"]), rows=s["rows"], heads=c["heads"],
                                 ldx=s["x"].shape[1], ldq=s["q"].shape[1], x_f32=int(c["wide"]), rope_len=s["rope"].shape[0], rot_dim=c["rot"],
                                 rope_kind=T.ROPE_HALVES if c["halves"] else T.ROPE_PAIRS)
    elif c["kind"] in ("decode", "prefill"):
        args = T.PagedAttnArgs(q=_ptr(s["q"]), out=_ptr(s["out"]), row_start=None if c["kind"] == "decode" else _ptr(s["start"]), rows=s["rows"],
                               heads=c["heads"], ldq=s["q"].shape[1], ldo=s["out"].shape[1], max_len=s["longest"], scale=1.0 / math.sqrt(c["dim"]),
                               softcap=c["cap"], slopes=_ptr(s["slopes"]), first=_ptr(s["first"]), prefix=_ptr(s["prefix"]), window=c["window"])
        n = L.ti_paged_workspace_bytes(ref, ctypes.byref(args))
        extra = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        args.workspace, args.workspace_bytes = extra.data_ptr(), n
    return L, T.check, ref, None if args is None else ctypes.byref(args), (cache, args, extra)


def _own(s):
    if "handles" not in s:
        s["handles"] = _handles(s)
    L, check, cache, args, _ = s["handles"]
    stream = torch.cuda.current_stream().cuda_stream
    kind = s["c"]["kind"]
    if kind == "append":
        check(L.ti_paged_append(cache, args, stream))
        if s["ks"] is None:
            return {"q": s["q"], "k": s["k"], "v": s["v"]}
        w = s["kr"].shape[1]
        check(L.ti_paged_read(cache, s["back"].data_ptr(), s["back_rows"], s["kr"].data_ptr(), w, s["vr"].data_ptr(), w, stream))
        return {"q": s["q"], "k": s["kr"], "v": s["vr"]}
    if kind == "read":
        w = s["kr"].shape[1]
        check(L.ti_paged_read(cache, s["start"].data_ptr(), s["rows"], s["kr"].data_ptr(), w, s["vr"].data_ptr(), w, stream))
        return {"k": s["kr"], "v": s["vr"]}
    check((L.ti_paged_decode if kind == "decode" else L.ti_paged_prefill)(cache, args, stream))
    return {"out": s["out"]}


# ---------------------------------------------------------------- plain forms
def _places(s, start, rows):
    """(sequence, position, page, place) of every row."""
    m = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), m.to(torch.int32), right=True)
    pos = s["len"][seq].long() - start[seq + 1].long() + m
    page = s["c"]["page"]
    return seq, pos, s["table"][seq, pos // page].long(), pos % page


def _rotate(x, cs, halves):
    """x [rows][heads][dim] fp32 by cs [rows][rot / 2][2]."""
    rot = 2 * cs.shape[1]
    co, si = cs[:, None, :, 0], cs[:, None, :, 1]
    r = x[..., :rot]
    if halves:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat([a * co - b * si, a * si + b * co], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack([a * co - b * si, a * si + b * co], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _put_i8(s, cache, scale, x, seq, pos, page, place):
    """Rows x [rows][kv_heads][dim] into an int8 cache."""
    c = s["c"]
    kvh, dim, nb = c["kv_heads"], c["dim"], c["page"] // BLOCK
    begin = s["len"].long() - (s["start"][1:] - s["start"][:-1]).long()   # each sequence's first new position
    blk = page * nb + place // BLOCK
    flat = scale.transpose(1, 2).reshape(-1, kvh)      # [page][block][head]
    old = ((begin[seq] // BLOCK == pos // BLOCK) & (begin[seq] % BLOCK > 0))[:, None]
    most = torch.zeros_like(flat).index_reduce_(0, blk, torch.maximum(x.abs().amax(-1) / 127.0, flat[blk] * old).clamp_min(TINY), "amax")
    # the blocks that hold older tokens: one a sequence
    at = begin.clamp_max(s["table"].shape[1] * c["page"] - 1)
    pg, pl = s["table"][torch.arange(c["seqs"], device="cuda"), at // c["page"]].long(), at % c["page"]
    b0 = pg * nb + pl // BLOCK
    cells = cache.view(-1, kvh, nb, BLOCK, dim)
    have = cells[pg, :, pl // BLOCK].float()
    is_old = (torch.arange(BLOCK, device="cuda")[None] < (begin % BLOCK)[:, None])[:, None, :, None] & (most[b0] > 0)[:, :, None, None]
    ratio = torch.where(most[b0] > 0, flat[b0] / most[b0], 1.0)[:, :, None, None]
    cells[pg, :, pl // BLOCK] = torch.where(is_old, (have * ratio).round(), have).to(torch.int8)
    cells[page, :, place // BLOCK, place % BLOCK] = (x / most[blk][..., None]).round().to(torch.int8)
    scale[page, :, place // BLOCK] = most[blk]


def _append(s):
    c = s["c"]
    qd, kvd, dim = c["heads"] * c["dim"], c["kv_heads"] * c["dim"], c["dim"]
    seq, pos, page, place = _places(s, s["start"], s["rows"])
    x = s["x"].float()
    cs = s["rope"][pos]
    s["q"].copy_(_rotate(x[:, :qd].unflatten(1, (-1, dim)), cs, c["halves"]).flatten(1))
    k, v = _rotate(x[:, qd:qd + kvd].unflatten(1, (-1, dim)), cs, c["halves"]), x[:, qd + kvd:].unflatten(1, (-1, dim))
    if s["ks"] is None:
        s["k"][page, :, place] = k.to(s["dt"])
        s["v"][page, :, place] = v.to(s["dt"])
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    _put_i8(s, s["k"], s["ks"], k, seq, pos, page, place)
    _put_i8(s, s["v"], s["vs"], v, seq, pos, page, place)
    return {"q": s["q"], **_read(s, s["back"], s["back_rows"])}


def _values(s, cache, scale, page, place):
    """The cache's values [...][kv_heads][dim] fp32 at these places."""
    v = cache[page, :, place].float()
    return v if scale is None else v * scale[page, :, place // BLOCK][..., None]


def _read(s, start, rows):
    _, _, page, place = _places(s, start, rows)
    return {n: _values(s, s[n], s[n + "s"], page, place).to(s["dt"]).flatten(1) for n in ("k", "v")}


def _attend(s):
    c = s["c"]
    B, H, kvh, dim, L, N = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["longest"], s["most"]
    j = torch.arange(L, device="cuda")
    page = s["table"][:, j // c["page"]].long()
    place = (j % c["page"])[None].expand(B, -1)
    k, v = (_values(s, s[n], s[n + "s"], page, place).transpose(1, 2) for n in ("k", "v"))       # [B][kv_heads][L][dim]
    # rows as [sequence][place among its new ones], the places behind a sequence's last one repeating it
    n = (s["start"][1:] - s["start"][:-1]).long()
    i = torch.minimum(torch.arange(N, device="cuda")[None], n[:, None] - 1)
    m = s["start"][:-1].long()[:, None] + i
    p = (s["len"].long() - n)[:, None] + i
    q = s["q"][m].float().view(B, N, kvh, H // kvh, dim).permute(0, 2, 3, 1, 4).reshape(B, kvh, -1, dim)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, kvh, H // kvh, N, L)
    sc *= 1.0 / math.sqrt(dim)
    if c["cap"]:
        sc = torch.tanh_(sc.div_(c["cap"])).mul_(c["cap"])
    if s["slopes"] is not None:
        sc += s["slopes"].view(1, kvh, -1, 1, 1) * (j[None, None] - p[:, :, None]).float()[:, None, None]
    hi = p if s["prefix"] is None else torch.maximum(p, s["prefix"].long()[:, None] - 1)
    lo = torch.zeros_like(p) if s["first"] is None else s["first"].long()[m]
    if c["window"]:
        lo = torch.maximum(lo, p - c["window"] + 1)
    seen = (j >= lo[..., None]) & (j <= hi[..., None]) & (j < s["len"][:, None, None])
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True).clamp_min(-3e38)
    w = torch.exp_(sc.sub_(top))
    v.masked_fill_((j >= s["len"][:, None])[:, None, :, None], 0.0)
    o = torch.matmul(w.view(B, kvh, -1, L), v.contiguous()).view(B, kvh, -1, N, dim)
    o /= w.sum(-1, keepdim=True).clamp_min(1e-37)
    o = o.permute(0, 3, 1, 2, 4).reshape(B * N, H * dim).to(s["dt"])
    keep = (torch.arange(N, device="cuda")[None] < n[:, None]).flatten().nonzero()[:, 0] if int(s["rows"]) != B * N else slice(None)
    s["out"].copy_(o[keep])
    return {"out": s["out"]}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    return {"append": _exact_append, "read": _exact_read}.get(c["kind"], _exact_attention)(s, c)


def _exact_cache(s, name):
    """The cache as float64 values [pages][kv_heads][page][dim]."""
    x = s[name].double()
    return x if s[name + "s"] is None else x * s[name + "s"].double().repeat_interleave(BLOCK, 2)[..., None]


def _exact_rows(s, c, values, b, t0, t1):
    """Tokens [t0, t1) of sequence b: [tokens][kv_heads][dim]."""
    u = -(-t1 // c["page"])
    return values[s["table"][b, :u].long()].transpose(1, 2).reshape(u * c["page"], c["kv_heads"], c["dim"])[t0:t1]


def _exact_read(s, c):
    k, v = _exact_cache(s, "k"), _exact_cache(s, "v")
    new, ln = _lengths(c)
    return {n: torch.cat([_exact_rows(s, c, x, b, l - w, l).flatten(1) for b, (w, l) in enumerate(zip(new, ln))]) for n, x in (("k", k), ("v", v))}


def _exact_rotate(x, pos, c):
    f = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    # (the table that the call is given holds fp32 values)
    z = torch.complex((pos[:, None] * f).cos().float().double(), (pos[:, None] * f).sin().float().double())[:, None]
    h = c["rot"] // 2
    a, b = (slice(0, h), slice(h, 2 * h)) if c["halves"] else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
    y = x.clone()
    w = torch.complex(x[..., a], x[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y


def _exact_append(s, c):
    new, ln = _lengths(c)
    qd, kvd = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
    x, at, page = s["x"].double(), 0, c["page"]
    cache, got = {n: s[n].double() for n in "kv"}, {n: [] for n in "qkv"}
    for b, (n, l) in enumerate(zip(new, ln)):
        r, p0 = x[at:at + n], l - n
        at += n
        pos = torch.arange(p0, l, device="cuda", dtype=torch.float64)
        got["q"].append(_exact_rotate(r[:, :qd].reshape(n, -1, c["dim"]), pos, c).flatten(1))
        kv = {"k": _exact_rotate(r[:, qd:qd + kvd].reshape(n, -1, c["dim"]), pos, c), "v": r[:, qd + kvd:].reshape(n, -1, c["dim"])}
        for name, y in kv.items():
            if c["kv"] == "same":
                t = torch.arange(p0, l, device="cuda")
                cache[name][s["table"][b, t // page].long(), :, t % page] = y
                continue
            o = p0 % BLOCK   # older tokens of the first block, then whole blocks
            have = _exact_rows(s, c, cache[name], b, p0 - o, p0)
            scale = s[name + "s"][s["table"][b, min(p0, l - 1) // page].long(), :, p0 % page // BLOCK].double()
            pad = -(o + n) % BLOCK
            z = torch.cat([torch.zeros_like(have), y, torch.zeros(pad, *y.shape[1:], dtype=torch.float64, device="cuda")])
            z = z.view(-1, BLOCK, *y.shape[1:])
            most = z.abs().amax((1, 3)) / 127.0
            if o:
                most[0] = torch.maximum(most[0], scale)
            most = most.clamp_min(TINY)[:, None, :, None]
            q = torch.round(z / most)
            if o:
                q[0, :o] = torch.round(have * (scale[:, None] / most[0]))
            got[name].append((q * most).flatten(0, 1)[:o + n].flatten(1))
    if c["kv"] == "same":
        return {"q": torch.cat(got["q"]), **cache}
    return {n: torch.cat(got[n]) for n in "qkv"}


def _exact_attention(s, c):
    new, ln = _lengths(c)
    first, prefix = _masks(c)
    k, v = s["k"], s["v"]
    out, at, G = [], 0, c["heads"] // c["kv_heads"]
    for b, (n, l) in enumerate(zip(new, ln)):
        pick = lambda name, x: _exact_rows(s, c, x, b, 0, l).double() if s[name + "s"] is None else _exact_rows(  # noqa: E731
            s, c, x, b, 0, l).double() * s[name + "s"][s["table"][b, :-(-l // c["page"])].long()].double().transpose(1, 2).flatten(0, 1).repeat_interleave(BLOCK, 0)[:l, :, None]
        kk, vv = pick("k", k).permute(1, 2, 0).contiguous(), pick("v", v).transpose(0, 1).contiguous()
        p = torch.arange(l - n, l, device="cuda")[:, None]
        j = torch.arange(l, device="cuda")[None]
        see = j <= p if prefix is None else (j <= p) | (j < prefix[b])
        if first is not None:
            see &= j >= torch.tensor(first[at:at + n], device="cuda")[:, None]
        if c["window"]:
            see &= p - j < c["window"]
        q = s["q"][at:at + n].double().view(n, c["kv_heads"], G, c["dim"])
        at += n
        o = torch.empty_like(q)
        for h in range(G):
            a = torch.bmm(q[:, :, h].transpose(0, 1).contiguous(), kk) / math.sqrt(c["dim"])
            if c["cap"]:
                a = c["cap"] * torch.tanh(a / c["cap"])
            if s["slopes"] is not None:
                a += s["slopes"].double().view(-1, G)[:, h, None, None] * (j - p)
            a = torch.softmax(a.masked_fill(~see, -math.inf), -1).nan_to_num(0.0)   # (a row that sees nothing: 0)
            o[:, :, h] = torch.bmm(a, vv).transpose(0, 1)
        out.append(o.view(n, -1))
    return {"out": torch.cat(out)}
