"""Measured cases of the paged key/value cache operators: rotary positions with
the cache write ("append"), attention of new tokens over the cache ("attend"),
the page bookkeeping of one decode turn ("fork": beam reorder, fork and free,
then growth) and the compaction of a cache ("compact").

Each case runs either in its plain form (elementary torch operations in 32
bits) or, where `own` is true, through pulsar_b200.kv.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}

# the most that a drawn case may cost: the largest listed cases' key bytes, rotated values and moved page bytes
MOST_KV = 2.2e9
MOST_PADDED = 1.1e9
MOST_ROPE = 6.5e8
MOST_PAGES = 7.0e8


def listed():
    return [
        # one user's first decode steps: a single short sequence, where the call's latency is all there is
        dict(name="attend 1 x 100", op="attend", rows=1, n_q=1, max_len=100, hq=32, hkv=8, d=128, page=16, q="bf16",
             kv="bf16", window=0, sinks=False),
        # a small batch with f32 activations (the expert layer's type) over an f16 cache, odd ragged lengths
        dict(name="attend 8 x 4001 f32", op="attend", rows=8, n_q=1, max_len=4001, hq=16, hkv=4, d=128, page=32,
             q="f32", kv="f16", window=0, sinks=False),
        # windowed layers with attention sinks, 64 heads of 64 over 8 key heads, a decode batch of 64
        dict(name="attend 64 x 2048 window", op="attend", rows=64, n_q=1, max_len=2048, hq=64, hkv=8, d=64, page=16,
             q="bf16", kv="bf16", window=128, sinks=True),
        # four drafted tokens verified at once, seven query heads to a key head
        dict(name="attend 16 x 9001 drafts", op="attend", rows=16, n_q=4, max_len=9001, hq=28, hkv=4, d=128, page=64,
             q="f16", kv="f16", window=0, sinks=False),
        # long contexts in an 8-bit cache: the length is what there is to split
        dict(name="attend 4 x 131071 e4m3", op="attend", rows=4, n_q=1, max_len=131071, hq=64, hkv=8, d=128, page=64,
             q="bf16", kv="e4m3", window=0, sinks=False),
        # the large decode batch (256 sequences) with ragged lengths
        dict(name="attend 256 x 4096", op="attend", rows=256, n_q=1, max_len=4096, hq=32, hkv=8, d=128, page=16,
             q="bf16", kv="bf16", window=0, sinks=False),
        # one token of one sequence: latency
        dict(name="append 1", op="append", rows=1, n_q=1, hq=32, hkv=8, d=128, rot=128, inter=False, page=16, x="bf16",
             kv="bf16"),
        # a decode batch of 256 in f32, half of each head rotated
        dict(name="append 256 part", op="append", rows=256, n_q=1, hq=32, hkv=4, d=128, rot=64, inter=False, page=16,
             x="f32", kv="bf16"),
        # prompts: 8 sequences of 2048 tokens, interleaved pairs
        dict(name="append 8 x 2048 inter", op="append", rows=8, n_q=2048, hq=64, hkv=8, d=128, rot=128, inter=True,
             page=64, x="f16", kv="f16"),
        # a turn of a small beam search: 2 searches of 4 beams, 4 layers
        dict(name="fork 2 x 4", op="fork", groups=2, beams=4, layers=4, max_len=500, hkv=4, d=64, page=16, kv="bf16"),
        # a turn of 32 searches of 8 beams over 20 layers
        dict(name="fork 32 x 8", op="fork", groups=32, beams=8, layers=20, max_len=300, hkv=2, d=64, page=32, kv="f16"),
        # a cache half of whose sequences have left, 16 layers
        dict(name="compact 128", op="compact", rows=128, layers=16, max_len=1000, hkv=2, d=64, page=32, kv="bf16"),
    ]


def _spread(rng, lo, hi):
    """a whole number of [lo, hi], even over its logarithm"""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if any(v == 3072 for v in c.values()):
            continue
        if c["op"] == "attend" and (w["bytes"] > MOST_KV or c["rows"] * c["max_len"] * c["hkv"] * c["d"] > MOST_PADDED
                                    or c["rows"] * c["max_len"] * c["hq"] * c["n_q"] > 2.5e8):
            continue
        if c["op"] == "append" and w["bytes"] > MOST_ROPE:
            continue
        if c["op"] in ("fork", "compact") and (w["bytes"] > MOST_PAGES or _pool_values(c) > 4e8):
            continue
        return c


def _draw(rng):
    op = rng.choice(("attend", "attend", "append", "fork", "compact"))
    if op == "attend":
        hkv = rng.choice((1, 2, 4, 8))
        kv = rng.choice(("bf16", "f16", "e4m3"))
        return dict(op=op, rows=_spread(rng, 1, 256), n_q=rng.choice((1, 1, 1, 2, 3, 5)),
                    max_len=_spread(rng, 1, 131072), hq=hkv * rng.choice((1, 2, 3, 4, 5, 7, 8, 12, 16)), hkv=hkv,
                    d=rng.choice((64, 80, 96, 128, 192, 256)), page=rng.choice((8, 16, 24, 32, 64, 128)),
                    q=rng.choice(("f32", "bf16", "f16")), kv=kv, window=rng.choice((0, 0, _spread(rng, 1, 4096))),
                    sinks=rng.choice((False, True)))
    if op == "append":
        d = rng.choice((64, 80, 96, 128, 192, 256))
        return dict(op=op, rows=_spread(rng, 1, 256), n_q=rng.choice((1, _spread(rng, 1, 4096))),
                    hq=rng.choice((4, 7, 16, 32, 64)), hkv=rng.choice((1, 2, 4, 8)), d=d,
                    rot=rng.choice((d, d // 2, d // 4)), inter=rng.choice((False, True)),
                    page=rng.choice((8, 16, 24, 32, 64, 128)), x=rng.choice(("f32", "bf16", "f16")),
                    kv=rng.choice(("bf16", "f16")))
    c = dict(op=op, layers=_spread(rng, 1, 48), max_len=_spread(rng, 1, 2000), hkv=rng.choice((1, 2, 4)),
             d=rng.choice((64, 80, 128)), page=rng.choice((8, 16, 24, 32)), kv=rng.choice(("bf16", "f16")))
    if op == "fork":
        c.update(groups=_spread(rng, 1, 64), beams=rng.choice((1, 2, 3, 4, 5, 8)))
    else:
        c.update(rows=_spread(rng, 2, 256))
    return c


# ------------------------------------------------------------- shapes of a case (the same for every seed)

def _rng(c):
    return random.Random("%s %s %s" % (c["op"], c["max_len"], c.get("rows", c.get("groups"))))


def _lens(c, rows):
    """ragged lengths: the first is the longest, the rest between a fifth of it and all of it"""
    r = _rng(c)
    return [c["max_len"]] + [max(1, int(c["max_len"] * r.uniform(0.2, 1.0))) for _ in range(rows - 1)]


def _seen(c, n):
    """(first, last) key seen by each of the n_q tokens of a sequence of n keys"""
    out = []
    for i in range(c["n_q"]):
        hi = n - (c["n_q"] - 1 - i)
        lo = max(0, hi - c["window"]) if c["window"] else 0
        out.append((lo, max(lo, hi)))
    return out


def _turn(c):
    """lengths, the row that each row continues (-1: its sequence ends) and the tokens by which it grows"""
    rows = c["groups"] * c["beams"]
    r = _rng(c)
    lens, src, new = [], [], []
    for g in range(c["groups"]):
        n = max(1, int(c["max_len"] * r.uniform(0.2, 1.0)))
        ends = c["groups"] > 3 and r.random() < 0.1
        for b in range(c["beams"]):
            lens.append(n)
            src.append(-1 if ends else g * c["beams"] + min(r.randrange(c["beams"]), r.randrange(c["beams"])))
            new.append(1)
    assert len(src) == rows
    return lens, src, new


def _pages(n, page):
    return -(-n // page)


def _pool_values(c):
    p = c["page"]
    if c["op"] == "fork":
        lens, _, _ = _turn(c)
        n_pages = sum(_pages(n, p) for n in lens) + 2 * len(lens)
    else:
        n_pages = sum(_pages(n, p) for n in _lens(c, c["rows"])) + 7
    return n_pages * c["layers"] * 2 * c["hkv"] * p * c["d"]


def _copies(c):
    """pages that a fork copies: a partly filled page has one holder"""
    lens, src, _ = _turn(c)
    stays = {s for i, s in enumerate(src) if s == i}
    n, took = 0, set()
    for i, s in enumerate(src):
        if s < 0 or lens[s] % c["page"] == 0 or s == i:
            continue
        if s in stays or s in took:
            n += 1
        took.add(s)
    return n


def _left(c):
    """the rows of a compact case that have left"""
    r = _rng(c)
    return [r.random() < 0.5 for _ in range(c["rows"])]


def work(c):
    if c["op"] == "attend":
        lens = _lens(c, c["rows"])
        spans = [_seen(c, n) for n in lens]
        keys = sum(max(h for _, h in s) - min(lo for lo, _ in s) for s in spans)
        seen = sum(h - lo for s in spans for lo, h in s)
        io = 2 * c["rows"] * c["n_q"] * c["hq"] * c["d"] * SIZE[c["q"]] + 4 * c["rows"] * c["n_q"] * c["hq"]
        return {"bytes": 2 * keys * c["hkv"] * c["d"] * SIZE[c["kv"]] + io, "flops": 4 * c["d"] * c["hq"] * seen}
    if c["op"] == "append":
        t = c["rows"] * c["n_q"]
        return {"bytes": t * c["d"] * (2 * c["hq"] * SIZE[c["x"]] + 2 * c["hkv"] * (SIZE[c["x"]] + SIZE[c["kv"]]))
                + 4 * t * c["rot"], "flops": 3 * t * (c["hq"] + c["hkv"]) * c["rot"]}
    page = c["layers"] * 2 * c["hkv"] * c["page"] * c["d"] * SIZE[c["kv"]]
    if c["op"] == "fork":
        lens, src, _ = _turn(c)
        rows = sum(_pages(lens[s], c["page"]) for s in src if s >= 0)
        return {"bytes": 2 * _copies(c) * page + 2 * 4 * rows, "flops": 0}
    lens, left = _lens(c, c["rows"]), _left(c)
    total = sum(_pages(n, c["page"]) for n in lens) + 7
    live = sum(_pages(n, c["page"]) for n, gone in zip(lens, left) if not gone)
    # live pages lie evenly over the pool: those above `live` move
    moved = live * (total - live) // total
    return {"bytes": 2 * moved * page + 8 * total, "flops": 0}


# ------------------------------------------------------------- inputs

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": c}

    def normal(shape, dtype, mul=1.0):
        x = torch.empty(shape, device="cuda", dtype=torch.float16 if dtype == "e4m3" else DT[dtype])
        x.normal_(0.0, mul, generator=g)
        return x.to(DT[dtype])

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32)

    def table_of(counts, n_pages, width):
        """rows of `counts` pages each, from anywhere in the pool"""
        ids, tab = shuffled(n_pages), torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
        n = torch.tensor(counts, device="cuda")
        used = torch.arange(width, device="cuda")[None] < n[:, None]
        tab[used] = ids[:sum(counts)]
        return tab

    if c["op"] == "attend":
        lens = _lens(c, c["rows"])
        counts = [_pages(n, c["page"]) for n in lens]
        n_pages = sum(counts) + 5
        s["k"] = normal((n_pages, c["hkv"], c["page"], c["d"]), c["kv"])
        s["v"] = normal((n_pages, c["hkv"], c["page"], c["d"]), c["kv"])
        s["table"] = table_of(counts, n_pages, max(counts))
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["q"] = normal((c["rows"], c["n_q"], c["hq"], c["d"]), c["q"], 2.0)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((c["rows"], c["n_q"], c["hq"]), dtype=torch.float32, device="cuda")
        s["sinks"] = normal((c["hq"],), "f32") if c["sinks"] else None
        s["ks"] = s["vs"] = None
        if c["kv"] == "e4m3":
            s["ks"] = torch.rand((c["hkv"],), generator=g, device="cuda") * 0.5 + 0.5
            s["vs"] = torch.rand((c["hkv"],), generator=g, device="cuda") * 0.5 + 0.5
        return s
    if c["op"] == "append":
        t = c["rows"] * c["n_q"]
        start = torch.randint(0, 8192, (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        s["pos"] = (start[:, None] + torch.arange(c["n_q"], device="cuda", dtype=torch.int32)[None]).reshape(-1).contiguous()
        s["seq"] = torch.arange(c["rows"], device="cuda", dtype=torch.int32).repeat_interleave(c["n_q"])
        # only the pages that the new tokens reach are held; those before them belong to another part of the pool
        per = c["n_q"] // c["page"] + 2
        n_pages = c["rows"] * per
        width = (8192 + c["n_q"]) // c["page"] + 2
        s["table"] = torch.full((c["rows"], width), -1, dtype=torch.int32, device="cuda")
        at = (start // c["page"]).long()[:, None] + torch.arange(per, device="cuda")[None]
        at = at.clamp(max=width - 1)
        s["table"].scatter_(1, at, shuffled(n_pages).view(c["rows"], per))
        s["k"] = normal((n_pages, c["hkv"], c["page"], c["d"]), c["kv"])
        s["v"] = normal((n_pages, c["hkv"], c["page"], c["d"]), c["kv"])
        qkv = normal((t, (c["hq"] + 2 * c["hkv"]) * c["d"]), c["x"])  # one projection's rows: q, k and v side by side
        s["qkv"] = qkv
        cut = [c["hq"] * c["d"], c["hkv"] * c["d"], c["hkv"] * c["d"]]
        q, k, v = qkv.split(cut, dim=1)
        s["q_in"], s["k_in"], s["v_in"] = q.unflatten(1, (-1, c["d"])), k.unflatten(1, (-1, c["d"])), v.unflatten(1, (-1, c["d"]))
        s["q_out"] = torch.empty((t, c["hq"], c["d"]), device="cuda", dtype=DT[c["x"]])
        half = c["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        ang = torch.arange(8192 + c["n_q"], device="cuda", dtype=torch.float64)[:, None] * freq[None]
        s["cos_sin"] = torch.stack((ang.cos(), ang.sin()), 1).to(torch.float32).contiguous()  # [pos][cos, sin][half]
        return s
    p = c["page"]
    if c["op"] == "fork":
        lens, src, new = _turn(c)
        counts = [_pages(n, p) for n in lens]
        n_pages, width = sum(counts) + 2 * len(lens), max(counts) + 2
        s["src"] = torch.tensor(src, dtype=torch.int32, device="cuda")
        s["rows"] = torch.arange(len(lens), dtype=torch.int32, device="cuda")
        s["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        held = counts
    else:
        lens, left = _lens(c, c["rows"]), _left(c)
        counts = [_pages(n, p) for n in lens]
        n_pages, width = sum(counts) + 7, max(counts)
        held = [0 if gone else n for n, gone in zip(counts, left)]
        lens = [0 if gone else n for n, gone in zip(lens, left)]
    tab = table_of(counts, n_pages, width)
    tab[torch.arange(width, device="cuda")[None] >= torch.tensor(held, device="cuda")[:, None]] = -1
    rows = len(lens)
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[tab[tab >= 0].long()] = 1
    # table, lengths and reference counts in one buffer, so that one copy takes a pass back to where it began
    s["book0"] = torch.cat((tab.reshape(-1), torch.tensor(lens, dtype=torch.int32, device="cuda"), refs))
    s["book"] = s["book0"].clone()
    s["table"] = s["book"][:rows * width].view(rows, width)
    s["lens"] = s["book"][rows * width:rows * width + rows]
    s["refs"] = s["book"][rows * width + rows:]
    s["data"] = normal((c["layers"], 2, n_pages, c["hkv"], p, c["d"]), c["kv"])
    return s


# ------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    if c["op"] in ("fork", "compact"):
        s["book"].copy_(s["book0"])
    return (_run_own if own else _run_plain)(s, c)


def _run_own(s, c):
    from pulsar_b200 import kv
    h = s.get("handle")
    if c["op"] == "attend":
        if h is None:
            h = s["handle"] = kv.PagedKv(s["k"], s["v"], s["table"], k_scale=s["ks"], v_scale=s["vs"])
        h.attend(s["q"], s["lens"], s["out"], window=c["window"], sinks=s["sinks"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if c["op"] == "append":
        if h is None:
            h = s["handle"] = kv.PagedKv(s["k"], s["v"], s["table"])
        h.append(s["q_in"], s["k_in"], s["v_in"], s["seq"], s["pos"], s["cos_sin"], s["q_out"], interleaved=c["inter"])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if h is None:
        h = s["handle"] = kv.KvPool(s["data"], s["table"], s["lens"], s["refs"])
    if c["op"] == "fork":
        h.fork(s["src"], s["rows"])
        h.grow(s["new"], s["rows"])
    else:
        h.compact()
    return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "data": s["data"]}


def _run_plain(s, c):
    return {"attend": _attend, "append": _append, "fork": _fork, "compact": _compact}[c["op"]](s, c)


def _attend(s, c):
    rows, n_q, hq, hkv, d, page = (c[x] for x in ("rows", "n_q", "hq", "hkv", "d", "page"))
    width = s["table"].shape[1]
    at = s["table"].clamp(min=0).long()
    keys = width * page
    k = s["k"][at].permute(0, 2, 1, 3, 4).reshape(rows, hkv, keys, d).float()
    v = s["v"][at].permute(0, 2, 1, 3, 4).reshape(rows, hkv, keys, d).float()
    if s["ks"] is not None:
        k, v = k * s["ks"].view(1, -1, 1, 1), v * s["vs"].view(1, -1, 1, 1)
    j = torch.arange(keys, device="cuda")
    hi = s["lens"][:, None] - (n_q - 1 - torch.arange(n_q, device="cuda"))[None]     # [rows][n_q]
    lo = (hi - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(hi)
    seen = (j >= lo[..., None]) & (j < hi[..., None])                                 # [rows][n_q][keys]
    group = hq // hkv
    q = s["q"].float().view(rows, n_q, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(rows, hkv, n_q * group, d)
    sc = (q @ k.transpose(2, 3)).view(rows, hkv, n_q, group, keys) * (d ** -0.5)
    sc = torch.where(seen[:, None, :, None, :], sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(sc - m)
    den = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        den = den + torch.exp(s["sinks"].view(1, hkv, 1, group, 1) - m)
    o = (p.view(rows, hkv, n_q * group, keys) @ v).view(rows, hkv, n_q, group, d)
    o = torch.where(den > 0, o / den, 0.0)
    lse = torch.log(den) + m
    empty = ~seen.any(-1)[:, None, :, None, None]
    lse = torch.where(empty, -math.inf, lse)
    s["out"].copy_(o.permute(0, 2, 1, 3, 4).reshape(rows, n_q, hq, d))
    s["lse"].copy_(lse[..., 0].permute(0, 2, 1, 3).reshape(rows, n_q, hq))
    return {"out": s["out"], "lse": s["lse"]}


def _rotated(x, cos, sin, rot, inter):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    y, z = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((y, z), -1).flatten(-2) if inter else torch.cat((y, z), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _append(s, c):
    pos, seq = s["pos"].long(), s["seq"].long()
    cs = s["cos_sin"][pos]
    cos, sin = cs[:, 0][:, None], cs[:, 1][:, None]
    s["q_out"].copy_(_rotated(s["q_in"].float(), cos, sin, c["rot"], c["inter"]))
    k = _rotated(s["k_in"].float(), cos, sin, c["rot"], c["inter"])
    at, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k"][at, :, slot] = k.to(s["k"].dtype)
    s["v"][at, :, slot] = s["v_in"].float().to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _fork(s, c):
    tab, lens, refs, p = s["table"], s["lens"], s["refs"], c["page"]
    rows, width = tab.shape
    src, dst = s["src"].long(), s["rows"].long()
    i = torch.arange(rows, device="cuda")
    j = torch.arange(width, device="cuda")
    from_row = src.clamp(min=0)
    n = torch.where(src >= 0, lens[from_row], 0)
    new, old = tab[from_row], tab[dst]
    used, had = j[None] < ((n + p - 1) // p)[:, None], j[None] < ((lens[dst] + p - 1) // p)[:, None]
    part = (n % p != 0) & (src >= 0)
    # a partly filled page stays with its own row, or with the first row that continues it
    stays = torch.zeros(rows + 1, dtype=torch.bool, device="cuda")
    stays[torch.where(src == dst, src, rows)] = True
    first = torch.full((rows,), rows, device="cuda").scatter_reduce(0, from_row, torch.where(src >= 0, i, rows), "amin")
    keeps = (src == dst) | (~stays[:rows][from_row] & (first[from_row] == i))
    need = part & ~keeps
    free = torch.sort((refs != 0).to(torch.int32), stable=True).indices
    fresh = free[(need.cumsum(0) - 1).clamp(min=0)]
    last = (n // p).clamp(max=width - 1)
    was = new.gather(1, last[:, None].long())[:, 0]
    now = torch.where(need, fresh.to(torch.int32), was)
    move = need.nonzero()[:, 0]
    s["data"][:, :, now[move].long()] = s["data"][:, :, was[move].long()]
    new = torch.where(need[:, None] & (j[None] == last[:, None]), now[:, None], new)
    count = torch.zeros_like(refs)
    count.index_add_(0, torch.where(used, new, 0).reshape(-1).long(), used.reshape(-1).to(torch.int32))
    count.index_add_(0, torch.where(had, old, 0).reshape(-1).long(), -had.reshape(-1).to(torch.int32))
    refs += count
    tab[dst] = torch.where(used, new, -1)
    lens[dst] = n.to(torch.int32)
    # growth: fresh pages for the new tokens, lowest first
    n, more = lens[dst], s["new"]
    a, b = (n + p - 1) // p, (n + more + p - 1) // p
    free = torch.sort((refs != 0).to(torch.int32), stable=True).indices.to(torch.int32)
    off = (b - a).cumsum(0) - (b - a)
    want = (j[None] >= a[:, None]) & (j[None] < b[:, None])
    pick = free[(off[:, None] + j[None] - a[:, None]).clamp(0, refs.numel() - 1).long()]
    tab[dst] = torch.where(want, pick, tab[dst])
    refs.index_add_(0, torch.where(want, pick, 0).reshape(-1).long(), want.reshape(-1).to(torch.int32))
    lens[dst] = n + more
    return {"table": tab, "lens": lens, "refs": refs, "data": s["data"]}


def _compact(s, c):
    tab, lens, refs, p = s["table"], s["lens"], s["refs"], c["page"]
    live = refs > 0
    ids = torch.arange(refs.numel(), device="cuda")
    n_live = live.sum()
    movers, holes = (live & (ids >= n_live)).nonzero()[:, 0], (~live & (ids < n_live)).nonzero()[:, 0]
    to = ids.to(torch.int32)
    to[movers] = holes.to(torch.int32)
    s["data"][:, :, holes] = s["data"][:, :, movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    used = torch.arange(tab.shape[1], device="cuda")[None] < ((lens + p - 1) // p)[:, None]
    tab.copy_(torch.where(used, to[tab.clamp(min=0).long()], tab))
    return {"table": tab, "lens": lens, "refs": refs, "data": s["data"]}


# ------------------------------------------------------------- in 64 bits, from the definitions

def exact(c, seed):
    s = prepare(c, seed)
    return {"attend": _exact_attend, "append": _exact_append, "fork": _exact_pages, "compact": _exact_pages}[c["op"]](s, c)


def _exact_attend(s, c):
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    out = torch.zeros((c["rows"], c["n_q"], hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((c["rows"], c["n_q"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lens(c, c["rows"])):
        ids = s["table"][r, :_pages(n, page)].long()
        k = s["k"][ids].double().transpose(0, 1).reshape(hkv, -1, d)
        v = s["v"][ids].double().transpose(0, 1).reshape(hkv, -1, d)
        if s["ks"] is not None:
            k, v = k * s["ks"].double()[:, None, None], v * s["vs"].double()[:, None, None]
        for i, (lo, hi) in enumerate(_seen(c, n)):
            if hi <= lo:
                continue
            q = s["q"][r, i].double().view(hkv, hq // hkv, d)
            a = torch.einsum("hgd,hkd->hgk", q, k[:, lo:hi]) / math.sqrt(d)
            if s["sinks"] is not None:
                a = torch.cat((a, s["sinks"].double().view(hkv, -1, 1)), 2)
            lse[r, i] = torch.logsumexp(a, 2).reshape(-1)
            out[r, i] = torch.einsum("hgk,hkd->hgd", torch.softmax(a, 2)[..., :hi - lo], v[:, lo:hi]).reshape(hq, d)
    return {"out": out, "lse": lse}


def _exact_append(s, c):
    cs = s["cos_sin"].double()[s["pos"].long()]
    turn = torch.complex(cs[:, 0], cs[:, 1])[:, None]                  # [T][1][rot / 2]
    half, rot = c["rot"] // 2, c["rot"]

    def turned(x):
        x = x.double().clone()
        i = torch.arange(half, device="cuda")
        a, b = (2 * i, 2 * i + 1) if c["inter"] else (i, i + half)
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
        return x

    assert rot <= c["d"]
    k, v = s["k"].double(), s["v"].double()
    where = s["table"].cpu()[s["seq"].cpu().long(), s["pos"].cpu().long() // c["page"]].cuda().long()
    flat = where * c["page"] + s["pos"].long() % c["page"]
    for cache, x in ((k, turned(s["k_in"])), (v, s["v_in"].double())):
        tokens = cache.permute(0, 2, 1, 3).reshape(-1, c["hkv"], c["d"])
        tokens[flat] = x
        cache.copy_(tokens.view(-1, c["page"], c["hkv"], c["d"]).permute(0, 2, 1, 3))
    return {"q": turned(s["q_in"]), "k": k, "v": v}


def _exact_pages(s, c):
    """the moved pages as values; the tables are whole numbers and need no 64-bit form"""
    p, data = c["page"], s["data"]
    tab, lens, refs = s["table"].cpu().tolist(), s["lens"].cpu().tolist(), s["refs"].cpu().tolist()
    moves = []
    if c["op"] == "fork":
        src = s["src"].cpu().tolist()
        free = [i for i, n in enumerate(refs) if n == 0]
        taken = set(i for i, r in enumerate(src) if i == r)
        for i, r in enumerate(src):
            if r < 0 or lens[r] % p == 0 or r == i:
                continue
            if r in taken:
                moves.append((tab[r][lens[r] // p], free.pop(0)))
            taken.add(r)
    else:
        live = [i for i, n in enumerate(refs) if n > 0]
        holes = [i for i, n in enumerate(refs[:len(live)]) if n == 0]
        moves = list(zip([i for i in live if i >= len(live)], holes))
    at = list(range(len(refs)))
    for a, b in moves:
        at[b] = a
    return {"table": None, "lens": None, "refs": None, "data": data[:, :, torch.tensor(at, device="cuda")].double()}
