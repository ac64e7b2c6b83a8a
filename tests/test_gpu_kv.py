"""The paged cache on the GPU: attention, rotary append and the page
bookkeeping against plain 64-bit forms and a Python model of the pages.

Attention's bound, per value, from the arithmetic alone (u = unit roundoff of
the output type, eps = 2^-24):
  scores   f32 sums of D exact products in chunks: |ds| <= (D / 16 + 20) eps spread,
           plus the split of q (bf16 caches with f32 or f16 q: three bf16 parts, 2^-24; else
           two f16 parts, 2^-22, or exact): 2^-21 spread covers both
  weights  p in two parts: 2^-16 (bf16 cache), 2^-22 (f16 parts); three bf16 parts 2^-23
  sums     (n / 16 + 64) eps of sum p |v|
  |do| <= u |o| + weight * (2 |ds| + parts + sums), and the type's least step
"""
import math

import pytest

import kv_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
EPS = 2.0 ** -24
STEP = {F32: 1e-37, BF16: 1e-37, F16: 2.0 ** -24}


@pytest.fixture(scope="module")
def kv():
    from pulsar_b200 import kv as m
    m.kv_error()
    return m


def values(shape, dtype, gen, mul=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * mul).to(dtype)


def cache(lens, n_kv, D, page, dtype, gen, stale=True, tokens_first=False, spare=3):
    """pages scattered over a pool, unheld pages and the ends of last pages full of NaN (e4m3: too)"""
    counts = [-(-max(n, 0) // page) for n in lens]
    n_pages = sum(counts) + spare
    shape = (n_pages, page, n_kv, D) if tokens_first else (n_pages, n_kv, page, D)
    k, v = (values(shape, F32, gen).to(dtype) for _ in range(2))
    if tokens_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(counts + [1]) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    if stale:
        nan = torch.tensor(math.nan, device="cuda").to(dtype)
        seen = torch.zeros((n_pages, page), dtype=torch.bool, device="cuda")
        for r, n in enumerate(lens):
            for j in range(counts[r]):
                seen[table[r, j].long(), :n - j * page] = True
        for t in (k, v):
            x = t.transpose(1, 2)
            if dtype == E4M3:
                x = x.view(torch.uint8)
                x[~seen] = nan.view(torch.uint8)
            else:
                x[~seen] = nan
    return k, v, table


def held(got, lse, want, q_type, c_type, n_max, D):
    out, ref_lse, wgt, spr = want
    ds = (D / 16 + 20) * EPS * spr + 2.0 ** -21 * spr
    parts = {BF16: 2.0 ** -23 if q_type != BF16 else 2.0 ** -16}.get(c_type, 2.0 ** -22)
    rel = 2 * ds[..., None] + parts + (n_max / 16 + 64) * EPS
    err = (got.double().cpu() - out).abs()
    top = kv_ref.U[q_type] * out.abs() + wgt * rel + STEP[q_type]
    assert torch.isfinite(got).all()
    assert (err <= top).all(), float((err / top).max())
    if lse is not None:
        x = lse.double().cpu()
        assert torch.equal(torch.isinf(x), torch.isinf(ref_lse))
        fine = ~torch.isinf(ref_lse)
        e = (x - ref_lse)[fine].abs()
        bound = (ds + (n_max / 16 + 64) * EPS + 4 * EPS * ref_lse.abs())[fine]
        assert (e <= bound).all(), float((e / bound).max())


# (lens, n_q, n_head, n_kv, D, page, window, sinks, q type, cache type)
CASES = [
    ([1], 1, 1, 1, 16, 1, 0, False, F32, F16),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 129], 1, 8, 2, 64, 16, 0, False, BF16, BF16),
    ([0, 5, 100, 1000], 1, 8, 8, 128, 16, 0, True, F32, BF16),
    ([7, 300, 41], 1, 9, 3, 80, 7, 0, False, F32, F16),
    ([257, 0, 511], 1, 16, 1, 128, 24, 100, True, F16, F16),
    ([1030, 77], 1, 33, 1, 48, 64, 0, False, BF16, BF16),
    ([500, 499, 3], 3, 14, 2, 96, 32, 0, False, F16, BF16),
    ([2, 1, 0, 90], 5, 12, 4, 112, 8, 0, True, F32, F16),
    ([64, 2000], 4, 32, 2, 128, 16, 50, False, BF16, E4M3),
    ([333, 12, 1], 1, 8, 1, 192, 33, 0, False, F32, E4M3),
    ([700, 130], 1, 20, 2, 256, 16, 0, True, BF16, BF16),
    ([190, 65], 2, 24, 2, 256, 128, 1, False, F32, F16),
    ([4097, 9000], 1, 16, 2, 128, 64, 0, False, F32, BF16),
    ([9001, 4, 20000], 1, 8, 1, 64, 16, 0, True, F16, E4M3),
    ([40] * 70, 1, 4, 2, 32, 16, 0, False, BF16, F16),
    ([130, 131], 64, 4, 1, 64, 16, 0, False, F32, F16),
    ([30] * 3 + [1] * 9 + [2500], 1, 64, 8, 64, 16, 128, True, BF16, BF16),
    # the workers' three ways of sharing a call: whole short segments a warp, segments cut among CTAs, equal slices;
    # batches beyond what a CTA keeps of the lengths
    ([20 + 3 * i % 90 for i in range(200)], 1, 24, 2, 64, 16, 0, False, BF16, F16),
    ([1 + 7 * i % 40 for i in range(300)], 1, 2, 1, 128, 16, 0, True, F32, F16),
    ([i % 5 for i in range(5000)], 1, 1, 1, 16, 4, 0, False, BF16, BF16),
    ([250 + 61 * i % 2250 for i in range(40)], 1, 8, 8, 64, 16, 0, False, F16, F16),
    ([250 + 61 * i % 2250 for i in range(40)], 1, 80, 8, 128, 32, 0, False, BF16, BF16),
    ([900 + 331 * i % 2000 for i in range(30)], 2, 10, 10, 256, 16, 700, False, F32, E4M3),
    ([100000], 1, 2, 1, 128, 64, 0, False, F32, BF16),
    # heads of 129 to 192, pages of multiples of 8 and of none
    ([700, 33, 2041], 2, 12, 2, 192, 24, 0, False, F32, BF16),
    ([190, 65, 16, 15], 1, 3, 3, 176, 8, 50, True, F16, F16),
    ([500, 77, 31], 1, 20, 2, 256, 10, 0, False, BF16, BF16),
    ([900, 9], 1, 5, 1, 144, 3, 0, True, F32, F16),
    ([1200, 640], 3, 16, 2, 64, 8, 0, False, F32, E4M3),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_attend(kv, i):
    lens, n_q, H, n_kv, D, page, window, with_sinks, qt, ct = CASES[i]
    gen = torch.Generator(device="cuda").manual_seed(100 + i)
    k, v, table = cache(lens, n_kv, D, page, ct, gen)
    q = values((len(lens), n_q, H, D), qt, gen, 1.5)
    sinks = values((H,), F32, gen) if with_sinks else None
    ks = vs = None
    if ct == E4M3:
        ks, vs = (torch.rand(n_kv, generator=gen, device="cuda") + 0.25 for _ in range(2))
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, math.nan)
    lse = torch.full((len(lens), n_q, H), math.nan, device="cuda")
    c = kv.PagedKv(k, v, table, ks, vs)
    c.attend(q, n, out, window=window, sinks=sinks, lse=lse)
    assert kv.kv_error() == 0
    want = kv_ref.attend(q, k, v, table, lens, window=window, sinks=sinks, k_scale=ks, v_scale=vs)
    held(out, lse, want, qt, ct, max(lens), D)
    assert int(c._ws[:kv.WS_ZEROED].to(torch.int32).sum()) == 0
    again = torch.zeros_like(out)
    c.attend(q, n, again, window=window, sinks=sinks)
    assert torch.equal(out, again)  # the order of the sums is fixed


def test_attend_strides_rows_and_padding(kv):
    """q and out inside wider buffers, tokens-first cache pages, rows that share a table row, padding rows, a
    prompt's tokens as rows of their own"""
    gen = torch.Generator(device="cuda").manual_seed(7)
    lens, H, n_kv, D, page = [50, 200], 8, 2, 64, 16
    k, v, table = cache(lens, n_kv, D, page, BF16, gen, tokens_first=True)
    seq = torch.tensor([1, -1, 0, 1, 1, 0], dtype=torch.int32, device="cuda")
    rows = [200, 9, 50, 199, 1, 17]
    wide = values((6, 3 * H * D), BF16, gen)
    q = wide[:, H * D:2 * H * D].unflatten(1, (H, D))
    o_wide = torch.full((6, 2 * H * D + 8), 7.0, dtype=BF16, device="cuda")
    out = o_wide[:, 8:8 + H * D].unflatten(1, (H, D))
    c = kv.PagedKv(k, v, table)
    lse = torch.zeros((6, H), device="cuda")
    c.attend(q, torch.tensor(rows, dtype=torch.int32, device="cuda"), out, seq=seq, lse=lse)
    # the stale bytes past a row's shorter length are another length's keys here, so NaN free
    want = kv_ref.attend(q.unsqueeze(1), k, v, table, rows, seq=seq.tolist())
    held(out.unsqueeze(1), lse.unsqueeze(1), want, BF16, BF16, 200, D)
    assert (o_wide[:, :8] == 7).all() and (o_wide[:, 8 + H * D:] == 7).all()
    assert (out[1] == 0).all() and torch.isinf(lse[1]).all()


def test_attend_extreme_scores(kv):
    """scores of +-500 (no overflow, one key takes all), equal scores (a plain mean), a -inf key (weight 0), and
    NaN or inf in a seen key spreads to its row alone"""
    gen = torch.Generator(device="cuda").manual_seed(8)
    lens, H, n_kv, D, page = [300, 300, 300, 300], 4, 1, 64, 16
    k, v, table = cache(lens, n_kv, D, page, F16, gen)
    q = values((4, 1, H, D), F32, gen)
    q[0] *= 400.0
    q[1] = 0.0
    q[2] = q[2].abs() + 0.1
    k[table[2, 3].long(), 0, 5, 0] = -math.inf
    k[table[3, 0].long(), 0, 0, 0] = math.nan
    c = kv.PagedKv(k, v, table)
    out = torch.zeros_like(q)
    c.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), out)
    want = kv_ref.attend(q[:2], k, v, table, lens[:2])
    held(out[:2], None, want, F32, F16, 300, D)
    mean = torch.cat([v[p, 0].double() for p in table[1, :19].long()])[:300].mean(0).cpu()
    assert (out[1, 0, 0].double().cpu() - mean).abs().max() < 1e-6
    assert torch.isfinite(out[2]).all()
    k2 = k.clone()
    k2[table[2, 3].long(), 0, 5, 0] = -60000.0  # as good as -inf
    w2 = kv_ref.attend(q[2:3], k2, v, table, lens[:1], seq=[2])
    assert (out[2].double().cpu() - w2[0][0]).abs().max() < 1e-5
    assert torch.isnan(out[3]).all()


@pytest.mark.parametrize("ct,H,n_kv,D,n_q,window", [(BF16, 4, 2, 128, 3, 0), (F16, 12, 1, 64, 4, 40), (E4M3, 8, 2, 80, 3, 0),
                                                    (BF16, 3, 1, 256, 5, 33), (E4M3, 20, 2, 192, 2, 64), (F16, 2, 1, 192, 3, 0)])
def test_drafts_do_not_share_their_faults(kv, ct, H, n_kv, D, n_q, window):
    """NaN (e4m3: NaN, 16 bits: infinities too) in keys and values that only some of a sequence's new tokens see: the
    others' outputs are what they are without"""
    gen = torch.Generator(device="cuda").manual_seed(60)
    lens, page = [70, 2, 200], 8
    k, v, table = cache(lens, n_kv, D, page, ct, gen)
    q = values((3, n_q, H, D), BF16, gen)
    ks = torch.ones(n_kv, device="cuda") if ct == E4M3 else None
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    bad = torch.tensor([math.nan if ct == E4M3 else math.inf, math.nan], device="cuda").to(ct)
    want = kv_ref.attend(q, k, v, table, lens, window=window, k_scale=ks, v_scale=ks)
    sees = torch.ones((3, n_q), dtype=torch.bool)
    for b, m in enumerate(lens):
        spots = [m - 1]                                   # the last new token's own key
        if window and m > window + n_q:
            spots.append(m - n_q - window + 1)            # the first token's window begins there, the others' later
        for x, j in enumerate(spots):
            p, o = table[b, j // page].long(), j % page
            for t in (k, v):
                raw = t.view(torch.uint8) if ct == E4M3 else t
                raw[p, :, o, 5 + x] = bad[x].view(torch.uint8) if ct == E4M3 else bad[x]
        for i in range(n_q):
            hi = m - (n_q - 1 - i)
            lo = max(0, hi - window) if window else 0
            sees[b, i] = any(lo <= j < hi for j in spots)
    out = torch.zeros_like(q)
    kv.PagedKv(k, v, table, ks, ks).attend(q, n, out, window=window)
    got = out.cpu()
    assert (~sees).any()
    for b in range(3):
        for i in range(n_q):
            if sees[b, i]:
                assert not torch.isfinite(got[b, i].float()).all(-1).any()
            else:
                w = tuple(z[b:b + 1, i:i + 1] for z in want)
                held(got[b:b + 1, i:i + 1], None, w, BF16, ct, 200, D)


def test_attend_past_32_bits(kv):
    """pages whose offsets pass 2^32 values, in a cache of 2^32 + values"""
    D, page, n_kv, H = 128, 64, 8, 16
    n_pages = (1 << 32) // (D * page * n_kv) + 4
    gen = torch.Generator(device="cuda").manual_seed(9)
    k = torch.empty((n_pages, n_kv, page, D), dtype=E4M3, device="cuda")
    v = torch.empty_like(k)
    ids = [n_pages - 1, 3, n_pages - 3, 0, n_pages // 2]
    for t in (k, v):
        for i in ids:
            t[i] = values((n_kv, page, D), F32, gen).to(E4M3)
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    q = values((1, 1, H, D), BF16, gen)
    out = torch.zeros_like(q)
    kv.PagedKv(k, v, table).attend(q, torch.tensor([300], dtype=torch.int32, device="cuda"), out)
    held(out, None, kv_ref.attend(q, k, v, table, [300]), BF16, E4M3, 300, D)
    pos = torch.arange(256, 259, dtype=torch.int32, device="cuda")
    x = values((3, n_kv, D), F32, gen)
    kv.PagedKv(k, v, table[:, :].flip(1).contiguous()).append(None, x, x, torch.zeros_like(pos), pos, None, None)
    got = k[n_pages - 1, :, :3].float()
    assert (got - x.transpose(0, 1)).abs().max() <= 2.0 ** -4 * x.abs().max()


@pytest.mark.parametrize("rows", [None, [3, 0, 3, 9, 1, 2, 3, 4, 5, 9, 7, 8, 0]])
def test_attend_in_several_launches(kv, rows):
    """rows so long (by the table's width) that the call takes a few of them at a time"""
    D, page, n_kv, n = 16, 1 << 20, 8, 10
    gen = torch.Generator(device="cuda").manual_seed(12)
    k, v = (values((3, n_kv, page, D), F32, gen).to(E4M3) for _ in range(2))
    table = torch.full((n, 2047), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(n, device="cuda", dtype=torch.int32) % 3
    lens = [40 + 9 * i for i in range(n if rows is None else len(rows))]
    q = values((len(lens), 1, n_kv, D), BF16, gen)
    out, lse = torch.zeros_like(q), torch.zeros((len(lens), 1, n_kv), device="cuda")
    seq = None if rows is None else torch.tensor(rows, dtype=torch.int32, device="cuda")
    kv.PagedKv(k, v, table).attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, lse=lse, seq=seq)
    small = torch.stack([t[:, :, :200].contiguous() for t in (k, v)])
    held(out, lse, kv_ref.attend(q, small[0], small[1], table[:, :1], lens, seq=rows), BF16, E4M3, 200, D)


def test_attend_streams_and_graph(kv):
    """on a side stream, and captured once and replayed over a growing cache"""
    gen = torch.Generator(device="cuda").manual_seed(10)
    lens, H, n_kv, D, page = [90, 400], 8, 2, 128, 16
    k, v, table = cache(lens, n_kv, D, page, BF16, gen)
    q = values((2, H, D), BF16, gen)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, first = torch.zeros_like(q), torch.zeros_like(q)
    c = kv.PagedKv(k, v, table)
    c.attend(q, n, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.attend(q, n, out, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attend(q, n, out)
    for step in ([90, 400], [1, 17], [64, 399]):
        n.copy_(torch.tensor(step, dtype=torch.int32))
        g.replay()
        held(out.unsqueeze(1), None, kv_ref.attend(q.unsqueeze(1), k, v, table, step), BF16, BF16, 400, D)


def test_attend_device_checks(kv):
    """out-of-range pages, lengths and rows are not followed, and are told"""
    gen = torch.Generator(device="cuda").manual_seed(11)
    lens, H, n_kv, D, page = [64, 64, 64], 4, 2, 64, 16
    k, v, table = cache(lens, n_kv, D, page, BF16, gen)
    q = values((3, 1, H, D), BF16, gen)
    good = table.clone()
    table[1, 2] = 1 << 30
    out = torch.zeros_like(q)
    c = kv.PagedKv(k, v, table)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.attend(q, n, out)
    assert kv.kv_error() == kv.ERR_PAGE and kv.kv_error() == 0
    held(out[:1], None, kv_ref.attend(q[:1], k, v, good, lens[:1]), BF16, BF16, 64, D)
    # the 16 keys of the missing page are left out
    short = good.clone()
    short[1, 2] = good[1, 3]
    held(out[1:2], None, kv_ref.attend(q[1:2], k, v, short, [48], seq=[1]), BF16, BF16, 64, D)
    c2 = kv.PagedKv(k, v, good[:, :4].contiguous())
    c2.attend(q, torch.tensor([64, 65, 1 << 30], dtype=torch.int32, device="cuda"), out)
    assert kv.kv_error() == kv.ERR_SPAN
    held(out, None, kv_ref.attend(q, k, v, good, lens), BF16, BF16, 64, D)
    c2.attend(q, n, out, seq=torch.tensor([0, 3, 2], dtype=torch.int32, device="cuda"))
    assert kv.kv_error() == kv.ERR_ROW and (out[1] == 0).all()


# ------------------------------------------------------------------ append

# (T, n_head, n_kv, D, rot, interleaved, page, x type, q_out type, cache type)
APPENDS = [
    (1, 4, 1, 64, 64, False, 16, BF16, BF16, BF16),
    (33, 7, 2, 80, 20, True, 7, F32, BF16, F16),
    (100, 8, 4, 128, 64, False, 16, F32, F32, BF16),
    (257, 3, 1, 96, 24, False, 1, F16, F16, F16),
    (64, 16, 2, 256, 256, True, 32, BF16, F32, E4M3),
    (20, 2, 2, 16, 2, False, 5, F32, F16, E4M3),
    (20, 2, 1, 48, 6, True, 5, F16, BF16, BF16),
    (9, 5, 3, 112, 0, False, 24, BF16, BF16, F16),
    (700, 32, 8, 128, 128, False, 64, F32, F32, F16),
]


@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append(kv, i):
    T, H, n_kv, D, rot, inter, page, xt, qt, ct = APPENDS[i]
    gen = torch.Generator(device="cuda").manual_seed(200 + i)
    n_seq = 3
    per = -(-T // n_seq)
    seq = torch.arange(T, device="cuda", dtype=torch.int32) % n_seq
    pos = torch.arange(T, device="cuda", dtype=torch.int32) // n_seq + 5
    width = (per + 5) // page + 1
    n_pages = n_seq * width
    table = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32).view(n_seq, width)
    skip = [0, 2] if T > 5 else []
    if skip:
        pos[skip[0]] = -1
        seq[skip[1]] = -4
    k, v = (torch.zeros((n_pages, n_kv, page, D), device="cuda").to(ct) for _ in range(2))
    qkv = values((T, (H + 2 * n_kv) * D), xt, gen, 2.0)
    q, kx, vx = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, n_kv * D, n_kv * D], 1))
    ks = vs = None
    if ct == E4M3:
        ks, vs = (torch.rand(n_kv, generator=gen, device="cuda") * 0.02 + 0.01 for _ in range(2))
    cs = kv.rope_table(per + 6, rot) if rot else None
    q_out = torch.full((T, H, D), 3.0, device="cuda", dtype=qt)
    kv.PagedKv(k, v, table, ks, vs).append(q, kx, vx, seq, pos, cs, q_out, interleaved=inter)
    assert kv.kv_error() == 0
    keep = [t for t in range(T) if t not in skip]
    # one product pair and a sum: three roundings of at most the terms' size, then the output's
    want, mag = kv_ref.turn(q, pos, cs, inter)
    err = (q_out.double().cpu() - want).abs()
    top = kv_ref.U[qt] * want.abs() + 3 * EPS * mag + STEP[qt]
    assert (err[keep] <= top[keep]).all()
    assert (q_out[skip] == 3).all()
    seqs, ps = seq.tolist(), pos.tolist()
    tab = table.cpu()
    for name, got, x, sc in (("k", k, kx, ks), ("v", v, vx, vs)):
        want, mag = kv_ref.turn(x, pos, cs if name == "k" else None, inter)
        if sc is not None:
            want, mag = want / sc.double().cpu()[:, None], mag / sc.double().cpu()[:, None]
            want, mag = want.clamp(-448, 448), mag.clamp(max=900)
        got = got.double().cpu()
        left = got.abs().sum()
        for t in keep:
            g = got[tab[seqs[t], ps[t] // page].long(), :, ps[t] % page]
            step = 2.0 ** -10 if ct == E4M3 else STEP[ct]
            top = kv_ref.U[ct] * want[t].abs() + 5 * EPS * mag[t] * (1 + kv_ref.U[ct]) + step
            assert ((g - want[t]).abs() <= top).all(), (name, t)
            left = left - g.abs().sum()
        assert abs(float(left)) <= 1e-9 * float(got.abs().sum())  # nothing else was written


def test_append_in_place_strided_and_told(kv):
    gen = torch.Generator(device="cuda").manual_seed(31)
    T, H, n_kv, D, page = 12, 3, 1, 32, 4
    x = values((T, 5 * D + 1), F32, gen)  # odd stride: no wide loads
    q, k, v = x[:, :3 * D].unflatten(1, (3, D)), x[:, 3 * D:4 * D].unflatten(1, (1, D)), x[:, 4 * D:5 * D].unflatten(1, (1, D))
    ck, cv = (torch.zeros((4, n_kv, page, D), device="cuda", dtype=F16) for _ in range(2))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    pos, seq = torch.arange(T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    cs = kv.rope_table(T, D)
    want, _ = kv_ref.turn(q, pos, cs, False)
    c = kv.PagedKv(ck, cv, table)
    c.append(q, k, v, seq, pos, cs, q)  # q_out is q
    assert (q.double().cpu() - want).abs().max() < 1e-5
    assert torch.equal(cv[[2, 0, 1]].transpose(1, 2).reshape(T, n_kv, D), v.to(F16))
    before = ck.clone(), cv.clone()
    bad = torch.full((1,), 12, dtype=torch.int32, device="cuda")
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.append(None, k[:1], v[:1], one, bad, None, None)          # past the table
    assert kv.kv_error() == kv.ERR_SPAN
    c.append(None, k[:1], v[:1], one + 1, one, None, None)      # no such row
    assert kv.kv_error() == kv.ERR_ROW
    c.append(q[:1], k[:1], v[:1], one, one, kv.rope_table(1, D), q[:1].clone())
    assert kv.kv_error() == 0
    kept = ck.clone(), cv.clone()
    c.append(q[:1], k[:1], v[:1], one, one + 1, kv.rope_table(1, D), q[:1].clone())  # past the angles
    assert kv.kv_error() == kv.ERR_SPAN
    assert torch.equal(ck, kept[0]) and torch.equal(cv, kept[1])
    table[0, 0] = 4
    c.append(None, k[:1], v[:1], one, one, None, None)
    assert kv.kv_error() == kv.ERR_PAGE
    assert torch.equal(ck[[2, 0, 1, 3]][1:], before[0][[2, 0, 1, 3]][1:]) and torch.equal(cv[0], before[1][0])


# ------------------------------------------------------------------ pages

def same(pool, model):
    table, lens, refs = pool.table.tolist(), pool.lens.tolist(), pool.refs.tolist()
    assert lens == model.lens
    assert refs == model.refs
    for got, want in zip(table, model.table):
        assert got[:len(want)] == want


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("page,n_pages,n_rows,width,seed", [(4, 40, 6, 12, 1), (1, 64, 8, 20, 2), (16, 300, 70, 9, 3),
                                                            (3, 2500, 33, 200, 4)])
def test_pages_follow_the_model(kv, page, n_pages, n_rows, width, seed):
    """random turns: every call's table, lengths, counts and status, and each row's tokens by their bytes"""
    import random
    rng = random.Random(seed)
    pool = kv.KvPool.empty(2, n_pages, page, 1, 16, n_rows, width, dtype=F32 if seed == 1 else F16)
    model = kv_ref.Pages(n_rows, width, n_pages, page)
    story = [[] for _ in range(n_rows)]  # each row's tokens
    stamp = 1
    seen = set()
    for step in range(60):
        what = rng.choice(("grow", "grow", "grow", "fork", "fork", "free", "compact"))
        if what == "grow":
            rows = rng.sample(range(n_rows), rng.randint(1, n_rows))
            n_new = [rng.choice((0, 1, 1, page, rng.randint(0, 3 * page))) for _ in rows]
            st = model.grow(rows, n_new)
            pool.grow(i32(n_new), i32(rows))
            if st == 0:
                for r, n in zip(rows, n_new):
                    for _ in range(n):
                        j = len(story[r])
                        story[r].append(stamp % 2000)
                        pool.data[:, :, model.table[r][j // page], :, j % page] = stamp % 2000
                        stamp += 1
        elif what in ("fork", "free"):
            dst = rng.sample(range(n_rows), rng.randint(1, n_rows))
            src = [-1 if what == "free" or rng.random() < 0.1 else rng.randrange(n_rows) for _ in dst]
            st, _ = model.fork(src, dst)
            if what == "free":
                pool.free(i32(dst))
            else:
                pool.fork(i32(src), i32(dst))
            if st == 0:
                old = [list(x) for x in story]
                for s, d in zip(src, dst):
                    story[d] = list(old[s]) if s >= 0 else []
        else:
            st = 0
            model.compact()
            pool.compact()
        seen.add((what, st))
        assert int(pool.status[{"grow": 0, "fork": 1, "free": 1, "compact": 2}[what], 0]) == st, (step, what)
        same(pool, model)
        if step % 5 == 4:
            data = pool.data[:, :, :, 0, :, 0].cpu()
            for r in range(n_rows):
                got = [data[:, :, model.table[r][j // page], j % page] for j in range(len(story[r]))]
                assert all((g == x).all() for g, x in zip(got, story[r])), (step, r)
    assert ("compact", 0) in seen and ("fork", 0) in seen and ("grow", 0) in seen
    assert kv.kv_error() == 0


@pytest.mark.parametrize("n_rows", [4000, 9000])
def test_pages_of_many_rows(kv, n_rows):
    """more rows than a plan keeps in shared memory (fork's marks, growth's too)"""
    import random
    rng = random.Random(n_rows)
    pool = kv.KvPool.empty(1, 3 * n_rows, 2, 1, 16, n_rows, 4, dtype=F16)
    model = kv_ref.Pages(n_rows, 4, 3 * n_rows, 2)
    for step in range(4):
        rows = rng.sample(range(n_rows), n_rows if step == 0 else 2500)
        n_new = [rng.randint(0, 1 if step else 3) for _ in rows]
        assert model.grow(rows, n_new) == 0
        pool.grow(i32(n_new), i32(rows))
        dst = rng.sample(range(n_rows), 900)
        src = [rng.choice((-1, rng.randrange(n_rows), dst[0], dst[1])) for _ in dst]
        assert model.fork(src, dst)[0] == 0
        pool.fork(i32(src), i32(dst))
        pool.check()
        same(pool, model)
    model.compact()
    pool.compact()
    same(pool, model)
    # a row named twice is found among many
    rows[-1] = rows[0]
    pool.grow(i32(n_new), i32(rows))
    assert int(pool.status[0, 0]) == 3
    dst[-1] = dst[0]
    pool.fork(i32(src), i32(dst))
    assert int(pool.status[1, 0]) == 3
    same(pool, model)


def test_python_refusals(kv):
    """what the wrappers refuse before a launch"""
    gen = torch.Generator(device="cuda").manual_seed(50)
    k, v, table = cache([20, 9], 2, 64, 8, BF16, gen)
    c = kv.PagedKv(k, v, table)
    n = torch.tensor([20, 9], dtype=torch.int32, device="cuda")
    q = values((2, 4, 64), BF16, gen)
    out = torch.zeros_like(q)
    bad = [dict(q=q.double()), dict(out=out.float()), dict(q=q[:, :, :32], out=out[:, :, :32]), dict(lens=n.long()),
           dict(lens=n[:1]), dict(lens=n.cpu()), dict(q=q.transpose(0, 1), out=out.transpose(0, 1)), dict(window=-1),
           dict(sinks=torch.zeros(3, device="cuda")), dict(lse=torch.zeros(2, device="cuda")), dict(q=q.cpu()),
           dict(seq=n.cpu()), dict(q=q[:, ::2], out=out[:, ::2])]
    for kw in bad:
        a = dict(q=q, lens=n, out=out)
        a.update(kw)
        with pytest.raises(ValueError):
            c.attend(a.pop("q"), a.pop("lens"), a.pop("out"), **a)
    with pytest.raises(kv.KernelError):
        c.attend(q[:, :3].contiguous(), n, out[:, :3].contiguous())       # 3 query heads over 2 key heads
    with pytest.raises(kv.KernelError):
        c.attend(q.repeat(2, 1, 1), n.repeat(2), out.repeat(2, 1, 1))      # more rows than the table
    with pytest.raises(kv.KernelError):
        c.attend(q, n, out, ws=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    x, pos = values((2, 2, 64), BF16, gen), torch.zeros(2, dtype=torch.int32, device="cuda")
    cs = kv.rope_table(4, 64)
    for a in ((None, x.float(), x, pos, pos, cs, None), (None, x, x[:1], pos, pos, cs, None), (None, x, x, pos.long(), pos, cs, None),
              (None, x, x, pos, pos, cs.half(), None), (q[:, :, :32], x, x, pos, pos, cs, q), (q, x, x, pos, pos, cs, q[:1])):
        with pytest.raises(ValueError):
            c.append(*a)
    with pytest.raises(kv.KernelError):
        c.append(None, x, x, pos, pos, kv.rope_table(4, 128), None)        # wider than the head
    for a in ((k.float(), v.float(), table), (k, v[:1], table), (k, v, table.long()), (k, v, table[:1].expand(2, -1)),
              (k.transpose(2, 3), v.transpose(2, 3), table), (k, v, table, torch.ones(2, device="cuda"))):
        with pytest.raises(ValueError):
            kv.PagedKv(*a)
    empty = torch.zeros((0, 4, 64), dtype=BF16, device="cuda")
    assert c.attend(empty, n[:0], empty.clone()).numel() == 0 and c.append(None, x[:0], x[:0], pos[:0], pos[:0], cs, None) is None
    assert kv.kv_error() == 0


def test_pages_refusals_change_nothing(kv):
    pool = kv.KvPool.empty(1, 6, 4, 1, 16, 4, 3)
    pool.grow(i32([6, 3]), i32([0, 2]))
    keep = pool.table.clone(), pool.lens.clone(), pool.refs.clone()

    def unchanged(i, code):
        assert int(pool.status[i, 0]) == code
        assert torch.equal(keep[0], pool.table) and torch.equal(keep[1], pool.lens) and torch.equal(keep[2], pool.refs)

    pool.grow(i32([12, 12]), i32([1, 3]))          # six pages of three
    unchanged(0, 1)
    with pytest.raises(kv.KernelError):
        pool.check()
    pool.grow(i32([7]), i32([0]))                  # 13 tokens in 3 pages of 4
    unchanged(0, 2)
    for rows, n in (([0, 0], [1, 1]), ([4], [1]), ([-1], [1]), ([1], [-1])):
        pool.grow(i32(n), i32(rows))
        unchanged(0, 3)
    for src, dst in (([0, 0], [1, 1]), ([4], [1]), ([-2], [1]), ([0], [4]), ([0], [-1])):
        pool.fork(i32(src), i32(dst))
        unchanged(1, 3)
    pool.grow(i32([10]), i32([1]))
    pool.grow(i32([0]), i32([0]))
    keep = pool.table.clone(), pool.lens.clone(), pool.refs.clone()
    pool.fork(i32([0]), i32([3]))                  # one copy, no free page
    unchanged(1, 1)
    pool.fork(i32([2, 0, 1, -1]), i32([0, 1, 2, 3]))  # a rotation copies nothing
    assert pool.status[1, :2].tolist() == [0, 0]
    assert pool.lens.tolist() == [3, 6, 10, 0]
    pool.lens[0] = 999
    pool.fork(i32([0]), i32([3]))
    assert int(pool.status[1, 0]) == 3


def test_pages_of_odd_bytes(kv):
    """page bytes that are no multiple of 16: copied by bytes"""
    pool = kv.KvPool.empty(3, 9, 3, 1, 1, 3, 4, dtype=F16)
    pool.data.copy_(torch.arange(pool.data.numel(), device="cuda").view(pool.data.shape) % 1999)
    pool.grow(i32([5]), i32([0]))
    was = pool.data.clone()
    pool.fork(i32([0, 0]), i32([1, 2]))
    pool.check()
    t = pool.table.tolist()
    for r in (1, 2):
        assert t[r][0] == t[0][0] and t[r][1] != t[0][1]
        assert torch.equal(pool.data[:, :, t[r][1]], was[:, :, t[0][1]])


def test_pool_calls_in_a_graph(kv):
    """a decode turn (fork, grow) captured once: the replays follow the model"""
    pool = kv.KvPool.empty(1, 64, 4, 1, 16, 4, 8)
    model = kv_ref.Pages(4, 8, 64, 4)
    src, dst, one = i32([0, 0, 2, 2]), i32([0, 1, 2, 3]), i32([1, 1, 1, 1])
    pool.grow(i32([5, 0, 3, 0]))
    model.grow([0, 1, 2, 3], [5, 0, 3, 0])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        pool.fork(src, dst)
        pool.grow(one, dst)
    for parents in ([0, 0, 2, 2], [1, 0, 3, 3], [3, 2, 1, 0]):
        src.copy_(torch.tensor(parents, dtype=torch.int32))
        g.replay()
        assert model.fork(parents, [0, 1, 2, 3])[0] == 0 and model.grow([0, 1, 2, 3], [1] * 4) == 0
        same(pool, model)
    pool.check()


def test_chained_calls_see_each_other(kv):
    """growth, append, attention and forks one behind the other on a stream, nothing between them (the kernels
    overlap): the same bits as with the device waited for after every call"""
    D, n_kv, H, rows, page = 64, 2, 8, 24, 8
    gen = torch.Generator(device="cuda").manual_seed(40)
    steps = 40
    x = values((steps, rows, (H + 2 * n_kv) * D), BF16, gen)
    ids = torch.arange(rows, dtype=torch.int32, device="cuda")
    one = torch.ones(rows, dtype=torch.int32, device="cuda")
    perm = torch.stack([torch.randint(0, rows, (rows,), generator=gen, device="cuda") for _ in range(steps)]).to(torch.int32)
    cs = kv.rope_table(steps + 1, D)

    def run(wait):
        pool = kv.KvPool.empty(1, 600, page, n_kv, D, rows, 8)
        layer, outs = pool.layer(0), []
        turned = torch.zeros((rows, H, D), dtype=BF16, device="cuda")
        pos = [torch.full((rows,), t, dtype=torch.int32, device="cuda") for t in range(steps)]
        cut = [[z.unflatten(1, (-1, D)) for z in x[t].split([H * D, n_kv * D, n_kv * D], 1)] for t in range(steps)]
        outs = [torch.zeros((rows, H, D), dtype=BF16, device="cuda") for _ in range(steps)]
        torch.cuda.synchronize()
        for t in range(steps):
            for f in (lambda: pool.grow(one, ids), lambda: layer.append(*cut[t], ids, pos[t], cs, turned),
                      lambda: layer.attend(turned, pool.lens, outs[t]), lambda: pool.fork(perm[t], ids),
                      lambda: pool.compact() if t % 5 == 4 else None):
                f()
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        pool.check()
        return torch.stack(outs), pool.table.clone(), pool.refs.clone()

    a, b = run(True), run(False)
    assert torch.isfinite(a[0]).all() and kv.kv_error() == 0
    assert all(torch.equal(p, q) for p, q in zip(a, b))
