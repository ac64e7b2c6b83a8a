"""Calls of the paged cache off the beaten track, against the model of the
pages and the plain 64-bit forms."""
import math
import random

import pytest

import kv_ref
from test_gpu_kv import BF16, E4M3, F16, cache, held, i32, same, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from pulsar_b200 import kv as m
    m.kv_error()
    return m


@pytest.mark.parametrize("n,width,layers", [(256, 4, 1), (507, 2, 1), (508, 2, 1), (600, 3, 1), (600, 2, 0), (1024, 2, 1),
                                            (2048, 1, 1), (2048, 1, 0)])
def test_turns_of_many_rows_of_few_pages(kv, n, width, layers):
    """fork and free of up to 2048 rows at once, with slabs and without, against the model and by the pages' bytes"""
    rng = random.Random(n + width + layers)
    page, n_pages = 4, n * width + n
    pool = kv.KvPool.empty(layers, n_pages, page, 1, 16, n, width, dtype=F16)
    model = kv_ref.Pages(n, width, n_pages, page)
    pool.data.copy_((torch.arange(n_pages, device="cuda") % 2000).to(F16).view(1, 1, -1, 1, 1, 1).expand_as(pool.data))
    rows = list(range(n))
    n_new = [rng.randint(0, width * page) for _ in rows]
    assert model.grow(rows, n_new) == 0
    pool.grow(i32(n_new))
    for _ in range(2):
        src = [-1 if rng.random() < 0.1 else rng.choice((r, rng.randrange(n))) for r in rows]
        was = pool.data.clone()
        st, copies = model.fork(src, rows)
        assert st == 0
        pool.fork(i32(src), i32(rows))
        pool.check()
        same(pool, model)
        for a, b in copies:
            was[:, :, b] = was[:, :, a]
        assert torch.equal(pool.data, was)
    assert model.fork([-1] * n, rows)[0] == 0
    pool.free(i32(rows))
    pool.check()
    same(pool, model)
    assert kv.kv_error() == 0


def allocations():
    return torch.cuda.memory_stats()["allocation.all.allocated"]


def test_free_on_another_stream(kv):
    """rows freed on a stream of their own while the current one is busy, and without an allocation"""
    pool = kv.KvPool.empty(1, 64, 4, 1, 16, 8, 8, dtype=F16)
    model = kv_ref.Pages(8, 8, 64, 4)
    side, n_new, gone = torch.cuda.Stream(), i32([5, 9, 1, 32, 4, 0, 7, 12]), i32([6, 1, 3])
    pool.grow(n_new)
    assert model.grow(list(range(8)), n_new.tolist()) == 0
    torch.cuda.synchronize()
    before = allocations()
    torch.cuda._sleep(100_000_000)                       # some 50 ms
    pool.free(gone, stream=side)
    assert allocations() == before
    side.synchronize()
    assert model.fork([-1] * 3, [6, 1, 3])[0] == 0
    same(pool, model)
    pool.check()
    # more rows than there are: refused, not read past the end
    with pytest.raises(kv.KernelError):
        pool.free(i32(list(range(8)) + [0]))
    same(pool, model)


def test_free_of_more_rows_than_a_fork_takes(kv):
    """releases do not depend on one another: any number of rows is one call of free(); a fork says its limit"""
    n = kv.MAX_FORK + 300
    pool = kv.KvPool.empty(1, 3 * n, 2, 1, 16, n, 3, dtype=F16)
    model = kv_ref.Pages(n, 3, 3 * n, 2)
    rows = list(range(n))
    n_new = [r % 6 for r in rows]
    assert model.grow(rows, n_new) == 0
    pool.grow(i32(n_new))
    with pytest.raises(kv.KernelError, match=str(kv.MAX_FORK)):
        pool.fork(i32(rows), i32(rows))
    same(pool, model)
    order = random.Random(3).sample(rows, n - 50)
    for r in order:
        assert model.fork([-1], [r])[0] == 0
    pool.free(i32(order))
    pool.check()
    same(pool, model)
    # what one piece refuses is told, whichever it is
    for at in (5, kv.MAX_FORK + 5, n - 60):
        bad = list(order)
        bad[at] = n
        pool.free(i32(bad))
        with pytest.raises(kv.KernelError):
            pool.check()
        pool.free(i32(order))
        pool.check()
    same(pool, model)
    assert kv.kv_error() == 0


def test_first_attend_on_another_stream(kv):
    """the first call of an object, with segments that several CTAs share, on a stream of its own while the current one
    is busy, and in a capture that is not replayed before the next call: the bits of any other call"""
    gen = torch.Generator(device="cuda").manual_seed(70)
    lens, H, n_kv, D, page = [4000, 2500], 8, 2, 64, 16
    k, v, table = cache(lens, n_kv, D, page, BF16, gen)
    q, n = values((2, 1, H, D), BF16, gen), i32(lens)
    first = torch.zeros_like(q)
    c = kv.PagedKv(k, v, table)
    c.attend(q, n, first)
    held(first, None, kv_ref.attend(q, k, v, table, lens), BF16, BF16, max(lens), D)
    size = c.workspace().numel()

    def fresh():
        used = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # what the allocator hands out next
        del used
        return kv.PagedKv(k, v, table)

    side, out = torch.cuda.Stream(), torch.zeros_like(q)
    c = fresh()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)                       # some 50 ms
    c.attend(q, n, out, stream=side)
    side.synchronize()
    assert torch.equal(out, first)
    c, out, g = fresh(), torch.zeros_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attend(q, n, out)
    again = torch.zeros_like(q)
    c.attend(q, n, again)
    assert torch.equal(again, first)
    g.replay()
    assert torch.equal(out, first)
    # layers of a pool share one
    pool = kv.KvPool.empty(2, 4, 8, 1, 64, 2, 2)
    a, b = pool.layer(0), pool.layer(1)
    assert a._ws.data_ptr() == b._ws.data_ptr()
    assert kv.kv_error() == 0


def test_lengths_as_positions_of_an_overlapped_call(kv):
    """the pool's lengths, which a growth just wrote, as the positions of the next append, nothing between them: every
    token is where the same calls put it with the device waited for"""
    rows, page, n_kv, D, steps = 48, 8, 2, 64, 30
    gen = torch.Generator(device="cuda").manual_seed(71)
    x = values((steps, rows, 2 * n_kv * D), BF16, gen)
    cut = [[z.unflatten(1, (-1, D)) for z in x[t].split(n_kv * D, 1)] for t in range(steps)]
    ids, one = i32(list(range(rows))), i32([1] * rows)
    cs = kv.rope_table(steps + 2, D)

    def run(wait):
        pool = kv.KvPool.empty(1, rows * 4, page, n_kv, D, rows, 4)
        pool.grow(i32([4 * page] * rows))
        count = kv.KvPool.empty(0, rows * 4, page, n_kv, D, rows, 4)  # whose lengths are the positions
        layer = pool.layer(0)
        torch.cuda.synchronize()
        for t in range(steps):
            for f in (lambda: count.grow(one, ids), lambda: layer.append(None, *cut[t], ids, count.lens, cs, None)):
                f()
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert count.lens.tolist() == [steps] * rows
        return pool

    a, b = run(True), run(False)
    assert torch.equal(a.data, b.data) and kv.kv_error() == 0
    # token t of the calls is at position t + 1
    v = torch.stack([a.data[0, 1, a.table[:, (t + 1) // page].long(), :, (t + 1) % page] for t in range(steps)])
    assert torch.equal(v, torch.stack([c[1] for c in cut]))


def test_compaction_leaves_pages_that_no_count_holds(kv):
    """a table entry of a page with a zero count is not in the plan's map: it stays and is told, whatever the workspace
    held before"""
    for fill in (0, 1, -1, 7):
        pool = kv.KvPool.empty(1, 16, 2, 1, 16, 3, 4, dtype=F16)
        pool.grow(i32([4, 4, 4]))
        pool.free(i32([0]))
        assert pool.table[2, :2].tolist() == [4, 5]
        pool.refs[5] = 0
        pool._ws[:pool._ws.numel() // 4 * 4].view(torch.int32).fill_(fill)
        pool.compact()
        pool.check()
        # pages 2, 3, 4 are live: 3 and 4 move to 0 and 1
        assert pool.table[1, :2].tolist() == [2, 0] and pool.table[2, :2].tolist() == [1, 5]
        assert pool.refs.tolist() == [1, 1, 1] + [0] * 13
        assert kv.kv_error() == kv.ERR_PAGE and kv.kv_error() == 0


@pytest.mark.parametrize("ct,H,n_kv,D,n_q,window", [(BF16, 4, 2, 128, 3, 0), (F16, 12, 1, 64, 4, 40), (E4M3, 8, 2, 80, 3, 0),
                                                    (BF16, 3, 1, 256, 5, 33), (E4M3, 20, 2, 192, 2, 64), (F16, 2, 1, 192, 3, 0)])
def test_lse_does_not_depend_on_the_values(kv, ct, H, n_kv, D, n_q, window):
    """NaN and infinite values (not keys) that some drafts of a sequence see: the outputs of those are not numbers, the
    others' and every lse are the formula's"""
    gen = torch.Generator(device="cuda").manual_seed(61)
    lens, page = [70, 2, 200, 3000], 8
    k, v, table = cache(lens, n_kv, D, page, ct, gen)
    q = values((len(lens), n_q, H, D), BF16, gen)
    ks = torch.ones(n_kv, device="cuda") if ct == E4M3 else None
    want = kv_ref.attend(q, k, v, table, lens, window=window, k_scale=ks, v_scale=ks)
    raw = v.view(torch.uint8) if ct == E4M3 else v
    bad = torch.tensor([math.nan if ct == E4M3 else math.inf, math.nan], device="cuda").to(ct)
    sees = torch.ones((len(lens), n_q), dtype=torch.bool)
    for b, m in enumerate(lens):
        spots = [m - 1]                                   # the last new token's own key
        if window and m > window + n_q:
            spots.append(m - n_q - window + 1)            # the first token's window begins there, the others' later
        for x, j in enumerate(spots):
            raw[table[b, j // page].long(), :, j % page, 5 + x] = bad[x].view(torch.uint8) if ct == E4M3 else bad[x]
        for i in range(n_q):
            hi = m - (n_q - 1 - i)
            lo = max(0, hi - window) if window else 0
            sees[b, i] = any(lo <= j < hi for j in spots)
    out, lse = torch.zeros_like(q), torch.zeros((len(lens), n_q, H), device="cuda")
    kv.PagedKv(k, v, table, ks, ks).attend(q, i32(lens), out, window=window, lse=lse)
    got, seen_lse = out.cpu(), lse.cpu()
    for b in range(len(lens)):
        for i in range(n_q):
            w = tuple(z[b:b + 1, i:i + 1] for z in want)
            if sees[b, i]:
                assert torch.isnan(got[b, i].float()).any(-1).all()
                held(w[0].to(BF16), seen_lse[b:b + 1, i:i + 1], w, BF16, ct, max(lens), D)
            else:
                held(got[b:b + 1, i:i + 1], seen_lse[b:b + 1, i:i + 1], w, BF16, ct, max(lens), D)
    assert kv.kv_error() == 0


def test_workspaces_that_are_refused(kv):
    """attend's ws, given with the call: bytes beside the cache, as the object's own"""
    gen = torch.Generator(device="cuda").manual_seed(72)
    k, v, table = cache([20, 9], 2, 64, 8, BF16, gen)
    c, n, q = kv.PagedKv(k, v, table), i32([20, 9]), values((2, 4, 64), BF16, gen)
    out, size = torch.zeros_like(q), kv.PagedKv(k, v, table).workspace().numel()
    for ws in (torch.zeros(size, dtype=torch.uint8), torch.zeros(size, dtype=torch.uint8).pin_memory(),
               torch.zeros(size, device="cuda"), torch.zeros(2 * size, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError):
            c.attend(q, n, out, ws=ws)
        with pytest.raises(ValueError):
            kv.PagedKv(k, v, table, ws=ws)
    assert (out == 0).all()
    want = torch.zeros_like(q)
    c.attend(q, n, want)
    c.attend(q, n, out, ws=c.workspace())
    assert torch.equal(out, want)
    # a zeroed one at an address that is no multiple of 16 is the library's to refuse
    with pytest.raises(kv.KernelError):
        c.attend(q, n, out, ws=torch.zeros(size + 8, dtype=torch.uint8, device="cuda")[8:])
