"""Calls of the paged cache off the beaten track, against the model of the
pages and the plain 64-bit forms."""
import random

import pytest

import kv_ref
from test_gpu_kv import F16, i32, same

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
