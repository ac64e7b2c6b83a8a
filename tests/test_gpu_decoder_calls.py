"""The decoder example off the beaten track."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def make():
    import pulsar_b200 as p
    from pulsar_b200.decoder import Decoder, DecoderSpec
    moe = p.LayerSpec(n_embd=256, n_ff=256, n_expert=8, n_used=2, quant=p.QUANT_Q4_K)

    def f(n_pages=0, max_tokens=96, **kw):
        spec = dict(moe=moe, n_layer=2, n_head=8, n_kv=2, head_dim=32, cache=torch.float16, page_size=8)
        spec.update(kw)
        return Decoder(DecoderSpec(**spec), n_rows=6, max_tokens=max_tokens, seed=3, n_pages=n_pages)
    return f


def hidden(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, 256), generator=g, device="cuda")


def test_on_a_stream_and_in_a_capture(make):
    """prompt, decode steps and a fork on a stream of their own while the default one is busy, and a decode step captured
    and replayed: the bits of the same calls on the default stream"""
    def run(d, between):
        outs = [d.forward(hidden(19, 1), *d.extend([2], [19]))]
        between()
        outs.append(d.forward(hidden(31, 2), *d.extend([2, 0], [1, 30])))
        d.pool.fork(torch.tensor([2, 2], dtype=torch.int32, device="cuda"), torch.tensor([1, 4], dtype=torch.int32, device="cuda"))
        outs.append(d.forward(hidden(3, 3), *d.extend([1, 2, 4], [1, 1, 1])))
        return outs

    want = run(make(), lambda: None)
    d, side = make(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = run(d, lambda: torch.cuda.default_stream().synchronize())
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    x = hidden(3, 4)
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)                       # the default stream is busy for some 50 ms
    with torch.cuda.stream(side):
        seq, pos = d.extend([1, 2, 4], [1, 1, 1])
        a = d.forward(x, seq, pos)
    side.synchronize()
    # the same step (its keys and values are written again) in a graph
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b = d.forward(x, seq, pos)
    for new in (x.clone(), hidden(3, 5)):
        x.copy_(new)
        b.zero_()
        g.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            c = d.forward(x, seq, pos)
        torch.cuda.synchronize()
        assert torch.equal(b, c)
        if torch.equal(new, hidden(3, 4)):
            assert torch.equal(a, b)
    d.pool.check()


def test_refused_growth_touches_no_cache(make):
    """too few free pages, and rows past their table: the new tokens are padding, and no byte of any sequence's keys and
    values changes; the next growth that has room goes on where the sequence ended"""
    from pulsar_b200 import KernelError
    d, free = make(n_pages=5), make()
    beams = torch.tensor([1, 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    for x in (d, free):                                  # 2 full pages shared by three beams, 3 pages of their own
        x.forward(hidden(21, 1), *x.extend([1], [21]))
        x.pool.fork(*beams)
        x.pool.check()
    was, lens = d.pool.data.clone(), d.pool.lens.clone()
    for rows, n_new in (([0, 1, 3], [1, 4, 2]), ([1], [90])):
        seq, pos = d.extend(rows, n_new)
        assert pos.tolist() == [-1] * sum(n_new)
        trace = []
        d.forward(hidden(sum(n_new), 2), seq, pos, trace)
        with pytest.raises(KernelError):
            d.pool.check()
        assert torch.equal(d.pool.data, was) and torch.equal(d.pool.lens, lens)
        assert all((a == 0).all() for _, a, _, _ in trace)
    same = [x.forward(hidden(3, 4), *x.extend([0, 1, 3], [1, 1, 1])) for x in (d, free)]
    d.pool.check()
    assert torch.equal(*same)


def test_rows_reach_the_end_of_their_pages(make):
    """max_tokens that is no multiple of the page: a row holds whole pages, and every token of them has its angles"""
    from pulsar_b200 import kv_error
    kv_error()
    short, whole = make(max_tokens=20), make(max_tokens=24)
    a, b = (x.forward(hidden(24, 5), *x.extend([2], [24])) for x in (short, whole))
    assert kv_error() == 0
    short.pool.check()
    assert torch.equal(a, b)
    assert torch.equal(short.pool.data[:, :, short.pool.table[2, :3].long()], whole.pool.data[:, :, whole.pool.table[2, :3].long()])


def test_refusals(make):
    """rows and positions of another type, width or place: refused before any launch"""
    d = make()
    seq, pos = d.extend([1], [5])
    x, was = hidden(5, 1), d.pool.data.clone()
    for a in ((x.bfloat16(), seq, pos), (x.double(), seq, pos), (x[:, :128].contiguous(), seq, pos), (hidden(10, 1)[::2], seq, pos),
              (x.T.contiguous().T, seq, pos), (x.cpu(), seq, pos), (x[0], seq, pos), (x, seq[:4], pos), (x, seq, pos[:4]),
              (x, seq.long(), pos), (x, seq, pos.long()), (x, seq.cpu(), pos), (x, seq, torch.stack((pos, pos), 1)[:, 0])):
        with pytest.raises(ValueError):
            d.forward(*a)
    assert torch.equal(d.pool.data, was)
    a, b = d.forward(x, seq, pos), d.forward(x, seq.view(5, 1), pos.view(1, 5))
    assert torch.isfinite(a).all() and torch.equal(a, b)


def test_no_tokens(make):
    """a step in which no sequence has a new token"""
    d = make()
    d.forward(hidden(5, 1), *d.extend([1], [5]))
    was = d.pool.data.clone()
    for rows, n_new in (([], []), ([1, 2], [0, 0])):
        seq, pos = d.extend(rows, n_new)
        assert d.forward(hidden(0, 1), seq, pos).shape == (0, 256)
    d.pool.check()
    assert d.pool.lens.tolist() == [0, 5, 0, 0, 0, 0] and torch.equal(d.pool.data, was)
