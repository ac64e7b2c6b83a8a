"""The decoder example: rotary append, paged attention, growth and fork with
the expert layer, against 64-bit attention over the same rows."""
import pytest

import kv_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def make():
    import pulsar_b200 as p
    from pulsar_b200.decoder import Decoder, DecoderSpec
    moe = p.LayerSpec(n_embd=256, n_ff=256, n_expert=8, n_used=2, quant=p.QUANT_Q4_K)

    def f(**kw):
        spec = dict(moe=moe, n_layer=2, n_head=8, n_kv=2, head_dim=32, cache=torch.float16, page_size=8)
        spec.update(kw)
        return Decoder(DecoderSpec(**spec), n_rows=6, max_tokens=96, seed=3)
    return f


def hidden(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, 256), generator=g, device="cuda")


@pytest.mark.parametrize("kw", [dict(), dict(window=9, interleaved=True, rot_dim=16), dict(cache=torch.bfloat16)])
def test_layers_against_64_bits(make, kw):
    """a prompt, a second prompt beside a decode step, and decode steps: every layer's attention output, from the
    layer's own input.  The keys in the cache are rounded to its type u; a rounding of a key moves a score by u
    spread, of a value the output by u weight; projections are f32 dots of 256 terms."""
    d = make(**kw)
    s = d.spec
    u = kv_ref.U[s.cache]
    story = {}  # (sequence, layer) -> inputs so far
    for step, (rows, n_new) in enumerate((([2], [19]), ([2, 0], [1, 30]), ([0, 2], [1, 1]))):
        seq, pos = d.extend(rows, n_new)
        assert pos.tolist() == [len(story.get((r, 0), [])) + i for r, n in zip(rows, n_new) for i in range(n)]
        trace = []
        out = d.forward(hidden(sum(n_new), step), seq, pos, trace)
        assert torch.isfinite(out).all()
        d.pool.check()
        for i, (x, a, mid, y) in enumerate(trace):
            for t, r in enumerate(seq.tolist()):
                story.setdefault((r, i), []).append(x[t].double().cpu())
            for r in set(seq.tolist()):
                xs = torch.stack(story[r, i])
                nx = xs / (xs.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
                qkv = nx @ d.wqkv[i].double().cpu().T
                P = torch.arange(len(xs))
                q, k, v = (z.unflatten(1, (-1, 32)) for z in qkv.split([256, 64, 64], 1))
                q, k = (kv_ref.turn(z, P, d.cos_sin, s.interleaved)[0] for z in (q, k))
                mine = [t for t in range(len(seq)) if int(seq[t]) == r]
                where = pos[mine].cpu()
                # one page of all keys; each row sees up to its own
                pages = (z.transpose(0, 1).unsqueeze(0) for z in (k, v))
                kk, vv = pages
                table = torch.zeros((1, 1), dtype=torch.int32)
                want, _, wgt, spr = kv_ref.attend(q[where].unsqueeze(1), kk, vv, table, (where + 1).tolist(),
                                                  seq=[0] * len(mine), window=s.window)
                # 4 u: both factors of a score and its weight's two sides; 600 eps: the projections' and the norm's sums
                rel = (4 * u + 600 * EPS) * (spr[..., None] + 1)
                err = (a[mine].double().cpu().unsqueeze(1) - want).abs()
                assert (err <= wgt * rel + 600 * EPS).all(), (step, i, r, float((err / (wgt * rel + 600 * EPS)).max()))
            ws = torch.zeros(d.moe[i].workspace_bytes(len(seq)), dtype=torch.uint8, device="cuda")
            from pulsar_b200.ops import rms_norm
            n, again = torch.empty_like(mid), torch.empty_like(mid)
            rms_norm(n, mid)
            d.moe[i].forward(n, again, ws, residual=mid)
            assert torch.equal(again, y)


def test_forked_beams_continue_alike(make):
    d = make()
    d.forward(hidden(21, 1), *d.extend([1], [21]))
    d.pool.fork(torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda"),
                torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda"))
    same = hidden(1, 2).expand(4, -1).contiguous()
    a = d.forward(same, *d.extend([0, 1, 3, 4], [1] * 4))
    assert all(torch.equal(a[0], a[i]) for i in range(1, 4))
    # other tokens: the beams part, and a reorder takes their caches along
    b = d.forward(hidden(4, 3), *d.extend([0, 1, 3, 4], [1] * 4))
    assert not torch.equal(b[0], b[1])
    d.pool.fork(torch.tensor([3, 3, 0, 1], dtype=torch.int32, device="cuda"),
                torch.tensor([0, 1, 3, 4], dtype=torch.int32, device="cuda"))
    c = d.forward(same, *d.extend([0, 1, 3, 4], [1] * 4))
    assert torch.equal(c[0], c[1]) and not torch.equal(c[0], c[2]) and not torch.equal(c[2], c[3])
    d.pool.check()
    d.pool.compact()
    e = d.forward(same, *d.extend([0, 1, 3, 4], [1] * 4))
    assert torch.equal(e[0], e[1]) and torch.isfinite(e).all()
