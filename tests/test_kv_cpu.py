"""The paged cache's C boundary and host side without a GPU: exported symbols,
struct layouts, refusals before any launch, and the rotary tables."""
import ctypes
import math
import os
import re
import subprocess

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "pulsar_kv.h")


@pytest.fixture(scope="module")
def L():
    import pulsar_b200
    pulsar_b200.build()
    return pulsar_b200.lib()


def test_exports_every_declared_symbol(L):
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(?:int|size_t|uint32_t)\s+(pulsar_kv_\w+)\s*\(", src)))
    assert len(names) == 8
    for n in names:
        assert hasattr(L, n)


def test_struct_layouts():
    from pulsar_b200._lib import KvAppendArgs, KvAttendArgs, KvDesc, KvPoolDesc
    pairs = [("pulsar_kv_desc", KvDesc, "dtype"), ("pulsar_kv_append_args", KvAppendArgs, "interleaved"),
             ("pulsar_kv_attend_args", KvAttendArgs, "q_type"), ("pulsar_kv_pool", KvPoolDesc, "n_slab")]
    fields = ",".join(f"sizeof({c}),offsetof({c},{f})" for c, _, f in pairs)
    src = '#include "pulsar_kv.h"\n#include <stdio.h>\nint main(){size_t a[]={%s};for(int i=0;i<8;i++)printf("%%zu ",a[i]);}'
    exe = os.path.join("/tmp", "pk_layout_probe")
    subprocess.run(["gcc", "-x", "c", "-", "-I", os.path.dirname(HEADER), "-o", exe], input=src % fields, text=True,
                   check=True)
    got = list(map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()))
    want = [x for _, s, f in pairs for x in (ctypes.sizeof(s), getattr(s, f).offset)]
    assert got == want


def desc(**kw):
    from pulsar_b200._lib import KvDesc
    d = KvDesc()
    d.k = d.v = d.table = 4096
    d.n_pages, d.page_size, d.n_kv, d.head_dim, d.n_rows, d.max_pages, d.dtype = 8, 16, 2, 64, 3, 4, 1
    d.table_stride, d.page_stride, d.head_stride, d.tok_stride = 4, 2048, 1024, 64
    for k, v in kw.items():
        setattr(d, k, v)
    return d


DESC_FAULTS = [dict(k=None), dict(table=None), dict(dtype=0), dict(dtype=4), dict(n_pages=0), dict(page_size=0),
               dict(n_kv=0), dict(n_rows=0), dict(max_pages=0), dict(head_dim=0), dict(head_dim=72),
               dict(head_dim=272), dict(table_stride=3), dict(k=4104), dict(tok_stride=65), dict(head_stride=1020),
               dict(k_scale=4096), dict(max_pages=1 << 28, table_stride=1 << 28), dict(tok_stride=1 << 28)]


def append_args(**kw):
    from pulsar_b200._lib import KvAppendArgs
    a = KvAppendArgs()
    a.q = a.k = a.v = a.q_out = a.seq = a.pos = a.cos_sin = 4096
    a.q_stride = a.q_out_stride = 4 * 64
    a.k_stride = a.v_stride = 128
    a.n_tok, a.n_head, a.rot_dim, a.n_pos, a.x_type, a.q_out_type = 5, 4, 64, 9, 1, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attend_args(**kw):
    from pulsar_b200._lib import KvAttendArgs
    a = KvAttendArgs()
    a.q = a.out = a.lens = 4096
    a.q_stride = a.out_stride = 4 * 64
    a.scale, a.n_rows, a.n_q, a.n_head, a.q_type = 0.125, 3, 1, 4, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_refusals_before_any_launch(L):
    ref = ctypes.byref
    big = 1 << 40
    for kw in DESC_FAULTS:
        assert L.pulsar_kv_append(ref(desc(**kw)), ref(append_args()), None) == 0, kw
        assert L.pulsar_kv_attend(ref(desc(**kw)), ref(attend_args()), 4096, big, None) == 0, kw
        assert L.pulsar_kv_attend_workspace(ref(desc(**kw)), ref(attend_args())) == 0, kw
    for kw in (dict(k=None), dict(seq=None), dict(pos=None), dict(q=None), dict(q_out=None), dict(x_type=3),
               dict(q_out_type=3), dict(rot_dim=7), dict(rot_dim=66), dict(cos_sin=None), dict(n_pos=0),
               dict(n_tok=0), dict(q_stride=255), dict(k_stride=127), dict(q_out_stride=1)):
        assert L.pulsar_kv_append(ref(desc()), ref(append_args(**kw)), None) == 0, kw
    for kw in (dict(q=None), dict(out=None), dict(lens=None), dict(q_type=3), dict(n_head=0), dict(n_head=5),
               dict(n_rows=0), dict(n_q=0), dict(n_rows=4), dict(q_stride=255), dict(out_stride=0)):
        assert L.pulsar_kv_attend(ref(desc()), ref(attend_args(**kw)), 4096, big, None) == 0, kw
    assert L.pulsar_kv_attend(ref(desc()), ref(attend_args()), None, big, None) == 0
    need = L.pulsar_kv_attend_workspace(ref(desc()), ref(attend_args()))
    assert need >= 32768
    assert L.pulsar_kv_attend(ref(desc()), ref(attend_args()), 4096, need - 1, None) == 0
    assert L.pulsar_kv_attend(ref(desc()), ref(attend_args()), 4104, big, None) == 0
    # enough for any arguments: the widest tiles of as many workers
    for kw in (dict(), dict(n_head=64, q_stride=64 * 64, out_stride=64 * 64), dict(n_q=9, q_type=0), dict(window=3)):
        assert L.pulsar_kv_attend_workspace(ref(desc()), None) >= L.pulsar_kv_attend_workspace(ref(desc()), ref(attend_args(**kw)))


def test_pool_refusals_before_any_launch(L):
    from pulsar_b200._lib import KvPoolDesc
    ref = ctypes.byref

    def pool(**kw):
        p = KvPoolDesc()
        p.table = p.len = p.refs = p.data = 4096
        p.slab_stride, p.page_bytes, p.table_stride = 1 << 20, 4096, 8
        p.n_rows, p.max_pages, p.n_pages, p.page_size, p.n_slab = 4, 8, 16, 4, 2
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    big = 1 << 40
    for kw in (dict(table=None), dict(len=None), dict(refs=None), dict(n_rows=0), dict(max_pages=0), dict(n_pages=0),
               dict(page_size=0), dict(table_stride=7), dict(data=None), dict(page_bytes=0),
               dict(max_pages=1 << 30, table_stride=1 << 30)):
        assert L.pulsar_kv_pool_workspace(ref(pool(**kw)), 4) == 0, kw
        assert L.pulsar_kv_grow(ref(pool(**kw)), None, 4096, 4, 4096, 4096, big, None) == 0, kw
        assert L.pulsar_kv_fork(ref(pool(**kw)), 4096, 4096, 4, 4096, 4096, big, None) == 0, kw
        assert L.pulsar_kv_compact(ref(pool(**kw)), 4096, 4096, big, None) == 0, kw
    need = L.pulsar_kv_pool_workspace(ref(pool()), 4)
    assert L.pulsar_kv_grow(ref(pool()), None, 4096, 4, 4096, 4096, need - 1, None) == 0
    assert L.pulsar_kv_grow(ref(pool()), None, 4096, 5, 4096, 4096, big, None) == 0
    assert L.pulsar_kv_grow(ref(pool()), None, None, 4, 4096, 4096, big, None) == 0
    assert L.pulsar_kv_grow(ref(pool()), None, 4096, 0, 4096, 4096, big, None) == 0
    assert L.pulsar_kv_fork(ref(pool()), 4096, None, 4, 4096, 4096, big, None) == 0
    assert L.pulsar_kv_fork(ref(pool(n_rows=5000)), 4096, 4096, 4097, 4096, 4096, big, None) == 0
    assert L.pulsar_kv_fork(ref(pool()), 4096, 4096, 4, None, 4096, big, None) == 0
    assert L.pulsar_kv_compact(ref(pool()), 4096, None, big, None) == 0


def test_rope_tables():
    from pulsar_b200.kv import rope_table
    t = rope_table(50, 8, device="cpu").double()
    assert t.shape == (50, 2, 4)
    for p in (0, 1, 49):
        for i in range(4):
            a = p * 10000.0 ** (-i / 4)
            assert abs(t[p, 0, i] - math.cos(a)) < 1e-7 and abs(t[p, 1, i] - math.sin(a)) < 1e-7
    far = rope_table(100001, 64, device="cpu")[100000].double()  # angles in 64 bits: no drift at long positions
    assert abs(far[1, 0] - math.sin(100000.0)) < 1e-7

    def freq(scaling, n=64, base=10000.0):
        t = rope_table(2, n, base, scaling, device="cpu").double()[1]
        return torch.atan2(t[1], t[0]), (t ** 2).sum(0).sqrt()

    f0, _ = freq(None)
    f, r = freq(dict(kind="linear", factor=4.0))
    assert torch.allclose(f, f0 / 4, rtol=1e-5) and torch.allclose(r, torch.ones_like(r), atol=1e-6)
    f, _ = freq(dict(kind="ntk", factor=4.0))
    assert abs(f[0] - f0[0]) < 1e-6 and abs(f[-1] / f0[-1] - 0.25) < 1e-4  # fast pair kept, slowest scaled by s
    f, r = freq(dict(kind="yarn", factor=8.0, trained=4096))
    assert abs(f[0] - f0[0]) < 1e-6 and abs(f[-1] * 8 / f0[-1] - 1) < 1e-4
    assert torch.allclose(r, torch.full_like(r, 1 + 0.1 * math.log(8.0)), atol=1e-6)
    share = f / f0
    assert (share[1:] <= share[:-1] + 1e-5).all()
    f, r = freq(dict(kind="bands", factor=8.0, trained=8192, low=1.0, high=4.0), base=500000.0)
    f0, _ = freq(None, base=500000.0)
    turns = 8192 * f0 / (2 * math.pi)
    assert torch.allclose(f[turns > 4.01], f0[turns > 4.01], rtol=1e-5)
    assert torch.allclose(f[turns < 0.99], f0[turns < 0.99] / 8, rtol=1e-3)
    for bad in (dict(n_pos=4, rot_dim=7), dict(n_pos=0, rot_dim=8), dict(n_pos=4, rot_dim=8, scaling=dict(kind="x", factor=2))):
        with pytest.raises(ValueError):
            rope_table(device="cpu", **bad)
