"""The paged cache's host side without a GPU: rotary tables, the package's import."""
import math
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("rot,base,trained,factor", [(64, 10000.0, 131072, 4.0), (64, 10000.0, 65536, 16.0),
                                                     (128, 10000.0, 32768, 4.0), (64, 10000.0, 4096, 8.0),
                                                     (128, 500000.0, 8192, 8.0), (32, 1000.0, 1 << 20, 2.0)])
def test_yarn_blends_as_published(rot, base, trained, factor):
    """every pair's rate against the published ramp: from the pair that turns 32 times over the trained context to the
    one that turns once, ends rounded outwards and kept within [0, rot - 1], so that it may end behind the last pair.
    The table's sines and cosines are f32: a rate is within 2^-23 of itself, with the rounding of the table's 64 bits"""
    from pulsar_b200.kv import rope_table
    t = rope_table(2, rot, base, dict(kind="yarn", factor=factor, trained=trained), device="cpu").double()[1]
    got = torch.atan2(t[1], t[0])

    def pair(turns):
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        ramp = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        want = f * (1 - ramp) + f / factor * ramp
        assert abs(float(got[i]) - want) <= 2.0 ** -22 * want, (i, float(got[i]), want)


def test_package_imports_beside_a_torch_without_cuda():
    """a torch built for the CPU has no CUDA bindings: the package, the layer builder's host side and the rotary tables
    need none"""
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]: delattr(torch._C, n)\n"
            "import pulsar_b200\n"
            "assert pulsar_b200.row_bytes(pulsar_b200.QUANT_Q4_K, 256) == 144\n"
            "assert pulsar_b200.rope_table(4, 8, device='cpu').shape == (4, 2, 4)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


def test_star_import_has_the_cache():
    import pulsar_b200
    from pulsar_b200 import decoder, kv
    for m in (kv, decoder):
        for n in ("KvPool", "PagedKv", "kv_error", "rope_table") if m is kv else ("Decoder", "DecoderSpec"):
            assert n in pulsar_b200.__all__ and getattr(pulsar_b200, n) is getattr(m, n)
