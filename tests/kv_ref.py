"""Plain 64-bit forms of the paged cache operators and the Python model of its
pages, for the tests."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}


def attend(q, k, v, table, lens, seq=None, scale=None, window=0, sinks=None, k_scale=None, v_scale=None):
    """(out, lse, weight, spread) in float64 on the CPU, all of q's shape
    [B][n_q][H][D] (lse without D).  weight = sum p |v| per value, spread = the
    most that a rounding unit of the products moves a score: scale * sum |q||k|
    at its largest over the seen keys, |score| included."""
    B, n_q, H, D = q.shape
    n_kv, P = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros((B, n_q, H, D), dtype=torch.float64)
    wgt, spr = torch.zeros_like(out), torch.zeros((B, n_q, H), dtype=torch.float64)
    lse = torch.full((B, n_q, H), -math.inf, dtype=torch.float64)
    qd = q.double().cpu()
    for b in range(B):
        r = b if seq is None else int(seq[b])
        n = int(lens[b])
        if r < 0 or n <= 0:
            continue
        ids = table[r, :-(-n // P)].long()
        kk = k[ids].double().cpu().transpose(0, 1).reshape(n_kv, -1, D)[:, :n]
        vv = v[ids].double().cpu().transpose(0, 1).reshape(n_kv, -1, D)[:, :n]
        if k_scale is not None:
            kk = kk * k_scale.double().cpu()[:, None, None]
        if v_scale is not None:
            vv = vv * v_scale.double().cpu()[:, None, None]
        for i in range(n_q):
            hi = n - (n_q - 1 - i)
            lo = max(0, hi - window) if window else 0
            if hi <= lo:
                continue
            for h in range(H):
                g = h // (H // n_kv)
                s = (kk[g, lo:hi] @ qd[b, i, h]) * scale
                spr[b, i, h] = ((kk[g, lo:hi].abs() @ qd[b, i, h].abs()) * scale).max() + s.abs().max()
                m = s.max()
                e = torch.exp(s - m)
                den = e.sum()
                if sinks is not None:
                    den = den + math.exp(float(sinks[h]) - float(m))
                out[b, i, h] = e @ vv[g, lo:hi] / den
                wgt[b, i, h] = e @ vv[g, lo:hi].abs() / den
                lse[b, i, h] = m + torch.log(den)
    return out, lse, wgt, spr


def turn(x, pos, cos_sin, interleaved):
    """x [T][H][D] turned, in float64, and sum |terms| of each value"""
    x = x.double().cpu()
    y, mag = x.clone(), x.abs().clone()
    if cos_sin is None:
        return y, mag
    half = cos_sin.shape[2]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    cs = cos_sin.double().cpu()[pos.long().cpu().clamp(min=0)]
    c, s = cs[:, 0][:, None], cs[:, 1][:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    mag[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    mag[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, mag


class Pages:
    """What the pool calls do, in Python lists."""

    def __init__(self, n_rows, max_pages, n_pages, page):
        self.table, self.lens = [[] for _ in range(n_rows)], [0] * n_rows
        self.refs, self.page, self.max_pages = [0] * n_pages, page, max_pages

    def _free(self):
        return [p for p, n in enumerate(self.refs) if n == 0]

    def grow(self, rows, n_new):
        """the status word, as of pulsar_kv.h"""
        if len(set(rows)) < len(rows) or any(not 0 <= r < len(self.table) for r in rows) or any(n < 0 for n in n_new):
            return 3
        if any(self.lens[r] + n > self.max_pages * self.page for r, n in zip(rows, n_new)):
            return 2
        need = [-(-(self.lens[r] + n) // self.page) - len(self.table[r]) for r, n in zip(rows, n_new)]
        free = self._free()
        if sum(need) > len(free):
            return 1
        for r, n, k in zip(rows, n_new, need):
            for _ in range(k):
                self.table[r].append(free.pop(0))
                self.refs[self.table[r][-1]] = 1
            self.lens[r] += n
        return 0

    def fork(self, src, dst):
        """(status, copies)"""
        if len(set(dst)) < len(dst) or any(not 0 <= d < len(self.table) for d in dst) or any(
                not -1 <= s < len(self.table) for s in src):
            return 3, []
        stays = {r for r in range(len(self.table)) if r not in dst} | {s for s, d in zip(src, dst) if s == d}
        new, copies, free = [], [], self._free()
        for i, (s, d) in enumerate(zip(src, dst)):
            row = list(self.table[s]) if s >= 0 else []
            n = self.lens[s] if s >= 0 else 0
            if n % self.page and s != d and (s in stays or src.index(s) != i):
                if not free:
                    return 1, []
                copies.append((row[-1], free.pop(0)))
                row[-1] = copies[-1][1]
            new.append((row, n))
        for row, _ in new:
            for p in row:
                self.refs[p] += 1
        for d in dst:
            for p in self.table[d]:
                self.refs[p] -= 1
        for d, (row, n) in zip(dst, new):
            self.table[d], self.lens[d] = row, n
        return 0, copies

    def compact(self):
        live = [p for p, n in enumerate(self.refs) if n > 0]
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        refs = [0] * len(self.refs)
        for p in live:
            refs[to.get(p, p)] = self.refs[p]
        self.refs = refs
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return to
