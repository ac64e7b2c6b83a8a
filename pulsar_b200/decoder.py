"""A decoder of the expert layers with attention over a paged cache.

Each layer computes
  x + wo . attend(turn(wqkv . rms_norm(x)))   (its keys and values appended)
  x + moe(rms_norm(x))                        (MoeLayer)
in f32 rows, as the expert layer takes them.  Any mix of prompts and decode
steps is one call: every new token is a row with its sequence and position,
and sees the keys up to its own.  Weights are seeded synthetic values, like
make_layer's.

  d = Decoder(spec, n_rows=8, max_tokens=4096, seed=1)
  x = d.forward(prompt, *d.extend([0], [len(prompt)]))   # sequence 0's prompt
  d.pool.fork(src, dst)                                  # beams
  x = d.forward(next_rows, *d.extend([0, 1, 2, 3], [1, 1, 1, 1]))
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .kv import KvPool, rope_table
from .layer import LayerSpec, make_layer
from .ops import add, matmul_f32, rms_norm


@dataclass
class DecoderSpec:
    moe: LayerSpec                # the expert layers; moe.n_embd is the model's width
    n_layer: int
    n_head: int
    n_kv: int
    head_dim: int
    window: int = 0               # keys that a token sees (0 = all)
    rot_dim: int | None = None    # None: the whole head
    rope_base: float = 10000.0
    rope_scaling: dict | None = None
    interleaved: bool = False
    cache: torch.dtype = torch.bfloat16
    page_size: int = 16


class Decoder:
    def __init__(self, spec: DecoderSpec, n_rows: int, max_tokens: int, seed: int, n_pages: int = 0, device="cuda"):
        s = self.spec = spec
        dev = torch.device(device)
        width = -(-max_tokens // s.page_size)
        self.pool = KvPool.empty(s.n_layer, n_pages or n_rows * width, s.page_size, s.n_kv, s.head_dim, n_rows, width,
                                 s.cache, dev)
        self.caches = [self.pool.layer(i) for i in range(s.n_layer)]
        # a row holds whole pages, and each of their tokens has its angles
        self.cos_sin = rope_table(width * s.page_size, s.head_dim if s.rot_dim is None else s.rot_dim, s.rope_base,
                                  s.rope_scaling, dev)
        self.moe = [make_layer(s.moe, seed * 1009 + i, dev) for i in range(s.n_layer)]
        self.wqkv, self.wo = [], []
        q, kv, h = s.n_head * s.head_dim, s.n_kv * s.head_dim, s.moe.n_embd
        for i in range(s.n_layer):
            g = torch.Generator(device=dev).manual_seed(seed * 2003 + i)
            self.wqkv.append(torch.randn((q + 2 * kv, h), generator=g, device=dev) * h ** -0.5)
            self.wo.append(torch.randn((h, q), generator=g, device=dev) * q ** -0.5)

    def extend(self, rows: list[int], n_new: list[int]):
        """room for n_new[i] more tokens of sequence rows[i]; (seq, pos) of all new tokens, int32 [sum(n_new)].  Where
        the pool has no room for all of them no sequence grows and every position is -1, which makes the tokens
        padding: forward() writes no cache for them (pool.check() raises)."""
        dev = self.pool.device
        r = torch.tensor(rows, dtype=torch.int32, device=dev)
        n = torch.tensor(n_new, dtype=torch.int32, device=dev)
        self.pool.grow(n, r)
        total = sum(n_new)
        seq = torch.repeat_interleave(r, n.long(), output_size=total)
        first = torch.repeat_interleave(self.pool.lens[r.long()] - n.cumsum(0, dtype=torch.int32), n.long(),
                                        output_size=total)
        pos = first + torch.arange(total, dtype=torch.int32, device=dev)
        return seq, torch.where(self.pool.status[0, 0] == 0, pos, -1)  # growth's status, on the device

    def forward(self, x: torch.Tensor, seq: torch.Tensor, pos: torch.Tensor, trace: list | None = None) -> torch.Tensor:
        """the last layer's rows of new tokens x [T][n_embd] (f32) at pos[t] of sequence seq[t], on torch's current
        stream (and so in a capture, behind one call outside it); trace collects each layer's (input, attention's
        output, row between the halves, output)"""
        s, T, dev = self.spec, x.shape[0], x.device
        st = torch.cuda.current_stream()
        q, kv, h = s.n_head * s.head_dim, s.n_kv * s.head_dim, s.moe.n_embd
        if x.shape != (T, h) or x.dtype != torch.float32 or dev != self.pool.device or not x.is_contiguous():
            raise ValueError(f"Decoder: x is f32 [T][{h}], contiguous, beside the cache")
        for t in (seq, pos):
            if t.numel() != T or t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
                raise ValueError("Decoder: seq and pos are int32 [T], contiguous, beside the cache")
        if T == 0:
            return torch.empty_like(x)
        n, y = torch.empty_like(x), torch.empty_like(x)
        qkv = torch.empty((T, q + 2 * kv), dtype=torch.float32, device=dev)
        turned = torch.empty((T, s.n_head, s.head_dim), dtype=torch.float32, device=dev)
        a = torch.empty_like(turned)
        qx, kx, vx = (t.unflatten(1, (-1, s.head_dim)) for t in qkv.split([q, kv, kv], 1))
        seen = pos + 1
        ws = torch.zeros(max(m.workspace_bytes(T) for m in self.moe), dtype=torch.uint8, device=dev)
        for i in range(s.n_layer):
            mid, out = torch.empty_like(x), torch.empty_like(x)
            rms_norm(n, x)
            matmul_f32(qkv, self.wqkv[i], n, h, q + 2 * kv, T, st)
            self.caches[i].append(qx, kx, vx, seq, pos, self.cos_sin, turned, s.interleaved)
            self.caches[i].attend(turned, seen, a, window=s.window, seq=seq)
            matmul_f32(y, self.wo[i], a, q, h, T, st)
            add(mid, x, y, T * h, st)
            rms_norm(n, mid)
            self.moe[i].forward(n, out, ws, residual=mid)
            if trace is not None:
                trace.append((x, a.clone(), mid, out))
            x = out
        return x
