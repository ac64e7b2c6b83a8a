"""The paged key/value cache: rotary positions with the cache write, attention
over the pages, and the pages' bookkeeping (include/pulsar_kv.h).

PagedKv is one layer's cache (append, attend), KvPool a whole cache's pages
shared by its layers (grow, fork, free, compact), rope_table() the angles.
All work on preallocated torch CUDA tensors as the caller's device buffers, on
the current stream unless one is given; the objects make their buffers when
they are made, no call allocates, and none synchronises but check() and
kv_error().  Tensors of the wrong kind raise ValueError, what the library
refuses KernelError.  What the device finds out of range (a page id, a length)
it does not follow; kv_error() tells and clears.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import KernelError, KvAppendArgs, KvAttendArgs, KvDesc, KvPoolDesc, check, lib

__all__ = ["PagedKv", "KvPool", "rope_table", "kv_error", "KernelError"]

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3}
WS_ZEROED = 32768
MAX_FORK = 4096

ERR_PAGE, ERR_SPAN, ERR_ROW = 1, 2, 4


def kv_error() -> int:
    """the device-side error word of the cache's kernels, read and cleared (synchronous); 0 = none"""
    return int(lib().pulsar_kv_error())


# current_stream() builds an object: 3 us a call.  (A torch without CUDA has neither; nor can it make a cache.)
_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _stream(stream, dev):
    """the cudaStream_t to launch on: dev is the buffers' device index"""
    if _device() != dev:
        raise ValueError("the buffers' device is not the current one")
    # torch's default stream goes by the runtime's handle for it (1): 0 would be the calling thread's own,
    # which is ordered with it, but by an event each way
    return (_raw_stream(dev) if stream is None else stream.cuda_stream) or 1


def _i32(t, n, dev, what):
    if t.dtype is not torch.int32 or t.device != dev or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what}: {n} contiguous int32 values on {dev}")
    return t.data_ptr()


def _heads(t, n_tok, n_head, d, dtype, dev, what):
    """(pointer, token stride) of [n_tok][n_head][d] values, heads d apart"""
    if t.shape != (n_tok, n_head, d) or t.dtype is not dtype or t.device != dev:
        raise ValueError(f"{what}: {n_tok} x {n_head} x {d} values of {dtype} on {dev}")
    s0, s1, s2 = t.stride()
    if (s2 != 1 and d > 1) or (s1 != d and n_head > 1):
        raise ValueError(f"{what}: a token's heads are {d} values apart and contiguous")
    return t.data_ptr(), s0


def _tokens(t, n, n_q, n_head, d):
    """the one stride between the n * n_q tokens of attend's q or out"""
    st = t.stride()
    if st[-1] != 1 or (n_head > 1 and st[-2] != d):
        raise ValueError(f"attend: a token's heads are {d} values apart and contiguous")
    if n_q == 1:
        return st[0] if n > 1 else n_head * d
    if n > 1 and st[0] != n_q * st[1]:
        raise ValueError("attend: one stride between all tokens")
    return st[1]


# ------------------------------------------------------------------ positions

def rope_table(n_pos: int, rot_dim: int, base: float = 10000.0, scaling: dict | None = None,
               device="cuda") -> torch.Tensor:
    """f32 [n_pos][2][rot_dim / 2]: cosines and sines of p * f_i, f_i =
    base^(-2 i / rot_dim), computed in 64 bits.  scaling, for contexts s =
    "factor" times the trained one:
      kind "linear": f_i / s
      kind "ntk":    base * s^(rot_dim / (rot_dim - 2)) in place of base
      kind "yarn":   f_i up to the pair that turns "fast" (32) times over the
        trained context ("trained"), f_i / s from the one that turns "slow"
        (1) times, a linear ramp over the pairs between; cosines and sines
        are times "mscale" (1 + 0.1 ln s)
      kind "bands":  f_i for pairs that turn "high" (4) times or more over the
        trained context, f_i / s for "low" (1) times or fewer, a blend linear
        in the turns between
    """
    _need(rot_dim >= 2 and rot_dim % 2 == 0 and n_pos >= 1, "rope_table: an even rot_dim and at least one position")
    half = rot_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    mul = 1.0
    kind = None if scaling is None else scaling["kind"]
    s = 1.0 if scaling is None else float(scaling["factor"])
    _need(s > 0 and base > 0, "rope_table: positive base and factor")
    if kind == "ntk":
        _need(rot_dim > 2, "rope_table: ntk needs more than one pair")
        base = base * s ** (rot_dim / (rot_dim - 2))
    f = base ** (-i / half)
    if kind == "linear":
        f = f / s
    elif kind == "yarn":
        trained = float(scaling["trained"])

        def pair_of(turns):  # the (fractional) pair that turns so often over the trained context
            return half * math.log(trained / (2 * math.pi * turns)) / math.log(base)

        lo = max(math.floor(pair_of(scaling.get("fast", 32.0))), 0)
        hi = min(math.ceil(pair_of(scaling.get("slow", 1.0))), rot_dim - 1)  # behind the last pair, where none turns so slowly
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - ramp) + f / s * ramp
        mul = float(scaling.get("mscale", 1.0 + 0.1 * math.log(s) if s > 1 else 1.0))
    elif kind == "bands":
        turns = float(scaling["trained"]) * f / (2 * math.pi)
        lo, hi = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        share = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
        f = f * share + f / s * (1.0 - share)
    else:
        _need(kind in (None, "ntk"), f"rope_table: unknown scaling {kind!r}")
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * f.to(device)[None]
    return (torch.stack((ang.cos(), ang.sin()), 1) * mul).to(torch.float32).contiguous()


# ------------------------------------------------------------------ one layer

class PagedKv:
    """One layer's cache: k, v [n_pages][n_kv][page_size][head_dim] (any
    strides whose head rows are contiguous and 16-byte aligned), bf16, f16 or
    float8_e4m3fn; table int32 [n_rows][max_pages].  k_scale, v_scale: f32
    [n_kv], e4m3 only.  ws: attend's workspace (workspace()), which any number
    of layers share on one stream; without one the object makes its own, on the
    current stream, like any tensor (so that a call on another stream, or in a
    capture, is ordered behind its zeros like behind the cache's bytes).
    An object serves one thread, and its workspace one stream, at a time."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, ws: torch.Tensor | None = None):
        _need(k.is_cuda and k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and k.dtype == v.dtype
              and v.device == k.device, "PagedKv: k and v alike, [n_pages][n_kv][page_size][head_dim] on one GPU")
        _need(k.dtype in TYPES and k.dtype != torch.float32, "PagedKv: caches are bf16, f16 or float8_e4m3fn")
        _need(k.stride(3) == 1, "PagedKv: a head's values are contiguous")
        _need(table.dim() == 2 and table.dtype == torch.int32 and table.device == k.device and table.stride(1) == 1,
              "PagedKv: table is int32 [n_rows][max_pages] beside the cache")
        _need(table.shape[0] == 1 or table.stride(0) >= table.shape[1], "PagedKv: table rows overlap")
        _need(k.dtype == torch.float8_e4m3fn or (k_scale is None and v_scale is None), "PagedKv: scales belong to e4m3 caches")
        for s in (k_scale, v_scale):
            _need(s is None or (s.dtype == torch.float32 and s.device == k.device and s.is_contiguous()
                                and s.numel() == k.shape[1]), "PagedKv: scales are f32 [n_kv] beside the cache")
        self.k, self.v, self.table, self.k_scale, self.v_scale = k, v, table, k_scale, v_scale
        self.device, self.n_kv, self.head_dim, self._index = k.device, k.shape[1], k.shape[3], k.device.index
        d = KvDesc()
        d.k, d.v, d.table = k.data_ptr(), v.data_ptr(), table.data_ptr()
        d.k_scale = None if k_scale is None else k_scale.data_ptr()
        d.v_scale = None if v_scale is None else v_scale.data_ptr()
        d.page_stride, d.head_stride, d.tok_stride = k.stride(0), k.stride(1), k.stride(2)
        d.table_stride = max(table.stride(0), table.shape[1])
        d.n_pages, d.n_kv, d.page_size, d.head_dim = k.shape
        d.n_rows, d.max_pages = table.shape
        d.dtype = TYPES[k.dtype]
        self._desc, self._pdesc = d, ctypes.addressof(d)
        self._args, self._append = KvAttendArgs(), KvAppendArgs()
        self._pargs, self._pappend = ctypes.addressof(self._args), ctypes.addressof(self._append)
        self._lib = lib()
        self._take(self.workspace() if ws is None else ws)
        self._c_append, self._c_attend = self._lib.pulsar_kv_append, self._lib.pulsar_kv_attend

    def append(self, q, k, v, seq, pos, cos_sin, q_out, interleaved: bool = False, stream=None):
        """Turn q [T][n_head][D] into q_out and write turned k and v [T][n_kv][D]
        at token pos[t] of table row seq[t] (both int32 [T]; negative =
        padding, skipped).  cos_sin: rope_table(), or None for no rotation; q
        and q_out None: keys and values only."""
        a, dev, D = self._append, self.device, self.head_dim
        n_tok = k.shape[0]
        if n_tok == 0:
            return q_out
        if k.dtype not in TYPES or k.dtype == torch.float8_e4m3fn:
            raise ValueError("append: values are f32, bf16 or f16")
        a.k, a.k_stride = _heads(k, n_tok, self.n_kv, D, k.dtype, dev, "append: k")
        a.v, a.v_stride = _heads(v, n_tok, self.n_kv, D, k.dtype, dev, "append: v")
        a.n_head, a.q, a.q_out = 0, None, None
        if q is not None:
            a.n_head = q.shape[1]
            a.q, a.q_stride = _heads(q, n_tok, a.n_head, D, k.dtype, dev, "append: q")
            a.q_out, a.q_out_stride = _heads(q_out, n_tok, a.n_head, D, q_out.dtype, dev, "append: q_out")
            a.q_out_type = TYPES[q_out.dtype]
        a.seq, a.pos = _i32(seq, n_tok, dev, "append: seq"), _i32(pos, n_tok, dev, "append: pos")
        a.cos_sin, a.rot_dim, a.n_pos = None, 0, 0
        if cos_sin is not None:
            if (cos_sin.dim() != 3 or cos_sin.shape[1] != 2 or cos_sin.dtype != torch.float32 or cos_sin.device != dev
                    or not cos_sin.is_contiguous()):
                raise ValueError("append: cos_sin is f32 [n_pos][2][rot_dim / 2]")
            a.cos_sin, a.n_pos, a.rot_dim = cos_sin.data_ptr(), cos_sin.shape[0], 2 * cos_sin.shape[2]
        a.n_tok, a.x_type, a.interleaved = n_tok, TYPES[k.dtype], int(interleaved)
        if not self._c_append(self._pdesc, self._pappend, _stream(stream, self._index)):
            raise KernelError("kv_append")
        return q_out

    def attend(self, q, lens, out, scale: float | None = None, window: int = 0, sinks=None, lse=None, seq=None,
               stream=None, ws: torch.Tensor | None = None):
        """out = attention of q over the cache.  q, out: [B][n_q][n_head][D], or
        [B][n_head][D] for one token a sequence; row b has lens[b] keys (its
        new ones among them) in table row seq[b] (None: b).  Token i of n_q
        sees lens[b] - (n_q - 1 - i) keys, the last `window` of them if that is
        not 0.  sinks f32 [n_head]; lse f32 [B][n_q][n_head].  scale: D^-1/2
        unless given.  ws: another workspace than the object's, zeroed before
        its first use (workspace())."""
        a, dev, D = self._args, self.device, self.head_dim
        shape, dtype = q.shape, q.dtype
        kind = TYPES.get(dtype, 3)
        if len(shape) == 4:
            n, n_q, n_head, d = shape
        else:
            (n, n_head, d), n_q = shape, 1
        if n == 0 or n_q == 0:
            return out
        if kind == 3 or dtype is not out.dtype or out.shape != shape or d != D or q.device != dev or out.device != dev:
            raise ValueError("attend: q and out alike, f32, bf16 or f16 [B][n_q][n_head][head_dim], beside the cache")
        a.q, a.out = q.data_ptr(), out.data_ptr()
        a.q_stride, a.out_stride = _tokens(q, n, n_q, n_head, D), _tokens(out, n, n_q, n_head, D)
        a.lens = _i32(lens, n, dev, "attend: lens")
        a.seq = None if seq is None else _i32(seq, n, dev, "attend: seq")
        a.sinks = a.lse = None
        if sinks is not None:
            if sinks.dtype is not torch.float32 or sinks.numel() != n_head or sinks.device != dev or not sinks.is_contiguous():
                raise ValueError("attend: sinks is f32 [n_head]")
            a.sinks = sinks.data_ptr()
        if lse is not None:
            if lse.dtype is not torch.float32 or lse.numel() != n * n_q * n_head or lse.device != dev or not lse.is_contiguous():
                raise ValueError("attend: lse is f32 [B][n_q][n_head]")
            a.lse = lse.data_ptr()
        if not 0 <= window <= 0x7fffffff:
            raise ValueError("attend: window is 0 (none) or a number of keys")
        a.scale = D ** -0.5 if scale is None else scale
        a.n_rows, a.n_q, a.n_head, a.window, a.q_type = n, n_q, n_head, window, kind
        if ws is not None:
            where = self._bytes(ws)
        else:
            where = self._where
        if not self._c_attend(self._pdesc, self._pargs, *where, _stream(stream, self._index)):
            raise KernelError("kv_attend")
        return out

    def workspace(self) -> torch.Tensor:
        """a zeroed workspace for attend() over caches of this shape, whatever its arguments (about 5 MB)"""
        n = int(self._lib.pulsar_kv_attend_workspace(self._pdesc, None))
        _need(n > 0, "PagedKv: shape refused")
        return torch.zeros(n, dtype=torch.uint8, device=self.device)

    def _bytes(self, ws: torch.Tensor):
        _need(ws.dtype == torch.uint8 and ws.device == self.device and ws.is_contiguous(),
              "PagedKv: a workspace is contiguous bytes beside the cache")
        return ws.data_ptr(), ws.numel()

    def _take(self, ws: torch.Tensor) -> None:
        self._ws, self._where = ws, self._bytes(ws)


# ------------------------------------------------------------------ all layers

class KvPool:
    """The pages of a cache.  data [n_layer][2][n_pages][n_kv][page_size][D]
    (keys and values of each layer; contiguous), table int32 [n_rows]
    [max_pages], lens int32 [n_rows], refs int32 [n_pages] (holders of each
    page).  KvPool.empty() makes all four."""

    def __init__(self, data: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor):
        _need(data.is_cuda and data.dim() == 6 and data.shape[1] == 2 and data.is_contiguous(),
              "KvPool: data is [n_layer][2][n_pages][n_kv][page_size][head_dim], contiguous")
        n_rows = table.shape[0]
        for t, n, what in ((table, table.numel(), "table"), (lens, n_rows, "lens"), (refs, data.shape[2], "refs")):
            _i32(t, n, data.device, "KvPool: " + what)
        _need(table.dim() == 2, "KvPool: table is [n_rows][max_pages]")
        self.data, self.table, self.lens, self.refs = data, table, lens, refs
        self.device, self.n_rows, self.page_size, self._index = data.device, n_rows, data.shape[4], data.device.index
        p = KvPoolDesc()
        p.table, p.len, p.refs, p.data = table.data_ptr(), lens.data_ptr(), refs.data_ptr(), data.data_ptr()
        p.slab_stride = data.stride(1) * data.element_size()
        p.page_bytes = data.stride(2) * data.element_size()
        p.table_stride = table.shape[1]
        p.n_rows, p.max_pages = table.shape
        p.n_pages, p.page_size, p.n_slab = data.shape[2], data.shape[4], 2 * data.shape[0]
        self._desc, self._p = p, ctypes.addressof(p)
        self._lib = lib()
        need = int(self._lib.pulsar_kv_pool_workspace(self._p, n_rows))
        _need(need > 0, "KvPool: shape refused")
        self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        self._where = self._ws.data_ptr(), need
        self._attend_ws = None
        self._none = torch.full((min(n_rows, MAX_FORK),), -1, dtype=torch.int32, device=self.device)  # free()'s sources
        #: what the last grow, fork and compact did (pulsar_kv.h's status words)
        self.status = torch.zeros((3, 4), dtype=torch.int32, device=self.device)
        self._status = [self.status[i].data_ptr() for i in range(3)]
        # of a free() in pieces: those behind the first
        self._more = torch.zeros((max(0, -(-n_rows // MAX_FORK) - 1), 4), dtype=torch.int32, device=self.device)
        self._n_more = 0

    @classmethod
    def empty(cls, n_layer, n_pages, page_size, n_kv, head_dim, n_rows, max_pages, dtype=torch.bfloat16, device="cuda"):
        data = torch.zeros((n_layer, 2, n_pages, n_kv, page_size, head_dim), dtype=dtype, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(data, torch.full((n_rows, max_pages), -1, **i32), torch.zeros(n_rows, **i32),
                   torch.zeros(n_pages, **i32))

    def layer(self, i: int, k_scale=None, v_scale=None) -> PagedKv:
        """layer i's cache; the layers share one attend workspace"""
        kv = PagedKv(self.data[i, 0], self.data[i, 1], self.table, k_scale, v_scale, self._attend_ws)
        self._attend_ws = kv._ws
        return kv

    def grow(self, n_new: torch.Tensor, rows: torch.Tensor | None = None, stream=None) -> None:
        """rows[i] (None: i) gets n_new[i] more tokens and the pages for them"""
        n = n_new.numel()
        if n == 0:
            return
        r = None if rows is None else _i32(rows, n, self.device, "grow: rows")
        check(self._lib.pulsar_kv_grow(self._p, r, _i32(n_new, n, self.device, "grow: n_new"), n, self._status[0],
                                       *self._where, _stream(stream, self._index)), "kv_grow")

    def _fork(self, src, dst, status, stream) -> None:
        n = src.numel()
        check(self._lib.pulsar_kv_fork(self._p, _i32(dst, n, self.device, "fork: dst"),
                                       _i32(src, n, self.device, "fork: src"), n, status, *self._where,
                                       _stream(stream, self._index)), "kv_fork")

    def fork(self, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
        """row dst[i] becomes what row src[i] was (src -1: empty), all i at once; at most 4096 (MAX_FORK) rows"""
        if src.numel() == 0:
            return
        if src.numel() > MAX_FORK:
            raise KernelError(f"kv_fork: more than {MAX_FORK} rows at once")
        self._n_more = 0
        self._fork(src, dst, self._status[1], stream)

    def free(self, rows: torch.Tensor, stream=None) -> None:
        """rows become empty; more than 4096 (MAX_FORK) go in pieces, each all or nothing by itself"""
        n = rows.numel()
        if n == 0:
            return
        if n > self.n_rows:
            raise KernelError("kv_free: more rows than the table has")
        _i32(rows, n, self.device, "free: rows")
        self._n_more = (n - 1) // MAX_FORK
        for i in range(0, n, MAX_FORK):
            piece = rows.view(-1)[i:i + MAX_FORK]
            self._fork(self._none[:piece.numel()], piece,
                       self._status[1] if i == 0 else self._more[i // MAX_FORK - 1].data_ptr(), stream)

    def compact(self, stream=None) -> None:
        """live pages move to the low ids"""
        check(self._lib.pulsar_kv_compact(self._p, self._status[2], *self._where, _stream(stream, self._index)),
              "kv_compact")

    def check(self) -> None:
        """raise if the last grow, fork or compact was refused on the device (synchronous)"""
        rest = self._more[:self._n_more].tolist() if self._n_more else []
        for name, s in zip(("grow", "fork", "compact") + ("fork",) * len(rest), self.status.tolist() + rest):
            if s[0]:
                why = {1: "too few free pages", 2: "a row would outgrow its table"}.get(s[0], "invalid rows or lengths")
                raise KernelError(f"kv_{name}: {why}")
