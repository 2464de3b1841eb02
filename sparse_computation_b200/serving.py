"""Serving operators between the products of a transformer.

The weights of such a model run as ``SpMMPlan`` products on feature-major
activations (features x tokens, fp32).  What a decoding step needs besides:

    cache = PagedKVCache.allocate(num_pages, page_size, kv_heads, head_dim, torch.bfloat16)
    rope = RotaryTable(cos, sin)
    attention = DecodeAttention(cache, q_heads, max_seqs)
    adapters = LowRankAdapters(down, up, scales)

    q = adapters.apply(x, ids, base=wq.spmm(x))           # low-rank adapters beside the shared projection
    rows = lambda y, h: y.view(h, head_dim, -1).permute(2, 0, 1)
    q = cache.append(rows(k, kv_heads), rows(v, kv_heads), positions, page_table, rope=rope, q=rows(q, q_heads))
    out = attention.attend(q, page_table, positions + 1)

Activations are fp32, fp16 or bf16 CUDA tensors with any strides; the cache is
fp32, fp16 or bf16 of its own.  All calls are asynchronous on torch's current
stream of the handle's device, or on ``stream``: that does not wait for the
current one, and what the call allocates comes from its memory.  There is no
CPU fallback.
The reference (hosseinal/sparse-computation) ends at the products.
"""
from __future__ import annotations

import ctypes
from struct import Struct
from typing import Optional, Sequence

import torch

from . import SC_ERR_ARG, SC_ERR_DEVICE, ScError, _check, lib

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# The argument structures of the C calls are all 8-byte fields.
_POOL = Struct("13q")
_APPEND = Struct("31q")
_ATTEND = Struct("15q")
_ADAPT = Struct("14q")


def _fail(what: str):
    raise ScError(SC_ERR_ARG, what)


def _rows(t, name: str, device: int, shape, dtype) -> tuple:
    if t.dtype != dtype or t.get_device() != device or t.shape != shape:
        _fail(f"{name} must be a {tuple(shape)} {dtype} tensor on cuda:{device}, "
              f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    return (t.data_ptr(), *t.stride())


def _apart(t, name: str) -> None:
    strides = t.stride()
    if 0 in strides and any(st == 0 and n > 1 for st, n in zip(strides, t.shape)):
        _fail(f"{name} has elements that share memory")


def _ints(t, name: str, device: int, n: int) -> int:
    if t.dtype != torch.int32 or t.get_device() != device or t.dim() != 1 or t.shape[0] != n or \
            (n > 1 and t.stride(0) != 1):
        _fail(f"{name} must be a contiguous int32 vector of length {n} on cuda:{device}")
    return t.data_ptr()


def _table(t, device: int) -> tuple:
    """(pointer, rows, columns, row stride) of a page table."""
    if t.dtype != torch.int32 or t.get_device() != device or t.dim() != 2:
        _fail(f"page_table must be a 2-D int32 tensor on cuda:{device}")
    (n, c), (s, unit) = t.shape, t.stride()
    if c > 1 and unit != 1:
        _fail("page_table needs a unit column stride")
    return t.data_ptr(), n, c, s


def _on(stream, device: int, given, call, *args):
    """call(*args) with ``stream`` current, so that outputs and scratch come from that stream's memory: a block that is free
    on the stream that is current here may still have its last kernel ahead of it, and ``stream`` does not wait for
    that.  The tensors of the call are kept from reuse until both streams are done with them."""
    if stream.device.index != device:
        _fail(f"the stream is on {stream.device}, the call on cuda:{device}")
    here = torch.cuda.current_stream(device)
    if stream == here:
        return call(*args)
    with torch.cuda.stream(stream):
        got = call(*args)
    for t in given:
        if t is not None:
            t.record_stream(stream)
    for t in got if isinstance(got, tuple) else (got,):
        if t is not None:
            t.record_stream(here)
    return got


# torch.cuda.current_stream builds an object (1.2 us a call); the raw handle is all that a launch needs.
_current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


class _Handle:
    _free = ""
    _status = ""
    _run = ""
    _h: Optional[ctypes.c_void_p] = None

    def status(self) -> int:
        """Device-side status since the last call (waits for the device, then
        clears it): 0 = none, 8 = a page-table entry or place outside the
        cache, 9 = a position without a rotation row, 10 = an adapter id
        beyond the set.  What it concerns was skipped."""
        v = ctypes.c_int32()
        _check(getattr(lib(), self._status)(self._h, ctypes.byref(v)))
        return v.value

    def check(self) -> None:
        """Raises ScError(SC_ERR_DEVICE) when status() is non-zero."""
        v = self.status()
        if v:
            raise ScError(SC_ERR_DEVICE, f"a kernel skipped entries that were out of range (status {v})")

    def _own(self, h: ctypes.c_void_p, *memory) -> None:
        """``memory``: device tensors that only the handle keeps alive.  They come from the stream that is current now."""
        self._h = h
        self._kept, self._streams = memory, {_current(self.device)}
        self._release = getattr(lib(), self._free)  # module globals may be gone when the interpreter ends
        self._call = getattr(lib(), self._run)

    def _keep(self, raw: int) -> None:
        """Keeps the handle's memory from reuse until the current stream, ``raw``, is done with it, however early the
        handle is dropped.  Once for each stream is enough, as the allocator looks when the memory is freed."""
        for t in self._kept:
            t.record_stream(torch.cuda.current_stream(self.device))
        self._streams.add(raw)

    def __del__(self):
        if self._h is not None:
            self._release(self._h)
            self._h = None


class RotaryTable:
    """cos and sin, [positions, rotary / 2] fp32 on one device; pair i of a
    head is dims (i, i + rotary / 2), or (2i, 2i + 1) when ``interleaved``."""

    def __init__(self, cos, sin, interleaved: bool = False):
        if cos.dtype != torch.float32 or cos.dim() != 2 or not cos.is_cuda or cos.stride(1) != 1 or \
                cos.shape[0] == 0 or cos.shape[1] == 0:
            _fail("cos must be a non-empty 2-D float32 CUDA tensor with unit column stride")
        if sin.dtype != torch.float32 or sin.shape != cos.shape or sin.stride() != cos.stride() or \
                sin.device != cos.device:
            _fail("sin must be like cos in type, shape, strides and device")
        self.cos, self.sin = cos, sin
        self.rotary = 2 * cos.shape[1]
        self.device = cos.device.index
        self._args = (cos.data_ptr(), sin.data_ptr(), cos.shape[0], cos.stride(0), self.rotary, int(interleaved))


class PagedKVCache(_Handle):
    """Keys and values of many sequences in pages.

    ``k`` and ``v``: [num_pages, kv_heads, page_size, head_dim] tensors of one
    type (fp32, fp16, bf16) on one GPU, head_dim contiguous and every row on a
    16-byte boundary; a permuted [num_pages, page_size, kv_heads, head_dim]
    pool is taken too.  Row i of a page table lists the pages of sequence i.
    """
    _free, _status, _run = "sc_kv_cache_free", "sc_kv_cache_status", "sc_kv_append"

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            _fail("k and v must be 4-D and alike in shape, type and device")
        if k.dtype not in _TYPES or not k.is_cuda:
            _fail("the cache must be float32, float16 or bfloat16 on a GPU")
        if (k.stride(3) != 1 or v.stride(3) != 1) and k.shape[3] > 1:
            _fail("head_dim must be contiguous in the cache")
        self.k, self.v = k, v
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device.index
        pool = _POOL.pack(k.data_ptr(), v.data_ptr(), self.num_pages, self.page_size, self.kv_heads, self.head_dim,
                          *k.stride()[:3], *v.stride()[:3], _TYPES[k.dtype])
        h = ctypes.c_void_p()
        _check(lib().sc_kv_cache_create(pool, self.device, ctypes.byref(h)))
        self._own(h, k, v)

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.float32,
                 device: int = 0) -> "PagedKVCache":
        shape = (num_pages, kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=f"cuda:{device}"),
                   torch.zeros(shape, dtype=dtype, device=f"cuda:{device}"))

    def append(self, k, v, positions, page_table, seq_ids=None, rope: Optional[RotaryTable] = None, q=None,
               q_out=None, stream=None):
        """Stores the rows k and v ([tokens, kv_heads, head_dim]) of new tokens
        at ``positions`` of their sequences (``seq_ids``; token t is of
        sequence t without them) and rotates k, and q ([tokens, heads,
        head_dim]) when given, by ``rope`` on the way.  Returns the rotated q
        (``q_out``, or a new contiguous tensor; q itself may be the output).  A
        token with a negative position is skipped: nothing is stored, its q
        rows become zero.  positions, seq_ids and page_table are int32."""
        dev, dtype = self.device, k.dtype
        if stream is not None:
            return _on(stream, dev, (k, v, positions, seq_ids, page_table, q, q_out,
                                     *((rope.cos, rope.sin) if rope is not None else ())),
                       self.append, k, v, positions, page_table, seq_ids, rope, q, q_out)
        kind = _TYPES.get(dtype)
        if kind is None or k.dim() != 3:
            _fail("k must be a 3-D float32, float16 or bfloat16 tensor")
        n = k.shape[0]
        shape = (n, self.kv_heads, self.head_dim)
        ka = _rows(k, "k", dev, shape, dtype)
        va = _rows(v, "v", dev, shape, dtype)
        pos = _ints(positions, "positions", dev, n)
        ids = 0 if seq_ids is None else _ints(seq_ids, "seq_ids", dev, n)
        tab, seqs, cols, tstride = _table(page_table, dev)
        if seq_ids is None and seqs < n:
            _fail(f"{n} tokens without seq_ids need a page table of as many rows, got {seqs}")
        heads, qa, oa = 0, (0, 0, 0, 0), (0, 0, 0, 0)
        if q is not None:
            if q.dim() != 3:
                _fail("q must be 3-D")
            heads = q.shape[1]
            qshape = (n, heads, self.head_dim)
            qa = _rows(q, "q", dev, qshape, dtype)
            if q_out is None:
                q_out = q.new_empty(qshape)
                oa = (q_out.data_ptr(), heads * self.head_dim, self.head_dim, 1)
            else:
                oa = _rows(q_out, "q_out", dev, qshape, dtype)
                _apart(q_out, "q_out")
            if n and oa[0] == qa[0] and oa != qa:
                _fail("q_out may only share q's memory with the same strides")
        elif q_out is not None:
            _fail("q_out without q")
        ra = (0, 0, 0, 0, 0, 0)
        if rope is not None:
            if rope.device != dev or rope.rotary > self.head_dim:
                _fail("the rotation table is on another device or wider than head_dim")
            ra = rope._args
        if n == 0 or seqs == 0:
            if n:
                _fail("an empty page table")
            return q_out
        s = _current(dev)
        if s not in self._streams:
            self._keep(s)
        bad = self._call(self._h, _APPEND.pack(n, heads, kind, *ka, *va, *qa, *oa, pos, ids, tab, seqs, cols, tstride,
                                               *ra), s)
        if bad:
            _check(bad)
        return q_out


class DecodeAttention(_Handle):
    """Attention of one new token per sequence over a PagedKVCache: a plan for
    ``q_heads`` query heads (a multiple of the cache's kv_heads; neighbouring
    heads share a kv head) and at most ``max_seqs`` sequences a call.
    ``scale`` defaults to 1/sqrt(head_dim); ``window`` > 0 limits a sequence
    to its last ``window`` keys.  Calls share the plan's workspace: use one
    plan per stream."""
    _free, _status, _run = "sc_attn_free", "sc_attn_status", "sc_attn_decode"

    def __init__(self, cache: PagedKVCache, q_heads: int, max_seqs: int, scale: Optional[float] = None,
                 window: int = 0):
        if scale is not None and not scale > 0:
            _fail("scale must be positive")
        self.cache, self.q_heads, self.max_seqs, self.window = cache, q_heads, max_seqs, window
        self.device = cache.device
        h, size = ctypes.c_void_p(), ctypes.c_int64()
        _check(lib().sc_attn_workspace(cache._h, q_heads, max_seqs, ctypes.byref(size)))
        # from torch's allocator: a cudaMalloc and cudaFree for each plan took ten times as long as the rest
        self._work = torch.empty(size.value + 256, dtype=torch.uint8, device=cache.k.device)
        torch.cuda.current_stream(self.device).synchronize()  # whatever used that memory before is done
        at = (self._work.data_ptr() + 255) // 256 * 256
        _check(lib().sc_attn_create_in(cache._h, q_heads, max_seqs, scale or 0.0, window, at, size.value, ctypes.byref(h)))
        self._own(h, self._work, cache.k, cache.v)
        self._streams &= cache._streams  # the cache may come from another stream's memory

    def attend(self, q, page_table, seq_lens, out=None, return_lse: bool = False, stream=None):
        """out[s] = softmax(scale q[s] k^T) v over the ``seq_lens[s]`` first
        keys of sequence s, whose pages row s of ``page_table`` lists.  q and
        out: [seqs, q_heads, head_dim] of one type, apart in memory.  A sequence
        of length 0 gives zeros (lse -inf).  Returns out, or (out, lse [seqs, q_heads])."""
        dev, dtype = self.device, q.dtype
        if stream is not None:
            return _on(stream, dev, (q, page_table, seq_lens, out), self.attend, q, page_table, seq_lens, out, return_lse)
        kind = _TYPES.get(dtype)
        if kind is None or q.dim() != 3:
            _fail("q must be a 3-D float32, float16 or bfloat16 tensor")
        n = q.shape[0]
        if n > self.max_seqs:
            _fail(f"{n} sequences, the plan has max_seqs {self.max_seqs}")
        shape = (n, self.q_heads, self.cache.head_dim)
        qa = _rows(q, "q", dev, shape, dtype)
        if out is None:
            out = q.new_empty(shape)
            oa = (out.data_ptr(), self.q_heads * self.cache.head_dim, self.cache.head_dim, 1)
        else:
            oa = _rows(out, "out", dev, shape, dtype)
            _apart(out, "out")
        tab, rows, cols, tstride = _table(page_table, dev)
        if rows < n:
            _fail(f"{n} sequences need a page table of as many rows, got {rows}")
        lens = _ints(seq_lens, "seq_lens", dev, n)
        lse = q.new_empty((n, self.q_heads), dtype=torch.float32) if return_lse else None
        if n:
            s = _current(dev)
            if s not in self._streams:
                self._keep(s)
            bad = self._call(self._h, _ATTEND.pack(n, kind, *qa, *oa, lse.data_ptr() if return_lse else 0, tab, cols,
                                                   tstride, lens), s)
            if bad:
                _check(bad)
        return (out, lse) if return_lse else out


class LowRankAdapters(_Handle):
    """A set of low-rank adapters of one projection (out_features x
    in_features): adapter i adds scales[i] * up[i] @ (down[i] @ x), with
    down[i] [rank_i, in_features] and up[i] [out_features, rank_i] of one type
    (fp32, fp16, bf16) and ranks of 0 to 256.  The weights are copied into the
    set's own layout once."""
    _free, _status, _run = "sc_adapters_free", "sc_adapters_status", "sc_adapters_apply"

    def __init__(self, down: Sequence, up: Sequence, scales: Sequence[float]):
        n = len(down)
        if n == 0 or len(up) != n or len(scales) != n:
            _fail("down, up and scales must be non-empty lists of one length")
        dtype, where = down[0].dtype, down[0].device
        if down[0].dim() != 2 or up[0].dim() != 2:
            _fail("adapter weights must be 2-D, of one type and on one device")
        if dtype not in _TYPES or where.type != "cuda":
            _fail("adapter weights must be float32, float16 or bfloat16 CUDA tensors")
        self.in_features, self.out_features = down[0].shape[-1], up[0].shape[0]
        self.device, self.dtype, self.count = where.index, dtype, n
        ranks = []
        for a, b in zip(down, up):
            if a.dim() != 2 or b.dim() != 2 or a.dtype != dtype or b.dtype != dtype or a.device != where or \
                    b.device != where:
                _fail("adapter weights must be 2-D, of one type and on one device")
            if a.shape[1] != self.in_features or b.shape[0] != self.out_features or a.shape[0] != b.shape[1]:
                _fail(f"adapter shapes do not match: down {tuple(a.shape)}, up {tuple(b.shape)}")
            ranks.append(a.shape[0])
        # rows that lie apart, as the packing reads them; expanded or overlapping ones are copied first
        plain = lambda w: w if w.stride(1) == 1 and (w.shape[0] == 1 or w.stride(0) >= w.shape[1]) else w.contiguous()
        down, up = [plain(a) for a in down], [plain(b) for b in up]
        i64, vp = ctypes.c_int64 * n, ctypes.c_void_p * n
        # a single row's stride means nothing: give the row length
        dl = [a.stride(0) if a.shape[0] > 1 else max(a.shape[1], 1) for a in down]
        ul = [b.stride(0) if b.shape[0] > 1 else max(b.shape[1], 1) for b in up]
        h, size, r = ctypes.c_void_p(), ctypes.c_int64(), i64(*ranks)
        _check(lib().sc_adapters_size(self.in_features, self.out_features, n, r, _TYPES[dtype], ctypes.byref(size)))
        self._memory = torch.empty(size.value + 256, dtype=torch.uint8, device=where)
        at = (self._memory.data_ptr() + 255) // 256 * 256
        _check(lib().sc_adapters_create_in(
            self.device, self.in_features, self.out_features, n, r, _TYPES[dtype],
            vp(*[a.data_ptr() for a in down]), i64(*dl), vp(*[b.data_ptr() for b in up]), i64(*ul),
            (ctypes.c_float * n)(*[float(x) for x in scales]), _current(self.device), at, size.value, ctypes.byref(h)))
        self._own(h, self._memory)
        self.ranks = ranks
        self._scratch = (-1, 0)

    def _workspace(self, n: int) -> int:
        tokens, size = self._scratch  # read once: another thread may put its own pair there
        if tokens != n:
            b = ctypes.c_int64()
            _check(lib().sc_adapters_workspace(self._h, n, ctypes.byref(b)))
            size = b.value
            self._scratch = (n, size)
        return size

    def apply(self, x, ids, base=None, out=None, stream=None):
        """out = base + the adapters' part of each token: x [in_features,
        tokens], base (zeros without one) and out [out_features, tokens] of one
        type with any strides, as SpMMPlan.spmm's B and C; ids [tokens] int32,
        negative for a token without an adapter.  out may be base."""
        dev, dtype = self.device, x.dtype
        if stream is not None:
            return _on(stream, dev, (x, ids, base, out), self.apply, x, ids, base, out)
        kind = _TYPES.get(dtype)
        if kind is None or x.dim() != 2:
            _fail("x must be a 2-D float32, float16 or bfloat16 tensor")
        n = x.shape[1]
        xa = _rows(x, "x", dev, (self.in_features, n), dtype)
        shape = (self.out_features, n)
        ba = (0, 0, 0) if base is None else _rows(base, "base", dev, shape, dtype)
        if out is None:
            # laid out as x is: feature-major, or token-major from a transposed x
            out = x.new_empty((n, self.out_features)).t() if xa[1] == 1 and n > 1 else x.new_empty(shape)
            oa = (out.data_ptr(), *out.stride())
        else:
            oa = _rows(out, "out", dev, shape, dtype)
            _apart(out, "out")
        if n and oa[0] == ba[0] and oa != ba:
            _fail("out may only share base's memory with the same strides")
        if n and oa[0] == xa[0]:
            _fail("out may not be x")
        idp = _ints(ids, "ids", dev, n)
        if n:
            size = self._workspace(n)
            work = x.new_empty(size, dtype=torch.uint8) if size else None
            s = _current(dev)
            if s not in self._streams:
                self._keep(s)
            bad = self._call(self._h, _ADAPT.pack(n, kind, *xa, *ba, *oa, idp, work.data_ptr() if size else 0, size),
                             s)
            if bad:
                _check(bad)
        return out
