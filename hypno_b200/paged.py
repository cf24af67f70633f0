"""Paged KV cache on torch tensors: append with rotation, and attention of new
tokens over the pages.

    PagedKV             one layer's pool of pages (any strides), the handle a
                        program keeps with it
    PagedBatch          one step's packed rows: block table, row starts, lengths
    append              rotated keys (and queries), values -> pages
    attention           softmax attention of the rows over their pages
    rope_table          the model's cos/sin table on the device
    PageTable           host-side owner of pages: sequences grow and are released

A step of a serving loop packs the new tokens of all its sequences (chunks of
prompts and single tokens alike) into rows, appends them, and attends:

    batch = PagedBatch(table, q_start, kv_len, max_q_len, max_kv_len)
    q = append(kv, batch, k, v, q=q, rope=rope)
    out = attention(kv, batch, q)

The operators run on torch's current stream of the pool's device, whichever
device is current, and do not synchronize; use `with torch.cuda.stream(...)`
(or an ExternalStream of HypnoModel.stream) for another one.  Errors raise
HypnoCudaError, ValueError or TypeError.  They call hc_paged_append_dev and
hc_paged_attention_dev.
"""
import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import (DTYPE_FP16, DTYPE_FP32, HC_PAGED_BATCH, HC_ROWS, KV_FP16, KV_FP32, HcPagedKV, call, check, load, raw_stream)

__all__ = ["PagedKV", "PagedBatch", "append", "attention", "rope_table", "PageTable"]

_DTYPE = {torch.float32: DTYPE_FP32, torch.float16: DTYPE_FP16}
_KV = {torch.float32: KV_FP32, torch.float16: KV_FP16}
_pack = HC_ROWS.pack


class PagedKV:
    """One layer's pages: k_pages and v_pages are [n_pages, n_kv_heads,
    page_size, head_dim] views of float32 or float16 memory with the last
    dimension contiguous; the other strides are free (a [n_pages, page_size,
    n_kv_heads, head_dim] pool is passed as pool.transpose(1, 2))."""

    __slots__ = ("_k", "_v", "struct", "ref", "device", "index", "n_kv_heads", "head_dim", "page_size", "n_pages")

    def __init__(self, k_pages, v_pages):
        for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            if not isinstance(t, torch.Tensor) or t.dim() != 4 or not t.is_cuda:
                raise TypeError(f"{name} must be a 4-dimensional CUDA tensor")
            if t.dtype not in _KV:
                raise TypeError(f"{name} must be float32 or float16, not {t.dtype}")
            if t.shape[3] > 1 and t.stride(3) != 1:
                raise ValueError(f"the last dimension of {name} must be contiguous")
        if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device:
            raise ValueError("k_pages and v_pages must have one shape, type and device")
        self._k, self._v = k_pages, v_pages
        self.device, self.index = k_pages.device, k_pages.device.index
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k_pages.shape
        self.struct = HcPagedKV(k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], *v_pages.stride()[:3],
                                _KV[k_pages.dtype], self.n_pages, self.page_size, self.n_kv_heads, self.head_dim, 0)
        self.ref = ctypes.addressof(self.struct)

    # (the struct holds their addresses: another pool is another PagedKV)
    k = property(lambda self: self._k, doc="The keys' pages.")
    v = property(lambda self: self._v, doc="The values' pages.")

    @classmethod
    def alloc(cls, n_pages, page_size, n_kv_heads, head_dim, dtype=torch.float16, device="cuda"):
        """A pool of its own, zeroed."""
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


def _int32(t, name, dim, index):
    """Raises for what PagedBatch does not take."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.dim() != dim or t.get_device() != index or index < 0:
        raise TypeError(f"{name} must be a {dim}-dimensional int32 CUDA tensor on the device of kv_len")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")


class PagedBatch:
    """The new tokens of a step.  block_table [n_seqs, max_pages] (an entry
    outside the pool is a hole), q_start [n_seqs + 1] (the packed rows of
    sequence b are q_start[b] .. q_start[b + 1] - 1), kv_len [n_seqs] (its
    positions, the new ones included), all int32 on the pool's device.
    max_q_len and max_kv_len are the host's upper bounds on a sequence's rows
    and positions: they choose launches, not results.  The tensors' contents may
    change between calls; other tensors or bounds are another batch."""

    __slots__ = ("_tensors", "_bounds", "index", "n_rows", "blob")

    def __init__(self, block_table, q_start, kv_len, max_q_len, max_kv_len):
        index = kv_len.get_device()
        _int32(kv_len, "kv_len", 1, index)
        _int32(block_table, "block_table", 2, index)
        _int32(q_start, "q_start", 1, index)
        n = block_table.shape[0]
        if kv_len.shape[0] != n or q_start.shape[0] != n + 1:
            raise ValueError(f"a block_table of {n} rows needs {n} lengths and {n + 1} row starts")
        if max_q_len < 0 or max_kv_len < 0:
            raise ValueError("max_q_len and max_kv_len must not be negative")
        self._tensors, self._bounds, self.index = (block_table, q_start, kv_len), (max_q_len, max_kv_len), index
        self.n_rows = -1

    # (read only: what pack() made of them is kept)
    block_table = property(lambda self: self._tensors[0])
    q_start = property(lambda self: self._tensors[1])
    kv_len = property(lambda self: self._tensors[2])
    max_q_len = property(lambda self: self._bounds[0])
    max_kv_len = property(lambda self: self._bounds[1])

    def pack(self, n_rows):
        """The batch with so many rows as the C ABI takes it."""
        if n_rows != self.n_rows:
            t, starts, lengths = self._tensors
            n, pages = t.shape
            self.blob = HC_PAGED_BATCH.pack(t.data_ptr(), starts.data_ptr(), lengths.data_ptr(), t.stride(0), n, pages, n_rows,
                                            *self._bounds, 0)
            self.n_rows = n_rows
        return self.blob


def _rows(t, name, kv, dtype, n):
    shape = t.shape
    if len(shape) != 3 or t.dtype is not dtype or t.get_device() != kv.index:
        raise TypeError(f"{name} must be a 3-dimensional {dtype} tensor on {kv.device}")
    rs, hs, ds = t.stride()
    d = shape[2]
    if d != kv.head_dim or shape[0] != n:
        raise ValueError(f"{name} of shape {tuple(shape)}: the cache has heads of {kv.head_dim}, the call {n} rows")
    if ds != 1 and d > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return _pack(t.data_ptr(), rs, hs)


def _same_device(kv, batch):
    if batch.index != kv.index:
        raise ValueError(f"the batch is on cuda:{batch.index}, the pool on {kv.device}")


def append(kv, batch, k, v, q=None, rope=None, pairs="adjacent", q_out=None):
    """Stores the rows' keys and values ([n_rows, n_kv_heads, head_dim]) in
    their pages, rotating keys, and queries ([n_rows, n_heads, head_dim]) if
    given, by rope ([positions, rot / 2, 2] float32 cos/sin; None: no
    rotation).  pairs: "adjacent" turns elements (2j, 2j + 1) together, the
    model's form; "halves" turns (j, j + rot / 2).  Elements past rot pass
    through.  Returns the rotated queries (in q_out, which may be q), or None.
    k, v and q have one type, float32 or float16, and any row and head
    strides; no two rows of one call may name the same position."""
    if _lib.current_device() != kv.index:
        with _lib.on_device(kv.index):
            return append(kv, batch, k, v, q, rope, pairs, q_out)
    _same_device(kv, batch)
    dtype = k.dtype
    code = _DTYPE.get(dtype)
    if code is None:
        raise TypeError(f"k must be float32 or float16, not {dtype}")
    n = k.shape[0]
    ks, vs = _rows(k, "k", kv, dtype, n), _rows(v, "v", kv, dtype, n)
    if k.shape[1] != kv.n_kv_heads or v.shape[1] != kv.n_kv_heads:
        raise ValueError(f"k and v need the cache's {kv.n_kv_heads} heads")
    if pairs != "adjacent" and pairs != "halves":
        raise ValueError(f"pairs must be 'adjacent' or 'halves', not {pairs!r}")
    qs = os_ = None
    heads = 0
    if q is not None:
        qs = _rows(q, "q", kv, dtype, n)
        heads = q.shape[1]
        if q_out is None:
            q_out = q.new_empty(q.shape)
        elif q_out.shape != q.shape:
            raise ValueError("q_out must have the shape of q")
        os_ = _rows(q_out, "q_out", kv, dtype, n)
    elif q_out is not None:
        raise ValueError("q_out without q")
    table, table_rows, rot = None, 0, 0
    if rope is not None:
        shape = rope.shape
        if rope.dtype is not torch.float32 or len(shape) != 3 or shape[2] != 2 or rope.get_device() != kv.index:
            raise TypeError(f"rope must be a [positions, rot / 2, 2] float32 tensor on {kv.device}")
        if not rope.is_contiguous():
            raise ValueError("rope must be contiguous")
        table, table_rows, rot = rope.data_ptr(), shape[0], 2 * shape[1]
    check(load().hc_paged_append_dev(kv.ref, batch.pack(n), ks, vs, qs, os_, heads, code, table, table_rows, rot,
                                     pairs == "halves", raw_stream(kv.index)))
    return q_out


def attention(kv, batch, q, out=None, scale=None, window=0, lse=None):
    """out[r, h] = softmax(scale * q[r, h] . K) V over the positions up to the
    row's own (window > 0: the last `window` of them), scale = head_dim ** -0.5
    by default; query head h reads KV head h // (n_heads // n_kv_heads).  A row
    that sees nothing gives zeros.  q is [n_rows, n_heads, head_dim] float32 or
    float16, out the same; lse, if given, is a contiguous [n_rows, n_heads]
    float32 tensor for the log of the sums.  The softmax is exact (the
    flat-cache forward passes keep the reference's polynomial).  Scores and sums
    are float32; float16 queries over a float16 cache round the weights to 11
    bits for their product with V (an error like the output's own rounding),
    float32 ones keep 22 bits."""
    if _lib.current_device() != kv.index:
        with _lib.on_device(kv.index):
            return attention(kv, batch, q, out, scale, window, lse)
    _same_device(kv, batch)
    dtype = q.dtype
    code = _DTYPE.get(dtype)
    if code is None:
        raise TypeError(f"q must be float32 or float16, not {dtype}")
    n, heads, dim = q.shape
    qs = _rows(q, "q", kv, dtype, n)
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape:
        raise ValueError("out must have the shape of q")
    os_ = _rows(out, "out", kv, dtype, n)
    lse_ptr = None
    if lse is not None:
        if lse.dtype != torch.float32 or lse.shape != (n, heads) or not lse.is_contiguous() or lse.device != kv.device:
            raise TypeError(f"lse must be a contiguous [{n}, {heads}] float32 tensor on {kv.device}")
        lse_ptr = lse.data_ptr()
    lib, ref = load(), batch.pack(n)
    need = ctypes.c_size_t()
    check(lib.hc_paged_attention_workspace(kv.ref, ref, heads, code, window, ctypes.byref(need)))
    # the workspace lives until the stream's later allocations reuse it: torch orders them after this call
    ws = torch.empty(need.value, dtype=torch.uint8, device=kv.device) if need.value else None
    check(lib.hc_paged_attention_dev(kv.ref, ref, qs, os_, lse_ptr, heads, code, dim ** -0.5 if scale is None else scale,
                                     window, ws.data_ptr() if ws is not None else None, need.value, raw_stream(kv.index)))
    return out


def rope_table(positions, head_dim, theta, device="cuda"):
    """The model's own cos/sin table (transformer.rs:317-343) as the [positions,
    head_dim / 2, 2] float32 tensor that append() takes."""
    t = np.empty((positions, head_dim // 2, 2), np.float32)
    call("hc_rope_table_host", positions, head_dim, float(theta), t.ctypes.data)
    return torch.from_numpy(t).to(device)


class PageTable:
    """Owner of a pool's pages: sequences take pages as they grow and give them
    back together.  `table` is the [max_seqs, max_pages] int32 host array of
    every sequence's pages, -1 where it has none."""

    def __init__(self, n_pages, page_size, max_seqs, max_pages):
        if min(n_pages, page_size, max_seqs, max_pages) < 1:
            raise ValueError("PageTable sizes must be positive")
        self.page_size, self.max_pages = page_size, max_pages
        self.free = list(range(n_pages - 1, -1, -1))
        self.table = np.full((max_seqs, max_pages), -1, np.int32)
        self.lengths = np.zeros(max_seqs, np.int32)

    def can_grow(self, seq, tokens):
        need = -(-(int(self.lengths[seq]) + tokens) // self.page_size)
        held = -(-int(self.lengths[seq]) // self.page_size)
        return need <= self.max_pages and need - held <= len(self.free)

    def grow(self, seq, tokens):
        """Takes the pages for `tokens` more positions; returns the new length."""
        if tokens < 0:
            raise ValueError("tokens must not be negative")
        if not self.can_grow(seq, tokens):
            raise ValueError(f"sequence {seq}: no pages for {tokens} more positions")
        held = -(-int(self.lengths[seq]) // self.page_size)
        self.lengths[seq] += tokens
        for i in range(held, -(-int(self.lengths[seq]) // self.page_size)):
            self.table[seq, i] = self.free.pop()
        return int(self.lengths[seq])

    def release(self, seq):
        """Gives the sequence's pages back; its length becomes 0."""
        row = self.table[seq]
        self.free.extend(int(p) for p in row[row >= 0][::-1])
        row[:] = -1
        self.lengths[seq] = 0
