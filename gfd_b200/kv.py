"""Paged KV cache: append with rotation, attention, attention behind a shared prefix, merge.

The operators that fill and read the KV blocks which the gathers fetch (gfd_kv_* in
include/gfd_b200.h, where shapes, masks and errors are specified).  Arrays are device
tensors -- anything with data_ptr(), shape, stride(), dtype and device as torch tensors
have; nothing is copied or made contiguous, strides are passed on.

    cache = kv.PagedCache(ctx, blocks[:, 0], blocks[:, 1])   # blocks: [n, 2, tokens, heads, dim]
    batch = kv.Batch(row_start, kv_len, table)               # int32 device tensors
    cache.fetch(host_pool_ptr, host_ids, block_ids)          # host blocks -> cache blocks
    cache.append(batch, k, v, q=q, q_out=q_rot, inv_freq=inv_freq, stream=s)
    cache.attend(batch, q_rot, out, workspace=ws, stream=s)

`stream`: 0 (the context's stream), a stream handle, or a torch stream object (whose
default stream is passed as the legacy default stream).
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np

from . import Context, entries_array

BF16, FP16, FP32 = 0, 1, 2
BAD_PAGE, BAD_LENGTH, GAVE_UP = 1, 2, 4  # bits of *status
MAX_SEQS = 4096
_VP = ctypes.c_void_p
_TYPES = {"torch.bfloat16": BF16, "torch.float16": FP16, "torch.float32": FP32}


class _Cache(ctypes.Structure):
    _fields_ = [("k", _VP), ("v", _VP)] + [(n, ctypes.c_int64) for n in ("blocks", "block_stride", "token_stride",
                                                                         "head_stride")] + [
        (n, ctypes.c_int32) for n in ("block_tokens", "heads", "head_dim", "dtype")]


class _Batch(ctypes.Structure):
    _fields_ = [("row_start", _VP), ("kv_len", _VP), ("table", _VP), ("table_stride", ctypes.c_int64),
                ("rows", ctypes.c_int64), ("seqs", ctypes.c_int32), ("table_width", ctypes.c_int32)]


class _Rows(ctypes.Structure):
    _fields_ = [("data", _VP), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _Append(ctypes.Structure):
    _fields_ = [("k", _Rows), ("v", _Rows), ("q", _Rows), ("q_out", _Rows), ("inv_freq", _VP), ("positions", _VP),
                ("status", _VP)] + [(n, ctypes.c_int32) for n in ("q_heads", "rot_dim", "interleaved", "_pad")]


class _Attend(ctypes.Structure):
    _fields_ = [("q", _Rows), ("out", _Rows), ("lse", _VP), ("alibi", _VP), ("prefix_len", _VP), ("workspace", _VP),
                ("workspace_bytes", ctypes.c_size_t), ("status", _VP)] + [
        (n, ctypes.c_int32) for n in ("q_heads", "out_dtype", "max_q_len", "causal", "window")] + [
        ("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("_pad", ctypes.c_int32)]


class _Merge(ctypes.Structure):
    _fields_ = [("parts", _Rows), ("part_stride", ctypes.c_int64), ("part_lse", _VP), ("out", _Rows), ("lse", _VP),
                ("rows", ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ("part_count", "heads", "head_dim", "part_dtype", "out_dtype", "_pad")]


def _format(c) -> str:
    """struct format of a ctypes structure (all fields aligned, so nothing is padded)."""
    one = {_VP: "Q", ctypes.c_size_t: "Q", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}
    return "".join(one[t] if t in one else _format(t) for _, t in c._fields_)


def _packer(c):
    p = struct.Struct("=" + _format(c))
    assert p.size == ctypes.sizeof(c)

    def pack(*values) -> bytes:
        try:
            return p.pack(*values)
        except (struct.error, OverflowError) as e:
            raise ValueError(f"an argument is out of range: {e}") from None

    return pack


# A call packs its arguments in one go: a ctypes structure, field by field, costs as much as the launch.
_pack_batch, _pack_append, _pack_attend, _pack_merge = (_packer(c) for c in (_Batch, _Append, _Attend, _Merge))


def _stream(s) -> int:
    if isinstance(s, int):
        return s
    return s.cuda_stream or 1  # 1: the legacy default stream, which torch calls 0


_codes = {}  # dtype object -> code or None: naming a type costs as much as a whole call


def _code(dtype):
    if dtype not in _codes:
        _codes[dtype] = _TYPES.get(str(dtype), str(dtype))
    return _codes[dtype]


def _dtype(x, what: str) -> int:
    d = _code(x.dtype)
    if not isinstance(d, int):
        raise ValueError(f"{what}: unsupported type {x.dtype}")
    return d


def _rows(x, what: str, rows: int, heads: int, dim: int, dtype: int):
    """Address, row stride and head stride of a row array."""
    if x.shape != (rows, heads, dim):
        raise ValueError(f"{what}: shape {tuple(x.shape)}, expected {(rows, heads, dim)}")
    if _code(x.dtype) != dtype:
        raise ValueError(f"{what}: type {x.dtype} does not match")
    row, head, one = x.stride()
    if one != 1:
        raise ValueError(f"{what}: the elements of a head must be contiguous")
    return x.data_ptr(), row if rows > 1 else 0, head if heads > 1 else 0


def _vector(x, what: str, shape, dtype) -> int:
    """Address of a contiguous vector or matrix (None: 0)."""
    if x is None:
        return 0
    if x.shape != shape or _code(x.dtype) != dtype or not x.is_contiguous():
        raise ValueError(f"{what}: expected contiguous {'torch.float32' if dtype == FP32 else dtype} of shape {tuple(shape)}, "
                         f"got {x.dtype} {tuple(x.shape)}")
    return x.data_ptr()


class Batch:
    """The sequences of a call: row_start [seqs + 1], kv_len [seqs], table [seqs, width]; int32
    device tensors that the kernels read when they run."""

    def __init__(self, row_start, kv_len, table):
        seqs = kv_len.shape[0]
        if table.dim() != 2 or table.shape[0] != seqs or _code(table.dtype) != "torch.int32":
            raise ValueError(f"table: expected int32 of shape ({seqs}, width), got {table.dtype} {tuple(table.shape)}")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("table: the entries of a row must be contiguous")
        self.arrays = (row_start, kv_len, table)
        self.seqs = seqs
        self._head = (_vector(row_start, "row_start", (seqs + 1,), "torch.int32"), _vector(kv_len, "kv_len", (seqs,), "torch.int32"),
                      table.data_ptr(), table.stride(0) if seqs > 1 else table.shape[1])
        self._tail = (seqs, table.shape[1])

    def _c(self, rows: int) -> bytes:
        return _pack_batch(*self._head, rows, *self._tail)


class PagedCache:
    """K and V of a paged cache: [blocks, block_tokens, heads, head_dim] views of equal strides
    (for example of one tensor [blocks, 2, block_tokens, heads, head_dim])."""

    def __init__(self, ctx: Context, k, v):
        if k.dim() != 4 or tuple(k.shape) != tuple(v.shape) or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError("k and v must be [blocks, block_tokens, heads, head_dim] of one type and equal strides")
        if k.stride(3) != 1:
            raise ValueError("the elements of a head must be contiguous")
        self.ctx = ctx
        self.k, self.v = k, v
        self.blocks, self.block_tokens, self.heads, self.head_dim = k.shape
        self.dtype = _dtype(k, "k")
        st = k.stride()
        self._c = bytes(_Cache(k.data_ptr(), v.data_ptr(), self.blocks, st[0], st[1], st[2] if self.heads > 1 else 0,
                               self.block_tokens, self.heads, self.head_dim, self.dtype))

    # -- moving blocks between host memory and the cache ----------------------------------
    def _block_entries(self, host_ptr: int, host_ids, block_ids, to_host: bool) -> np.ndarray:
        st, item = self.k.stride(), 2
        dense = self.block_tokens * self.heads * self.head_dim
        if st[2] != self.head_dim and self.heads > 1 or st[1] != self.heads * self.head_dim:
            raise ValueError("fetch and offload need the tokens of a block contiguous")
        host_ids, block_ids = (np.asarray(x) for x in (host_ids, block_ids))
        if host_ids.shape != block_ids.shape or host_ids.ndim != 1:
            raise ValueError("host_ids and block_ids must be vectors of one length")
        if host_ids.size:
            if host_ids.dtype.kind not in "iu" or block_ids.dtype.kind not in "iu":
                raise ValueError("host_ids and block_ids must be whole numbers")
            if int(host_ids.min()) < 0 or int(host_ptr) + (int(host_ids.max()) + 1) * 2 * dense * item >= 1 << 64:
                raise ValueError("a host block is outside the address space")
            if int(block_ids.min()) < 0 or int(block_ids.max()) >= self.blocks:
                raise ValueError("a block id is outside the cache")
        host_ids, block_ids = host_ids.astype(np.uint64), block_ids.astype(np.uint64)
        nbytes = np.uint64(dense * item)
        host = np.uint64(host_ptr) + host_ids * np.uint64(2) * nbytes
        parts = []
        for x, at in ((self.k, np.uint64(0)), (self.v, nbytes)):
            dev = np.uint64(x.data_ptr()) + block_ids * np.uint64(st[0] * item)
            parts.append(entries_array(host + at, dev, nbytes) if to_host else entries_array(dev, host + at, nbytes))
        # K and V of a block side by side, so that their copies merge where they continue each other
        return np.stack(parts, 1).reshape(-1)

    def fetch(self, host_ptr: int, host_ids, block_ids, stream=0):
        """Gathers host blocks (block h: K then V of all its tokens, at host_ptr + h * block bytes
        in pinned memory) into the cache's blocks, asynchronously on `stream`.  No block of the cache is named twice."""
        e = self._block_entries(host_ptr, host_ids, block_ids, False)
        self.ctx._check(self.ctx.gather(e, _stream(stream)))

    def offload(self, host_ptr: int, host_ids, block_ids, stream=0):
        """The reverse of fetch: cache blocks to host blocks, none of which is named twice."""
        e = self._block_entries(host_ptr, host_ids, block_ids, True)
        self.ctx._check(self.ctx.scatter(e, _stream(stream)))

    # -- operators ------------------------------------------------------------------------
    def append(self, batch: Batch, k, v, q=None, q_out=None, inv_freq=None, interleaved: bool = False, positions=None,
               status=None, stream=0):
        """gfd_kv_append: stores k, v [rows, heads, dim] at the ends of the sequences, k (and q
        into q_out) rotated by position when inv_freq [rot_dim / 2] is given."""
        rows, heads, dim, dtype = k.shape[0], self.heads, self.head_dim, self.dtype
        if (q is None) != (q_out is None):
            raise ValueError("q and q_out go together")
        q_heads, q_args, out_args = 0, (0, 0, 0), (0, 0, 0)
        if q is not None:
            q_heads = q.shape[1]
            q_args = _rows(q, "q", rows, q_heads, dim, dtype)
            out_args = _rows(q_out, "q_out", rows, q_heads, dim, dtype)
        half = 0 if inv_freq is None else inv_freq.shape[0]
        a = _pack_append(*_rows(k, "k", rows, heads, dim, dtype), *_rows(v, "v", rows, heads, dim, dtype), *q_args, *out_args,
                         _vector(inv_freq, "inv_freq", (half,), FP32), _vector(positions, "positions", (rows,), "torch.int32"),
                         _vector(status, "status", (1,), "torch.int32"), q_heads, 2 * half, bool(interleaved), 0)
        ctx = self.ctx
        ctx._check(ctx.lib.gfd_kv_append(ctx.handle, self._c, batch._c(rows), a, _stream(stream)))

    def workspace_bytes(self, rows: int, q_heads: int, seqs: int, max_q_len: int = 0, shared_len: int = 0) -> int:
        """Bytes of workspace that attend / attend_shared need for these shapes."""
        b, a, n = _Batch(rows=rows, seqs=seqs), _Attend(q_heads=q_heads, max_q_len=max_q_len), ctypes.c_size_t()
        self.ctx._check(self.ctx.lib.gfd_kv_attend_workspace(self.ctx.handle, self._c, ctypes.byref(b),
                                                             ctypes.byref(a), shared_len, ctypes.byref(n)))
        return n.value

    def _attend(self, batch, q, out, lse, scale, causal, window, softcap, alibi, prefix_len, max_q_len, workspace, status):
        rows, heads, dim = q.shape[0], q.shape[1], self.head_dim
        out_dtype = _dtype(out, "out")
        room, room_bytes = 0, 0
        if workspace is not None:
            if not workspace.is_contiguous():
                raise ValueError("workspace: must be contiguous")
            room, room_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        return batch._c(rows), _pack_attend(
            *_rows(q, "q", rows, heads, dim, self.dtype), *_rows(out, "out", rows, heads, dim, out_dtype),
            _vector(lse, "lse", (rows, heads), FP32), _vector(alibi, "alibi", (heads,), FP32),
            _vector(prefix_len, "prefix_len", (batch.seqs,), "torch.int32"), room, room_bytes,
            _vector(status, "status", (1,), "torch.int32"), heads, out_dtype, max_q_len or 0, bool(causal), window,
            dim ** -0.5 if scale is None else scale, softcap, 0)

    def attend(self, batch: Batch, q, out, lse=None, scale=None, causal: bool = True, window: int = 0, softcap: float = 0.0,
               alibi=None, prefix_len=None, max_q_len=None, workspace=None, status=None, stream=0):
        """gfd_kv_attend: q [rows, q_heads, dim] over the cache into out (and lse [rows, q_heads])."""
        b, a = self._attend(batch, q, out, lse, scale, causal, window, softcap, alibi, prefix_len, max_q_len, workspace, status)
        ctx = self.ctx
        ctx._check(ctx.lib.gfd_kv_attend(ctx.handle, self._c, b, a, _stream(stream)))

    def attend_shared(self, batch: Batch, shared_table, shared_len: int, q, out, lse=None, scale=None, causal: bool = True,
                      window: int = 0, softcap: float = 0.0, alibi=None, prefix_len=None, max_q_len=None, workspace=None,
                      status=None, stream=0):
        """gfd_kv_attend_shared: the same behind shared_len tokens that every sequence starts with,
        in the blocks of shared_table."""
        b, a = self._attend(batch, q, out, lse, scale, causal, window, softcap, alibi, prefix_len, max_q_len, workspace, status)
        need = -(-shared_len // self.block_tokens)
        if shared_table.dim() != 1 or shared_table.shape[0] < need:
            raise ValueError(f"shared_table: {need} block ids needed for {shared_len} tokens")
        table = _vector(shared_table, "shared_table", shared_table.shape, "torch.int32")
        ctx = self.ctx
        ctx._check(ctx.lib.gfd_kv_attend_shared(ctx.handle, self._c, b, table, shared_len, a, _stream(stream)))


def merge(ctx: Context, parts, part_lse, out, lse=None, stream=0):
    """gfd_kv_merge: joins parts [parts, rows, heads, dim] with part_lse [parts, rows, heads]."""
    if parts.dim() != 4 or parts.stride(3) != 1:
        raise ValueError("parts must be [parts, rows, heads, dim], the elements of a head contiguous")
    n, rows, heads, dim = parts.shape
    part, row, head, _ = parts.stride()
    out_dtype = _dtype(out, "out")
    a = _pack_merge(parts.data_ptr(), row if rows > 1 else 0, head if heads > 1 else 0, part if n > 1 else 0,
                    _vector(part_lse, "part_lse", (n, rows, heads), FP32), *_rows(out, "out", rows, heads, dim, out_dtype),
                    _vector(lse, "lse", (rows, heads), FP32), rows, n, heads, dim, _dtype(parts, "parts"), out_dtype, 0)
    ctx._check(ctx.lib.gfd_kv_merge(ctx.handle, a, _stream(stream)))
