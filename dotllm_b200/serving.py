"""Serving operators over the C ABI: an 8-bit paged KV pool (write, read), attention of a batch over
a shared prefix and its own pages, and the verification of drafted tokens.

Arguments are CUDA tensors; a call runs on the calling thread's current torch stream of their
device, asynchronously, and returns new tensors (outputs and scratch come from torch's allocator on
that stream).  Wrong types, shapes, strides or devices raise ``ValueError`` before the call; what
the library refuses raises ``CudaBackendError``.  There is no other path: without the library or a
device every call fails.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import native
from .native import check, lib

PAGE = 64
KVQ_I8, KVQ_E4M3 = 0, 1
_FORMATS = {torch.int8: KVQ_I8, torch.float8_e4m3fn: KVQ_E4M3}
_raw_stream = torch._C._cuda_getCurrentRawStream
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 25}


def _bad(text: str):
    raise ValueError(text)


def _count(n: int) -> int:
    """n for a 32-bit count of the library, which refuses (or bounds) what does not fit; ctypes would keep its low bits.
    (Rows, heads and pages of tensors that fit a device stay below.)"""
    return max(-(1 << 31), min(n, (1 << 31) - 1))


def _int32(name: str, t: torch.Tensor, shape: tuple, device: int) -> int:
    if t.dtype is not torch.int32 or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        _bad(f"{name}: needs a contiguous int32 tensor of shape {shape} on cuda:{device}")
    return t.data_ptr()


class KvqPool:
    """Pages of 8-bit K and V: codes ``[n_pages, heads_kv, 64, head_dim]`` (int8 or float8_e4m3fn) and
    fp32 scales ``[n_pages, heads_kv, 64]``.  Holds the tensors; many batches share one pool."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "device", "n_pages", "heads_kv", "head_dim", "_c")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        fmt, shape, device = _FORMATS.get(k.dtype), k.shape, k.get_device()
        if fmt is None or v.dtype is not k.dtype:
            _bad("KvqPool: codes must be int8 or float8_e4m3fn, K and V alike")
        if len(shape) != 4 or shape[2] != PAGE or v.shape != shape:
            _bad("KvqPool: codes must be [n_pages, heads_kv, 64, head_dim], K and V alike")
        self.n_pages, self.heads_kv, _, self.head_dim = shape
        if k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32 or k_scale.shape != shape[:3] \
                or v_scale.shape != shape[:3]:
            _bad("KvqPool: scales must be float32 [n_pages, heads_kv, 64]")
        if device < 0 or v.get_device() != device or k_scale.get_device() != device or v_scale.get_device() != device:
            _bad("KvqPool: all tensors must be on one CUDA device")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            _bad("KvqPool: tensors must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, device
        self._c = native.KvqPool(fmt, self.head_dim, self.heads_kv, self.n_pages, k.data_ptr(), v.data_ptr(),
                                 k_scale.data_ptr(), v_scale.data_ptr())

    @classmethod
    def empty(cls, n_pages: int, heads_kv: int, head_dim: int, dtype: torch.dtype = torch.int8, device="cuda") -> "KvqPool":
        """A new pool; its contents are undefined until written."""
        shape = (n_pages, heads_kv, PAGE, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                   torch.empty(shape[:3], dtype=torch.float32, device=device),
                   torch.empty(shape[:3], dtype=torch.float32, device=device))


class KvqBatch:
    """Sequences over a pool: ``pages[b, i]`` holds positions 64 i .. 64 i + 63 of sequence b,
    ``seq_len[b]`` is its length, and rows ``row_start[b] .. row_start[b + 1]`` of a call are its last
    positions.  ``max_rows`` bounds the rows of any one sequence; rows beyond it, and rows of no sequence, leave
    their part of a call's (new) outputs undefined."""

    __slots__ = ("row_start", "seq_len", "pages", "device", "max_rows", "_sizes", "_ptrs")

    def __init__(self, row_start: torch.Tensor, seq_len: torch.Tensor, pages: torch.Tensor, max_rows: int):
        shape = pages.shape
        if len(shape) != 2:
            _bad("KvqBatch: pages must be [batch, max_pages]")
        device = pages.get_device()
        if device < 0:
            _bad("KvqBatch: tensors must be on a CUDA device")
        if max_rows < 0:
            _bad("KvqBatch: max_rows is negative")
        self.row_start, self.seq_len, self.pages, self.device, self.max_rows = row_start, seq_len, pages, device, max_rows
        self._sizes = shape[0], max_rows, shape[1]
        if max(self._sizes) >= 1 << 31:
            self._sizes = tuple(map(_count, self._sizes))
        self._ptrs = (_int32("row_start", row_start, (shape[0] + 1,), device), _int32("seq_len", seq_len, (shape[0],), device),
                      _int32("pages", pages, shape, device))

    def _c(self, rows: int) -> native.KvqBatch:
        return native.KvqBatch(self._sizes[0], rows, self._sizes[1], self._sizes[2], *self._ptrs)


def _rows(name: str, t: torch.Tensor, heads: int, dim: int, device: int) -> int:
    """ld of a [rows, heads, dim] tensor whose rows may be strided; its heads and values are dense."""
    s = t.shape
    if len(s) != 3 or s[1] != heads or s[2] != dim or t.get_device() != device:
        _bad(f"{name}: needs [rows, {heads}, {dim}] on cuda:{device}")
    ld, st_head, st_value = t.stride()
    if st_value != 1 or (st_head != dim and heads > 1) or (ld < heads * dim and s[0] > 1):
        _bad(f"{name}: heads and values of a row must be dense and rows must not overlap")
    return ld


def _call(fn, device: int, *args) -> None:
    """fn(*args, stream) on torch's current stream of the tensors' device, made the current device."""
    stream = _raw_stream(device)
    if torch.cuda.current_device() == device:
        check(fn(*args, stream))
    else:
        with torch.cuda.device(device):
            check(fn(*args, stream))


def kvq_write(pool: KvqPool, batch: KvqBatch, k: torch.Tensor, v: torch.Tensor) -> None:
    """Quantise the rows ``k`` and ``v`` ([rows, heads_kv, head_dim], float32, float16 or bfloat16; rows
    may be strided) into their positions' slots of the pool."""
    if k.dtype not in _TYPES or v.dtype is not k.dtype or v.shape != k.shape:
        _bad("kvq_write: K and V must be float32, float16 or bfloat16, alike")
    if batch.device != pool.device:
        _bad("kvq_write: pool and batch are on different devices")
    ld_k = _rows("k", k, pool.heads_kv, pool.head_dim, pool.device)
    ld_v = _rows("v", v, pool.heads_kv, pool.head_dim, pool.device)
    _call(lib().llmdot_cuda_kvq_write, pool.device, pool._c, batch._c(k.shape[0]), k.data_ptr(), v.data_ptr(), _TYPES[k.dtype],
          ld_k, ld_v)


def kvq_read(pool: KvqPool, batch: KvqBatch, rows: int, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows' positions as values: K and V, each [rows, heads_kv, head_dim]."""
    if dtype not in _TYPES:
        _bad("kvq_read: dtype must be float32, float16 or bfloat16")
    if rows < 0 or batch.device != pool.device:
        _bad("kvq_read: negative rows, or pool and batch on different devices")
    out = pool.k_scale.new_empty((2, rows, pool.heads_kv, pool.head_dim), dtype=dtype)
    ld = pool.heads_kv * pool.head_dim
    k, v = out.unbind(0)
    _call(lib().llmdot_cuda_kvq_read, pool.device, pool._c, batch._c(rows), k.data_ptr(), v.data_ptr(), _TYPES[dtype], ld, ld)
    return k, v


def kvq_attention(pool: KvqPool, batch: KvqBatch, q: torch.Tensor, prefix_pages: Optional[torch.Tensor] = None,
                  prefix_len: int = 0, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0,
                  return_lse: bool = False):
    """Attention of the rows ``q`` ([rows, heads, head_dim]; rows may be strided) over the shared prefix
    (``prefix_len`` positions in the pages ``prefix_pages``) and their sequences' own positions.  Returns the
    output in q's type, and with ``return_lse`` the log of the exponentials' sum, [rows, heads] fp32.
    ``scale`` defaults to head_dim ** -0.5."""
    if q.dtype not in _TYPES or q.dim() != 3:
        _bad("kvq_attention: q must be float32, float16 or bfloat16 [rows, heads, head_dim]")
    rows, heads = q.shape[0], q.shape[1]
    device = pool.device
    if batch.device != device:
        _bad("kvq_attention: pool and batch are on different devices")
    ld = _rows("q", q, heads, pool.head_dim, device)
    prefix = 0
    if prefix_len > 0:
        if prefix_pages is None:
            _bad("kvq_attention: prefix_len without prefix_pages")
        if prefix_pages.dim() != 1 or prefix_pages.shape[0] * PAGE < prefix_len:
            _bad("kvq_attention: prefix_pages holds fewer than prefix_len positions")
        prefix = _int32("prefix_pages", prefix_pages, prefix_pages.shape, device)
    if not (-1 < window < 1 << 31 and -1 < prefix_len < 1 << 31):
        window, prefix_len = _count(window), _count(prefix_len)
    L, p, b = lib(), pool._c, batch._c(rows)
    a = native.KvqAttn(heads, _TYPES[q.dtype], prefix_len, window, pool.head_dim ** -0.5 if scale is None else scale, softcap,
                       prefix)
    need = C.c_size_t()
    check(L.llmdot_cuda_kvq_attention_workspace(p, b, a, need))
    out = q.new_empty(q.shape)
    lse = q.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    work, size = None, need.value
    if size:
        work = q.new_empty(size, dtype=torch.uint8)
    _call(L.llmdot_cuda_kvq_attention, device, p, b, a, q.data_ptr(), ld, out.data_ptr(), heads * pool.head_dim,
          lse.data_ptr() if return_lse else None, work.data_ptr() if size else None, size)
    return (out, lse) if return_lse else out


def verify_draft(p: torch.Tensor, q: Optional[torch.Tensor], draft: torch.Tensor, uniform: torch.Tensor,
                 n_draft: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Verify drafted tokens against the target's probabilities.

    ``p`` [batch, k + 1, vocab] and ``q`` [batch, k, vocab] (None: drafts without probabilities, as from a
    lookup) are float32; ``draft`` [batch, k] int32; ``uniform`` [batch, k + 1] float32 in [0, 1), the last of a
    row for the drawn token; ``n_draft`` [batch] int32 counts a sequence's drafts (None: k).  Returns
    ``tokens`` [batch, k + 1] int32 -- the accepted drafts, the drawn token, then -1 -- and ``accepted`` [batch]."""
    if p.dtype is not torch.float32 or p.dim() != 3 or not p.is_cuda:
        _bad("verify_draft: p must be a float32 CUDA tensor [batch, drafts + 1, vocab]")
    B, k1, V = p.shape
    device, k = p.get_device(), k1 - 1
    if k < 0:
        _bad("verify_draft: p holds no row")

    def ld(name, t, n):
        """From one of the B * n rows to the next: the sequences' stride where each has one row."""
        s0, s1, s2 = t.stride()
        row = s1 if n > 1 else s0
        if t.dtype is not torch.float32 or t.shape != (B, n, V) or t.get_device() != device or (s2 != 1 and V > 1) \
                or (s0 != n * s1 and n > 1 and B > 1) or (row < V and B * n > 1):
            _bad(f"verify_draft: {name} must be float32 [{B}, {n}, {V}] on cuda:{device} with evenly strided rows that do not overlap")
        return row if B * n > 1 else V

    ld_p = ld("p", p, k1)
    if q is not None and k == 0:
        if q.shape != (B, 0, V):
            _bad(f"verify_draft: q must be [{B}, 0, {V}]")
        q = None  # no draft, nothing to subtract
    ld_q = ld("q", q, k) if q is not None else 0
    if uniform.dtype is not torch.float32 or uniform.shape != (B, k1) or uniform.get_device() != device or not uniform.is_contiguous():
        _bad(f"verify_draft: uniform must be contiguous float32 [{B}, {k1}] on cuda:{device}")
    if p.shape.numel() >= 1 << 31:
        k, V = _count(k), _count(V)
    tokens, accepted = p.new_empty((B, k1), dtype=torch.int32), p.new_empty((B,), dtype=torch.int32)
    _call(lib().llmdot_cuda_verify_draft, device,
          native.Verify(B, k, V, 0, p.data_ptr(), q.data_ptr() if q is not None else None, ld_p, ld_q,
                        _int32("draft", draft, (B, k1 - 1), device), uniform.data_ptr(),
                        _int32("n_draft", n_draft, (B,), device) if n_draft is not None else None, tokens.data_ptr(),
                        accepted.data_ptr()))
    return tokens, accepted
