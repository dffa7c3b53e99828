"""The paged K / V cache as calls on device tensors: a batch of new tokens (whole prompts, chunks of
prompts, single decode tokens, packed) normalised, rotated and written into pages (``paged_prep``),
their attention over the pages (``paged_attention``) and cache rows back out (``paged_read``).

Beside the contiguous caches of ``units.decode_prep`` / ``units.decode_attention`` /
``units.attention_strided`` (one slab a sequence, one position for the batch): sequences of any
lengths, rows in pages of one pool, int16 or int8.  The reference has no counterpart; the arithmetic
is its units' (rowops_spec.py's NORM and ROPE, the pow2 contraction, the softmax unit's exponential).

A ``PagedCache`` (one layer's pool), a ``PagedBatch`` (the step's packing, shared by every layer) and a
``PagedPrep`` (a layer's rotation and norms) check their tensors once; the calls then check what
they are given and enqueue on the current torch stream of the cache's device.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from . import _lib
from .units import _require


def block_bytes(page: int, head_dim: int, int8: bool = False) -> int:
    """Bytes of one KV head of a page (cm_paged_block_bytes)."""
    return page * (2 * head_dim + 6 if int8 else 4 * head_dim + 4)


class PagedCache:
    """One layer's pool: ``pages`` pages of ``page`` rows (a power of two, 16 .. 4096) for ``kv_heads``
    heads of ``head_dim`` (64 or 128), held as int16 (two byte planes) or, with ``int8``, as int8 rows
    with a power-of-two scale a row.  ``data``: the pool's bytes (uint8, cm_paged_cache's layout), by
    default zeroed memory on ``device``."""

    def __init__(self, pages: int, page: int, kv_heads: int, head_dim: int, int8: bool = False,
                 data: Optional[torch.Tensor] = None, device="cuda"):
        if page < 16 or page > 4096 or page & (page - 1):
            raise ValueError(f"PagedCache: pages of {page} rows (a power of two, 16 .. 4096)")
        if head_dim not in (64, 128):
            raise ValueError(f"PagedCache: head_dim {head_dim} (64 or 128)")
        if pages < 1 or not 1 <= kv_heads <= 1024:
            raise ValueError(f"PagedCache: {pages} pages of {kv_heads} heads")
        self.pages, self.page, self.kv_heads, self.head_dim, self.int8 = pages, page, kv_heads, head_dim, bool(int8)
        nbytes = pages * kv_heads * block_bytes(page, head_dim, self.int8)
        self.data = torch.zeros(nbytes, dtype=torch.uint8, device=device) if data is None else data
        _require(self.data, "PagedCache: data", torch.uint8, nbytes)
        self.width, self.device, self.index = kv_heads * head_dim, self.data.device, self.data.get_device()
        self._c = _lib.CmPagedCache(self.data.data_ptr(), pages, page, kv_heads, head_dim, int(self.int8))
        self._ref = ctypes.byref(self._c)


class PagedBatch:
    """A step's packed tokens: sequence b's are rows q_start[b] .. q_start[b+1] - 1 (int32 [batch + 1]
    from 0), kv_len[b] (int32 [batch]) its length with them, table[b] (int32 [batch][max_pages], rows
    any stride apart) its pages in order; ``tokens`` rows in every operand (q_start[batch] or more: the
    rows behind the last sequence are left alone).  The tensors may change between calls (and replays
    of a captured call), their sizes not."""

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, table: torch.Tensor, tokens: int):
        batch = kv_len.numel() if kv_len is not None else 0
        _require(kv_len, "PagedBatch: kv_len", torch.int32, batch)
        _require(q_start, "PagedBatch: q_start", torch.int32, batch + 1)
        if not table.is_cuda or table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] < batch or \
                table.shape[1] < 1 or table.stride(1) != 1:
            raise ValueError("PagedBatch: table must be a GPU int32 [batch][max_pages] tensor with contiguous rows")
        if batch < 1 or tokens < 0:
            raise ValueError(f"PagedBatch: {batch} sequences, {tokens} tokens")
        if not (kv_len.device == q_start.device == table.device):
            raise ValueError("PagedBatch: q_start, kv_len and table on different devices")
        self.q_start, self.kv_len, self.table, self.tokens, self.batch = q_start, kv_len, table, tokens, batch
        self.device = kv_len.device
        self._c = _lib.CmPagedBatch(q_start.data_ptr(), kv_len.data_ptr(), table.data_ptr(), batch, tokens,
                                    table.shape[1], table.stride(0))
        self._ref = ctypes.byref(self._c)


class PagedPrep:
    """A layer's rotation and norms: ``table`` int32 [positions][2 rotary] (cos then sin at 2^-23:
    rowops_nodes.rope_table's rows; with ``interleaved`` its own, each angle on a pair of neighbouring
    columns), ``params_q`` / ``params_k`` the ROPE jobs' parameter bytes (one 16-byte entry, or one
    per column), ``norm_q`` / ``norm_k`` the per-head RMSNorms' entries [head_dim] (None: no norm)
    with ``eps_q`` / ``eps_k`` (rowops_nodes.norm_params, rms)."""

    def __init__(self, table: torch.Tensor, params_q: torch.Tensor, params_k: torch.Tensor, interleaved: bool = False,
                 norm_q: Optional[torch.Tensor] = None, norm_k: Optional[torch.Tensor] = None, eps_q: int = 0,
                 eps_k: int = 0):
        if not (0 <= eps_q <= 1 << 61 and 0 <= eps_k <= 1 << 61):            # the ABI's words would drop bits from 2^63 on
            raise ValueError(f"PagedPrep: eps {eps_q}, {eps_k} outside 0 .. 2^61")
        if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 32 or table.shape[1] % 32:
            raise ValueError("PagedPrep: a table [positions][2 rotary], rotary a multiple of 16")
        _require(table, "PagedPrep: table", torch.int32, 2)
        for name, p in (("params_q", params_q), ("params_k", params_k)):
            _require(p, f"PagedPrep: {name}", torch.uint8, 16)
        self.table, self.params_q, self.params_k, self.norm_q, self.norm_k = table, params_q, params_k, norm_q, norm_k
        self.rotary, self.interleaved = table.shape[1] // 2, bool(interleaved)
        self.eps_q, self.eps_k = int(eps_q), int(eps_k)
        self.device = table.device
        if any(t is not None and t.device != self.device for t in (params_q, params_k, norm_q, norm_k)):
            raise ValueError("PagedPrep: the table and the parameter blocks on different devices")
        ptr = lambda t: None if t is None else t.data_ptr()         # noqa: E731
        self._args = _lib.CmPagedPrepArgs(rope=table.data_ptr(), rope_rows=table.shape[0], rotary=self.rotary,
                                          interleaved=int(self.interleaved), rope_q=params_q.data_ptr(),
                                          rope_k=params_k.data_ptr(), rope_q_cols=int(params_q.numel() != 16),
                                          rope_k_cols=int(params_k.numel() != 16), norm_q=ptr(norm_q),
                                          norm_k=ptr(norm_k), eps_q=self.eps_q, eps_k=self.eps_k)
        self._tail = bytes(self._args)[_OPERANDS.size:]
        self._checked = None

    def _check(self, heads: int, kv_heads: int, head_dim: int) -> None:
        """The blocks against a cache's heads (once for each head layout)."""
        if self.rotary > head_dim:
            raise ValueError(f"paged_prep: {self.rotary} rotated columns of a head of {head_dim}")
        for name, p, n in (("params_q", self.params_q, heads), ("params_k", self.params_k, kv_heads)):
            if p.numel() != 16 and p.numel() != 16 * n * head_dim:
                raise ValueError(f"paged_prep: {name} holds {p.numel()} bytes (16, or 16 for each of {n} x {head_dim} columns)")
        for name, p in (("norm_q", self.norm_q), ("norm_k", self.norm_k)):
            if p is not None:
                _require(p, f"paged_prep: {name}", torch.uint8, 16 * head_dim)
        self._checked = (heads, kv_heads, head_dim)


_OPERANDS = struct.Struct("@4P4QI")         # cm_paged_prep_args up to heads: q, k, v, qr, their strides, heads


def _rows(t: torch.Tensor, name: str, tokens: int, width: int) -> int:
    """The row stride of a [tokens][>= width] int16 operand (rows of contiguous columns)."""
    if t.dtype is not torch.int16 or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU int16 tensor")
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] < tokens or shape[1] < width or stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name} must be [{tokens}][{width}] rows of contiguous columns, got {list(shape)} "
                         f"at strides {list(stride)}")
    return stride[0] if shape[0] > 1 else shape[1]


def _on(cache: PagedCache, *on) -> int:
    """The current stream of the cache's device, which every operand must be on and which must be current."""
    index = cache.index
    for t in on:
        if t.get_device() != index:
            raise ValueError(f"the cache is on {cache.device}, an operand on {t.device}")
    if index != torch.cuda.current_device():
        raise ValueError(f"the cache is on {cache.device}, the current device is cuda:{torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(index)         # torch.cuda.current_stream() takes 2.8 us of a 10 us call


def paged_prep(cache: PagedCache, batch: PagedBatch, prep: PagedPrep, q: torch.Tensor, k: torch.Tensor,
               v: torch.Tensor, qr: torch.Tensor) -> torch.Tensor:
    """cm_paged_prep: q [tokens][heads hd] normalised per head and rotated into ``qr`` (it may be q), k
    likewise and v as they are into the cache rows of the tokens' positions.  Rows may be strided
    (views of a fused projection)."""
    n, hd = batch.tokens, cache.head_dim
    heads = qr.shape[-1] // hd
    if qr.shape[-1] % hd or heads < 1:
        raise ValueError(f"paged_prep: qr rows of {qr.shape[-1]} columns are no heads of {hd}")
    lds = [_rows(q, "q", n, heads * hd), _rows(k, "k", n, cache.width), _rows(v, "v", n, cache.width),
           _rows(qr, "qr", n, heads * hd)]
    if prep._checked != (heads, cache.kv_heads, hd):
        prep._check(heads, cache.kv_heads, hd)
    if q.data_ptr() == qr.data_ptr() and lds[0] != lds[3]:
        raise ValueError("paged_prep: qr is q at another stride")
    stream = _on(cache, batch.kv_len, prep.table, q, k, v, qr)
    a = _OPERANDS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), qr.data_ptr(), *lds, heads) + prep._tail
    _lib.check(_lib.lib().cm_paged_prep(cache._ref, batch._ref, a, stream), "cm_paged_prep")
    return qr


def paged_attention(cache: PagedCache, batch: PagedBatch, q: torch.Tensor, o: torch.Tensor, heads: int, smx_cm: int,
                    smx_cfg: int, window: int = 0) -> torch.Tensor:
    """cm_paged_attention: the causal attention of the batch's tokens, q / o [tokens][heads hd] (apart), over
    their sequences' cache rows (the last ``window`` of them, 0: all); smx_cm / smx_cfg as the softmax
    unit's registers (graph.softmax_regs), o at 2^-(f_p + f_v - 8) as the unit's P . V.  Any call may use the
    device's workspace: one at a time a device, and one of the same sizes before a capture.  The kernels are
    chosen by the sizes (the table's width among them), not by the sequences' lengths."""
    n, hd = batch.tokens, cache.head_dim
    if heads < 1 or heads % cache.kv_heads or not 0 <= window < 1 << 30:       # the ABI's word would drop bits from 2^32 on
        raise ValueError(f"paged_attention: {heads} heads over {cache.kv_heads} KV heads, window {window} (below 2^30)")
    q_ld, o_ld = _rows(q, "q", n, heads * hd), _rows(o, "o", n, heads * hd)
    q_at, o_at = q.data_ptr(), o.data_ptr()
    if q_at == o_at and n:                      # a tile's rows are read by several workgroups, and by two kernels
        raise ValueError("paged_attention: o is q")
    stream = _on(cache, batch.kv_len, q, o)
    _lib.check(_lib.lib().cm_paged_attention(cache._ref, batch._ref, q_at, o_at, q_ld, o_ld, heads,
                                             window, smx_cm & 0xFFFFFFFF, smx_cfg & 0xFFFFFFFF, stream),
               "cm_paged_attention")
    return o


def paged_read(cache: PagedCache, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor) -> None:
    """cm_paged_read: the cache rows of the batch's tokens as int16 rows k / v [tokens][kv_heads hd]."""
    n = batch.tokens
    lds = _rows(k, "k", n, cache.width), _rows(v, "v", n, cache.width)
    stream = _on(cache, batch.kv_len, k, v)
    _lib.check(_lib.lib().cm_paged_read(cache._ref, batch._ref, k.data_ptr(), v.data_ptr(), *lds, stream),
               "cm_paged_read")


__all__ = ["PagedCache", "PagedBatch", "PagedPrep", "paged_prep", "paged_attention", "paged_read", "block_bytes"]
