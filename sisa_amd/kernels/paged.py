"""A generation cache in pages on the HIP kernels of csrc/paged.hip and csrc/evict.hip (``include/sisa_hip_cache.h``):

* :class:`PagePool`: the memory, ``pages`` pages of ``page_size`` positions of every head;
* :func:`sisa_paged_write_hip`: new positions of every sequence into its pages;
* :func:`sisa_paged_decode_hip`: the attention of new tokens over the pages, with the semantics of
  :func:`sisa_amd.kernels.decode.sisa_decode_hip`, and, on request, every position's accumulated softmax weight;
* :func:`sisa_cache_evict_hip`: a cache cut down to its last and its most attended positions.

Position ``j`` of sequence ``n`` lives in slot ``j % page_size`` of page ``table[n, j // page_size]``. Tables, lengths and
counts are int32 tensors on the GPU, so that calls can be captured into a graph and replayed with others; their values are
not seen by the host. No memory outside the pool is touched whatever they are; the functions say what the answer then is.
Sequences may share pages that are only read (a common prefix). Inference only.

The reference has no such cache; its own (src/sisa/generation.py:34-100) keeps one tensor per layer for sequences of
one length.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from ..config import HIP_D_HEAD, HIP_D_STATE
from . import _lib

__all__ = ["PagePool", "Evicted", "sisa_paged_write_hip", "sisa_paged_decode_hip", "sisa_cache_evict_hip"]

MIN_PAGE_SIZE = 16             # SISA_MIN_PAGE_SIZE
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_NO_VIEW = (0, 0, 0, 0)

_write = _lib.Packed("sisa_paged_write", _lib.PagedWriteArgs)
_decode = _lib.Packed("sisa_paged_decode", _lib.PagedDecodeArgs)
_evict = _lib.Packed("sisa_cache_evict", _lib.CacheEvictArgs)


def row_view(t: Tensor) -> tuple[Tensor, int, int, int, int]:
    """``t`` ``(B, H, L, .)``, its address and its three outer strides; of a copy where 16-byte loads cannot read its rows.
    (A copy in any case then: ``contiguous()`` hands back a tensor of one row wherever it begins.)"""
    s0, s1, s2, s3 = t.stride()
    address = t.data_ptr()
    if s3 != 1 or (address | (s0 | s1 | s2) * t.element_size()) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, s2, _ = t.stride()
        address = t.data_ptr()
    return t, address, s0, s1, s2


def inference_only(name: str) -> None:
    raise RuntimeError(f"{name} is for inference: call it under torch.no_grad() or on detached tensors")


def check_ints(name: str, what: str, t: Tensor, shape: tuple, device: int) -> None:
    if t.dtype is not torch.int32 or t.shape != shape or t.get_device() != device:
        raise ValueError(f"{name}: {what} must be an int32 tensor of shape {shape} on the GPU of the others, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: {what} must be contiguous along its last axis")


class PagePool:
    """Pages of cached positions: ``k, v`` ``(P, H, S, 64)`` and ``b`` ``(P, H, S, 32)`` in bf16, fp16 or fp32, ``g, fgate``
    ``(P, H, S)`` float32 (``fgate`` may be ``None``: no forget term), all on one GPU. ``S``, the positions of a page, is a
    power of two of at least 16. Rows must be readable with 16-byte loads; the tensors may be views of a larger one. The
    handle keeps the tensors and checks them once."""

    __slots__ = ("k", "v", "b", "g", "fgate", "pages", "heads", "page_size", "dtype", "dtype_code", "device_index",
                 "packed")

    def __init__(self, k: Tensor, v: Tensor, b: Tensor, g: Tensor, fgate: Tensor | None = None):
        if k.dim() != 4 or k.shape[-1] != HIP_D_HEAD or v.shape != k.shape:
            raise ValueError(f"PagePool: k and v must be (pages, heads, page_size, {HIP_D_HEAD}), got {tuple(k.shape)} and "
                             f"{tuple(v.shape)}")
        P, H, S, _ = k.shape
        if b.shape != (P, H, S, HIP_D_STATE):
            raise ValueError(f"PagePool: b must be {(P, H, S, HIP_D_STATE)}, got {tuple(b.shape)}")
        if any(t is not None and t.shape != (P, H, S) for t in (g, fgate)):
            raise ValueError(f"PagePool: g and fgate must be {(P, H, S)}")
        if not (P and H) or S < MIN_PAGE_SIZE or S & (S - 1):
            raise ValueError(f"PagePool: {P} pages of {S} positions of {H} heads: the page size must be a power of two of at "
                             f"least {MIN_PAGE_SIZE}, and there must be a page and a head")
        if k.dtype not in _DTYPES or v.dtype != k.dtype or b.dtype != k.dtype:
            raise TypeError(f"PagePool: k, v, b must share one of bf16, fp16, fp32, got {k.dtype}, {v.dtype}, {b.dtype}")
        if any(t is not None and t.dtype != torch.float32 for t in (g, fgate)):
            raise TypeError("PagePool: g and fgate must be float32")
        device = _lib.device_index(k)
        if any(t is not None and t.get_device() != device for t in (v, b, g, fgate)):
            raise ValueError("PagePool: the tensors are on different devices")
        if any(row_view(t)[0] is not t for t in (k, v, b)):
            raise ValueError("PagePool: k, v, b need rows that 16-byte loads can read (unit last stride, 16-byte aligned)")
        self.k, self.v, self.b, self.g, self.fgate = k, v, b, g, fgate
        self.pages, self.heads, self.page_size, self.dtype, self.device_index = P, H, S, k.dtype, device
        self.dtype_code = _lib.dtype_code(k.dtype)
        self.packed = bytes(_lib.PagePoolArgs(P, H, S, self.dtype_code, *(_lib.view(t) for t in (k, v, b, g, fgate))))

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, dtype: torch.dtype, device) -> "PagePool":
        """A pool of uninitialised pages with a forget term."""
        def new(*tail, dt=dtype):
            return torch.empty((pages, heads, page_size, *tail), dtype=dt, device=device)
        return cls(new(HIP_D_HEAD), new(HIP_D_HEAD), new(HIP_D_STATE), new(dt=torch.float32), new(dt=torch.float32))


def _rows(name: str, what: str, t: Tensor, shape: tuple, pool: PagePool) -> tuple:
    """:func:`row_view` of ``t`` checked against the pool."""
    if t.shape != shape or t.dtype is not pool.dtype or t.get_device() != pool.device_index:
        raise ValueError(f"{name}: {what} must be {shape} in {pool.dtype} on the pool's GPU, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device}")
    return row_view(t)


def _gates(name: str, what: str, t: Tensor | None, shape: tuple, pool: PagePool) -> tuple:
    """Address and strides of a float32 ``(B, H, .)`` tensor checked against the pool."""
    if t is None:
        return _NO_VIEW
    if t.shape != shape or t.dtype is not torch.float32 or t.get_device() != pool.device_index:
        raise ValueError(f"{name}: {what} must be {shape} float32 on the pool's GPU, got {tuple(t.shape)} {t.dtype} on "
                         f"{t.device}")
    return t.data_ptr(), *t.stride()


def _forget(name: str, f: Tensor | None, pool: PagePool) -> None:
    if (f is None) != (pool.fgate is None):
        raise ValueError(f"{name}: the new rows and the pool must both have a forget term, or neither")


def sisa_paged_write_hip(pool: PagePool, table: Tensor, start: Tensor, k: Tensor, v: Tensor, b: Tensor, g: Tensor,
                         fgate: Tensor | None, count: Tensor | None = None) -> None:
    """Write row ``m < count[n]`` (default: every row) of ``k, v`` ``(B, H, M, 64)``, ``b`` ``(B, H, M, 32)`` and
    ``g, fgate`` ``(B, H, M)`` to position ``start[n] + m`` of sequence ``n``; ``table`` ``(B, W)``, ``start, count``
    ``(B,)`` int32. A row whose position has no page of the pool is left out. The written pages of two sequences must
    differ."""
    name = "sisa_paged_write_hip"
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or b.requires_grad or g.requires_grad
                                    or (fgate is not None and fgate.requires_grad)):
        inference_only(name)
    if k.dim() != 4 or table.dim() != 2:
        raise ValueError(f"{name}: k must be (B, H, M, {HIP_D_HEAD}) and table (B, W), got {tuple(k.shape)} and "
                         f"{tuple(table.shape)}")
    (B, _, M, _), W, H, device = k.shape, table.shape[1], pool.heads, pool.device_index
    _forget(name, fgate, pool)
    k, *vk = _rows(name, "k", k, (B, H, M, HIP_D_HEAD), pool)
    v, *vv = _rows(name, "v", v, (B, H, M, HIP_D_HEAD), pool)
    b, *vb = _rows(name, "b", b, (B, H, M, HIP_D_STATE), pool)
    vg, vf = _gates(name, "g", g, (B, H, M), pool), _gates(name, "fgate", fgate, (B, H, M), pool)
    check_ints(name, "table", table, (B, W), device)
    check_ints(name, "start", start, (B,), device)
    if count is not None:
        check_ints(name, "count", count, (B,), device)
    if not B or not M:
        return
    if not W:
        raise ValueError(f"{name}: the table has no entries")
    _write(k, B, M, W, 0, pool.packed, table.data_ptr(), table.stride(0), start.data_ptr(),
           0 if count is None else count.data_ptr(), *vk, *vv, *vb, *vg, *vf)


def _weights_view(name: str, what: str, t: Tensor, B: int, H: int, max_len: int, pool: PagePool) -> tuple:
    if t.dim() != 3 or t.shape[0] != B or t.shape[1] != H or t.shape[2] < max_len or t.dtype is not torch.float32 \
            or t.get_device() != pool.device_index:
        raise ValueError(f"{name}: {what} must be ({B}, {H}, at least {max_len}) float32 on the pool's GPU, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr(), *t.stride()


def _max_len(name: str, max_len: int | None, W: int, pool: PagePool) -> int:
    held = W * pool.page_size
    if max_len is None:
        return held
    if not 1 <= max_len <= held:
        raise ValueError(f"{name}: max_len = {max_len} must be in 1 .. {held}, what {W} pages of {pool.page_size} hold")
    return max_len


def sisa_paged_decode_hip(q: Tensor, c: Tensor, g_q: Tensor, f_q: Tensor | None, lam: Tensor, pool: PagePool, table: Tensor,
                          lengths: Tensor, *, max_len: int | None = None, weights: Tensor | None = None,
                          weights_out: Tensor | None = None) -> Tensor:
    """Exact SISA attention of the last ``M`` cached positions of every sequence (written before the call) over the
    positions up to their own: ``q`` ``(B, H, M, 64)``, ``c`` ``(B, H, M, 32)`` in the pool's dtype, ``g_q, f_q``
    ``(B, H, M)`` and ``lam`` ``(H,)`` float32, ``table`` ``(B, W)`` and ``lengths`` ``(B,)`` int32, the new positions
    included. Returns ``(B, H, M, 64)`` float32.

    ``max_len`` bounds the lengths (default: what the table can hold): the launch is sized for it. ``weights``
    ``(B, H, >= max_len)`` float32: the accumulated weight of every position, to which the softmax weights of the ``M`` rows
    are added, in place or into ``weights_out``, for the sequence's ``lengths[n]`` positions; the others are left alone.

    A row that sees no position (an empty sequence) is 0. Every row of a sequence whose length is negative or above
    ``max_len``, or one of whose pages is not in the pool, is NaN."""
    name = "sisa_paged_decode_hip"
    if torch.is_grad_enabled() and (q.requires_grad or c.requires_grad or g_q.requires_grad or lam.requires_grad
                                    or (f_q is not None and f_q.requires_grad)
                                    or (weights is not None and weights.requires_grad)):
        inference_only(name)
    if q.dim() != 4 or table.dim() != 2:
        raise ValueError(f"{name}: q must be (B, H, M, {HIP_D_HEAD}) and table (B, W), got {tuple(q.shape)} and "
                         f"{tuple(table.shape)}")
    (B, _, M, _), W, H, device = q.shape, table.shape[1], pool.heads, pool.device_index
    _forget(name, f_q, pool)
    q, *vq = _rows(name, "q", q, (B, H, M, HIP_D_HEAD), pool)
    c, *vc = _rows(name, "c", c, (B, H, M, HIP_D_STATE), pool)
    vg, vf = _gates(name, "g_q", g_q, (B, H, M), pool), _gates(name, "f_q", f_q, (B, H, M), pool)
    if lam.shape != (H,) or lam.dtype is not torch.float32 or lam.get_device() != device:
        raise ValueError(f"{name}: lam must be ({H},) float32 on the pool's GPU, got {tuple(lam.shape)} {lam.dtype}")
    check_ints(name, "table", table, (B, W), device)
    check_ints(name, "lengths", lengths, (B,), device)
    out = lam.new_empty((B, H, M, HIP_D_HEAD))
    if not B or not M:
        return out
    if not W:
        raise ValueError(f"{name}: the table has no entries")
    max_len = _max_len(name, max_len, W, pool)
    if weights is None:
        if weights_out is not None:
            raise ValueError(f"{name}: weights_out goes with weights")
        w_in = w_out = _NO_VIEW
    else:
        w_in = _weights_view(name, "weights", weights, B, H, max_len, pool)
        w_out = w_in if weights_out is None else _weights_view(name, "weights_out", weights_out, B, H, max_len, pool)
        if any(step == 0 and size > 1 for step, size in zip(w_out[1:], (B, H, max_len))):
            raise ValueError(f"{name}: the weights that are written must not be an expanded tensor")
    size = _lib.floats("sisa_paged_decode_workspace_bytes", B, H, M, max_len, pool.dtype_code, weights is not None)
    ws = lam.new_empty((size,)) if size else None
    _decode(q, B, M, W, max_len, pool.packed, table.data_ptr(), table.stride(0), lengths.data_ptr(), *vq, *vc, *vg, *vf,
            lam.data_ptr(), lam.stride(0), *w_in, *w_out, out.data_ptr(), 0 if ws is None else ws.data_ptr())
    return out


class Evicted(NamedTuple):
    """Result of :func:`sisa_cache_evict_hip`: ``lengths`` ``(B,)`` int32 (-1: it could not be done), and per head the kept positions' ``weights``
    ``(B, H, keep)`` float32 (0 behind the last) and the ``positions`` ``(B, H, keep)`` int32 they had (-1 behind)."""
    lengths: Tensor
    weights: Tensor
    positions: Tensor


def sisa_cache_evict_hip(pool: PagePool, table: Tensor, lengths: Tensor, weights: Tensor, keep: int, recent: int,
                         new_pool: PagePool, new_table: Tensor, *, max_len: int | None = None) -> Evicted:
    """Cut every sequence down to at most ``keep`` positions per head: the last ``recent`` ones and, of the others, those
    with the largest ``weights`` ``(B, H, >= max_len)`` float32 (of equal ones the lowest position; NaN is above all). Their
    rows are copied, in order, to the pages of ``new_table`` ``(B, W')`` in ``new_pool`` (``pool`` or another with its heads
    and dtype); no page may be both read and written. The old pages are left as they are.

    The score of a SISA key depends on its own ``g`` and ``F``, not on how many keys lie between, so what follows attends
    exactly as a softmax over the kept keys. Lengths that are negative or above ``max_len``, too few new pages, and pages of
    kept rows outside their pool answer with a new length of -1, which :func:`sisa_paged_decode_hip` turns into NaN. It is not
    a length to count on from, -1 and a new position being an empty sequence: ``held = torch.where(n < 0, n, n + 1)``."""
    name = "sisa_cache_evict_hip"
    if weights.requires_grad and torch.is_grad_enabled():
        inference_only(name)
    if table.dim() != 2 or new_table.dim() != 2:
        raise ValueError(f"{name}: tables must be (B, W), got {tuple(table.shape)} and {tuple(new_table.shape)}")
    (B, W), H, W_new, device = table.shape, pool.heads, new_table.shape[1], pool.device_index
    if new_pool is not pool and (new_pool.heads != H or new_pool.dtype != pool.dtype or new_pool.device_index != device
                                 or (new_pool.fgate is None) != (pool.fgate is None)):
        raise ValueError(f"{name}: the pools must agree in heads, dtype, GPU and the forget term")
    if not 1 <= recent <= keep:
        raise ValueError(f"{name}: recent = {recent} must be in 1 .. keep = {keep}")
    check_ints(name, "table", table, (B, W), device)
    check_ints(name, "new_table", new_table, (B, W_new), device)
    check_ints(name, "lengths", lengths, (B,), device)
    if B:
        if not W or not W_new:
            raise ValueError(f"{name}: a table has no entries")
        max_len = _max_len(name, max_len, W, pool)
    w_in = _weights_view(name, "weights", weights, B, H, max_len if B else 0, pool)
    new_lengths = torch.empty_like(lengths, memory_format=torch.contiguous_format)
    new_weights, positions = weights.new_empty((B, H, keep)), table.new_empty((B, H, keep))
    if B:
        _evict(pool.k, B, W, W_new, max_len, keep, recent, pool.packed, new_pool.packed, table.data_ptr(), table.stride(0),
               new_table.data_ptr(), new_table.stride(0), lengths.data_ptr(), *w_in, new_lengths.data_ptr(),
               new_weights.data_ptr(), positions.data_ptr())
    return Evicted(new_lengths, new_weights, positions)
