"""Attention of sequences that have their first positions in common, on the HIP kernels of csrc/prefix.hip
(``include/sisa_hip_branch.h``): several continuations of one prompt, many prompts behind one text, or the drafted tokens of
a sequence. The cached rows of the common positions are read once for the query rows of a group, not once for each.

* :class:`PrefixGroups`: which sequences of a batch belong together;
* :func:`sisa_prefix_decode_hip`: :func:`sisa_amd.kernels.paged.sisa_paged_decode_hip` for them, over the same pages.

A softmax over a sequence's positions is joined from the one over the common positions and the one over its own; the score of
a SISA key depends on its own ``g``, ``F`` and rotated ``b`` alone, so a key means the same to every sequence that has it.
Inference only. The reference generates one continuation of a row (src/sisa/generation.py:137-191).
"""
from __future__ import annotations

from typing import Iterable

import torch
from torch import Tensor

from ..config import HIP_D_HEAD, HIP_D_STATE
from . import _lib
from .paged import PagePool, _forget, _gates, _max_len, _rows, check_ints, inference_only

__all__ = ["PrefixGroups", "sisa_prefix_decode_hip"]

_decode = _lib.Packed("sisa_prefix_decode", _lib.PrefixDecodeArgs)


class PrefixGroups:
    """Groups of neighbouring sequences: the first ``sizes[0]`` sequences of a batch, the next ``sizes[1]``, and so on. The
    handle keeps the tensors on the GPU that the kernels take: ``first`` ``(G + 1,)``, where each group begins, and ``group``
    ``(B,)``, the group of each sequence, both int32; they stay as they are."""

    __slots__ = ("sizes", "first", "group", "device_index")

    def __init__(self, sizes: Iterable[int], device):
        self.sizes = tuple(int(n) for n in sizes)
        if not self.sizes or min(self.sizes) < 1:
            raise ValueError(f"PrefixGroups: sizes = {self.sizes}: at least one group, of at least one sequence each")
        first, group = [0], []
        for r, n in enumerate(self.sizes):
            first.append(first[-1] + n)
            group += [r] * n
        self.first, self.group = (torch.tensor(x, dtype=torch.int32).to(device) for x in (first, group))
        self.device_index = _lib.device_index(self.first)

    @property
    def sequences(self) -> int:
        return self.group.shape[0]

    def __len__(self) -> int:
        """How many groups."""
        return len(self.sizes)


def sisa_prefix_decode_hip(q: Tensor, c: Tensor, g_q: Tensor, f_q: Tensor | None, lam: Tensor, pool: PagePool, table: Tensor,
                           lengths: Tensor, groups: PrefixGroups, shared: Tensor, *, max_len: int | None = None,
                           max_shared: int | None = None) -> Tensor:
    """Exact SISA attention of the last ``M`` cached positions of every sequence over the positions up to their own, with the
    arguments and the answers of :func:`sisa_amd.kernels.paged.sisa_paged_decode_hip`, for sequences in ``groups``: the first
    ``shared[r]`` positions (``(G,)`` int32, on the GPU) of the sequences of group ``r`` are those of its first sequence, the
    others each sequence's own. Returns ``(B, H, M, 64)`` float32.

    ``max_len`` bounds the lengths and ``max_shared`` the common positions (default: what the table can hold, and ``max_len``):
    the launch is sized for them. Every row of a group whose ``shared[r]`` is negative or above ``max_shared`` is NaN; so may a
    row be that sees an infinite ``v``. Of the table rows of a group, only the first one's entries for the common positions are
    read. Drafted tokens of a sequence are a group of one, with everything before them in common."""
    name = "sisa_prefix_decode_hip"
    if torch.is_grad_enabled() and (q.requires_grad or c.requires_grad or g_q.requires_grad or lam.requires_grad
                                    or (f_q is not None and f_q.requires_grad)):
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
    G = len(groups)
    if groups.sequences != B or groups.device_index != device:
        raise ValueError(f"{name}: groups of {groups.sequences} sequences on GPU {groups.device_index} for {B} on GPU {device}")
    check_ints(name, "table", table, (B, W), device)
    check_ints(name, "lengths", lengths, (B,), device)
    check_ints(name, "shared", shared, (G,), device)
    out = lam.new_empty((B, H, M, HIP_D_HEAD))
    if not M:
        return out
    if not W:
        raise ValueError(f"{name}: the table has no entries")
    max_len = _max_len(name, max_len, W, pool)
    if max_shared is None:
        max_shared = max_len
    elif not 0 <= max_shared <= W * pool.page_size:
        raise ValueError(f"{name}: max_shared = {max_shared} must be in 0 .. {W * pool.page_size}, what {W} pages of "
                         f"{pool.page_size} hold")
    ws = lam.new_empty((_lib.floats("sisa_prefix_decode_workspace_bytes", B, H, M, G, max_len, max_shared),))
    _decode(q, B, M, W, G, max_len, max_shared, _lib.F32, 0, pool.packed, table.data_ptr(), table.stride(0),
            lengths.data_ptr(), groups.first.data_ptr(), groups.group.data_ptr(), shared.data_ptr(), *vq, *vc, *vg, *vf,
            lam.data_ptr(), lam.stride(0), out.data_ptr(), *out.stride()[:3], ws.data_ptr())
    return out
