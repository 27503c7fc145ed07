"""What the positions of a prompt have received from its queries, on the HIP kernels of csrc/attn_weights.hip
(``include/sisa_hip_cache.h``): the accumulated softmax weights from which :func:`sisa_amd.kernels.paged.
sisa_cache_evict_hip` chooses what stays in a cache. Inference only; no counterpart in the reference."""
from __future__ import annotations

import torch
from torch import Tensor

from ..config import HIP_D_HEAD, HIP_D_STATE
from . import _lib
from .paged import _DTYPES, _NO_VIEW, check_ints, inference_only, row_view

__all__ = ["sisa_attention_weights_hip"]

MAX_STRIDE = 1 << 24           # SISA_ATTN_WEIGHTS_MAX_STRIDE

_weights = _lib.Packed("sisa_attn_weights", _lib.AttnWeightsArgs)


def _rows(t: Tensor) -> tuple:
    """:func:`row_view`, of a copy also where positions are MAX_STRIDE elements or more apart."""
    return row_view(t if t.stride(2) < MAX_STRIDE else t.clone(memory_format=torch.contiguous_format))


def _gates(t: Tensor) -> tuple:
    """``t`` ``(B, H, L)``, its address and strides; of a copy where its positions are not neighbours."""
    if t.stride(2) != 1:
        t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), *t.stride()


def sisa_attention_weights_hip(q: Tensor, k: Tensor, c: Tensor, b: Tensor, g: Tensor, lam: Tensor,
                               fgate: Tensor | None = None, *, lengths: Tensor | None = None,
                               window: int | None = None) -> Tensor:
    """The softmax weights of SISA attention summed over its queries: ``out[n, h, j]`` is the sum, over the last ``window``
    queries ``i >= j`` of sequence ``n`` (default: all of its queries), of the weight that query ``i`` gives position ``j``.

    ``q, k`` ``(B, H, L, 64)`` and ``c, b`` ``(B, H, L, 32)`` in bf16, fp16 or fp32, ``g, fgate`` ``(B, H, L)`` and ``lam``
    ``(H,)`` float32, as :func:`sisa_amd.kernels.attention.sisa_attention_hip` takes them. ``lengths`` ``(B,)`` int32: the
    positions of each sequence of a right-padded batch (default ``L``; values outside ``0 .. L`` count as the nearer of the
    two); what lies behind is not looked at and receives 0. Returns ``(B, H, L)`` float32. The scores are formed twice and
    never stored. Gates that rise along the sequence are taken as they are (and more slowly where they rise by more than
    16), not refused."""
    name = "sisa_attention_weights_hip"
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or c.requires_grad or b.requires_grad or g.requires_grad
                                    or lam.requires_grad or (fgate is not None and fgate.requires_grad)):
        inference_only(name)
    if q.dim() != 4 or q.shape[-1] != HIP_D_HEAD or k.shape != q.shape:
        raise ValueError(f"{name}: q and k must be (B, H, L, {HIP_D_HEAD}), got {tuple(q.shape)} and {tuple(k.shape)}")
    B, H, L, _ = q.shape
    if c.shape != (B, H, L, HIP_D_STATE) or b.shape != c.shape:
        raise ValueError(f"{name}: c and b must be {(B, H, L, HIP_D_STATE)}, got {tuple(c.shape)} and {tuple(b.shape)}")
    if g.shape != (B, H, L) or (fgate is not None and fgate.shape != g.shape) or lam.shape != (H,):
        raise ValueError(f"{name}: g and fgate must be {(B, H, L)} and lam ({H},)")
    if q.dtype not in _DTYPES or not (q.dtype == k.dtype == c.dtype == b.dtype):
        raise TypeError(f"{name}: q, k, c, b must share one of bf16, fp16, fp32")
    if g.dtype is not torch.float32 or lam.dtype is not torch.float32 or (fgate is not None
                                                                         and fgate.dtype is not torch.float32):
        raise TypeError(f"{name}: g, fgate and lam must be float32")
    device = _lib.device_index(q)
    if k.get_device() != device or c.get_device() != device or b.get_device() != device or g.get_device() != device \
            or lam.get_device() != device or (fgate is not None and fgate.get_device() != device):
        raise ValueError(f"{name}: the tensors are on different devices")
    if window is not None and window < 1:
        raise ValueError(f"{name}: window = {window} must be positive or None")
    if lengths is not None:
        check_ints(name, "lengths", lengths, (B,), device)
    out = lam.new_empty((B, H, L))
    if not out.numel():
        return out
    q, *vq = _rows(q)
    k, *vk = _rows(k)
    c, *vc = _rows(c)
    b, *vb = _rows(b)
    g, *vg = _gates(g)
    fgate, *vf = (None, *_NO_VIEW) if fgate is None else _gates(fgate)
    window = 0 if window is None or window >= L else window
    ws = lam.new_empty((_lib.floats("sisa_attn_weights_workspace_bytes", B, H, L, window),))
    _weights(q, B, H, L, window, _lib.dtype_code(q.dtype), 0, *vq, *vk, *vc, *vb, *vg, *vf, lam.data_ptr(), lam.stride(0),
             0 if lengths is None else lengths.data_ptr(), out.data_ptr(), ws.data_ptr())
    return out
