"""Verification of drafted tokens on the HIP kernel of csrc/verify.hip (``include/sisa_hip_branch.h``): which of the tokens
that a draft proposed the target takes, and the token behind them, so that what comes out is distributed as if the target had
been sampled token by token. The random numbers are the caller's. The reference has no drafts (src/sisa/generation.py:137-191).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import _lib
from .paged import check_ints

__all__ = ["Verified", "sisa_verify_drafts_hip"]

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_VOCAB = 1 << 24            # SISA_VERIFY_MAX_V

_verify = _lib.Packed("sisa_verify", _lib.VerifyArgs)


class Verified(NamedTuple):
    """Result of :func:`sisa_verify_drafts_hip`: ``tokens`` ``(B, K + 1)`` int64, the accepted drafts of each row, the token that
    was drawn behind them, and -1; ``accepted`` ``(B,)`` int32, how many drafts that are."""
    tokens: Tensor
    accepted: Tensor


def _probabilities(name: str, what: str, t: Tensor, shape: tuple, device: int) -> Tensor:
    if t.shape != shape or t.dtype not in _DTYPES or t.get_device() != device:
        raise ValueError(f"{name}: {what} must be {shape} in bf16, fp16 or fp32 on the GPU of the others, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t if t.stride(-1) == 1 or shape[-1] == 1 else t.contiguous()


def sisa_verify_drafts_hip(p: Tensor, drafts: Tensor, u: Tensor, q: Tensor | None = None,
                           counts: Tensor | None = None) -> Verified:
    """Check ``drafts`` ``(B, K)`` int64 against the target's probabilities ``p`` ``(B, K + 1, V)``, ``p[n, i]`` those of what
    follows ``i`` drafts, with ``u`` ``(B, K + 1)`` float32, uniform in [0, 1). ``q`` ``(B, K, V)``: the probabilities that each
    draft was drawn from; None: it was not drawn (looked up, or the likeliest token). ``counts`` ``(B,)`` int32: how many
    drafts a row has (default ``K``).

    Draft ``i`` is accepted while all before it are and ``u[n, i] q[n, i, x] < p[n, i, x]``, exactly. The token behind the
    accepted ones is drawn with ``u[n, K]``: after a refused draft from ``max(p - q, 0)`` there, or from ``p`` where that is 0
    everywhere; after the last draft from ``p``: the lowest token up to which the weights' sum (in float64) is more than that
    share of all. Where ``p`` is 0 everywhere, or a sum is not finite, the token is -1. The probabilities need not sum to 1
    (``p`` and ``q`` should alike). bf16, fp16 and fp32 may be mixed."""
    name = "sisa_verify_drafts_hip"
    if p.dim() != 3 or drafts.dim() != 2 or p.shape[1] != drafts.shape[1] + 1 or not 1 <= p.shape[2] <= MAX_VOCAB:
        raise ValueError(f"{name}: p must be (B, K + 1, V), V at most {MAX_VOCAB}, and drafts (B, K), got {tuple(p.shape)} and "
                         f"{tuple(drafts.shape)}")
    device = _lib.device_index(p)
    (B, K), V = drafts.shape, p.shape[2]
    p = _probabilities(name, "p", p, (B, K + 1, V), device)
    if q is not None:
        q = _probabilities(name, "q", q, (B, K, V), device)
    if drafts.dtype is not torch.int64 or drafts.shape[0] != B or drafts.get_device() != device:
        raise ValueError(f"{name}: drafts must be ({B}, {K}) int64 on the GPU of the others, got {tuple(drafts.shape)} "
                         f"{drafts.dtype} on {drafts.device}")
    if u.shape != (B, K + 1) or u.dtype is not torch.float32 or u.get_device() != device:
        raise ValueError(f"{name}: u must be ({B}, {K + 1}) float32 on the GPU of the others, got {tuple(u.shape)} {u.dtype} on "
                         f"{u.device}")
    if counts is not None:
        check_ints(name, "counts", counts, (B,), device)
    tokens, accepted = drafts.new_empty((B, K + 1)), torch.empty((B,), dtype=torch.int32, device=p.device)
    if not B:
        return Verified(tokens, accepted)
    size = _lib.floats("sisa_verify_workspace_bytes", B, V)
    ws = torch.empty((size,), dtype=torch.float32, device=p.device) if size else None
    vq = (0, 0, 0) if q is None else (q.data_ptr(), *q.stride()[:2])
    _verify(p, B, K, V, _lib.dtype_code(p.dtype), _lib.dtype_code((p if q is None else q).dtype), 0, p.data_ptr(),
            *p.stride()[:2], *vq, drafts.data_ptr(), *drafts.stride(), u.data_ptr(), *u.stride(),
            0 if counts is None else counts.data_ptr(), tokens.data_ptr(), accepted.data_ptr(),
            0 if ws is None else ws.data_ptr())
    return Verified(tokens, accepted)
