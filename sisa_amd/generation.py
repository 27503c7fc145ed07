"""Incremental decoding: the per-layer cache and ``generate`` (the API of the reference's src/sisa/generation.py).

Per head and cached position a SISA layer keeps, besides ``k`` and ``v``, the rotated state write vector ``b~``
(``d_state`` values) and the cumulative decay ``g`` and forget ``F`` values; the running phase ``Phi`` is kept for the
last position only. A new token extends ``g``, ``F`` and ``Phi`` in float32 and attends to the whole cache with the
exact score (on the GPU through the HIP decode kernel, :mod:`sisa_amd.kernels.decode`, or, for a single new position
of a 16-bit model, together with the rest of its layer, :mod:`sisa_amd.kernels.step`).

The cache is a set of preallocated slabs per layer, ``(B, H, capacity, .)``, filled front to back: a decode step
writes its rows in place and the layer state handed to the attention is a view of the filled prefix, so a step costs
the new rows' bytes, not a copy of the whole cache. ``generate`` sizes the slabs for the prompt plus every new token
up front; a cache made without a capacity grows by doubling. When the appended rows carry autograd history the slab
is rebuilt out of place instead, so gradients still flow. Batched decoding with this cache assumes equal-length prompts
(there is no padding mask); prompts of unequal lengths, a bound on the positions that are kept, several continuations of a
prompt and tokens that a draft model proposes go through :class:`sisa_amd.paged.SISAPagedCache`.
"""
from __future__ import annotations

import numbers
from dataclasses import dataclass
from typing import TYPE_CHECKING, Iterable

import torch
from torch import Tensor

from .backends import hip_status
from .paged import SISAPagedCache

if TYPE_CHECKING:  # pragma: no cover
    from .modeling import SISAForCausalLM

__all__ = ["LayerState", "SISACache", "generate", "verify_drafts"]



@dataclass
class LayerState:
    """One layer's cached positions: ``k, v`` ``(B, H, T, d_head)`` and ``b`` ``(B, H, T, d_state)`` in the
    attention's compute dtype, ``g, fgate`` ``(B, H, T)`` float32, and ``phi`` ``(B, H, d_state // 2)`` float32 at the
    last position. The position tensors may be views of a larger slab."""

    k: Tensor
    v: Tensor
    b: Tensor
    g: Tensor
    fgate: Tensor
    phi: Tensor

    @property
    def length(self) -> int:
        return self.k.shape[2]


class _Slab:
    """Position-axis buffers of one layer with room for ``capacity`` positions, ``filled`` of them in use."""

    def __init__(self, buffers: dict[str, Tensor], filled: int, phi: Tensor):
        self.buffers, self.filled, self.phi = buffers, filled, phi

    @property
    def capacity(self) -> int:
        return self.buffers["k"].shape[2]

    def state(self) -> LayerState:
        return LayerState(**{n: t[:, :, :self.filled] for n, t in self.buffers.items()}, phi=self.phi)


class SISACache:
    """Decode cache: one slab of :class:`LayerState` tensors per layer. ``capacity``: positions to reserve per layer
    when a layer is first filled (default: what the first fill needs, then doubling)."""

    def __init__(self, capacity: int | None = None) -> None:
        if capacity is not None and capacity < 1:
            raise ValueError(f"SISACache capacity must be positive, got {capacity}")
        self.capacity = capacity
        self._slabs: dict[int, _Slab] = {}

    def get(self, layer_idx: int) -> LayerState | None:
        slab = self._slabs.get(layer_idx)
        return None if slab is None else slab.state()

    def update(self, layer_idx: int, *, k: Tensor, v: Tensor, b: Tensor, g: Tensor, fgate: Tensor,
               phi: Tensor) -> LayerState:
        """Append positions (dim 2 of ``k, v, b, g, fgate``) to a layer's cache, take ``phi`` as its new last phase,
        and return the layer's whole cached state."""
        new = dict(k=k, v=v, b=b, g=g, fgate=fgate)
        slab = self._slabs.get(layer_idx)
        n_new = k.shape[2]
        if any(t.shape[2] != n_new for t in new.values()):
            raise ValueError(f"SISACache.update: position counts differ: "
                             f"{ {n: t.shape[2] for n, t in new.items()} }")
        if torch.is_grad_enabled() and any(t.requires_grad for t in new.values()):
            old = None if slab is None else slab.state()
            bufs = new if old is None else {n: torch.cat([getattr(old, n), t], 2) for n, t in new.items()}
            slab = _Slab(bufs, bufs["k"].shape[2], phi)
        else:
            slab = self.room(layer_idx, n_new, new, phi)
            filled, need = slab.filled, slab.filled + n_new
            for n, t in new.items():
                slab.buffers[n][:, :, filled:need].copy_(t)
            slab.filled, slab.phi = need, phi
        self._slabs[layer_idx] = slab
        return slab.state()

    def room(self, layer_idx: int, n_new: int, like: dict[str, Tensor], phi: Tensor) -> _Slab:
        """The layer's slab with space for ``n_new`` more positions after its filled ones; made, or grown by doubling,
        where it lacks that. ``like``: tensors with the batch and head sizes, widths and dtypes of new buffers."""
        slab = self._slabs.get(layer_idx)
        filled = 0 if slab is None else slab.filled
        need = filled + n_new
        if slab is None or need > slab.capacity:
            room = max(need, self.capacity or 0, 2 * slab.capacity if slab is not None else 0)
            grown = {n: t.new_empty(t.shape[:2] + (room,) + t.shape[3:]) for n, t in like.items()}
            if slab is not None:
                for n, t in grown.items():
                    t[:, :, :filled].copy_(slab.buffers[n][:, :, :filled])
            slab = self._slabs[layer_idx] = _Slab(grown, filled, phi)
        return slab

    @property
    def seq_len(self) -> int:
        """How many positions the cache holds (0 before the prefill)."""
        slab = self._slabs.get(0)
        return 0 if slab is None else slab.filled

    def reset(self) -> None:
        self._slabs.clear()

    def __len__(self) -> int:
        return len(self._slabs)


def _eos_ids(eos_token_id: int | Iterable[int] | Tensor | None) -> list[int]:
    """The end-of-sequence ids as a list: from ``None``, an integer, a 0-d or 1-d integer tensor or numpy array, or
    an iterable of integers. Booleans, strings, floats and arrays of more than one dimension raise ``TypeError``."""
    if eos_token_id is None:
        return []
    err = TypeError(f"eos_token_id takes one token id or a flat collection of ids; {eos_token_id!r} "
                    f"({type(eos_token_id).__name__}) is neither")
    if isinstance(eos_token_id, (bool, str, bytes)):
        raise err
    if isinstance(eos_token_id, numbers.Integral):
        return [int(eos_token_id)]
    if torch.is_tensor(eos_token_id):
        integer = eos_token_id.dtype not in (torch.bool,) and not (eos_token_id.dtype.is_floating_point
                                                                   or eos_token_id.dtype.is_complex)
        if not integer or eos_token_id.dim() > 1:
            raise err
        return eos_token_id.reshape(-1).tolist()
    kind = getattr(getattr(eos_token_id, "dtype", None), "kind", None)       # numpy arrays and scalars
    if kind is not None:
        if kind not in "iu" or eos_token_id.ndim > 1:
            raise err
        return [int(t) for t in eos_token_id.reshape(-1).tolist()]
    try:
        ids = list(eos_token_id)
    except TypeError:
        raise err from None
    if not all(isinstance(t, numbers.Integral) and not isinstance(t, bool) for t in ids):
        raise err
    return [int(t) for t in ids]


def _pick(logits: Tensor, do_sample: bool, temperature: float, top_k: int | None,
          generator: torch.Generator | None) -> Tensor:
    """The next token per row: argmax, or a draw from ``softmax(logits / temperature)`` over the whole vocabulary
    with every logit below the row's ``top_k``-th largest set to -inf (the reference's sampling rule,
    src/sisa/generation.py:126-135: ties at the k-th value stay candidates, and a seeded generator yields the same
    draws as the reference's)."""
    if not do_sample:
        return logits.float().argmax(dim=-1)
    return torch.multinomial(_probabilities(logits, temperature, top_k), 1, generator=generator).squeeze(-1)


def _probabilities(logits: Tensor, temperature: float, top_k: int | None) -> Tensor:
    """What :func:`_pick` draws from."""
    scores = logits.float() / temperature
    if top_k is not None and top_k < scores.shape[-1]:
        floor = scores.topk(top_k, dim=-1).values[..., -1:]
        scores = torch.where(scores < floor, torch.full_like(scores, float("-inf")), scores)
    return scores.softmax(-1)


def verify_drafts(p: Tensor, drafts: Tensor, u: Tensor, q: Tensor) -> tuple[Tensor, Tensor]:
    """:func:`sisa_amd.kernels.verify.sisa_verify_drafts_hip` in plain PyTorch, on any device, for rows that all have ``K`` drafts
    drawn from ``q``: ``(tokens, accepted)``."""
    (B, K), V = drafts.shape, p.shape[2]
    row, i = torch.arange(B, device=p.device), torch.arange(K + 1, device=p.device)
    at, u = drafts.clamp(0, V - 1)[..., None], u.double()
    took = u[:, :K] * q.gather(2, at)[..., 0].double() < p[:, :K].gather(2, at)[..., 0].double()
    took &= (drafts >= 0) & (drafts < V)
    accepted = took.long().cumprod(1).sum(1)
    target = p[row, accepted].double()
    behind_all = torch.cat([q, q.new_zeros((B, 1, V))], 1)         # after the last draft nothing is taken off
    rest = (target - behind_all[row, accepted].double()).clamp(min=0.0)
    weights = torch.where((rest.sum(1) == 0)[:, None], target.clamp(min=0.0), rest)
    total, upto, some = weights.sum(1), weights.cumsum(1), weights > 0
    over = (upto > u[:, K:] * upto[:, -1:]) & some
    token = torch.where(over.any(1), over.int().argmax(1), V - 1 - some.flip(1).int().argmax(1))
    token = torch.where(total.isfinite() & (total > 0), token, -1)
    padded = torch.cat([drafts, drafts.new_full((B, 1), -1)], 1)
    behind, here = i > accepted[:, None], i == accepted[:, None]
    return torch.where(behind, -1, torch.where(here, token[:, None], padded)), accepted.to(torch.int32)


def _prompt_lengths(prompt_lengths, rows: Tensor) -> list[int] | None:
    """The prompts' lengths as a list, or None where every row is full."""
    if prompt_lengths is None:
        return None
    lengths = prompt_lengths.tolist() if torch.is_tensor(prompt_lengths) else list(prompt_lengths)
    if len(lengths) != rows.shape[0] or not all(isinstance(n, numbers.Integral) and 1 <= n <= rows.shape[1] for n in lengths):
        raise ValueError(f"prompt_lengths = {lengths}: expected an integer in 1 .. {rows.shape[1]} for each of the "
                         f"{rows.shape[0]} rows")
    lengths = [int(n) for n in lengths]
    return None if min(lengths) == rows.shape[1] else lengths


class _Budget:
    """When a cache is cut, and to what: to ``keep`` positions, of them the last ``recent``, once it has grown ``slack`` over
    them."""

    def __init__(self, keep: int, recent: int | None) -> None:
        if keep < 1:
            raise ValueError(f"cache_budget = {keep} must be positive")
        self.keep, self.recent = keep, max(1, keep // 4) if recent is None else recent
        if not 1 <= self.recent <= keep:
            raise ValueError(f"cache_recent = {recent} must be in 1 .. cache_budget = {keep}")
        self.slack = max(16, keep // 8)


def _paged_cache(lengths: list[int], new: int, budget: _Budget | None, samples: int = 1) -> SISAPagedCache:
    """A cache for prompts of these lengths and ``new`` more positions of each of their samples, or for what a budget lets them
    grow to. The whole pages of a prompt are held once."""
    rows, longest = len(lengths) * samples, max(lengths)
    size, each = 64, lambda n: -(-n // 64)  # noqa: E731
    if samples > 1:
        pages = sum(n // size + samples * (each(n + new) - n // size) for n in lengths)
        return SISAPagedCache(rows, longest + new, pages=pages, page_size=size)
    if budget is None:
        return SISAPagedCache(rows, longest + new)
    top = max(longest + 1, min(longest + new, budget.keep + budget.slack) + 1)
    return SISAPagedCache(rows, top, pages=rows * (each(top) + each(budget.keep)), page_size=size, track=True)


@torch.no_grad()
def generate(model: "SISAForCausalLM", input_ids: Tensor, max_new_tokens: int, temperature: float = 1.0,
             top_k: int | None = None, eos_token_id: int | Iterable[int] | Tensor | None = None,
             do_sample: bool = False, *, generator: torch.Generator | None = None,
             prompt_lengths: Iterable[int] | Tensor | None = None, cache_budget: int | None = None,
             cache_recent: int | None = None, samples: int = 1, draft: "SISAForCausalLM | None" = None,
             draft_tokens: int = 4) -> Tensor:
    """Continue the prompts ``input_ids`` (``(B, L)`` of equal-length rows, or ``(L,)``) by up to ``max_new_tokens``
    tokens: greedy, or sampled at ``temperature`` from the ``top_k`` most likely tokens with ``do_sample``.

    A row that emits an ``eos_token_id`` is finished and padded with the first such id (which need not be a token) from then on;
    generation ends when every row is finished. Returns ``(B, L + n)`` ids, ``n <= max_new_tokens``, with the rank of
    ``input_ids``.

    ``prompt_lengths``: the prompts are right-padded rows of these lengths (with anything). A row's tokens follow its prompt, and what is
    left of the row behind them is the first ``eos_token_id``, or 0 without one.

    ``cache_budget``: how many positions each layer and head keeps: the last ``cache_recent`` (default: a quarter) and those
    that have received the largest softmax weight. The cache is cut after the prompt, and whenever it has grown by an eighth
    (at least 16) over its budget; until a cut nothing is left out.

    ``samples``: every prompt is read once and continued that many times; the rows of a prompt are neighbours, ``(B * samples,
    L + n)`` (``(samples, L + n)`` for one prompt of rank 1). Their attention reads the prompt's cached positions once for all
    of them.

    ``draft``: a smaller model with the same vocabulary, which proposes ``draft_tokens`` tokens at a time; the model reads them
    in one pass and keeps those that it would have taken: with ``do_sample``, by random numbers such that what comes out is
    distributed as without the draft (not the same draws from a seed), else those that are its own likeliest. Neither goes with
    ``cache_budget``, and not with the other.
    """
    if max_new_tokens < 0:
        raise ValueError(f"max_new_tokens = {max_new_tokens} is negative")
    if do_sample and temperature <= 0:
        raise ValueError(f"sampling needs a positive temperature, got {temperature}")
    if top_k is not None and top_k <= 0:
        raise ValueError(f"top_k = {top_k}: expected a positive integer or None")
    rows = input_ids if input_ids.dim() == 2 else input_ids.unsqueeze(0)
    if rows.dim() != 2 or rows.shape[1] == 0:
        raise ValueError(f"generate needs at least one prompt token per row in a (B, L) or (L,) tensor, got shape "
                         f"{tuple(input_ids.shape)}")
    if cache_recent is not None and cache_budget is None:
        raise ValueError("cache_recent goes with cache_budget")
    if samples < 1 or draft_tokens < 1:
        raise ValueError(f"samples = {samples}, draft_tokens = {draft_tokens}: both must be positive")
    if (samples > 1) + (draft is not None) + (cache_budget is not None) > 1:
        raise ValueError("samples, draft and cache_budget do not go together")
    if draft is not None and draft.config.vocab_size != model.config.vocab_size:
        raise ValueError(f"the draft has {draft.config.vocab_size} tokens, the model {model.config.vocab_size}")
    lengths = _prompt_lengths(prompt_lengths, rows)
    budget = None if cache_budget is None else _Budget(cache_budget, cache_recent)
    stops = _eos_ids(eos_token_id)
    if draft is not None:
        result = _generate_drafted(model, draft, draft_tokens, rows, lengths, max_new_tokens, stops,
                                   (temperature, top_k) if do_sample else None, generator)
        return result if input_ids.dim() == 2 else result.squeeze(0)
    stop_ids = torch.tensor(stops, device=rows.device, dtype=rows.dtype) if stops else None
    pad_unread = bool(stops) and not 0 <= stops[0] < model.config.vocab_size       # what finished rows are padded with is no token
    prompt, prompts = rows.shape[1], rows.shape[0]
    first = [prompt] * prompts if lengths is None else lengths
    if samples > 1:
        rows = rows.repeat_interleave(samples, 0)
    out = rows.new_empty((rows.shape[0], prompt + max_new_tokens))
    out[:, :prompt] = rows
    length = prompt
    if max_new_tokens:
        if lengths is None and budget is None and samples == 1:
            cache = SISACache(capacity=prompt + max_new_tokens)
        else:
            cache = _paged_cache(first, max_new_tokens, budget, samples)
        finished = torch.zeros(rows.shape[0], dtype=torch.bool, device=rows.device)
        ends = None
        if samples > 1:
            some = cache[:prompts]
            n = torch.tensor(first, device=rows.device)
            some.expect(first)
            ids = rows[::samples].masked_fill(torch.arange(prompt, device=rows.device) >= n[:, None], 0)
            logits = model(ids, cache=some, logits_at=[m - 1 for m in first]).logits[:, -1].repeat_interleave(samples, 0)
            cache.branch(samples)
            if lengths is not None:
                ends = n.repeat_interleave(samples)[:, None]
                out[torch.arange(out.shape[1], device=rows.device) >= ends] = stops[0] if stops else 0
        elif lengths is None:
            logits = model(rows, cache=cache, logits_to_keep=1).logits[:, -1]
        else:
            # what pads the rows need not be a token; rows are laid out from their own ends
            n = torch.tensor(lengths, device=rows.device)
            behind = torch.arange(out.shape[1], device=rows.device) >= n[:, None]
            cache.expect(lengths)
            logits = model(rows.masked_fill(behind[:, :prompt], 0), cache=cache,
                           logits_at=[n - 1 for n in lengths]).logits[:, -1]
            out[behind] = stops[0] if stops else 0
            ends = n[:, None]
        while True:
            token = _pick(logits, do_sample, temperature, top_k, generator).to(rows.dtype)
            if stop_ids is not None:
                token = torch.where(finished, stop_ids[0], token)
                finished |= torch.isin(token, stop_ids)
            if ends is None:
                out[:, length] = token
            else:
                out.scatter_(1, ends + (length - prompt), token[:, None])
            length += 1
            if length == out.shape[1] or (stop_ids is not None and bool(finished.all())):
                break
            if budget is not None and (length == prompt + 1 or cache.seq_len >= budget.keep + budget.slack):
                cache.evict(budget.keep, budget.recent)
            if pad_unread:
                token = token.masked_fill(finished, 0)
            logits = model(token[:, None], cache=cache, logits_to_keep=1).logits[:, -1]
    result = out[:, :length].contiguous()
    return result if input_ids.dim() == 2 or samples > 1 else result.squeeze(0)


def _generate_drafted(model, draft, K: int, rows: Tensor, lengths: list[int] | None, new: int, stops: list[int],
                      sampling: tuple[float, int | None] | None, generator: torch.Generator | None) -> Tensor:
    """:func:`generate` with a draft. In each round the draft reads its last token and its own proposals, one by one, and the
    model all of them at once; both caches keep what was accepted. Rows that are done keep nothing more."""
    B, prompt = rows.shape
    first = [prompt] * B if lengths is None else lengths
    fill = stops[0] if stops else 0
    if not new:
        return rows.clone()
    n = torch.tensor(first, device=rows.device)
    ids = rows.masked_fill(torch.arange(prompt, device=rows.device) >= n[:, None], 0)
    caches = [SISAPagedCache(B, max(first) + new + K + 1) for _ in range(2)]
    logits = []
    for m, cache in zip((model, draft), caches):
        cache.expect(first)
        logits.append(m(ids, cache=cache, logits_at=[i - 1 for i in first]).logits[:, -1])
    target, proposals = caches
    token = _pick(logits[0], sampling is not None, *(sampling or (1.0, None)), generator).to(rows.dtype)
    out = [[t] for t in token.tolist()]
    done = [new == 1 or t[0] in stops for t in out]
    while not all(done):
        proposals.tentative(K + 1)
        target.tentative(K + 1)
        said, q, last = [token], [], token
        for i in range(K + 1):
            logits = draft(last[:, None], cache=proposals, logits_to_keep=1).logits[:, -1]
            if i == K:                                     # the last proposal is read for the draft's cache alone
                break
            if sampling is None:
                last = logits.float().argmax(dim=-1).to(rows.dtype)
            else:
                q.append(_probabilities(logits, *sampling))
                last = torch.multinomial(q[-1], 1, generator=generator).squeeze(-1).to(rows.dtype)
            said.append(last)
        logits = model(torch.stack(said, 1), cache=target).logits
        drafts = torch.stack(said[1:], 1).long()
        if sampling is None:
            own = logits.float().argmax(dim=-1)
            accepted = (own[:, :K] == drafts).long().cumprod(1).sum(1)
            tokens = torch.where(torch.arange(K + 1, device=rows.device) <= accepted[:, None], own, -1)
        else:
            p = _probabilities(logits, *sampling)
            u = torch.rand((B, K + 1), device=p.device, generator=generator)
            if p.is_cuda and hip_status(p.device)[0]:
                from .kernels.verify import sisa_verify_drafts_hip

                tokens, accepted = sisa_verify_drafts_hip(p, drafts, u, torch.stack(q, 1))
            else:
                tokens, accepted = verify_drafts(p, drafts, u, torch.stack(q, 1))
        got, took = tokens.tolist(), accepted.tolist()
        counts = []
        for i, row in enumerate(out):
            if done[i]:
                counts.append(0)
                got[i][0], took[i] = 0, 0                  # read and not kept (the fill need not be a token)
                continue
            if got[i][took[i]] < 0:
                raise RuntimeError("generate: the model's probabilities are not finite, or 0 everywhere")
            for t in got[i][:took[i] + 1]:
                row.append(t)
                done[i] = len(row) == new or t in stops
                if done[i]:
                    break
            counts.append(0 if done[i] else took[i] + 1)
        target.keep(counts)
        proposals.keep(counts)
        token = torch.tensor([row[a] for row, a in zip(got, took)], device=rows.device, dtype=rows.dtype)
    longest = max(len(row) for row in out)
    result = rows.new_full((B, prompt + longest), fill)
    result[:, :prompt] = torch.where(torch.arange(prompt, device=rows.device) < n[:, None], rows, fill)
    at = n[:, None] + torch.arange(longest, device=rows.device)
    return result.scatter_(1, at, torch.tensor([row + [fill] * (longest - len(row)) for row in out], device=rows.device,
                                               dtype=rows.dtype))
