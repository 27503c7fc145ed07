"""A decode cache in pages: sequences of unequal lengths in one batch, a bound on how many positions are kept, several
continuations of one prompt, and positions that can be taken back.

:class:`SISAPagedCache` stands where :class:`sisa_amd.generation.SISACache` does (``model(ids, cache=cache)``), with four
things that one has not:

* every sequence has its own length and takes its memory in pages from a common pool, so prompts of different lengths are
  one right-padded batch, a finished sequence gives its pages to the next, and ``cache[2]`` is the cache of sequence 2
  alone, to fill while the others stay;
* with ``track=True`` every position's softmax weight is accumulated over the queries that saw it, and :meth:`evict` cuts
  the sequences down to their last and their most attended positions. The score of a SISA key depends on its own ``g``,
  ``F`` and rotated ``b``, not on its distance, so what follows is exactly the softmax over the kept keys;
* :meth:`branch` continues every prompt several times: the branches hold the prompt's pages together, and their attention
  reads them once;
* after :meth:`tentative`, :meth:`keep` takes back what a draft proposed in vain.

On the GPU the operators are the HIP kernels of :mod:`sisa_amd.kernels.paged`, :mod:`sisa_amd.kernels.weights` and
:mod:`sisa_amd.kernels.prefix`;
elsewhere, and for head or state sizes those do not take, the plain PyTorch forms below, in float32 (float64 inputs:
float64). Inference only. The reference has no such cache.
"""
from __future__ import annotations

from typing import NamedTuple, Sequence

import torch
from torch import Tensor

from .config import HIP_D_HEAD, HIP_D_STATE
from .functional import autocast_disabled, working_dtype

__all__ = ["SISAPagedCache", "attention_weights", "paged_attention"]


#: Scores of a call of the attention kernel over pages that several new positions take: about 5 bytes of workspace each.
MAX_SCORES = 1 << 26
#: Rows, of every head, of a call of the one over common positions: about 530 bytes of workspace each, at most 420 MB in all.
MAX_ROWS = 1 << 19


# ------------------------------------------------------------------------------------------------ plain forms
class _Pages(NamedTuple):
    """The tensors of a pool, as :class:`sisa_amd.kernels.paged.PagePool` has them, on any device and of any head size."""
    k: Tensor
    v: Tensor
    b: Tensor
    g: Tensor
    fgate: Tensor


def _write(pool: _Pages, table: Tensor, start: Tensor, count: Tensor, rows: Sequence[Tensor]) -> None:
    S, M = pool.g.shape[2], rows[0].shape[2]
    m = torch.arange(M, device=table.device)
    pos, new = start.long()[:, None] + m, m < count[:, None]
    pos = torch.where(new, pos, 0)
    page, slot = table.long().gather(1, pos // S)[new], (pos % S)[new]
    for t, x in zip(pool, rows):
        t[page, :, slot] = x.transpose(1, 2)[new]


def _laid_out(pool: _Pages, table: Tensor, N: int, dtype: torch.dtype) -> list[Tensor]:
    """The first ``N`` positions of every sequence side by side, ``(B, H, N, .)``."""
    pages = table.long().clamp(min=0)
    return [t[pages].transpose(1, 2).flatten(2, 3)[:, :, :N].to(dtype) for t in pool]


def _softmax_weights(q, c, g, f, lam, k, b, g_k, f_k, seen: Tensor) -> Tensor:
    """Softmax over the keys that ``seen`` (broadcastable to ``(B, H, M, N)``) allows; 0 for the others, and in rows that see
    none."""
    with autocast_disabled(q.device.type):
        decay = torch.where(seen, g[..., :, None] - g_k[..., None, :], 0.0).exp()
        s = (q @ k.mT) * q.shape[-1] ** -0.5 + lam[:, None, None] * decay * (c @ b.mT)
        s = s + (f[..., :, None] - f_k[..., None, :])
        p = torch.where(seen, s, float("-inf")).softmax(-1)
    return torch.where(seen, p, 0.0)


def paged_attention(q: Tensor, c: Tensor, g_q: Tensor, f_q: Tensor, lam: Tensor, pool, table: Tensor, lengths: Tensor,
                    max_len: int, weights: Tensor | None = None) -> Tensor:
    """Exact attention of the last ``M`` cached positions of every sequence (``q`` ``(B, H, M, d_head)``) over the positions
    up to their own, in plain PyTorch; ``weights`` ``(B, H, >= max_len)`` gets the softmax weights added in place. Semantics
    of :func:`sisa_amd.kernels.paged.sisa_paged_decode_hip`, in the working precision."""
    wd, M = working_dtype(q.dtype), q.shape[2]
    k, v, b, g, f = _laid_out(pool, table, max_len, wd)
    m, j = torch.arange(M, device=q.device)[:, None], torch.arange(max_len, device=q.device)
    n = lengths.long()[:, None, None, None]
    seen = j < n - M + 1 + m
    v = torch.where((j < n[..., 0])[..., None], v, 0.0)          # what lies behind a sequence may be anything
    p = _softmax_weights(q.to(wd), c.to(wd), g_q.to(wd), f_q.to(wd), lam.to(wd), k, b, g, f, seen)
    if weights is not None:
        weights[:, :, :max_len] += p.sum(2).to(weights.dtype)
    with autocast_disabled(q.device.type):
        return p @ v


def attention_weights(q: Tensor, k: Tensor, c: Tensor, b: Tensor, g: Tensor, lam: Tensor, fgate: Tensor, lengths: Tensor,
                      block: int = 256) -> Tensor:
    """Every position's softmax weight summed over the queries of its sequence, ``(B, H, L)``, in plain PyTorch: semantics of
    :func:`sisa_amd.kernels.weights.sisa_attention_weights_hip` without a window, in the working precision, query block by
    query block."""
    wd, L = working_dtype(q.dtype), q.shape[2]
    qw, kw, cw, bw, gw, fw, lw = (t.to(wd) for t in (q, k, c, b, g, fgate, lam))
    j = torch.arange(L, device=q.device)
    out = torch.zeros_like(gw)
    for first in range(0, L, block):
        last = min(first + block, L)
        i = torch.arange(first, last, device=q.device)[:, None]
        seen = (j <= i) & (i < lengths.long()[:, None, None, None])
        out += _softmax_weights(qw[:, :, first:last], cw[:, :, first:last], gw[:, :, first:last], fw[:, :, first:last], lw,
                                kw, bw, gw, fw, seen).sum(2)
    return out


def _evict(pool: _Pages, table: Tensor, lengths: Tensor, weights: Tensor, keep: int, recent: int, new_table: Tensor,
           max_len: int) -> tuple[Tensor, Tensor]:
    """New lengths and weights ``(B, H, keep)``; the kept rows are copied to the pages of ``new_table``."""
    n, w = lengths.long()[:, None, None], weights[:, :, :max_len]
    j = torch.arange(max_len, device=table.device)
    order = torch.where(j < n, w, float("-inf")).sort(dim=-1, descending=True, stable=True).indices
    # the recent positions before all others, the others as they are
    late = (order >= n - recent) & (order < n)
    order = order.gather(-1, late.to(torch.int8).sort(dim=-1, descending=True, stable=True).indices)
    K = min(keep, max_len)
    kept = torch.arange(K, device=table.device) < n.clamp(max=keep)
    pos = torch.where(kept, order[..., :K], max_len).sort(-1).values.clamp(max=max_len - 1)
    ok = kept.expand_as(pos)
    S, H = pool.g.shape[2], pool.g.shape[1]
    i = torch.arange(K, device=table.device)
    page = table.long().clamp(min=0)[:, None].expand(-1, H, -1).gather(2, pos // S)
    to = new_table.long().clamp(min=0)[:, None, i // S].expand_as(pos)
    h = torch.arange(H, device=table.device)[:, None].expand_as(pos)
    for t in pool:
        t[to[ok], h[ok], (i % S).expand_as(pos)[ok]] = t[page[ok], h[ok], (pos % S)[ok]]
    new = weights.new_zeros((*weights.shape[:2], keep))
    new[..., :K] = torch.where(ok, w.gather(2, pos), 0.0)
    return lengths.clamp(max=keep), new


# ------------------------------------------------------------------------------------------------ the cache
def at_last(x: Tensor, count: Tensor | None) -> Tensor:
    """The last real position of ``x`` ``(B, H, M, ...)``, kept as an axis of one."""
    if count is None:
        return x[:, :, -1:]
    at = (count.long() - 1).view(-1, 1, 1, *[1] * (x.dim() - 3))
    return x.gather(2, at.expand(x.shape[0], x.shape[1], 1, *x.shape[3:]))


class _Last(NamedTuple):
    """What a layer's recurrences continue from: ``g, fgate`` ``(B, H, 1)`` and ``phi`` ``(B, H, d_state // 2)`` at the last
    position of every sequence."""
    g: Tensor
    fgate: Tensor
    phi: Tensor


class _Step(NamedTuple):
    """What a layer's step is given: the pool, the sequences' table rows, their lengths before and after, what the recurrences
    continue from (advanced in place), the accumulated weights, and a bound on the lengths."""
    pool: object
    table: Tensor
    start: Tensor
    end: Tensor
    last: _Last
    weights: Tensor | None
    max_len: int


class _Sharing(NamedTuple):
    """What :func:`sisa_amd.kernels.prefix.sisa_prefix_decode_hip` is told of the sequences: their groups, the positions that each
    has in common, and the most of them."""
    groups: object
    shared: Tensor
    most: int


class _Trial:
    """Positions that may be taken back: the sequences, how many positions there can be, where they begin, and per layer
    ``(sequences, H, room + 1, 2 + d_state // 2)`` what the recurrences continue from before the first and after each."""

    def __init__(self, lo: int, hi: int, room: int, starts: list[int]) -> None:
        self.lo, self.hi, self.room, self.starts = lo, hi, room, starts
        self.rows: dict[int, Tensor] = {}


class _Begun(NamedTuple):
    """A pass whose first layer is not written yet: its sequences, and what the store held for them before."""
    lo: int
    hi: int
    pages: list[int]
    starts: list[int]
    lengths: list[int]
    expected: list


class _Layer:
    """One layer: its pages, the last position's recurrences, how many positions each sequence holds, and the accumulated
    weights ``(sequences, H, max_length)`` of a tracked cache."""

    def __init__(self, pool, last: _Last, weights: Tensor | None, sequences: int) -> None:
        self.pool, self.last, self.weights, self.filled = pool, last, weights, [0] * sequences


class _Store:
    """What the cache and its parts (``cache[2:4]``) share."""

    def __init__(self, sequences: int, max_length: int, pages: int, page_size: int, track: bool) -> None:
        self.sequences, self.max_length, self.page_size, self.track = sequences, max_length, page_size, track
        self.pages = pages
        self.free = list(range(pages - 1, -1, -1))
        self.held: list[list[int]] = [[] for _ in range(sequences)]
        self.starts, self.lengths = [0] * sequences, [0] * sequences   # before and after the last forward pass
        self.widths = [0] * sequences                                  # that pass's positions, padding included
        self.expected: list[int | None] = [None] * sequences           # real positions of the next pass, if not all
        self.begun: _Begun | None = None
        self.trial: _Trial | None = None
        self.family: list[tuple[int, int] | None] = [None] * sequences    # a prompt's number, and its pages that are shared
        self.families = 0
        self.others: dict[int, int] = {}                   # of a shared page: how many sequences hold it beside one
        self.sharing: dict[tuple[int, int], _Sharing | None] = {}
        self.layers: dict[int, _Layer] = {}
        self.table = self.start = self.end = None          # on the model's device, made by the first pass

    def device_state(self, device: torch.device) -> None:
        if self.table is None:
            width = -(-self.max_length // self.page_size)
            self.table = torch.full((self.sequences, width), -1, dtype=torch.int32, device=device)
            self.start, self.end = (torch.zeros(self.sequences, dtype=torch.int32, device=device) for _ in range(2))
            if any(self.held):                             # reserved before the first pass
                self.show(range(self.sequences))
        elif self.table.device != device:
            raise ValueError(f"SISAPagedCache: filled on {self.table.device}, used on {device}")

    def take(self, lo: int, ends: Sequence[int]) -> list[int]:
        """Pages so that the sequences from ``lo`` on have room for ``ends`` positions, all of them or, where there are too few
        pages, none; the sequences that got any."""
        need = [max(0, -(-end // self.page_size) - len(held)) for end, held in zip(ends, self.held[lo:])]
        if sum(need) > len(self.free):
            raise RuntimeError(f"SISAPagedCache: {sum(need)} more pages of {self.page_size} positions are needed, "
                               f"{len(self.free)} of {self.pages} are free (evict, release a sequence, or make the pool "
                               f"larger)")
        for n, pages in enumerate(need, lo):
            self.held[n] += [self.free.pop() for _ in range(pages)]
        return [n for n, pages in enumerate(need, lo) if pages]

    def give(self, pages) -> None:
        """Pages of a sequence that holds them no more: free, where no other does."""
        for page in pages:
            left = self.others.pop(page, 0)
            if not left:
                self.free.append(page)
            elif left > 1:
                self.others[page] = left - 1

    def runs(self, lo: int, hi: int) -> list[tuple[int, int]]:
        """Neighbours that continue the same prompt: how many, and the positions that they share."""
        out, last = [], None
        for family in self.family[lo:hi]:
            if family is not None and family == last:
                out[-1] = (out[-1][0] + 1, out[-1][1])
            else:
                out.append((1, 0 if family is None else family[1] * self.page_size))
            last = family
        return out

    def grouped(self, lo: int, hi: int) -> _Sharing | None:
        """The sequences' groups for the kernels, or None where no two have pages in common."""
        if (lo, hi) not in self.sharing:
            runs, found = self.runs(lo, hi), None
            if any(size > 1 and shared for size, shared in runs):
                from .kernels.prefix import PrefixGroups

                shared = torch.tensor([n for _, n in runs], dtype=torch.int32).to(self.table.device)
                found = _Sharing(PrefixGroups([size for size, _ in runs], self.table.device), shared, max(n for _, n in runs))
            self.sharing[lo, hi] = found
        return self.sharing[lo, hi]

    def singles(self, lo: int, hi: int) -> object:
        """Every sequence a group of its own."""
        from .kernels.prefix import PrefixGroups

        key = (lo, hi, "singles")
        if key not in self.sharing:
            self.sharing[key] = PrefixGroups([1] * (hi - lo), self.table.device)
        return self.sharing[key]

    def undo(self) -> None:
        """Take back the pass that has begun and written nothing: the cache is as it was before."""
        was, self.begun = self.begun, None
        if was is None:
            return
        lo, hi = was.lo, was.hi
        for n in reversed(range(lo, hi)):
            pages = was.pages[n - lo]
            self.free += reversed(self.held[n][pages:])
            del self.held[n][pages:]
        self.starts[lo:hi], self.lengths[lo:hi], self.expected[lo:hi] = was.starts, was.lengths, was.expected
        self.end[lo:hi].copy_(torch.tensor(was.lengths, dtype=torch.int32))
        self.show(range(lo, hi))

    def show(self, sequences: Sequence[int]) -> None:
        """The device's table of these sequences, from the host's."""
        rows = [self.held[n] + [-1] * (self.table.shape[1] - len(self.held[n])) for n in sequences]
        lo, hi = sequences[0], sequences[-1] + 1
        self.table[lo:hi].copy_(torch.tensor(rows, dtype=torch.int32))


class _Writing:
    """:meth:`SISAPagedCache.failed` on an error."""
    __slots__ = ("cache", "layer_idx")

    def __init__(self, cache: "SISAPagedCache", layer_idx: int) -> None:
        self.cache, self.layer_idx = cache, layer_idx

    def __enter__(self) -> None:
        pass

    def __exit__(self, kind, *_) -> None:
        if kind is not None:
            self.cache.failed(self.layer_idx)


class SISAPagedCache:
    """Decode cache of ``sequences`` sequences of at most ``max_length`` positions each, in ``pages`` pages (default: what all
    of them can need, and with ``track`` as many more as one of them, for the rows that an eviction keeps) of ``page_size``
    positions per layer, a power of two of at least 16. ``track``: accumulate every position's softmax weight, for
    :meth:`evict`.

    The first pass of a sequence may be right-padded: ``cache.expect([5, 9])`` before it says how many of its positions are
    there. Later passes add the same number of positions to every sequence. ``cache[n]`` and ``cache[a:b]`` are the caches of
    some of the sequences, sharing everything with the whole.

    A pass that is refused, or fails before its first layer is written, leaves the cache as it was. One that fails later has
    reached some layers and not others: its sequences refuse further passes until they are released."""

    def __init__(self, sequences: int, max_length: int, *, pages: int | None = None, page_size: int = 64,
                 track: bool = False) -> None:
        if sequences < 1 or max_length < 1:
            raise ValueError(f"SISAPagedCache: {sequences} sequences of {max_length} positions: both must be positive")
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"SISAPagedCache: page_size = {page_size} must be a power of two of at least 16")
        each = -(-max_length // page_size)
        if pages is not None and pages < 1:
            raise ValueError(f"SISAPagedCache: pages = {pages} must be positive")
        self._store = _Store(sequences, max_length, (sequences + bool(track)) * each if pages is None else pages, page_size,
                             track)
        self._lo, self._hi = 0, sequences

    # -------------------------------------------------------------------------------------------- parts
    def __getitem__(self, which: int | slice) -> "SISAPagedCache":
        n = len(self)
        if isinstance(which, slice):
            lo, hi, step = which.indices(n)
            if step != 1 or lo >= hi:
                raise ValueError(f"SISAPagedCache: a part is a range of sequences in order, got {which}")
        else:
            if not -n <= which < n:
                raise IndexError(f"sequence {which} of {n}")
            lo = which % n
            hi = lo + 1
        part = object.__new__(SISAPagedCache)
        part._store, part._lo, part._hi = self._store, self._lo + lo, self._lo + hi
        return part

    def __len__(self) -> int:
        """How many sequences."""
        return self._hi - self._lo

    @property
    def lengths(self) -> list[int]:
        """Cached positions of every sequence."""
        return self._store.lengths[self._lo:self._hi]

    @property
    def seq_len(self) -> int:
        """The longest sequence's positions (0 before the first pass)."""
        return max(self.lengths)

    @property
    def free_pages(self) -> int:
        return len(self._store.free)

    @property
    def tracked(self) -> bool:
        return self._store.track

    def weights(self, layer_idx: int) -> Tensor:
        """A layer's accumulated weights ``(sequences, H, max_length)`` float32, 0 behind each sequence."""
        layer = self._store.layers.get(layer_idx)
        if layer is None or layer.weights is None:
            raise ValueError("SISAPagedCache: weights are there after the first pass of a cache made with track=True")
        return layer.weights[self._lo:self._hi]

    # -------------------------------------------------------------------------------------------- a forward pass
    def expect(self, counts: Sequence[int]) -> None:
        """How many positions of each row of the next, first pass are real; the others are padding on the right."""
        self._store.undo()                                 # of a pass that was given up between two calls, as below
        counts = [int(c) for c in counts]
        if len(counts) != len(self) or any(c < 1 for c in counts):
            raise ValueError(f"SISAPagedCache.expect: {counts}: a positive count for each of the {len(self)} sequences")
        if any(self.lengths):
            raise ValueError("SISAPagedCache.expect: only the first pass of a sequence may be padded")
        self._store.expected[self._lo:self._hi] = counts

    def last(self, layer_idx: int) -> _Last | None:
        """What the layer's recurrences continue from, or None before its first pass."""
        if self.empty(layer_idx):
            return None
        layer = self._store.layers[layer_idx]
        if not all(layer.filled[self._lo:self._hi]):
            raise ValueError("SISAPagedCache: some of these sequences are empty and some are not; fill the empty ones on "
                             "their own (cache[n])")
        return _Last(*(t[self._lo:self._hi] for t in layer.last))

    def writing(self, layer_idx: int) -> _Writing:
        """For a with statement around what a layer does between :meth:`begin` or :meth:`begin_step` and its end."""
        return _Writing(self, layer_idx)

    def failed(self, layer_idx: int) -> None:
        """An error in what a layer does for a pass that has begun: the pass is taken back, or the layer marked."""
        st = self._store
        if st.begun is not None:
            st.undo()
        else:                                              # some layers have this pass's positions, this one may have
            st.layers[layer_idx].filled[self._lo:self._hi] = [-1] * len(self)

    def _begin(self, layer: _Layer, M: int) -> None:
        """The positions of a pass of ``M``, at its first layer; the later ones find them there."""
        st, lo, hi = self._store, self._lo, self._hi
        if st.begun is not None:
            st.undo()
        filled = layer.filled[lo:hi]
        first = filled == st.lengths[lo:hi]
        if not first and filled == st.starts[lo:hi] and st.widths[lo:hi] == [M] * (hi - lo):
            return
        if not first or any(x.filled[lo:hi] != filled for x in st.layers.values()):
            raise RuntimeError("SISAPagedCache: an earlier forward pass did not reach every layer; release() the sequences")
        counts = [M if c is None else c for c in st.expected[lo:hi]]
        if max(counts) > M:
            raise ValueError(f"SISAPagedCache: {max(counts)} positions were expected, the pass has {M}")
        ends = [n + c for n, c in zip(self.lengths, counts)]
        if max(ends) > st.max_length:
            raise ValueError(f"SISAPagedCache: {max(ends)} positions exceed max_length = {st.max_length}")
        trial = st.trial
        if trial is not None and lo < trial.hi and trial.lo < hi:
            if (lo, hi) != (trial.lo, trial.hi):
                raise ValueError("SISAPagedCache: a pass of tentative sequences takes all of them")
            if ends[0] - trial.starts[0] > trial.room:
                raise ValueError(f"SISAPagedCache: more than the {trial.room} positions that tentative() was told of")
        st.begun = _Begun(lo, hi, [len(pages) for pages in st.held[lo:hi]], st.starts[lo:hi], st.lengths[lo:hi],
                          st.expected[lo:hi])
        try:
            fresh = st.take(lo, ends)
            if fresh:
                st.show(fresh if len(fresh) == 1 else range(lo, hi))
            st.start[lo:hi].copy_(st.end[lo:hi])
            if counts == [M] * len(self):
                st.end[lo:hi].add_(M)
            else:
                st.end[lo:hi].copy_(torch.tensor(ends, dtype=torch.int32))
        except BaseException:
            st.undo()
            raise
        st.starts[lo:hi], st.lengths[lo:hi], st.widths[lo:hi] = self.lengths, ends, [M] * len(self)
        st.expected[lo:hi] = [None] * len(self)

    def _layer(self, layer_idx: int, k: Tensor, b: Tensor, hip: bool) -> _Layer:
        st = self._store
        layer = st.layers.get(layer_idx)
        if layer is not None:
            return layer
        H, D, s = k.shape[1], k.shape[3], b.shape[3]
        like = (st.pages, H, st.page_size)
        # pages begin as zeros: what a sequence leaves unwritten is read by the plain forms, and then masked
        tensors = (k.new_zeros((*like, D)), k.new_zeros((*like, D)), b.new_zeros((*like, s)),
                   k.new_zeros(like, dtype=torch.float32), k.new_zeros(like, dtype=torch.float32))
        if hip:
            from .kernels.paged import PagePool

            pool = PagePool(*tensors)
        else:
            pool = _Pages(*tensors)
        gates = k.new_zeros((st.sequences, H, 1), dtype=torch.float32)
        last = _Last(gates, gates.clone(), gates.new_zeros((st.sequences, H, s // 2)))
        weights = gates.new_zeros((st.sequences, H, st.max_length)) if st.track else None
        layer = st.layers[layer_idx] = _Layer(pool, last, weights, st.sequences)
        return layer

    def begin(self, layer_idx: int, k: Tensor, b: Tensor, hip: bool) -> Tensor | None:
        """Room in a layer for a pass of ``k.shape[2]`` positions of every sequence. Returns how many of them are real, a
        tensor, or None where all are."""
        st, lo, hi = self._store, self._lo, self._hi
        B, _, M, _ = k.shape
        if B != len(self):
            raise ValueError(f"SISAPagedCache: {B} rows for {len(self)} sequences")
        st.device_state(k.device)
        layer = self._layer(layer_idx, k, b, hip)
        if (layer.pool.k.dtype, layer.pool.k.shape[1]) != (k.dtype, k.shape[1]):
            raise ValueError(f"SISAPagedCache: filled in {layer.pool.k.dtype} with {layer.pool.k.shape[1]} heads, got "
                             f"{k.dtype} and {k.shape[1]}")
        if isinstance(layer.pool, _Pages) == hip:
            raise ValueError(f"SISAPagedCache: filled by the {'torch' if hip else 'HIP'} implementation, which cannot be changed "
                             f"while sequences are held; make a new cache")
        self._begin(layer, M)
        with self.writing(layer_idx):
            padded = [n - m for n, m in zip(self.lengths, layer.filled[lo:hi])] != [M] * B
            return st.end[lo:hi] - st.start[lo:hi] if padded else None

    def put(self, layer_idx: int, rows: Sequence[Tensor], phi: Tensor, count: Tensor | None, hip: bool) -> None:
        """The rows ``k, v, b, g, fgate`` of a pass that :meth:`begin` made room for, and the phase ``(B, H, d_state // 2)``
        at each sequence's last one."""
        st, lo, hi = self._store, self._lo, self._hi
        layer = st.layers[layer_idx]
        if hip:
            from .kernels.paged import sisa_paged_write_hip

            sisa_paged_write_hip(layer.pool, st.table[lo:hi], st.start[lo:hi], *rows, count)
        else:
            _write(layer.pool, st.table[lo:hi], st.start[lo:hi], st.end[lo:hi] - st.start[lo:hi], rows)
        for t, x in zip(layer.last, (*(at_last(x, count) for x in (rows[3], rows[4])), phi)):
            t[lo:hi].copy_(x)
        self._written(layer)

    def _written(self, layer: _Layer) -> None:
        layer.filled[self._lo:self._hi] = self.lengths
        self._store.begun = None

    def extend(self, layer_idx: int, p, hip: bool) -> None:
        """Write a pass's rows (``p``: :class:`sisa_amd.modeling.Prepared`) of one layer behind what its sequences hold."""
        if torch.is_grad_enabled() and (p.k.requires_grad or p.g.requires_grad):
            raise RuntimeError("SISAPagedCache is for inference: run the model under torch.no_grad()")
        count = self.begin(layer_idx, p.k, p.b, hip)
        with self.writing(layer_idx):
            self._note(layer_idx, p)
            self.put(layer_idx, (p.k, p.v, p.b, p.g.float(), p.fgate.float()), at_last(p.phi, count)[:, :, 0], count, hip)

    def _rows(self, layer_idx: int) -> tuple[Tensor, int] | None:
        """Of a pass of tentative positions that has begun: the layer's states, and the place of the one before it."""
        st = self._store
        trial = st.trial
        if trial is None or (trial.lo, trial.hi) != (self._lo, self._hi):
            return None
        rows, last = trial.rows.get(layer_idx), st.layers[layer_idx].last
        if rows is None:
            rows = trial.rows[layer_idx] = last.phi.new_empty((len(self), last.phi.shape[1], trial.room + 1,
                                                               2 + last.phi.shape[2]))
        return rows, st.starts[self._lo] - trial.starts[0]

    def _note(self, layer_idx: int, p) -> None:
        found = self._rows(layer_idx)
        if found is None:
            return
        (rows, at), M = found, p.k.shape[2]
        before = _Last(*(t[self._lo:self._hi] for t in self._store.layers[layer_idx].last))
        rows[:, :, at] = torch.cat([before.g, before.fgate, before.phi], -1)
        rows[:, :, at + 1:at + 1 + M] = torch.cat([p.g[..., None], p.fgate[..., None], p.phi], -1)

    def _sharing(self) -> _Sharing | None:
        """Which positions the sequences' new rows have in common: a prompt's with its other branches, or, for positions that may
        be taken back, all that lies before them with each other."""
        st, lo, hi = self._store, self._lo, self._hi
        found = st.grouped(lo, hi)
        if found is None and st.trial is not None and (st.trial.lo, st.trial.hi) == (lo, hi):
            found = _Sharing(st.singles(lo, hi), st.start[lo:hi], max(st.starts[lo:hi]))
        return found

    def attend(self, layer_idx: int, p, lam: Tensor, hip: bool) -> Tensor:
        """The attention of the rows that :meth:`extend` has just written, ``(B, H, M, d_head)`` float32 (float64 rows:
        float64), their softmax weights tracked."""
        st, lo, hi = self._store, self._lo, self._hi
        layer = st.layers[layer_idx]
        weights = None if layer.weights is None else layer.weights[lo:hi]
        with self.writing(layer_idx):
            if hip:
                return self._attend_hip(p, lam, layer.pool, weights)
            return paged_attention(p.q, p.c, p.g, p.fgate, lam, layer.pool, st.table[lo:hi], st.end[lo:hi], self.seq_len,
                                   weights)

    def _attend_hip(self, p, lam: Tensor, pool, weights: Tensor | None) -> Tensor:
        from .kernels.paged import sisa_paged_decode_hip

        st, lo, hi = self._store, self._lo, self._hi
        table, lengths, longest, (B, H, M, _) = st.table[lo:hi], st.end[lo:hi], self.seq_len, p.q.shape

        def parts(rows: int, attend) -> Tensor:
            """Some of the new rows at a time, for which the sequences end with the last of them."""
            if rows >= M:
                return attend(p.q, p.c, p.g, p.fgate, lengths)
            return torch.cat([attend(*(t[:, :, m:m + rows] for t in (p.q, p.c, p.g, p.fgate)), lengths - max(0, M - m - rows))
                              for m in range(0, M, rows)], 2)

        sharing = None if weights is not None else self._sharing()
        if sharing is not None:
            from .kernels.prefix import sisa_prefix_decode_hip

            return parts(max(1, MAX_ROWS // (B * H)), lambda q, c, g, f, ends: sisa_prefix_decode_hip(
                q, c, g, f, lam, pool, table, ends, sharing.groups, sharing.shared, max_len=longest, max_shared=sharing.most))
        return parts(max(1, MAX_SCORES // (B * H * longest)), lambda q, c, g, f, ends: sisa_paged_decode_hip(
            q, c, g, f, lam, pool, table, ends, max_len=longest, weights=weights))

    def receive(self, layer_idx: int, q: Tensor, k: Tensor, c: Tensor, b: Tensor, g: Tensor, lam: Tensor, fgate: Tensor,
                hip: bool) -> None:
        """Track the weights of a first pass, in which the rows attended to each other."""
        st, lo, hi = self._store, self._lo, self._hi
        with self.writing(layer_idx):
            if hip:
                from .kernels.weights import sisa_attention_weights_hip

                w = sisa_attention_weights_hip(q, k, c, b, g.float(), lam, fgate.float(), lengths=st.end[lo:hi])
            else:
                w = attention_weights(q, k, c, b, g, lam, fgate, st.end[lo:hi])
            N = min(k.shape[2], st.max_length)             # a padded batch may be wider than the cache
            st.layers[layer_idx].weights[lo:hi, :, :N] = w[:, :, :N]

    def empty(self, layer_idx: int) -> bool:
        """Whether no sequence holds a position in this layer."""
        layer = self._store.layers.get(layer_idx)
        return layer is None or not any(layer.filled[self._lo:self._hi])

    def kernel_layer(self, layer_idx: int, like: Tensor, heads: int) -> bool:
        """Whether every sequence holds positions in this layer, in a pool of the HIP kernels for rows of ``like``'s dtype and
        device with ``heads`` heads."""
        layer = self._store.layers.get(layer_idx)
        return (layer is not None and not isinstance(layer.pool, _Pages) and all(layer.filled[self._lo:self._hi])
                and (layer.pool.dtype, layer.pool.heads, layer.pool.device_index) == (like.dtype, heads, like.get_device())
                and len(self) == like.shape[0])

    def begin_step(self, layer_idx: int) -> "_Step":
        """One more position of every sequence of a :meth:`kernel_layer`: what a kernel that writes it, advances the
        recurrences and attends needs; :meth:`end_step` follows."""
        st, lo, hi = self._store, self._lo, self._hi
        layer = st.layers[layer_idx]
        self._begin(layer, 1)
        return _Step(layer.pool, st.table[lo:hi], st.start[lo:hi], st.end[lo:hi], _Last(*(t[lo:hi] for t in layer.last)),
                     None if layer.weights is None else layer.weights[lo:hi], self.seq_len)

    def end_step(self, layer_idx: int) -> None:
        self._written(self._store.layers[layer_idx])

    def shares(self) -> bool:
        """Whether the sequences of a :meth:`kernel_layer` are for the kernels of common positions: branches of a prompt, or
        positions that may be taken back."""
        st, lo, hi = self._store, self._lo, self._hi
        trial = st.trial
        return (trial is not None and (trial.lo, trial.hi) == (lo, hi)) or st.grouped(lo, hi) is not None

    def begin_rows(self, layer_idx: int, M: int) -> tuple["_Step", _Sharing, tuple[Tensor, int] | None]:
        """:meth:`begin_step` for ``M`` positions of every sequence of a cache that :meth:`shares`, with what they share and where
        their states go."""
        st, lo, hi = self._store, self._lo, self._hi
        layer = st.layers[layer_idx]
        self._begin(layer, M)
        with self.writing(layer_idx):
            at = _Step(layer.pool, st.table[lo:hi], st.start[lo:hi], st.end[lo:hi], _Last(*(t[lo:hi] for t in layer.last)), None,
                       self.seq_len)
            return at, self._sharing(), self._rows(layer_idx)

    # -------------------------------------------------------------------------------------------- branches and drafts
    def _settled(self, what: str) -> None:
        """A call between whole passes of a cache that is not tracked."""
        st = self._store
        st.undo()
        if st.track:
            raise ValueError(f"SISAPagedCache.{what}: a cache with track=True accumulates weights, which cannot be shared or taken "
                             f"back")
        if st.trial is not None and self._lo < st.trial.hi and st.trial.lo < self._hi:
            raise RuntimeError(f"SISAPagedCache.{what}: keep() the tentative positions first")
        for layer in st.layers.values():
            if layer.filled[self._lo:self._hi] != self.lengths:
                raise RuntimeError(f"SISAPagedCache.{what}: a forward pass has not reached every layer")

    def branch(self, n: int) -> None:
        """Continue every prompt ``n`` times. The first ``len(self) // n`` of these sequences hold the prompts, the others are
        empty; afterwards sequences ``i n .. i n + n - 1`` continue prompt ``i``. Its whole pages belong to all of them, and are
        read once for all of them by their attention; what lies in a page that is not full is copied."""
        st, lo, hi = self._store, self._lo, self._hi
        self._settled("branch")
        if n < 1 or len(self) % n:
            raise ValueError(f"SISAPagedCache.branch: {len(self)} sequences are not prompts of n = {n} each")
        k = len(self) // n
        lengths = self.lengths
        if not all(lengths[:k]) or any(lengths[k:]):
            raise ValueError(f"SISAPagedCache.branch: the first {k} sequences hold the prompts, the others must be empty; lengths "
                             f"are {lengths}")
        if n == 1:
            return
        S = st.page_size
        whole, old = [m // S for m in lengths[:k]], [st.held[lo + i] for i in range(k)]
        src = [old[i][whole[i]] for i in range(k) if lengths[i] % S for _ in range(n - 1)]
        free = [*st.free, *(page for i in range(lo + k, hi) for page in st.held[i])]       # some that reserve() has taken
        if len(src) > len(free):
            raise RuntimeError(f"SISAPagedCache.branch: {len(src)} pages are needed for the copies of pages that are not full, "
                               f"{len(free)} are free")
        dst = [free.pop() for _ in src]
        states = [[t[lo:lo + k].repeat_interleave(n, 0) for t in layer.last] for layer in st.layers.values()]
        if src:                                            # no sequence holds what is written yet
            a, b = (torch.tensor(x).to(st.table.device) for x in (src, dst))
            for layer in st.layers.values():
                pool = layer.pool
                for t in (pool.k, pool.v, pool.b, pool.g, pool.fgate):
                    t[b] = t[a]
        for layer, state in zip(st.layers.values(), states):
            for t, x in zip(layer.last, state):
                t[lo:hi] = x
        copies, held = iter(dst), []
        for i in range(k):
            for page in old[i][:whole[i]]:
                st.others[page] = st.others.get(page, 0) + n - 1
            held.append(old[i])
            held += [old[i][:whole[i]] + ([next(copies)] if lengths[i] % S else []) for _ in range(n - 1)]
        st.free[:], st.held[lo:hi] = free, held
        ends = [m for m in lengths[:k] for _ in range(n)]
        st.starts[lo:hi], st.lengths[lo:hi] = list(ends), list(ends)
        for i in range(k):
            st.families += 1
            st.family[lo + i * n:lo + i * n + n] = [(st.families, whole[i])] * n
        st.sharing.clear()
        for layer in st.layers.values():
            layer.filled[lo:hi] = list(ends)
        st.expected[lo:hi] = [None] * len(self)
        st.end[lo:hi].copy_(torch.tensor(ends, dtype=torch.int32))
        st.show(range(lo, hi))

    def tentative(self, positions: int) -> None:
        """The next passes, of up to ``positions`` positions of every sequence, are proposals, of which :meth:`keep` says what
        stays. They take all of these sequences together; :meth:`release` of any of them ends the trial, and what the others have
        taken stays."""
        self._settled("tentative")
        if positions < 1:
            raise ValueError(f"SISAPagedCache.tentative: positions = {positions} must be positive")
        if not all(self.lengths):
            raise ValueError("SISAPagedCache.tentative: an empty sequence has nothing to go back to")
        if self._store.trial is not None:
            raise RuntimeError("SISAPagedCache.tentative: other sequences' positions are tentative; keep() them first")
        self._store.trial = _Trial(self._lo, self._hi, positions, self.lengths)

    def keep(self, counts: Sequence[int]) -> None:
        """Keep the first ``counts[n]`` positions of every sequence since :meth:`tentative`, and go on from there."""
        st, lo, hi = self._store, self._lo, self._hi
        st.undo()
        trial, counts = st.trial, [int(c) for c in counts]
        if trial is None or (trial.lo, trial.hi) != (lo, hi):
            raise RuntimeError("SISAPagedCache.keep: tentative() comes first, for the same sequences")
        added = self.lengths[0] - trial.starts[0]
        if len(counts) != len(self) or any(not 0 <= c <= added for c in counts):
            raise ValueError(f"SISAPagedCache.keep: {counts}: for each of the {len(self)} sequences 0 .. {added} positions")
        for layer in st.layers.values():
            if layer.filled[lo:hi] != self.lengths:
                raise RuntimeError("SISAPagedCache.keep: a forward pass has not reached every layer; release() the sequences")
        if min(counts) < added:
            ends = [n + c for n, c in zip(trial.starts, counts)]
            row = torch.arange(len(self), device=st.table.device)
            at = torch.tensor(counts).to(st.table.device)
            for i, layer in st.layers.items():
                state = trial.rows[i][row, :, at]
                for t, x in zip(layer.last, (state[..., 0:1], state[..., 1:2], state[..., 2:])):
                    t[lo:hi] = x
            st.end[lo:hi].copy_(torch.tensor(ends, dtype=torch.int32))
            st.starts[lo:hi], st.lengths[lo:hi] = list(ends), list(ends)
            for layer in st.layers.values():
                layer.filled[lo:hi] = list(ends)
        st.trial = None

    # -------------------------------------------------------------------------------------------- memory
    def reserve(self, positions: int) -> None:
        """Take the pages that ``positions`` more positions of every sequence need now, not as they come."""
        st = self._store
        st.undo()
        ends = [min(n + positions, st.max_length) for n in self.lengths]
        if st.take(self._lo, ends) and st.table is not None:
            st.show(range(self._lo, self._hi))

    def release(self) -> None:
        """Empty these sequences: their pages are free for others."""
        st, lo, hi = self._store, self._lo, self._hi
        st.undo()
        for n in range(lo, hi):
            st.give(reversed(st.held[n]))
            st.held[n] = []
        st.family[lo:hi] = [None] * len(self)
        st.sharing.clear()
        if st.trial is not None and lo < st.trial.hi and st.trial.lo < hi:
            st.trial = None
        st.starts[lo:hi] = st.lengths[lo:hi] = [0] * (hi - lo)
        for layer in st.layers.values():
            layer.filled[lo:hi] = [0] * (hi - lo)
            if layer.weights is not None:
                layer.weights[lo:hi].zero_()
        if st.table is not None:
            st.table[lo:hi].fill_(-1)
            st.end[lo:hi].zero_()
        st.expected[lo:hi] = [None] * len(self)

    def evict(self, keep: int, recent: int) -> None:
        """Cut every sequence down to ``keep`` positions per layer and head: its last ``recent`` ones and, of the others,
        those that have received the largest weight (each head its own). Sequences of at most ``keep`` are left alone. The
        kept rows move to other pages, of which there must be enough for one sequence."""
        st = self._store
        st.undo()
        if not st.track:
            raise ValueError("SISAPagedCache.evict needs a cache made with track=True")
        if not 1 <= recent <= keep:
            raise ValueError(f"SISAPagedCache.evict: recent = {recent} must be in 1 .. keep = {keep}")
        for layer in st.layers.values():
            if layer.filled[self._lo:self._hi] != self.lengths:
                raise RuntimeError("SISAPagedCache.evict: a forward pass has not reached every layer")
        long = [n for n in range(self._lo, self._hi) if st.lengths[n] > keep]
        each = -(-keep // st.page_size)
        while long:
            # neighbours together, as many as there are free pages for
            run = 1
            while run < len(long) and long[run] == long[0] + run and (run + 1) * each <= len(st.free):
                run += 1
            self._evict_run(long[0], long[0] + run, keep, recent, each)
            long = long[run:]

    def _evict_run(self, lo: int, hi: int, keep: int, recent: int, each: int) -> None:
        st = self._store
        if (hi - lo) * each > len(st.free):
            raise RuntimeError(f"SISAPagedCache.evict: {each} free pages are needed for a sequence's kept rows, "
                               f"{len(st.free)} are there")
        new = [[st.free.pop() for _ in range(each)] for _ in range(lo, hi)]
        table, lengths, max_len, kept = st.table[lo:hi], st.end[lo:hi], max(st.lengths[lo:hi]), []
        try:                                               # the old pages and weights stay until every layer has its new ones
            new_table = torch.tensor(new, dtype=torch.int32).to(table.device)
            for layer in st.layers.values():
                w = layer.weights[lo:hi]
                if isinstance(layer.pool, _Pages):
                    kept.append(_evict(layer.pool, table, lengths, w, keep, recent, new_table, max_len)[1])
                else:
                    from .kernels.paged import sisa_cache_evict_hip

                    kept.append(sisa_cache_evict_hip(layer.pool, table, lengths, w, keep, recent, layer.pool, new_table,
                                                     max_len=max_len).weights)
        except BaseException:
            st.free += [page for pages in reversed(new) for page in reversed(pages)]
            raise
        for layer, w in zip(st.layers.values(), kept):
            layer.weights[lo:hi, :, :keep] = w
            layer.weights[lo:hi, :, keep:max_len].zero_()
            layer.filled[lo:hi] = [keep] * (hi - lo)
        for n, pages in zip(range(lo, hi), new):
            st.free += reversed(st.held[n])
            st.held[n], st.starts[n], st.lengths[n] = pages, keep, keep
        st.show(range(lo, hi))
        st.end[lo:hi].fill_(keep)


def takes_kernels(k: Tensor, b: Tensor) -> bool:
    """Whether the paged kernels are built for these rows."""
    return (k.shape[-1], b.shape[-1]) == (HIP_D_HEAD, HIP_D_STATE) and k.dtype in (torch.bfloat16, torch.float16, torch.float32)
