"""The cache operators of generation, as cases that a timing program can run and check against a plain form.

A generation cache in pages: ``k, v`` ``(P, H, S, 64)`` and ``b`` ``(P, H, S, 32)`` in the compute dtype, ``g, f``
``(P, H, S)`` in float32; position ``j`` of sequence ``n`` lives in slot ``j % S`` of page ``table[n, j // S]``. A case is
a dict of plain values; its ``"kind"`` names the operator:

* ``write``   -- new positions of every sequence into the pages: position ``start[n] + m`` for ``m < count[n]``;
* ``decode``  -- one new token per sequence against its cached positions, ``s_j = q.k_j / 8 + lam exp(g - g_j) (c.b_j) +
                 (F - F_j)``, ``out = softmax(s) v``; with ``tracked``, the token's softmax weights are added to every
                 position's accumulated weight;
* ``weights`` -- what each position of a prompt has received: the sum, over the last ``window`` queries of the sequence
                 (0: all of them), of the softmax weights that they give it;
* ``evict``   -- a cache cut down to ``keep`` positions per head: the last ``recent`` ones and, of the others, those of
                 the largest accumulated weight (ties: the lowest position), copied in order to other pages.

Head size 64 and state size 32 throughout (the only ones the kernels take); head counts are those of the presets in
``sisa_amd/config.py``; gates are distributed as in ``sisa_amd/workloads.py`` at its long-context configuration.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
D_HEAD, D_STATE = 64, 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # a step of continuous batching: the new position of 48 sequences, each at a length of its own
        dict(name="write_48x1_h12", kind="write", B=48, H=12, M=1, shortest=1, longest=4000, S=64, dtype="bf16"),
        # a right-padded batch of prompts filling an empty cache
        dict(name="write_6x1500_h16_fp16", kind="write", B=6, H=16, M=1500, shortest=0, longest=0, S=32, dtype="fp16"),
        # one chat's next token after a short exchange: latency
        dict(name="decode_1x900_h8", kind="decode", B=1, H=8, shortest=900, longest=900, S=64, dtype="bf16",
             tracked=False),
        # a served batch of unequal lengths, from a first token to a long document, small pages, heavy positions tracked
        dict(name="decode_24_to_6001_h12_fp16", kind="decode", B=24, H=12, shortest=1, longest=6001, S=16,
             dtype="fp16", tracked=True),
        # the accuracy path: a few sequences of an fp32 model
        dict(name="decode_3x2500_h16_fp32", kind="decode", B=3, H=16, shortest=2500, longest=2500, S=128, dtype="fp32",
             tracked=False),
        # long contexts side by side, tracked for eviction
        dict(name="decode_8x16384_h12", kind="decode", B=8, H=12, shortest=16384, longest=16384, S=64, dtype="bf16",
             tracked=True),
        # a short fp32 prompt, every query counted
        dict(name="weights_2x333_h4_fp32", kind="weights", B=2, H=4, L=333, shortest=200, window=0, dtype="fp32"),
        # a batch of prompts at the training length, every query counted
        dict(name="weights_4x2048_h12", kind="weights", B=4, H=12, L=2048, shortest=2048, window=0, dtype="bf16"),
        # a long prompt judged by its last 64 queries alone
        dict(name="weights_1x16384_h16_fp16", kind="weights", B=1, H=16, L=16384, shortest=16384, window=64,
             dtype="fp16"),
        # one chat's cache back to its budget
        dict(name="evict_1x1100_to_512_h8", kind="evict", B=1, H=8, shortest=1100, longest=1100, keep=512, recent=64,
             S=64, dtype="bf16"),
        # a served batch of unequal lengths, some of them within the budget already
        dict(name="evict_16_to_5003_h16_fp16", kind="evict", B=16, H=16, shortest=40, longest=5003, keep=1000,
             recent=250, S=16, dtype="fp16"),
        # long prompts cut to a quarter before generation begins
        dict(name="evict_8x16384_to_4096_h12", kind="evict", B=8, H=12, shortest=16384, longest=16384, keep=4096,
             recent=1024, S=64, dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["write", "decode", "decode", "weights", "weights", "evict"])
    H, S, dtype = rng.choice([4, 8, 12, 16]), rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    es = BYTES[dtype]
    B = _log_int(rng, 1, 48)
    if kind == "write":
        if rng.random() < 0.5:
            longest = _log_int(rng, 1, 4000)
            return dict(kind=kind, B=B, H=H, M=1, shortest=max(1, longest // rng.choice([1, 3, 50])), longest=longest,
                        S=S, dtype=dtype)
        M = _log_int(rng, 2, max(2, min(4000, 6 * 1500 * 16 * 2 // (B * H * es))))
        longest = rng.choice([0, rng.randint(1, 900)])
        return dict(kind=kind, B=B, H=H, M=M, shortest=0, longest=longest, S=S, dtype=dtype)
    if kind == "weights":
        window = rng.choice([0, 0, rng.randint(1, 300)])
        L = _log_int(rng, 1, 700 if dtype == "fp32" else 4096 if not window else 16384)
        room = 48 * 2048 ** 2 // (H * L * L) if not window else 16 * 16384 * 64 // (H * L * min(L, window))
        B = _log_int(rng, 1, max(1, min(24, room)))
        return dict(kind=kind, B=B, H=H, L=L, shortest=max(1, L // rng.choice([1, 1, 2, 20])), window=window, dtype=dtype)
    longest = _log_int(rng, 1, max(1, min(16384, 8 * 16384 * 12 * 2 // (B * H * es))))
    shortest = max(1, longest // rng.choice([1, 1, 4, 50]))
    if kind == "decode":
        return dict(kind=kind, B=B, H=H, shortest=shortest, longest=longest, S=S, dtype=dtype,
                    tracked=rng.random() < 0.6)
    keep = max(1, min(4096, int(longest * rng.uniform(0.05, 0.8))))
    return dict(kind=kind, B=B, H=H, shortest=shortest, longest=longest, keep=keep,
                recent=max(1, int(keep * rng.uniform(0.02, 0.6))), S=S, dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def _spread(shortest: int, longest: int, n: int) -> list[int]:
    """``n`` lengths from ``longest`` down to ``shortest``, even over their logarithm."""
    if n == 1 or shortest == longest:
        return [longest] * n
    lo, hi = math.log(max(shortest, 1)), math.log(max(longest, 1))
    out = [round(math.exp(hi + (lo - hi) * i / (n - 1))) for i in range(n)]
    return [longest] + out[1:-1] + [shortest]


def _lengths(case: dict) -> list[int]:
    """Cached positions of every sequence (of the prompt, for ``weights``), before a ``write``'s own."""
    if case["kind"] == "weights":
        return _spread(case["shortest"], case["L"], case["B"])
    return _spread(case["shortest"], case["longest"], case["B"])


def _counts(case: dict) -> list[int]:
    """New positions of every sequence in a ``write``: all of ``M``, or down to a third of it in a padded batch."""
    return _spread(max(1, case["M"] // 3), case["M"], case["B"])


def _gates(gen, B: int, H: int, N: int):
    """Cumulative log-decay and log-forget values: steps -softplus(N(-7, 1)) and logsigmoid(N(6, 1))."""
    g = -torch.nn.functional.softplus(torch.randn(B, H, N, generator=gen, device=DEVICE) - 7.0)
    f = -torch.nn.functional.softplus(torch.randn(B, H, N, generator=gen, device=DEVICE) - 6.0)
    return g.cumsum(2), f.cumsum(2)


def _pages(gen, n: int, H: int, S: int, dt) -> dict:
    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=dt)
    return dict(k=normal(n, H, S, D_HEAD), v=normal(n, H, S, D_HEAD), b=normal(n, H, S, D_STATE),
                g=-torch.rand(n, H, S, generator=gen, device=DEVICE),
                f=-torch.rand(n, H, S, generator=gen, device=DEVICE))


def _table(gen, pages: list[int], spare: int) -> tuple[torch.Tensor, int]:
    """A table in which every sequence has its own pages, in no order, -1 behind its last; and how many pages there are."""
    total, width = sum(pages) + spare, max(1, max(pages))
    order = torch.randperm(total, generator=gen, device=DEVICE)[:sum(pages)].to(torch.int32)
    has = torch.tensor(pages, device=DEVICE)[:, None] > torch.arange(width, device=DEVICE)
    table = torch.full((len(pages), width), -1, device=DEVICE, dtype=torch.int32)
    table[has] = order
    return table, total


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, B, H, dt = case["kind"], case["B"], case["H"], DTYPES[case["dtype"]]
    ints = dict(device=DEVICE, dtype=torch.int32)
    state = dict(case=case, lam=torch.full((H,), math.log1p(math.exp(-1.0)), device=DEVICE))
    lengths = _lengths(case)
    if kind == "weights":
        L = case["L"]

        def heads(width):          # (B, L, H, width) in memory, as a projection leaves them
            return torch.randn(B, L, H, width, generator=gen, device=DEVICE, dtype=dt).transpose(1, 2)
        g, f = _gates(gen, B, H, L)
        return state | dict(q=heads(D_HEAD), k=heads(D_HEAD), c=heads(D_STATE), b=heads(D_STATE), g=g, f=f,
                            lengths=torch.tensor(lengths, **ints))
    S = case["S"]
    counts = _counts(case) if kind == "write" else [0] * B
    held = [-(-(n + m) // S) for n, m in zip(lengths, counts)]
    table, total = _table(gen, held, 3)
    state |= dict(table=table, lengths=torch.tensor(lengths, **ints), pages=_pages(gen, total, H, S, dt))
    if kind == "write":
        M = case["M"]

        def rows(width):
            return torch.randn(B, M, H, width, generator=gen, device=DEVICE, dtype=dt).transpose(1, 2)
        g, f = _gates(gen, B, H, M)
        return state | dict(k=rows(D_HEAD), v=rows(D_HEAD), b=rows(D_STATE), g=g, f=f, counts=torch.tensor(counts, **ints))
    # the gates of a sequence fall along its positions, wherever its pages are
    N = table.shape[1] * S
    g, f = _gates(gen, B, H, N)
    has = table >= 0
    for name, x in (("g", g), ("f", f)):
        state["pages"][name][table[has].long()] = x.unflatten(2, (-1, S)).transpose(1, 2)[has]
    longest = case["longest"]
    if kind == "decode" and not case["tracked"]:
        state |= dict(old=None, new=None)
    else:                           # accumulated weights: a few heavy positions, many light ones
        state |= dict(old=torch.exp(2.0 * torch.randn(B, H, longest, generator=gen, device=DEVICE)),
                      new=torch.zeros(B, H, longest, device=DEVICE))
    if kind == "decode":
        def rows(width):
            return torch.randn(B, 1, H, width, generator=gen, device=DEVICE, dtype=dt).transpose(1, 2)
        last = (state["lengths"].long() - 1)[:, None, None].expand(B, H, 1)
        return state | dict(q=rows(D_HEAD), c=rows(D_STATE), g=g.gather(2, last), f=f.gather(2, last))
    state["to"], total = _table(gen, [-(-min(n, case["keep"]) // S) for n in lengths], 2)
    return state | dict(into={n: torch.zeros(total, *x.shape[1:], device=DEVICE, dtype=x.dtype)
                              for n, x in state["pages"].items()})


# ------------------------------------------------------------------------------------------------ one pass
def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        return {"write": _own_write, "decode": _own_decode, "weights": _own_weights, "evict": _own_evict}[kind](state)
    return {"write": _write, "decode": _decode, "weights": _weights, "evict": _evict}[kind](state)


def _pool(state: dict, which: str = "pages"):
    """The handle of a cache's pages, made when a program makes the cache."""
    held = state.get("pool of " + which)
    if held is None:
        from sisa_amd.kernels.paged import PagePool

        p = state[which]
        held = state["pool of " + which] = PagePool(p["k"], p["v"], p["b"], p["g"], p["f"])
    return held


def _own_write(s):
    from sisa_amd.kernels.paged import sisa_paged_write_hip

    sisa_paged_write_hip(_pool(s), s["table"], s["lengths"], s["k"], s["v"], s["b"], s["g"], s["f"], s["counts"])
    return s["pages"]


def _own_decode(s):
    from sisa_amd.kernels.paged import sisa_paged_decode_hip

    out = sisa_paged_decode_hip(s["q"], s["c"], s["g"], s["f"], s["lam"], _pool(s), s["table"], s["lengths"],
                                max_len=s["case"]["longest"], weights=s["old"], weights_out=s["new"])
    return dict(out=out, weights=s["new"])


def _own_weights(s):
    from sisa_amd.kernels.weights import sisa_attention_weights_hip

    return sisa_attention_weights_hip(s["q"], s["k"], s["c"], s["b"], s["g"], s["lam"], s["f"], lengths=s["lengths"],
                                      window=s["case"]["window"] or None)


def _own_evict(s):
    from sisa_amd.kernels.paged import sisa_cache_evict_hip

    case = s["case"]
    got = sisa_cache_evict_hip(_pool(s), s["table"], s["lengths"], s["old"], case["keep"], case["recent"],
                               _pool(s, "into"), s["to"], max_len=case["longest"])
    return dict(lengths=got.lengths, weights=got.weights, positions=got.positions, pages=s["into"])


# ------------------------------------------------------------------------------------------------ the plain forms
def _rows_of(x, table):
    """The pages of a table side by side: (P, H, S, .) -> (B, H, W S, .)."""
    return x[table.long().clamp(min=0)].transpose(1, 2).flatten(2, 3)


def _write(s):
    S, M = s["case"]["S"], s["case"]["M"]
    m = torch.arange(M, device=DEVICE)
    pos = s["lengths"].long()[:, None] + m
    new = m < s["counts"][:, None]
    page = s["table"].long().gather(1, (pos // S).clamp(max=s["table"].shape[1] - 1))[new]
    slot = (pos % S)[new]
    p = s["pages"]
    p["k"][page, :, slot] = s["k"].transpose(1, 2)[new]
    p["v"][page, :, slot] = s["v"].transpose(1, 2)[new]
    p["b"][page, :, slot] = s["b"].transpose(1, 2)[new]
    p["g"][page, :, slot] = s["g"].transpose(1, 2)[new]
    p["f"][page, :, slot] = s["f"].transpose(1, 2)[new]
    return p


def _decode(s):
    N, n = s["case"]["longest"], s["lengths"].long()
    there = (torch.arange(N, device=DEVICE) < n[:, None])[:, None, None]
    k, v, b, g, f = (_rows_of(s["pages"][x], s["table"])[:, :, :N].float() for x in ("k", "v", "b", "g", "f"))
    decay = torch.exp(s["g"] - torch.where(there[:, :, 0], g, s["g"]))[:, :, None]
    score = (s["q"].float() @ k.mT) / 8.0 + s["lam"][:, None, None] * decay * (s["c"].float() @ b.mT)
    score = torch.where(there, score + (s["f"] - f)[:, :, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    if s["old"] is not None:
        s["new"].copy_(torch.where(there[:, :, 0], s["old"] + p[:, :, 0], s["new"]))
    return dict(out=p @ v, weights=s["new"])


def _weights(s):
    case, n = s["case"], s["lengths"].long()
    L = case["L"]
    W = min(L, case["window"] or L)
    at = n[:, None] - W + torch.arange(W, device=DEVICE)             # the last W queries of each sequence
    real, row = at >= 0, at.clamp(min=0)[:, None].expand(-1, case["H"], -1)
    q = s["q"].gather(2, row[..., None].expand(-1, -1, -1, D_HEAD)).float()
    c = s["c"].gather(2, row[..., None].expand(-1, -1, -1, D_STATE)).float()
    g, f = s["g"].gather(2, row), s["f"].gather(2, row)
    seen = torch.arange(L, device=DEVICE) <= row[..., None]
    decay = torch.exp(torch.where(seen, g[..., None] - s["g"][:, :, None], 0.0))
    score = (q @ s["k"].float().mT) / 8.0 + s["lam"][:, None, None] * decay * (c @ s["b"].float().mT)
    score = torch.where(seen, score + (f[..., None] - s["f"][:, :, None]), float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.where(real[:, None, :, None], p, 0.0).sum(2)


def _evict(s):
    case, n = s["case"], s["lengths"].long()[:, None, None]
    H, S, N, keep = case["H"], case["S"], case["longest"], case["keep"]
    at = torch.arange(N, device=DEVICE).expand(case["B"], H, N)
    rank = torch.where(at >= n - case["recent"], float("inf"), s["old"])
    rank = torch.where(at < n, rank, float("-inf"))
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    K = min(keep, N)
    i = torch.arange(K, device=DEVICE)
    kept = i < n.clamp(max=keep)
    pos = torch.where(kept, order[:, :, :K], N).sort(dim=-1).values
    ok = kept.expand(-1, H, -1)
    at = pos.clamp(max=N - 1)
    page = s["table"].long().clamp(min=0)[:, None].expand(-1, H, -1).gather(2, at // S)
    to = s["to"].long()[:, None, i // S].expand(-1, H, -1)
    head = torch.arange(H, device=DEVICE)[:, None].expand_as(at)
    src, dst = (page[ok], head[ok], (at % S)[ok]), (to[ok], head[ok], (i % S).expand_as(at)[ok])
    p, q = s["pages"], s["into"]
    q["k"][dst], q["v"][dst], q["b"][dst] = p["k"][src], p["v"][src], p["b"][src]
    q["g"][dst], q["f"][dst] = p["g"][src], p["f"][src]
    weights, where = (torch.zeros(case["B"], H, keep, device=DEVICE),
                      torch.full((case["B"], H, keep), -1, device=DEVICE, dtype=torch.int32))
    weights[:, :, :K] = torch.where(ok, s["old"].gather(2, at), 0.0)
    where[:, :, :K] = torch.where(ok, pos, -1).to(torch.int32)
    return dict(lengths=n[:, 0, 0].clamp(max=keep).to(torch.int32), weights=weights, positions=where, pages=q)


# ------------------------------------------------------------------------------------------------ necessary work
def work(case: dict) -> dict:
    """Bytes and floating-point operations of one pass that no implementation can leave out: cached rows, queries and
    accumulated weights read once, rows and weights written once; a prompt's scores formed once."""
    kind, B, H, es = case["kind"], case["B"], case["H"], BYTES[case["dtype"]]
    row, total = 160 * es + 8, sum(_lengths(case))
    if kind == "write":
        return dict(bytes=2.0 * sum(_counts(case)) * H * row, flops=0.0)
    if kind == "decode":
        return dict(bytes=float(H * (total * (row + 8 * case["tracked"]) + B * (96 * es + 8 + 256))),
                    flops=320.0 * H * total)
    if kind == "weights":
        pairs = rows = 0
        for n in _lengths(case):
            w = min(n, case["window"] or n)
            pairs, rows = pairs + w * n - w * (w - 1) // 2, rows + w
        return dict(bytes=float(H * (total * (96 * es + 8) + rows * (96 * es + 8) + 4 * B * case["L"])),
                    flops=192.0 * H * pairs)
    kept = sum(min(n, case["keep"]) for n in _lengths(case))
    return dict(bytes=float(H * (4 * total + kept * (2 * row + 4) + 4 * B * case["keep"])), flops=0.0)


# ------------------------------------------------------------------------------------------------ 64-bit results
def exact(case: dict, seed: int):
    """What ``run`` returns, by the definitions in 64 bits, one sequence after the other."""
    s = prepare(case, seed)
    return {"write": _exact_write, "decode": _exact_decode, "weights": _exact_weights, "evict": _exact_evict}[
        case["kind"]](s, case)


def _places(s, n, first, last):
    """Pages and slots of the positions first .. last - 1 of sequence n."""
    pos = torch.arange(first, last, device=DEVICE)
    S = s["case"]["S"]
    return s["table"][n].long()[torch.div(pos, S, rounding_mode="floor")], pos.remainder(S)


def _exact_write(s, case):
    out = {name: x.double() for name, x in s["pages"].items()}
    for n in range(case["B"]):
        first, m = int(s["lengths"][n]), int(s["counts"][n])
        page, slot = _places(s, n, first, first + m)
        for name in out:
            out[name][page, :, slot] = s[name][n, :, :m].double().transpose(0, 1)
    return out


def _exact_decode(s, case):
    outs, new = [], None if s["new"] is None else s["new"].double()
    lam = s["lam"].double()[:, None]
    for n in range(case["B"]):
        N = int(s["lengths"][n])
        page, slot = _places(s, n, 0, N)
        k, v, b, g, f = (s["pages"][x][page, :, slot].double().transpose(0, 1) for x in ("k", "v", "b", "g", "f"))
        x = (k * s["q"][n].double()).sum(-1) * D_HEAD ** -0.5
        x = x + lam * (s["g"][n].double() - g).exp() * (b * s["c"][n].double()).sum(-1) + s["f"][n].double() - f
        p = (x - x.logsumexp(-1, keepdim=True)).exp()
        outs.append((p[..., None] * v).sum(1, keepdim=True))
        if new is not None:
            new[n, :, :N] = s["old"][n, :, :N].double() + p
    return dict(out=torch.stack(outs), weights=new)


def _exact_weights(s, case):
    L = case["L"]
    out = torch.zeros(case["B"], case["H"], L, device=DEVICE, dtype=torch.float64)
    for n in range(case["B"]):
        N = int(s["lengths"][n])
        first = max(0, N - (case["window"] or N))
        hidden = torch.ones(N - first, N, dtype=torch.bool, device=DEVICE).triu(first + 1)
        for h in range(case["H"]):
            q, c, g, f = (s[x][n, h, first:N].double() for x in ("q", "c", "g", "f"))
            k, b, gk, fk = (s[x][n, h, :N].double() for x in ("k", "b", "g", "f"))
            decay = (g[:, None] - gk[None, :]).masked_fill(hidden, 0.0).exp()
            x = q @ k.T * D_HEAD ** -0.5 + s["lam"][h].double() * decay * (c @ b.T) + f[:, None] - fk[None, :]
            out[n, h, :N] = x.masked_fill(hidden, -math.inf).softmax(-1).sum(0)
    return out


def _exact_evict(s, case):
    B, H, keep, recent = case["B"], case["H"], case["keep"], case["recent"]
    where = torch.full((B, H, keep), -1, device=DEVICE, dtype=torch.int32)
    weights = torch.zeros(B, H, keep, device=DEVICE, dtype=torch.float64)
    into = {name: x.double() for name, x in s["into"].items()}
    lengths = []
    for n in range(B):
        N = int(s["lengths"][n])
        lengths.append(min(N, keep))
        if N <= keep:
            chosen = torch.arange(N, device=DEVICE).expand(H, N)
        else:
            light = torch.argsort(s["old"][n, :, :N - recent].double(), dim=1, descending=True, stable=True)
            newest = torch.arange(N - recent, N, device=DEVICE).expand(H, recent)
            chosen = torch.cat([light[:, :keep - recent], newest], 1).sort(1).values
        K = chosen.shape[1]
        where[n, :, :K] = chosen.to(torch.int32)
        weights[n, :, :K] = s["old"][n].double().gather(1, chosen)
        page, slot = _places(s, n, 0, N)
        i = torch.arange(K, device=DEVICE)
        to = s["to"][n].long()[torch.div(i, case["S"], rounding_mode="floor")]
        for name in into:
            for h in range(H):
                into[name][to, h, i.remainder(case["S"])] = s["pages"][name][page[chosen[h]], h, slot[chosen[h]]].double()
    return dict(lengths=torch.tensor(lengths, device=DEVICE, dtype=torch.int32), weights=weights, positions=where,
                pages=into)
