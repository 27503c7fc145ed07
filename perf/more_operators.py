"""Operators of branched and drafted generation, as cases that a timing program can run and check against a plain form.

A generation cache in pages: ``k, v`` ``(P, H, S, 64)`` and ``b`` ``(P, H, S, 32)`` in the compute dtype, ``g, f``
``(P, H, S)`` in float32; position ``j`` of sequence ``n`` lives in slot ``j % S`` of page ``table[n, j // S]``. A case is
a dict of plain values; its ``"kind"`` names the operator:

* ``attend`` -- the last ``M`` positions of every sequence against the positions up to their own,
                ``s_mj = q_m.k_j / 8 + lam exp(g_m - g_j) (c_m.b_j) + (F_m - F_j)``, ``out_m = softmax_j(s_mj) v_j``.
                The sequences form groups of neighbours, of ``smallest`` to ``largest``; those of group ``r`` have their
                first ``shared[r]`` positions in common, which is what the operator reads once for all of them;
* ``verify`` -- tokens that a draft proposed against the target's probabilities, with given random numbers: draft ``i`` is
                accepted while ``u_i q_i(x_i) < p_i(x_i)``, the first token behind the accepted ones is drawn with the last
                random number from ``max(p - q, 0)`` at the position of the refused draft, or from ``p`` behind the last one.

Head size 64 and state size 32 throughout (the only ones the kernels take); head counts and the vocabulary are those of
the presets in ``sisa_amd/config.py``; gates are distributed as in ``sisa_amd/workloads.py`` at its long-context
configuration.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
D_HEAD, D_STATE = 64, 32
VOCAB = 50277
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------ the cases
def _attend(name, groups, smallest, largest, M, H, S, dtype, shared, suffix):
    """``shared`` and ``suffix``: the least and the most common positions of a group, and own positions of a sequence (the
    ``M`` new ones included)."""
    return dict(name=name, kind="attend", groups=groups, smallest=smallest, largest=largest, M=M, H=H, S=S, dtype=dtype,
                shared_least=shared[0], shared_most=shared[1], suffix_least=suffix[0], suffix_most=suffix[1])


def listed() -> list[dict]:
    return [
        # four answers to one short question, a few tokens in: latency
        _attend("attend_4_of_600_h8", 1, 4, 4, 1, 8, 64, "bf16", (600, 600), (9, 9)),
        # the best of sixteen: one prompt, sixteen answers of unequal lengths
        _attend("attend_16_of_2000_h12", 1, 16, 16, 1, 12, 64, "bf16", (2000, 2000), (30, 500)),
        # many questions about one long document
        _attend("attend_64_of_16384_h12", 1, 64, 64, 1, 12, 64, "bf16", (16384, 16384), (20, 700)),
        # one system prompt in front of a large served batch
        _attend("attend_256_of_1500_h12", 1, 256, 256, 1, 12, 64, "bf16", (1500, 1500), (1, 1000)),
        # a served batch in which requests ask for unequal numbers of answers, some with nothing in common, small pages
        _attend("attend_9_groups_h16_fp16", 9, 1, 24, 1, 16, 16, "fp16", (0, 3001), (1, 333)),
        # four drafted tokens and the one before them, one chat: all earlier positions are read once for the five
        _attend("attend_5_drafts_of_3000_h16", 1, 1, 1, 5, 16, 64, "bf16", (3000, 3000), (5, 5)),
        # drafts of a served batch, unequal lengths
        _attend("attend_24x8_drafts_h12_fp16", 24, 1, 1, 8, 12, 32, "fp16", (200, 6000), (8, 8)),
        # several answers to each of four prompts, drafted: both at once
        _attend("attend_4x8x4_drafts_h12", 4, 8, 8, 4, 12, 64, "bf16", (1000, 4000), (4, 900)),
        # the accuracy path: a few branches of an fp32 model
        _attend("attend_2_groups_h16_fp32", 2, 3, 6, 2, 16, 128, "fp32", (2400, 2500), (2, 77)),
        # one chat's drafts: latency
        dict(name="verify_1x4", kind="verify", B=1, K=4, V=VOCAB, dtype="fp32", top_k=0, proposal=True, ragged=False),
        # a served batch, unequal numbers of drafts, probabilities of the 50 likeliest tokens
        dict(name="verify_64x7_top50", kind="verify", B=64, K=7, V=VOCAB, dtype="fp32", top_k=50, proposal=True, ragged=True),
        # drafts looked up in the text, which have no probabilities of their own, against 16-bit ones
        dict(name="verify_200x3_bf16", kind="verify", B=200, K=3, V=VOCAB, dtype="bf16", top_k=0, proposal=False,
             ragged=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    if rng.random() < 0.3:
        B, K, V = _log_int(rng, 1, 200), rng.randint(1, 10), _log_int(rng, 1000, 131072)
        while B * (K + 1) * V > 200 * 4 * VOCAB:
            B = max(1, B // 2)
        return dict(kind="verify", B=B, K=K, V=V, dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    top_k=rng.choice([0, 0, 20, 200]), proposal=rng.random() < 0.7, ragged=rng.random() < 0.5)
    H, S, dtype = rng.choice([4, 8, 12, 16]), rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    M = rng.choice([1, 1, 1, 2, 3, rng.randint(4, 12)])
    groups, largest = _log_int(rng, 1, 24), _log_int(rng, 1, 128)
    smallest = max(1, largest // rng.choice([1, 1, 2, 10]))
    shared_most = rng.choice([0, *[_log_int(rng, 16, 16384)] * 9])
    suffix_most = M + _log_int(rng, 1, 1500) - 1
    # at most the largest listed cases' scores, and their rows
    size = DTYPES[dtype].itemsize / 2
    while (groups * largest * M * (shared_most + suffix_most) * H * size > 64 * 17000 * 12
           or (groups * shared_most + groups * largest * suffix_most) * H * size > 4.5e5):
        if groups > 1:
            groups = max(1, groups // 2)
        elif largest > 16:
            largest, smallest = largest // 2, max(1, smallest // 2)
        else:
            shared_most, suffix_most = shared_most // 2, max(M, suffix_most // 2)
    return dict(kind="attend", groups=groups, smallest=min(smallest, largest), largest=largest, M=M, H=H, S=S, dtype=dtype,
                shared_least=shared_most // rng.choice([1, 1, 3, 20]), shared_most=shared_most,
                suffix_least=max(M, suffix_most // rng.choice([1, 2, 30])), suffix_most=suffix_most)


# ------------------------------------------------------------------------------------------------ inputs
def _spread(least: int, most: int, n: int) -> list[int]:
    """``n`` integers from ``most`` down to ``least``, even over their logarithm."""
    if n == 1 or least == most:
        return [most] * n
    lo, hi = math.log(max(least, 1)), math.log(max(most, 1))
    out = [round(math.exp(hi + (lo - hi) * i / (n - 1))) for i in range(n)]
    return [most] + out[1:-1] + [least]


def _sizes(case: dict) -> list[int]:
    """Sequences of every group."""
    return _spread(case["smallest"], case["largest"], case["groups"])[::-1]


def _shared(case: dict) -> list[int]:
    """Positions that a group's sequences have in common."""
    return _spread(case["shared_least"], case["shared_most"], case["groups"])


def _suffixes(case: dict) -> list[int]:
    """Own positions of every sequence."""
    return _spread(case["suffix_least"], case["suffix_most"], sum(_sizes(case)))


def _counts(case: dict) -> list[int]:
    """How many drafts every row has: ``K``, or from ``K`` down to none."""
    return [case["K"] - n % (case["K"] + 1) if case["ragged"] else case["K"] for n in range(case["B"])]


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return dict(case=case) | (_prepare_attend if case["kind"] == "attend" else _prepare_verify)(case, gen)


def _prepare_attend(case: dict, gen) -> dict:
    H, S, M, dt = case["H"], case["S"], case["M"], DTYPES[case["dtype"]]
    sizes, shared, suffix = _sizes(case), _shared(case), _suffixes(case)
    group = [r for r, size in enumerate(sizes) for _ in range(size)]
    B, lengths = len(group), [shared[r] + suffix[n] for n, r in enumerate(group)]
    # whole pages of a group's common positions belong to all of its sequences; every other page to one
    whole = [n // S for n in shared]
    own_pages = [-(-lengths[n] // S) - whole[r] for n, r in enumerate(group)]
    total, width = sum(whole) + sum(own_pages) + 3, max(1, max(-(-n // S) for n in lengths))
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32).cpu()
    common, at, rows = [], 0, []
    for n in whole:
        common.append(order[at:at + n])
        at += n
    for n, r in enumerate(group):
        row = torch.cat([common[r], order[at:at + own_pages[n]]])
        rows.append(torch.nn.functional.pad(row, (0, width - len(row)), value=-1))
        at += own_pages[n]
    table = torch.stack(rows).to(DEVICE)

    def normal(*shape, dtype=dt):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)
    pages = dict(k=normal(total, H, S, D_HEAD), v=normal(total, H, S, D_HEAD), b=normal(total, H, S, D_STATE),
                 g=normal(total, H, S, dtype=torch.float32), f=normal(total, H, S, dtype=torch.float32))
    grp, length, common_n = (torch.tensor(x, device=DEVICE) for x in (group, lengths, shared))
    N, Ns = max(lengths), max(max(shared), 1)
    # gates fall along a sequence: steps -softplus(N(-7, 1)) and -softplus(N(-6, 1)); a group's common ones are the same
    pos = torch.arange(N, device=DEVICE).expand(B, N)
    in_common = pos < common_n[grp][:, None]
    last = {}
    for name, mean in (("g", -7.0), ("f", -6.0)):
        step = -torch.nn.functional.softplus(normal(B, H, N, dtype=torch.float32) + mean)
        first = -torch.nn.functional.softplus(normal(len(sizes), H, Ns, dtype=torch.float32) + mean)
        step[:, :, :Ns] = torch.where(in_common[:, None, :Ns], first[grp][:, :, :N], step[:, :, :Ns])
        x = step.double().cumsum(2).float()
        there = pos < length[:, None]
        page = table.long().clamp(min=0).gather(1, pos // S)[there]
        pages[name][page, :, (pos % S)[there]] = x.transpose(1, 2)[there]
        last[name] = x.gather(2, (length[:, None, None] - M + torch.arange(M, device=DEVICE)).expand(B, H, M))
    # the position behind a group's whole pages is each sequence's own copy, up to the end of what is common
    for r, n in enumerate(shared):
        first = group.index(r)
        if n % S and sizes[r] > 1:
            to = table[first + 1:first + sizes[r], whole[r]].long()
            for name in pages:
                pages[name][to, :, :n % S] = pages[name][table[first, whole[r]].long(), :, :n % S]

    def rows_of(width_):                                  # as a projection leaves them
        return normal(B, M, H, width_).transpose(1, 2)
    ints = dict(device=DEVICE, dtype=torch.int32)
    return dict(table=table, lengths=torch.tensor(lengths, **ints), shared=torch.tensor(shared, **ints), pages=pages,
                sizes=sizes, longest=max(lengths), common=max(shared), q=rows_of(D_HEAD), c=rows_of(D_STATE), g=last["g"],
                f=last["f"], lam=torch.full((H,), math.log1p(math.exp(-1.0)), device=DEVICE))


def _prepare_verify(case: dict, gen) -> dict:
    B, K, V, dt = case["B"], case["K"], case["V"], DTYPES[case["dtype"]]
    target = 3.0 * torch.randn(B, K + 1, V, generator=gen, device=DEVICE)
    draft = target[:, :K] + torch.randn(B, K, V, generator=gen, device=DEVICE)

    def probabilities(logits):
        if case["top_k"]:
            least = logits.topk(case["top_k"], dim=-1).values[..., -1:]
            logits = logits.masked_fill(logits < least, float("-inf"))
        return logits.softmax(-1)
    p, q = probabilities(target), probabilities(draft)
    drafts = torch.multinomial(q.flatten(0, 1), 1, generator=gen).view(B, K)
    counts = torch.tensor(_counts(case), device=DEVICE, dtype=torch.int32) if case["ragged"] else None
    return dict(p=p.to(dt), q=q.to(dt) if case["proposal"] else None, drafts=drafts, counts=counts,
                u=torch.rand(B, K + 1, generator=gen, device=DEVICE))


# ------------------------------------------------------------------------------------------------ one pass
def run(state: dict):
    if state["case"]["kind"] == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    return _own_verify(state) if own else _plain_verify(state)


def _own_attend(s):
    from sisa_amd.kernels.paged import PagePool
    from sisa_amd.kernels.prefix import PrefixGroups, sisa_prefix_decode_hip

    if "pool" not in s:                                   # the handles that a program keeps with its cache
        p = s["pages"]
        s["pool"] = PagePool(p["k"], p["v"], p["b"], p["g"], p["f"])
        s["grouped"] = PrefixGroups(s["sizes"], DEVICE)
    return sisa_prefix_decode_hip(s["q"], s["c"], s["g"], s["f"], s["lam"], s["pool"], s["table"], s["lengths"],
                                  s["grouped"], s["shared"], max_len=s["longest"], max_shared=s["common"])


def _own_verify(s):
    from sisa_amd.kernels.verify import sisa_verify_drafts_hip

    got = sisa_verify_drafts_hip(s["p"], s["drafts"], s["u"], s["q"], s["counts"])
    return dict(tokens=got.tokens, accepted=got.accepted)


# ------------------------------------------------------------------------------------------------ the plain forms
def _scores(s, q, c, g, f, k, b, gk, fk, seen):
    """Scores of query rows (.., R, .) against keys (.., N, .) in float32, -inf where they are not seen."""
    lam = s["lam"][:, None, None]
    decay = torch.exp(torch.where(seen, g[..., :, None] - gk[..., None, :], 0.0))
    score = (q @ k.mT) / 8.0 + lam * decay * (c @ b.mT) + (f[..., :, None] - fk[..., None, :])
    return torch.where(seen, score, float("-inf"))


def _plain_attend(s):
    """The common positions once for every group, the own ones once for every sequence, and the two parts of the softmax
    joined. Groups are filled up to the largest."""
    case, S = s["case"], s["case"]["S"]
    M, H, (B, _), G = case["M"], case["H"], s["table"].shape, len(s["sizes"])
    size = torch.tensor(s["sizes"], device=DEVICE)
    R, first = max(s["sizes"]), size.cumsum(0) - size
    group = torch.repeat_interleave(torch.arange(G, device=DEVICE), size, output_size=B)
    member = torch.arange(B, device=DEVICE) - first[group]
    shared, lengths, table = s["shared"].long(), s["lengths"].long(), s["table"].long()
    q, c, g, f = s["q"].float(), s["c"].float(), s["g"], s["f"]
    own_n = max(_suffixes(case))

    def cached(rows, pos):                                # (n, H, N, .) of the positions (n, N) of the table's rows
        page = rows.gather(1, (pos // S).clamp(max=rows.shape[1] - 1)).clamp(min=0)
        return [s["pages"][x][page, :, pos % S].transpose(1, 2).float() for x in ("k", "v", "b", "g", "f")]

    # own positions
    pos = shared[group][:, None] + torch.arange(own_n, device=DEVICE)
    k, v, b, gk, fk = cached(table, pos)
    at = lengths[:, None] - M + torch.arange(M, device=DEVICE)
    seen = pos[:, None, None, :] <= at[:, None, :, None]
    v = torch.where((pos < lengths[:, None])[:, None, :, None], v, 0.0)
    score = _scores(s, q, c, g, f, k, b, gk, fk, seen)
    top = score.amax(-1)
    if s["common"]:
        def grouped(x):                                   # (B, H, M, .) -> (G, H, R M, .), nothing in empty places
            y = x.new_zeros(G, R, *x.shape[1:])
            y[group, member] = x
            return y.transpose(1, 2).flatten(2, 3)

        def back(y):                                      # and back
            return y.unflatten(2, (R, M)).transpose(1, 2)[group, member]
        pos0 = torch.arange(s["common"], device=DEVICE).expand(G, -1)
        k0, v0, b0, g0, f0 = cached(table[first], pos0)
        seen0 = (pos0 < shared[:, None])[:, None, None, :]
        score0 = _scores(s, grouped(q), grouped(c), grouped(g), grouped(f), k0, b0, g0, f0, seen0)
        v0 = torch.where((pos0 < shared[:, None])[:, None, :, None], v0, 0.0)
        top = torch.maximum(top, back(score0.amax(-1)))
        weight0 = torch.exp(score0 - grouped(top)[..., None])
    weight = torch.exp(score - top[..., None])
    total, out = weight.sum(-1), weight @ v
    if s["common"]:
        total, out = total + back(weight0.sum(-1)), out + back(weight0 @ v0)
    return out / total[..., None]


def _plain_verify(s):
    """In 64 bits: a decision is a comparison of two products that may be next to each other."""
    p, q, drafts, u = s["p"], s["q"], s["drafts"], s["u"].double()
    B, K = drafts.shape
    rows = torch.arange(B, device=DEVICE)
    counts = torch.full((B,), K, device=DEVICE) if s["counts"] is None else s["counts"].long()
    at = drafts[..., None]
    px = p[:, :K].gather(2, at)[..., 0].double()
    qx = torch.ones_like(px) if q is None else q.gather(2, at)[..., 0].double()
    took = (u[:, :K] * qx < px) & (torch.arange(K, device=DEVICE) < counts[:, None])
    accepted = took.long().cumprod(1).sum(1)
    refused, i = accepted < counts, accepted.clamp(max=K - 1)
    target = p[rows, accepted].double()
    if q is None:
        rest = target.scatter(1, drafts[rows, i][:, None], 0.0)
    else:
        rest = (target - q[rows, i].double()).clamp(min=0.0)
    rest = torch.where((refused & (rest.sum(1) > 0))[:, None], rest, target)
    upto = rest.cumsum(1)
    over = upto > u[:, K:] * upto[:, -1:]
    token = torch.where(over.any(1), over.int().argmax(1), p.shape[2] - 1)
    k = torch.arange(K + 1, device=DEVICE)
    padded = torch.nn.functional.pad(drafts, (0, 1), value=-1)
    tokens = torch.where(k < accepted[:, None], padded, torch.where(k == accepted[:, None], token[:, None], -1))
    return dict(tokens=tokens, accepted=accepted.to(torch.int32))


# ------------------------------------------------------------------------------------------------ necessary work
def work(case: dict) -> dict:
    """Bytes and floating-point operations of one pass that no implementation can leave out: common rows read once for a
    group, own ones once, queries and outputs; the probabilities that decide about the drafts, and of one row to draw from."""
    if case["kind"] == "attend":
        es, H, M = BYTES[case["dtype"]], case["H"], case["M"]
        sizes, shared, suffix = _sizes(case), _shared(case), _suffixes(case)
        group = [r for r, size in enumerate(sizes) for _ in range(size)]
        pairs = sum(M * (shared[r] + suffix[n]) - M * (M - 1) // 2 for n, r in enumerate(group))
        rows = sum(shared) + sum(suffix)
        return dict(bytes=float(H * (rows * (160 * es + 8) + len(group) * M * (96 * es + 8 + 256))), flops=320.0 * H * pairs)
    es, B, K, V = BYTES[case["dtype"]], case["B"], case["K"], case["V"]
    return dict(bytes=float(B * (V * es * (2 if case["proposal"] else 1) + 8 * (2 * K + 1) + 4 * (K + 1))),
                flops=float(2 * B * V))


# ------------------------------------------------------------------------------------------------ 64-bit results
def exact(case: dict, seed: int):
    """What ``run`` returns, by the definitions in 64 bits, one sequence after the other."""
    s = prepare(case, seed)
    return _exact_attend(s, case) if case["kind"] == "attend" else _exact_verify(s, case)


def _exact_attend(s, case):
    S, M, outs = case["S"], case["M"], []
    lam = s["lam"].double()[:, None]
    for n in range(s["table"].shape[0]):
        N = int(s["lengths"][n])
        pos = torch.arange(N, device=DEVICE)
        page, slot = s["table"][n].long()[torch.div(pos, S, rounding_mode="floor")], pos.remainder(S)
        k, v, b, g, f = (s["pages"][x][page, :, slot].double().transpose(0, 1) for x in ("k", "v", "b", "g", "f"))
        row = []
        for m in range(M):
            e = N - M + m + 1
            q, c, gm, fm = (s[x][n, :, m].double() for x in ("q", "c", "g", "f"))
            x = (k[:, :e] * q[:, None]).sum(-1) * D_HEAD ** -0.5
            x = x + lam * (gm[:, None] - g[:, :e]).exp() * (b[:, :e] * c[:, None]).sum(-1) + fm[:, None] - f[:, :e]
            row.append((x.softmax(-1)[..., None] * v[:, :e]).sum(1))
        outs.append(torch.stack(row, 1))
    return torch.stack(outs)


def _exact_verify(s, case):
    K, V, counts = case["K"], case["V"], _counts(case)
    tokens, accepted = [], []
    for n in range(case["B"]):
        p, drafts, u = s["p"][n].double(), s["drafts"][n].tolist(), s["u"][n].double()
        q = None if s["q"] is None else s["q"][n].double()
        took = 0
        while took < counts[n] and float(u[took] * (1.0 if q is None else q[took, drafts[took]])) < float(p[took, drafts[took]]):
            took += 1
        w = p[took].clone()
        if took < counts[n]:
            if q is None:
                w[drafts[took]] = 0.0
            else:
                w = torch.maximum(w - q[took], torch.zeros_like(w))
            if float(w.sum()) == 0.0:
                w = p[took].clone()
        below = w.cumsum(0)
        token = int((below <= u[K] * below[-1]).sum())
        tokens.append(drafts[:took] + [min(token, V - 1)] + [-1] * (K - took))
        accepted.append(took)
    return dict(tokens=torch.tensor(tokens, device=DEVICE), accepted=torch.tensor(accepted, device=DEVICE, dtype=torch.int32))
