"""Attention over common first positions (csrc/prefix.hip) against a plain form in float64, and the verification of drafted
tokens (csrc/verify.hip) against one in float64 that goes through the vocabulary token by token.

Tolerance, norm-wise, of the attention's float32 results: a score is a sum of 64 + 32 products with operands of order 1 (exact
in 16 bits), so its rounding error is about sqrt(96) 2^-24 times the largest partial sum (about 10 here), plus a few 2^-24 of
|F - F'| (below 40) and of the exponents: under 3e-6 in all; a weight's relative error is that of its score and of its row's
sum, twice that; weights enter the products with values as two or three 16-bit terms, which leave out 2^-22 of a weight or
less. The results are averages of weights: 1e-5 is above it. Tokens and counts are compared exactly."""
import math

import pytest
import torch

DEV = "cuda:0"
TOL = 1e-5
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
pytestmark = pytest.mark.gpu


def _rel(x, ref):
    return float((x.double() - ref).norm() / ref.norm().clamp_min(1e-300))


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values):
    return torch.tensor(list(values), device=DEV, dtype=torch.int32)


def _gates(gen, *shape):
    steps = 0.02 * torch.rand(shape, generator=gen, device=DEV)
    return -steps.cumsum(-1)


class Grouped:
    """Sequences in groups with common first positions. ``rows``: (B, H, N, .) of every sequence, side by side. In the pool
    only the first sequence of a group has the common ones: where another one's table row would name them it says a page
    outside the pool, and the slots of its first own page in front of its own positions are NaN, like every slot that holds
    nothing."""

    def __init__(self, sizes, shared, own, H, S, dtype, seed=0, forget=True, nowhere=-1):
        from sisa_amd.kernels.paged import PagePool
        from sisa_amd.kernels.prefix import PrefixGroups
        gen = self.gen = _gen(seed)
        self.sizes, self.shared, self.H, self.S, self.dtype = sizes, shared, H, S, dtype
        self.group = [r for r, n in enumerate(sizes) for _ in range(n)]
        self.B = B = len(self.group)
        self.lengths = [shared[r] + own[i] for i, r in enumerate(self.group)]
        N, W = max(1, max(self.lengths)), max(1, max(-(-n // S) for n in self.lengths))
        new = lambda w: torch.randn(B, H, N, w, generator=gen, device=DEV).to(dtype)  # noqa: E731
        self.rows = dict(k=new(64), v=new(64), b=new(32), g=_gates(gen, B, H, N),
                         f=_gates(gen, B, H, N) if forget else None)
        self.first = [sum(sizes[:r]) for r in range(len(sizes))]
        for x in self.rows.values():
            if x is not None:
                for i, r in enumerate(self.group):
                    x[i, :, :shared[r]] = x[self.first[r], :, :shared[r]]
        total = B * W + 3
        order = torch.randperm(total, generator=gen, device=DEV).tolist()
        nan = lambda *s, dt=dtype: torch.full((total, H, S, *s), math.nan, device=DEV, dtype=dt)  # noqa: E731
        self.t = dict(k=nan(64), v=nan(64), b=nan(32), g=nan(dt=torch.float32),
                      f=nan(dt=torch.float32) if forget else None)
        table = torch.full((B, W), nowhere, dtype=torch.int32)
        for i, r in enumerate(self.group):
            lo = 0 if i == self.first[r] else shared[r]
            for at in range(lo // S, -(-self.lengths[i] // S)):
                if self.lengths[i] == lo:
                    break
                page = table[i, at] = order.pop()
                j0, j1 = max(lo, at * S), min(self.lengths[i], at * S + S)
                for name, x in self.rows.items():
                    if x is not None:
                        self.t[name][page, :, j0 - at * S:j1 - at * S] = x[i, :, j0:j1]
        self.table = table.to(DEV)
        self.pool = PagePool(*(self.t[x] for x in ("k", "v", "b", "g", "f")))
        self.groups = PrefixGroups(sizes, DEV)
        self.lam = torch.rand(H, generator=gen, device=DEV) + 0.1

    def queries(self, M=1):
        """q, c and the gates of the last M positions (of a sequence shorter than M: of any)."""
        new = lambda w: torch.randn(self.B, M, self.H, w, generator=self.gen,  # noqa: E731
                                    device=DEV).to(self.dtype).transpose(1, 2)
        at = torch.tensor([[max(0, n - M + m) for m in range(M)] for n in self.lengths], device=DEV)
        at = at[:, None].expand(self.B, self.H, M)
        return new(64), new(32), self.rows["g"].gather(2, at), None if self.rows["f"] is None else self.rows["f"].gather(2, at)

    def run(self, q, c, g, f, lengths=None, shared=None, **kw):
        from sisa_amd.kernels.prefix import sisa_prefix_decode_hip
        return sisa_prefix_decode_hip(q, c, g, f, self.lam, self.pool, self.table, _ints(lengths or self.lengths),
                                      self.groups, _ints(self.shared if shared is None else shared), **kw)

    def want(self, q, c, g, f, lengths=None):
        M = q.shape[2]
        out = torch.zeros(self.B, self.H, M, 64, device=DEV, dtype=torch.float64)
        for i, n in enumerate(lengths or self.lengths):
            for m in range(M):
                vis = max(0, n - M + m + 1)
                if vis:
                    r = {x: None if t is None else t[i, :, :vis].double() for x, t in self.rows.items()}
                    s = (r["k"] @ q[i, :, m].double()[..., None])[..., 0] / 8
                    s = s + self.lam.double()[:, None] * (g[i, :, m, None].double() - r["g"]).exp() * (
                        r["b"] @ c[i, :, m].double()[..., None])[..., 0]
                    if f is not None:
                        s = s + f[i, :, m, None].double() - r["f"]
                    out[i, :, m] = (s.softmax(-1)[..., None] * r["v"]).sum(1)
        return out


def _agrees(got, want):
    return got.shape == want.shape and got.dtype == torch.float32 and _rel(got, want) <= TOL


# one sequence and many; groups of one, and of more rows than a tile takes (16, 32, 64); common positions that end in a page
# and at its end, none, and one; own positions that begin inside a tile; pages smaller and larger than a tile; drafts of a
# group of one, and of several sequences; more drafts than a tile takes
CASES = [([1], [0], [1], 1, 16, 1), ([1], [33], [1], 2, 16, 1), ([2], [1], [1, 2], 1, 16, 1), ([4], [64], [1, 5, 31, 32], 3, 16, 1),
         ([3, 1, 2], [100, 0, 31], [1, 33, 64, 7, 1, 129], 2, 32, 1), ([17], [500], list(range(1, 18)), 2, 64, 1),
         ([40], [257], [3] * 40, 1, 128, 1), ([70, 1], [300, 20], [1 + i % 9 for i in range(71)], 2, 16, 1),
         ([150], [90], [1 + i % 70 for i in range(150)], 1, 32, 1), ([1], [1000], [5], 4, 64, 5),
         ([1, 1, 1], [700, 3, 0], [8, 8, 8], 2, 32, 8), ([5, 3], [400, 65], [3, 9, 40, 100, 4, 3, 3, 500], 3, 64, 3),
         ([1, 2], [40, 50], [33, 70, 90], 2, 16, 33), ([2], [100], [80, 300], 1, 64, 80), ([2, 2], [2500, 1300], [900, 1, 3, 64], 5, 1024, 1),
         ([1], [0], [40], 2, 16, 40), ([9], [4100], [600] * 9, 2, 64, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,shared,own,H,S,M", CASES)
def test_prefix_decode(sizes, shared, own, H, S, M, dtype):
    for forget in (True, False):
        case = Grouped(sizes, shared, own, H, S, dtype, seed=M + H, forget=forget, nowhere=-1 if forget else 1 << 30)
        rows = case.queries(M)
        want = case.want(*rows)
        assert _agrees(case.run(*rows), want)
        got = case.run(*rows, max_len=max(case.lengths), max_shared=max(shared))
        assert _agrees(got, want)
        assert torch.equal(got, case.run(*rows, max_len=max(case.lengths), max_shared=max(shared)))


def test_lengths_within_the_common_positions():
    """Empty sequences, sequences that end inside what their group has in common, and fewer positions than new rows."""
    case = Grouped([5, 2], [100, 40], [5, 5, 5, 5, 5, 9, 9], 2, 16, torch.bfloat16, seed=3)
    for M in (1, 4, 20):
        rows = case.queries(M)
        lengths = [105, 100, 37, 0, 3, 49, 1]
        got, want = case.run(*rows, lengths=lengths), case.want(*rows, lengths=lengths)
        assert _agrees(got, want)
        assert all(got[i, :, m].eq(0).all() for i, n in enumerate(lengths) for m in range(M) if n - M + m < 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_there_is_nan(dtype):
    """Lengths and common positions that the call does not take, and pages outside the pool: NaN for the rows concerned, and
    the others as they are."""
    case = Grouped([3, 2, 2], [70, 40, 0], [5, 9, 40, 3, 33, 20, 50], 2, 16, dtype, seed=4)
    rows = case.queries(2)
    want, plain = case.want(*rows), case.run(*rows)

    def only(got, bad):
        assert all(got[i].isnan().all() if i in bad else torch.equal(got[i], plain[i]) for i in range(case.B)), bad
    top = dict(max_len=max(case.lengths), max_shared=70)
    plain = case.run(*rows, **top)
    assert _agrees(plain, want)
    n = case.lengths
    only(case.run(*rows, lengths=[n[0], -1, *n[2:4], 111, *n[5:]], **top), {1, 4})
    only(case.run(*rows, shared=[70, -1, 0], **top), {3, 4})
    only(case.run(*rows, shared=[71, 40, 0], **top), {0, 1, 2})
    only(case.run(*rows, lengths=[-(1 << 31), (1 << 31) - 1, *n[2:]], shared=[70, (1 << 31) - 1, 0], **top), {0, 1, 3, 4})
    held = case.table.clone()
    case.table[3, 1] = case.pool.pages                    # the second group's common positions 16 .. 31
    only(case.run(*rows, **top), {3, 4})
    case.table.copy_(held)
    case.table[2, 105 // 16] = -5                         # an own page of the third sequence
    only(case.run(*rows, **top), {2})
    case.table.copy_(held)
    case.table[1, 0] = case.table[4, 0] = -(1 << 31)      # not read
    only(case.run(*rows, **top), set())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(value, dtype):
    """What a row does not see does not reach it: the positions of later drafts, and another sequence's own."""
    M = 6
    case = Grouped([2, 1], [50, 90], [40, 8, 20], 2, 16, dtype, seed=5)
    rows = case.queries(M)
    plain = case.run(*rows)
    for name in ("v", "k", "b", "g", "f"):
        held = case.t[name].clone()
        j = case.lengths[0] - 3                           # of six rows the last three see it
        case.t[name][case.table[0, j // 16], :, j % 16] = value
        got = case.run(*rows)
        assert torch.equal(got[1:], plain[1:]) and torch.equal(got[0, :, :3], plain[0, :, :3])
        if name == "v" or math.isnan(value):
            assert not got[0, :, 3:].isfinite().any()
        case.t[name].copy_(held)
    j = 7                                                 # common to the first group
    case.t["v"][case.table[0, 0], :, j] = value
    got = case.run(*rows)
    assert not got[:2].isfinite().any() and torch.equal(got[2], plain[2])


def test_no_positions_weigh_anything():
    """Scores that are all -inf have no softmax: NaN, as a plain form gives; one finite score among them takes everything."""
    case = Grouped([3], [40], [4, 4, 4], 1, 16, torch.bfloat16, seed=6)
    rows = list(case.queries())
    for i in range(3):
        for j in range(case.lengths[i]):
            own = i if j >= 40 else 0
            case.t["f"][case.table[own, j // 16], :, j % 16] = math.inf
    assert case.run(*rows).isnan().all()
    case.t["f"][case.table[1, 41 // 16], :, 41 % 16] = 0.5
    got = case.run(*rows)
    assert got[0].isnan().all() and got[2].isnan().all() and torch.allclose(got[1, 0, 0], case.rows["v"][1, 0, 41].float(), rtol=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steep_gates(dtype):
    """Decays that underflow, gates that rise, and weights over many orders of magnitude."""
    case = Grouped([20], [600], [1 + 7 * i for i in range(20)], 2, 32, dtype, seed=7)
    N = case.rows["g"].shape[2]
    g = -200.0 * torch.rand(case.B, 2, N, generator=case.gen, device=DEV)
    g[:, :, -300:] = torch.linspace(-30, -10, 300, device=DEV)
    for i in range(case.B):
        g[i, :, :600] = g[0, :, :600]
        for j in range(0 if i == 0 else 600, case.lengths[i]):
            case.t["g"][case.table[i, j // 32], :, j % 32] = g[i, :, j]
    case.rows["g"] = g
    rows = list(case.queries())
    rows[2] = g[:, :, 0:1] * 0 - 205.0
    # c.b of order sqrt(32), times exp(-205 + 200) at most: what the state term adds is small; 1 / 8 q.k is what it was
    assert _agrees(case.run(*rows), case.want(*rows))
    rows[0] = rows[0] * 6                                 # scores of up to 30, whose float32 rounding is up to 2^-20 each
    want = case.want(*rows)
    assert _rel(case.run(*rows), want) <= 2 * TOL


def test_strides_and_copies():
    """Operands of other strides, rows that 16-byte loads cannot read (copied), a table that is part of another, lam with a
    stride, and expanded gates."""
    case = Grouped([3, 2], [77, 20], [5, 9, 40, 3, 33], 3, 16, torch.float16, seed=8)
    q, c, g, f = case.queries(2)
    plain = case.run(q, c, g, f)
    off = torch.empty(case.B, 3, 2, 65, device=DEV, dtype=torch.float16)[..., 1:].copy_(q)
    wide = torch.full((case.B + 1, case.table.shape[1] + 5), -1, device=DEV, dtype=torch.int32)
    wide[1:, 2:-3] = case.table
    case.table = wide[1:, 2:-3]
    case.lam = torch.stack([case.lam, case.lam], 1)[:, 0]
    gt = g.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(case.run(off, c.contiguous(), gt, f), plain)
    g1 = g[:, :, :1].expand(-1, -1, 2)
    assert torch.equal(case.run(q, c, g1, f), case.run(q, c, g1.contiguous(), f))


def test_pages_beyond_32_bit_offsets():
    """Pages whose rows start past 2^31 elements, and 2^32 bytes, of their tensor."""
    from sisa_amd.kernels.paged import PagePool, sisa_paged_write_hip
    from sisa_amd.kernels.prefix import PrefixGroups, sisa_prefix_decode_hip
    S, H, P, M = 1024, 8, 4200, 1500                      # 4200 x 8 x 1024 x 64 = 2.2e9 elements
    dt, gen = torch.float16, _gen(1)
    new = lambda w: torch.randn(2, H, M, w, generator=gen, device=DEV).to(dt)  # noqa: E731
    k, v, b, g, f = new(64), new(64), new(32), _gates(gen, 2, H, M), _gates(gen, 2, H, M)
    lam, q, c = torch.rand(H, generator=gen, device=DEV), new(64)[:, :, :1], new(32)[:, :, :1]
    outs = []
    for pages, rows in ((P, [[P - 1, 3], [P - 1, P - 2]]), (5, [[1, 3], [1, 4]])):
        pool = PagePool.empty(pages, H, S, dt, DEV)
        table = torch.tensor(rows, device=DEV, dtype=torch.int32)
        sisa_paged_write_hip(pool, table, _ints([S, S]), k[:, :, S:], v[:, :, S:], b[:, :, S:], g[:, :, S:], f[:, :, S:])
        sisa_paged_write_hip(pool, table[:1], _ints([0]), *(x[:1, :, :S] for x in (k, v, b, g, f)))
        outs.append(sisa_prefix_decode_hip(q, c, g[:, :, -1:], f[:, :, -1:], lam, pool, table, _ints([M, M]),
                                           PrefixGroups([2], DEV), _ints([S])))
    assert torch.equal(*outs) and outs[0].isfinite().all()


def test_agrees_with_the_attention_of_single_sequences():
    from sisa_amd.kernels.paged import sisa_paged_decode_hip
    case = Grouped([1] * 6, [300, 5, 64, 0, 900, 33], [4, 40, 4, 4, 300, 9], 4, 32, torch.bfloat16, seed=9)
    rows = case.queries(4)
    one = sisa_paged_decode_hip(*rows, case.lam, case.pool, case.table, _ints(case.lengths))
    assert _rel(case.run(*rows), one.double()) <= 2 * TOL


def test_refusals():
    from sisa_amd.kernels.prefix import PrefixGroups
    case = Grouped([2, 1], [20, 5], [3, 4, 5], 2, 16, torch.bfloat16)
    q, c, g, f = case.queries()
    with pytest.raises(ValueError, match="groups of 2"):
        case.groups = PrefixGroups([1, 1], DEV)
        case.run(q, c, g, f)
    case.groups = PrefixGroups([2, 1], DEV)
    for bad, word in (((q.float(), c, g, f), "q must be"), ((q, c[:, :1], g, f), "c must be"), ((q, c, g.half(), f), "g_q must be"),
                      ((q, c, g, None), "forget term"), ((q[0], c, g, f), "q must be")):
        with pytest.raises(ValueError, match=word):
            case.run(*bad)
    with pytest.raises(ValueError, match="shared must be"):
        case.run(q, c, g, f, shared=[20])
    with pytest.raises(ValueError, match="max_len"):
        case.run(q, c, g, f, max_len=10_000)
    with pytest.raises(ValueError, match="max_shared"):
        case.run(q, c, g, f, max_shared=-1)
    with pytest.raises(RuntimeError, match="inference"):
        case.run(q.clone().requires_grad_(True), c, g, f)
    for sizes in ([], [0], [2, -1]):
        with pytest.raises(ValueError, match="at least one group"):
            PrefixGroups(sizes, DEV)


# ------------------------------------------------------------------------------------------------ verification
def _want(p, drafts, u, q=None, counts=None):
    """Tokens and accepted counts by the definition, token by token."""
    B, K = drafts.shape
    V = p.shape[2]
    p, u = p.double().cpu(), u.double().cpu()
    q = None if q is None else q.double().cpu()
    tokens, accepted = [], []
    for n in range(B):
        count = K if counts is None else min(max(int(counts[n]), 0), K)
        took = 0
        while took < count:
            x = int(drafts[n, took])
            if not 0 <= x < V or not float(u[n, took]) * (1.0 if q is None else float(q[n, took, x])) < float(p[n, took, x]):
                break
            took += 1
        ways = [p[n, took].clamp(min=0.0)]
        if took < count:
            if q is not None:
                ways.insert(0, (p[n, took] - q[n, took]).clamp(min=0.0))
            else:
                rest = ways[0].clone()
                if 0 <= int(drafts[n, took]) < V:
                    rest[int(drafts[n, took])] = 0.0
                ways.insert(0, rest)
        token = -1
        for w in ways:
            total = float(w.sum())
            if not math.isfinite(total):
                break
            if total > 0.0:
                up = w.cumsum(0)
                good = (up > float(u[n, K]) * float(up[-1])) & (w > 0)
                token = int(good.int().argmax()) if good.any() else int(w.nonzero()[-1])
                break
        tokens.append([int(x) for x in drafts[n, :took]] + [token] + [-1] * (K - took))
        accepted.append(took)
    return torch.tensor(tokens), torch.tensor(accepted, dtype=torch.int32)


def _verify(p, drafts, u, q=None, counts=None):
    from sisa_amd.kernels.verify import sisa_verify_drafts_hip
    got = sisa_verify_drafts_hip(p, drafts, u, q, counts)
    assert got.tokens.dtype == torch.int64 and got.accepted.dtype == torch.int32
    return got


def _same(got, want):
    assert got.accepted.tolist() == want[1].tolist()
    assert got.tokens.tolist() == want[0].tolist()


def _drafted(B, K, V, p_dtype, q_dtype, seed, top_k=0, sharp=3.0):
    gen = _gen(seed)
    target = sharp * torch.randn(B, K + 1, V, generator=gen, device=DEV)
    draft = target[:, :K] + torch.randn(B, K, V, generator=gen, device=DEV)

    def probabilities(x):
        if top_k:
            x = x.masked_fill(x < x.topk(min(top_k, V), -1).values[..., -1:], -math.inf)
        return x.softmax(-1)
    q = probabilities(draft)
    drafts = torch.multinomial(q.flatten(0, 1), 1, generator=gen).view(B, K) if K else torch.zeros(B, 0, device=DEV, dtype=torch.int64)
    return probabilities(target).to(p_dtype), drafts, torch.rand(B, K + 1, generator=gen, device=DEV), q.to(q_dtype or p_dtype)


# a vocabulary of one token, and at the edges of a wave's and a workgroup's loads; no drafts, one, and more than a wave has lanes
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 0, 5), (2, 3, 2), (5, 2, 63), (4, 4, 64), (4, 1, 65), (7, 5, 255), (9, 3, 257),
                                   (33, 4, 1000), (3, 70, 300), (16, 7, 1023), (16, 7, 1025), (6, 3, 4097), (5, 2, 50277), (2, 3, 131073)])
@pytest.mark.parametrize("types", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, torch.float32),
                                   (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16)])
def test_verify(B, K, V, types):
    for seed, top_k in ((0, 0), (1, 20)):
        p, drafts, u, q = _drafted(B, K, V, *types, seed=seed + V, top_k=top_k)
        counts = torch.tensor([(3 * n) % (K + 2) - (n == 1) for n in range(B)], device=DEV, dtype=torch.int32)
        for draft_p in (q, None):
            for c in (None, counts):
                _same(_verify(p, drafts, u, draft_p, c), _want(p, drafts, u, draft_p, c))


def test_verify_decides_exactly():
    """Random numbers next to and at the ratio: u q < p in exact arithmetic. 0.75 and 0.5 are exact in every type; the products
    of two 24-bit numbers are not exact in float32."""
    V = 8
    p, q = torch.zeros(4, 2, V, device=DEV), torch.zeros(4, 1, V, device=DEV)
    p[:, 0, 3], q[:, 0, 3] = 0.375, 0.75
    p[:, 0, 5], q[:, 0, 1] = 0.625, 0.25
    p[:, 1, 6] = 1.0
    drafts = torch.full((4, 1), 3, device=DEV)
    half = torch.tensor(0.5, device=DEV)
    below, above = torch.nextafter(half, torch.zeros_like(half)), torch.nextafter(half, torch.ones_like(half))
    u = torch.stack([torch.stack([below, half, above, torch.zeros_like(half)]), torch.zeros(4, device=DEV)], 1)
    got = _verify(p, drafts, u, q)
    assert got.accepted.tolist() == [1, 0, 0, 1] and got.tokens.tolist() == [[3, 6], [5, -1], [5, -1], [3, 6]]
    x = torch.tensor(1.0 + 2.0 ** -23, device=DEV)
    p[:, 0, 3] = float(x * x)                             # rounded down: below the product of the two
    q[:, 0, 3], u[:, 0] = x, x
    assert float(x * x) < float(x.double() * x.double())
    assert _verify(p, drafts, u, q).accepted.tolist() == [0] * 4


def test_verify_edges():
    """Weights that are 0 everywhere, sums that are not finite, drafts outside the vocabulary, random numbers at the ends of
    their range and outside it."""
    nan, inf, V = math.nan, math.inf, 100
    p, drafts, u, q = _drafted(16, 2, V, torch.float32, None, seed=5)
    u[:] = 0.99999994
    drafts[0, 0], drafts[1, 0], drafts[2, 1] = -1, V, 1 << 40
    p[3] = q[3, :1]                                       # refused by u = 1 alone, below: no residual is left
    u[3] = 1.0
    p[4] = 0.0                                            # nothing to draw from
    p[5, 0, 7], p[6, 0, 8], q[7, 0, 9] = nan, inf, nan
    p[8, 0, :], p[8, 0, 42] = 0.0, 1.0                    # one token that can be
    drafts[8, 0] = 42
    u[9, 2], u[10, 2], u[11, 2], u[12, 2] = 0.0, 1.0, -1.0, 2.0
    p[9:13, :, :5] = p[9:13, :, 95:] = 0.0                # first and last tokens that cannot be
    u[13, 0] = nan
    p[14] = -0.25                                         # not probabilities: below 0 counts as 0
    got, want = _verify(p, drafts, u, q), _want(p, drafts, u, q)
    _same(got, want)
    assert got.accepted[:3].tolist() == [0, 0, want[1][2]] and got.tokens[4].tolist() == [-1] * 3
    assert got.accepted[13] == 0
    _same(_verify(p, drafts, u), _want(p, drafts, u))


def test_verify_strides_and_determinism():
    p, drafts, u, q = _drafted(6, 3, 777, torch.bfloat16, None, seed=6)
    want = _want(p, drafts, u, q)
    wide = torch.zeros(6, 5, 800, device=DEV, dtype=torch.bfloat16)
    wide[:, 1:, 3:780] = p
    odd = torch.zeros(7, 6, 3, 777, device=DEV, dtype=torch.bfloat16)
    odd[3] = q
    across = p.transpose(1, 2).contiguous().transpose(1, 2)           # unit stride along the positions: copied
    for pp in (wide[:, 1:, 3:780], across):
        got = _verify(pp, drafts.t().contiguous().t(), u.t().contiguous().t(), odd[3])
        _same(got, want)
    counts = torch.tensor([2, 3, 0, 1, 3, 2], device=DEV, dtype=torch.int32)
    _same(_verify(p, drafts, u[:, :1].expand(-1, 4), q, counts), _want(p, drafts, u[:, :1].expand(-1, 4), q, counts))


def test_verify_keeps_the_targets_distribution():
    """Over many random numbers the first token is distributed as the target's, whatever the draft's: the formula's promise,
    by counting. With 200,000 rows a share x has the standard deviation sqrt(x (1 - x) / 200,000) < 0.0012: five of them."""
    gen, B, V = _gen(7), 200_000, 6
    t, d = torch.rand(V, generator=gen, device=DEV) + 0.05, torch.rand(V, generator=gen, device=DEV) + 0.05
    t, d = t / t.sum(), d / d.sum()
    drafts = torch.multinomial(d.expand(B, V), 1, generator=gen)
    u = torch.rand(B, 2, generator=gen, device=DEV)
    got = _verify(t.expand(B, 2, V), drafts, u, d.expand(B, 1, V))
    share = torch.bincount(got.tokens[:, 0], minlength=V) / B
    assert (share - t).abs().max() < 0.006
    assert abs(float(got.accepted.float().mean()) - float(torch.minimum(t, d).sum())) < 0.006


def test_verify_refusals():
    p, drafts, u, q = _drafted(2, 2, 10, torch.float32, None, seed=8)
    for args, word in (((p[:, :2], drafts, u, q), "K \\+ 1"), ((p, drafts.int(), u, q), "int64"), ((p, drafts, u[:, :2], q), "u must be"),
                       ((p, drafts, u.double(), q), "u must be"), ((p, drafts, u, q[:1]), "q must be"), ((p.double(), drafts, u, q), "p must be"),
                       ((p, drafts, u, q, torch.zeros(2, device=DEV)), "counts"), ((p, drafts.cpu(), u, q), "drafts must be"),
                       ((p.cpu(), drafts, u, q), "GPU")):
        with pytest.raises(ValueError, match=word):
            _verify(*args)
    empty = _verify(p[:0], drafts[:0], u[:0], q[:0])
    assert empty.tokens.shape == (0, 3) and empty.accepted.shape == (0,)


# ------------------------------------------------------------------------------------------------ both, as they are used
def test_captured_and_replayed():
    """A round of drafting in one graph (drafted rows written, attended to with everything before them in common, tokens
    verified, lengths cut back to what was accepted), replayed with other rows, with eager calls and a second graph beside."""
    from sisa_amd.kernels.paged import sisa_paged_write_hip
    M, V = 4, 500
    case = Grouped([3, 2], [70, 20], [10, 20, 30, 6, 50], 2, 16, torch.bfloat16, seed=10)
    W = case.table.shape[1]
    case.table = torch.arange(case.B * W, device=DEV, dtype=torch.int32).view(case.B, W).contiguous()
    for r, first in enumerate(case.first):                # pages of their own, the common ones as the first has them
        case.table[first:first + case.sizes[r], :case.shared[r] // 16] = case.table[first, :case.shared[r] // 16].clone()
    for t in case.t.values():
        t.copy_(torch.randn(t.shape, generator=case.gen, device=DEV) * 0.1)
    held = {n: t.clone() for n, t in case.t.items()}
    new = lambda *w: torch.randn(case.B, 2, M, *w, generator=case.gen, device=DEV)  # noqa: E731
    state = dict(k=new(64).bfloat16(), v=new(64).bfloat16(), b=new(32).bfloat16(), q=new(64).bfloat16(), c=new(32).bfloat16(),
                 g=-new().abs(), f=-new().abs())
    p, drafts, u, q = _drafted(case.B, M - 1, V, torch.float32, None, seed=11)
    start = _ints([60, 70, 80, 15, 50])
    lengths, shared = torch.empty_like(start), _ints([64, 16])

    def step():
        from sisa_amd.kernels.prefix import sisa_prefix_decode_hip
        from sisa_amd.kernels.verify import sisa_verify_drafts_hip
        sisa_paged_write_hip(case.pool, case.table, start, state["k"], state["v"], state["b"], state["g"], state["f"])
        torch.add(start, M, out=lengths)
        out = sisa_prefix_decode_hip(state["q"], state["c"], state["g"], state["f"], case.lam, case.pool, case.table, lengths,
                                     case.groups, shared)
        got = sisa_verify_drafts_hip(p, drafts, u, q)
        torch.add(start, got.accepted, out=lengths)
        lengths.add_(1)
        return out, got.tokens, got.accepted, lengths.clone()

    def other():
        return case.run(state["q"], state["c"], state["g"], state["f"], lengths=None)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(), other()
    torch.cuda.current_stream().wait_stream(side)
    graph, beside = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    fixed = _ints(case.lengths)
    with torch.cuda.graph(beside, stream=side):
        from sisa_amd.kernels.prefix import sisa_prefix_decode_hip
        second = sisa_prefix_decode_hip(state["q"], state["c"], state["g"], state["f"], case.lam, case.pool, case.table, fixed,
                                        case.groups, shared)
    for turn in range(4):
        for x in state.values():
            x.copy_(torch.randn(x.shape, generator=case.gen, device=DEV) * (0.3 + turn))
        u.uniform_(generator=case.gen)
        start.copy_(_ints([60 + turn, 64, 66 + 3 * turn, 16, 44]))
        shared.copy_(_ints([64 - turn, 16]))
        for n, t in case.t.items():
            t.copy_(held[n])
        want = step()
        again = other()
        for n, t in case.t.items():
            t.copy_(held[n])
        beside.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, want))
        assert second.isfinite().all() and again.shape == second.shape


def test_another_stream():
    """Calls on a stream other than the default one, on tensors that it has waited for."""
    case = Grouped([4], [200], [5, 6, 70, 8], 2, 16, torch.bfloat16, seed=12)
    rows = case.queries()
    p, drafts, u, q = _drafted(4, 3, 3000, torch.float32, None, seed=13)
    plain, want = case.run(*rows), _verify(p, drafts, u, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, verified = case.run(*rows), _verify(p, drafts, u, q)
    side.synchronize()
    assert torch.equal(got, plain) and torch.equal(verified.tokens, want.tokens)


@pytest.mark.parametrize("empty", [3, 5, 6])
def test_a_border_that_rounding_moves_past_tokens_without_weight(empty):
    """Sums of 1,024 tokens whose total up to a chunk depends on the order of its additions, 1 or 1 + 2^-52 for weights 2^-53,
    2^-53 and 1, with the goal 0.5 * 2 between them, and a chunk behind them that holds nothing: the token is one that has a
    weight, on either side of the border."""
    chunk = 1024
    p = torch.zeros((1, 1, 8 * chunk), device=DEV)
    weights = {empty - 3: 2.0 ** -53, empty - 2: 2.0 ** -53, empty - 1: 1.0, empty + 1: 1.0}
    for c, x in weights.items():
        p[0, 0, c * chunk + 17] = x
    got = _verify(p, torch.empty((1, 0), dtype=torch.int64, device=DEV), torch.tensor([[0.5]], device=DEV))
    assert got.tokens.item() in ((empty - 1) * chunk + 17, (empty + 1) * chunk + 17)


def test_verify_infinities_on_both_sides():
    """Where p and q are infinite at one token their difference is not a number, and so is the sum: no token, in the first
    1,024 tokens, behind them and at the end; beside an infinite p or q alone."""
    inf, V = math.inf, 2600
    for types in ((torch.float32, None), (torch.bfloat16, torch.float16)):
        p, drafts, u, q = _drafted(6, 2, V, *types, seed=14)
        u[:, 2] = torch.tensor([0.0, 0.3, 0.6, 0.9, 0.99999994, 0.5], device=DEV)
        for n, at in enumerate((5, 1030, V - 1, 700, 2047, 2048)):
            x = int(drafts[n, 0])
            p[n, 0, x] = 0.0                              # the first draft is refused
            at += at == x
            if at == V:
                at = V - 2
            p[n, 0, at] = inf if n != 4 else 0.1
            q[n, 0, at] = inf if n != 3 else 0.1
        want = _want(p, drafts, u, q)
        assert want[1].tolist() == [0] * 6 and [int(t) < 0 for t in want[0][:, 0]] == [True, True, True, True, False, True]
        _same(_verify(p, drafts, u, q), want)


@pytest.mark.parametrize("wide", ["k", "v", "b", "g", "f"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_far_apart_in_pages_of_16(wide, dtype):
    """Pages of 16 positions whose rows lie 2^20 bytes apart, every page's and head's beside each other, more than 4,096
    positions of them: the bytes of what is left of a range pass 2^32, those of a page do not."""
    from sisa_amd.kernels.paged import PagePool
    case = Grouped([2, 1, 1], [4119, 4112, 0], [9, 70, 5, 4125], 2, 16, dtype, seed=15)
    for x in (case.rows, case.t):
        for gate in "gf":
            x[gate] *= 0.01                               # flat enough for the first positions to weigh as much as the last
    rows = case.queries(2)
    plain = case.run(*rows)
    assert _rel(plain, case.want(*rows)) <= TOL
    t = case.t[wide]
    P, H, S = t.shape[:3]
    width = t[0, 0, 0].numel()
    far = torch.zeros(S * (1 << 20) // t.element_size(), device=DEV, dtype=t.dtype)
    assert P * H * width * t.element_size() <= 1 << 20
    far = far.as_strided(t.shape, (H * width, width, (1 << 20) // t.element_size(), *t.stride()[3:])).copy_(t)
    case.pool = PagePool(*(far if x == wide else case.t[x] for x in ("k", "v", "b", "g", "f")))
    assert torch.equal(case.run(*rows), plain)


def test_two_graphs_and_eager_calls():
    """Two graphs of the same calls on the same tensors, one over fewer groups, replayed in either order with eager calls between and
    beside them: each one's answers are those of the eager calls on what the tensors hold then, after the other's replay, too."""
    case = Grouped([3, 2], [70, 20], [10, 20, 30, 6, 50], 2, 16, torch.bfloat16, seed=16)
    q, c, g, f = case.queries(4)
    p, drafts, u, draft_p = _drafted(case.B, 3, 2500, torch.float32, None, seed=17)
    shared, fewer, lengths = _ints([70, 20]), _ints([70, 16]), _ints(case.lengths)
    from sisa_amd.kernels.prefix import sisa_prefix_decode_hip

    def step(common, n):
        got = _verify(p[:n], drafts[:n], u[:n], draft_p[:n])
        out = sisa_prefix_decode_hip(q, c, g, f, case.lam, case.pool, case.table, lengths, case.groups, common)
        return out, got.tokens, got.accepted
    calls = [(shared, case.B), (fewer, 2)]
    for x, t in case.t.items():                           # positions 16 .. 19 of the last sequence in its own page, too
        t[int(case.table[4, 1]), :, :4] = case.rows[x][4, :, 16:20]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for call in calls:
            step(*call)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in calls], []
    for graph, call in zip(graphs, calls):
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(*call))
    seen = []
    for turn in range(4):
        q.copy_(torch.randn(q.shape, generator=case.gen, device=DEV))
        u.uniform_(generator=case.gen)
        lengths.copy_(_ints([n - turn for n in case.lengths]))
        for i in (0, 1) if turn % 2 else (1, 0):
            graphs[i].replay()
            step(*calls[1 - i])
        want = [step(*call) for call in calls]
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert got[0].isfinite().all() and all(torch.equal(x, y) for x, y in zip(got, ref))
        seen.append(outs[0][0].clone())
    assert not any(torch.equal(x, y) for x, y in zip(seen, seen[1:]))
