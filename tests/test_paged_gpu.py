"""The paged generation cache (csrc/paged.hip, csrc/evict.hip) and the received attention weights (csrc/attn_weights.hip)
against plain forms in float64.

Tolerances, norm-wise, of the float32 results of ``decode`` and ``weights``: a score is a sum of 64 + 32 products with
operands of order 1 (exact in 16 bits), so its rounding error is about sqrt(96) 2^-24 times the largest partial sum (about
10 here), plus a few 2^-24 of |F - F'| (below 40) and of the exponents: under 3e-6 in all; a weight's relative error is that
of its score and of its row's sum, twice that, and the results are averages of weights: 1e-5 is above it. Everything that is
copied or chosen is compared bit for bit."""
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


def _ints(*values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def _gates(gen, *shape):
    steps = 0.02 * torch.rand(shape, generator=gen, device=DEV)
    return -steps.cumsum(-1)


class Cache:
    """Sequences in a pool and the same positions side by side, (B, H, N, .) in float64. Slots that hold no position and
    pages that no sequence has are NaN, and the table says -1, or a page out of range, where there is none."""

    def __init__(self, lengths, H, S, dtype, seed=0, forget=True, nowhere=-1, room=0):
        from sisa_amd.kernels.paged import PagePool
        gen = self.gen = _gen(seed)
        self.lengths, self.B, self.H, self.S, self.dtype = list(lengths), len(lengths), H, S, dtype
        held = [-(-(n + room) // S) for n in lengths]
        W, total = max(1, max(held)), sum(held) + 3
        order = torch.randperm(total, generator=gen, device=DEV).tolist()
        rows, at = [], 0
        for n in held:
            rows.append(order[at:at + n] + [nowhere] * (W - n))
            at += n
        self.table = torch.tensor(rows, device=DEV, dtype=torch.int32)
        self.held = held
        N = max(1, max(lengths))
        new = lambda w: torch.randn(self.B, H, N, w, generator=gen, device=DEV).to(dtype)  # noqa: E731
        self.rows = dict(k=new(64), v=new(64), b=new(32), g=_gates(gen, self.B, H, N),
                         f=_gates(gen, self.B, H, N) if forget else None)
        nan = lambda *s, dt=dtype: torch.full((total, H, S, *s), math.nan, device=DEV, dtype=dt)  # noqa: E731
        self.t = dict(k=nan(64), v=nan(64), b=nan(32), g=nan(dt=torch.float32),
                      f=nan(dt=torch.float32) if forget else None)
        for i, n in enumerate(lengths):
            for j0 in range(0, n, S):
                j1, page = min(n, j0 + S), rows[i][j0 // S]
                for name, x in self.rows.items():
                    if x is not None:
                        self.t[name][page, :, :j1 - j0] = x[i, :, j0:j1]
        self.pool = PagePool(*(self.t[x] for x in ("k", "v", "b", "g", "f")))
        self.lam = torch.rand(H, generator=gen, device=DEV) + 0.1

    def queries(self, M=1):
        """q, c and the gates of the last M positions (of a sequence shorter than M: of any)."""
        new = lambda w: torch.randn(self.B, M, self.H, w, generator=self.gen,  # noqa: E731
                                    device=DEV).to(self.dtype).transpose(1, 2)
        at = torch.tensor([[max(0, n - M + m) for m in range(M)] for n in self.lengths], device=DEV)
        at = at[:, None].expand(self.B, self.H, M)
        return new(64), new(32), self.rows["g"].gather(2, at), None if self.rows["f"] is None else self.rows["f"].gather(2, at)

    def decode64(self, q, c, g, f):
        """Outputs and the positions' weights summed over the rows."""
        M = q.shape[2]
        out = torch.zeros(self.B, self.H, M, 64, device=DEV, dtype=torch.float64)
        got = torch.zeros(self.B, self.H, max(1, max(self.lengths)), device=DEV, dtype=torch.float64)
        for i, n in enumerate(self.lengths):
            for m in range(M):
                vis = max(0, n - M + m + 1)
                if not vis:
                    continue
                r = {x: None if t is None else t[i, :, :vis].double() for x, t in self.rows.items()}
                s = (r["k"] @ q[i, :, m].double()[..., None])[..., 0] / 8
                s = s + self.lam.double()[:, None] * (g[i, :, m, None].double() - r["g"]).exp() * (
                    r["b"] @ c[i, :, m].double()[..., None])[..., 0]
                if f is not None:
                    s = s + f[i, :, m, None].double() - r["f"]
                p = s.softmax(-1)
                out[i, :, m] = (p[..., None] * r["v"]).sum(1)
                got[i, :, :vis] += p
        return out, got


def _decode(cache, q, c, g, f, **kw):
    from sisa_amd.kernels.paged import sisa_paged_decode_hip
    return sisa_paged_decode_hip(q, c, g, f, cache.lam, cache.pool, cache.table, _ints(*cache.lengths), **kw)


# lengths at the edges of a wave's 64, a workgroup's 256 and a page; an empty sequence among others; a page larger than a
# chunk and pages smaller than a wave's 64; the positions of one head and of many
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,H,S,M", [([1], 1, 16, 1), ([0, 5, 64], 2, 16, 1), ([15, 16, 17], 3, 16, 1),
                                           ([63, 65, 255, 256, 257], 2, 32, 1), ([700, 0, 3, 1030], 4, 64, 1),
                                           ([511, 2049], 5, 1024, 1), ([4100, 1, 257], 2, 128, 1),
                                           ([2, 40, 300], 3, 16, 3), ([0, 1, 600, 1100], 2, 64, 5), ([33], 12, 16, 33)])
def test_decode(lengths, H, S, M, dtype):
    for forget in (True, False):
        cache = Cache(lengths, H, S, dtype, seed=M + H, forget=forget, nowhere=-1 if forget else 1 << 30)
        rows = cache.queries(M)
        want, received = cache.decode64(*rows)
        plain = _decode(cache, *rows)
        assert plain.shape == want.shape and plain.dtype == torch.float32
        assert _rel(plain, want) <= TOL
        assert all(plain[i, :, m].eq(0).all() for i, n in enumerate(lengths) for m in range(M) if n - M + m < 0)
        N = max(1, max(lengths))
        old = torch.rand(cache.B, H, N + 5, generator=cache.gen, device=DEV)
        new = torch.full_like(old, 7.0)
        out = _decode(cache, *rows, max_len=N, weights=old, weights_out=new)
        assert _rel(out, want) <= TOL
        for i, n in enumerate(lengths):
            assert new[i, :, n:].eq(7.0).all()
            if n:
                # what old + p keeps of p: the sum is below 1 + M (old is below 1, a row's weights at most 1 each), so each
                # of the H n roundings is off by at most (1 + M) 2^-24, together sqrt(H n) times that in the norm
                lost = (1 + M) * 2 ** -24 * (H * n) ** 0.5 / float(received[i, :, :n].norm())
                assert _rel(new[i, :, :n] - old[i, :, :n], received[i, :, :n]) <= TOL + lost
        held = old.clone()
        assert torch.equal(_decode(cache, *rows, max_len=N, weights=held), out)      # in place, and bitwise again
        assert all(torch.equal(held[i, :, :n], new[i, :, :n]) and torch.equal(held[i, :, n:], old[i, :, n:])
                   for i, n in enumerate(lengths))


# rows that a workgroup of 4, 8 or 16 waves takes whole, or that are too many for it
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,H,S,M", [([256, 0, 31], 3, 16, 1), ([512, 300, 257, 1], 3, 64, 1), ([1000, 513, 0, 1024], 2, 128, 1),
                                           ([600, 513, 64, 1, 0, 257, 570, 599, 80], 30, 32, 1), ([500, 40], 3, 16, 2)])
def test_decode_of_rows_taken_whole(lengths, H, S, M, dtype):
    test_decode(lengths, H, S, M, dtype)


# more than 256 chunks a row. The positions whose F lies more than 40 away have weights below exp(-30) of the nearest ones'.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 2])
def test_decode_of_many_chunks(M, dtype):
    test_decode([70_000, 200, 65_537], 1, 1024, M, dtype)


@pytest.mark.parametrize("dtype,N", [(torch.bfloat16, 54560), (torch.bfloat16, 54561), (torch.float16, 60000), (torch.float32, 27700)])
def test_decode_at_the_streaming_line(dtype, N):
    """Caches just below and above 256 MiB (15 heads: 4,920 or 9,720 bytes a position) give each head what a pool of that head
    alone, far below it, gives: the loads' cache policy is all that changes."""
    from sisa_amd.kernels.paged import PagePool, sisa_paged_decode_hip
    gen, H, S = _gen(N), 15, 64
    W = -(-N // S)
    new = lambda *w: torch.randn(W, H, S, *w, generator=gen, device=DEV)  # noqa: E731
    k, v, b = new(64).to(dtype), new(64).to(dtype), new(32).to(dtype)
    table = torch.randperm(W, generator=gen, device=DEV)[None].to(torch.int32)
    g, f = (torch.empty(W, H, S, device=DEV) for _ in range(2))
    for t in (g, f):
        t[table[0].long()] = (0.02 * _gates(gen, 1, H, W * S)).view(H, W, S).transpose(0, 1)
    q, c, lam = new(64)[:1, :, :1].to(dtype), new(32)[:1, :, :1].to(dtype), torch.rand(H, generator=gen, device=DEV)
    page, slot = int(table[0, (N - 1) // S]), (N - 1) % S
    gq, fq = (t[page, :, slot].reshape(1, H, 1).clone() for t in (g, f))
    old, w = torch.rand(1, H, N, generator=gen, device=DEV), torch.zeros(1, H, N, device=DEV)
    out = sisa_paged_decode_hip(q, c, gq, fq, lam, PagePool(k, v, b, g, f), table, _ints(N), max_len=N, weights=old, weights_out=w)
    assert torch.equal(out, sisa_paged_decode_hip(q, c, gq, fq, lam, PagePool(k, v, b, g, f), table, _ints(N), max_len=N))
    one = torch.zeros(1, 1, N, device=DEV)
    for h in (0, 7, 14):
        s = slice(h, h + 1)
        pool = PagePool(*(t[:, s] for t in (k, v, b, g, f)))
        alone = sisa_paged_decode_hip(q[:, s], c[:, s], gq[:, s], fq[:, s], lam[s], pool, table, _ints(N), max_len=N,
                                      weights=old[:, s], weights_out=one)
        assert torch.equal(out[:, s], alone) and torch.equal(w[:, s], one)
    assert (w >= old).all() and (w > old).any(-1).all()


def test_decode_continues_the_contiguous_cache():
    """The same rows through sisa_decode_hip, whose cache is one tensor."""
    from sisa_amd.kernels.decode import sisa_decode_hip
    cache = Cache([777, 777], 4, 64, torch.bfloat16, seed=3)
    q, c, g, f = cache.queries(2)
    r = cache.rows
    there = sisa_decode_hip(q, r["k"], r["v"], c, r["b"], g, r["g"], cache.lam, f, r["f"], 775)
    assert _rel(_decode(cache, q, c, g, f), there.double()) <= 2 * TOL


def test_decode_of_views_and_shared_pages():
    """A pool that is a layer of a larger tensor, a table with columns of another, two sequences that share their prefix."""
    from sisa_amd.kernels.paged import PagePool, sisa_paged_decode_hip
    cache = Cache([100, 150], 3, 32, torch.float16, seed=5)
    big = {n: torch.full((x.shape[0], 2, *x.shape[1:]), math.nan, device=DEV, dtype=x.dtype) for n, x in cache.t.items()}
    for n, x in cache.t.items():
        big[n][:, 1] = x
    pool = PagePool(*(big[n][:, 1] for n in ("k", "v", "b", "g", "f")))
    rows = cache.queries()
    wide = torch.full((2, 9), -5, device=DEV, dtype=torch.int32)
    wide[:, 2:2 + cache.table.shape[1]] = cache.table
    got = sisa_paged_decode_hip(*rows, cache.lam, pool, wide[:, 2:2 + cache.table.shape[1]], _ints(100, 150))
    assert torch.equal(got, _decode(cache, *rows))
    # both rows read sequence 1: its whole cache, and its first three pages
    both = cache.table[1:].expand(2, -1)
    q, c, g, f = (x[1:].expand(2, *x.shape[1:]) for x in rows)
    got = sisa_paged_decode_hip(q, c, g, f, cache.lam, pool, both, _ints(150, 96))
    assert torch.equal(got[0], _decode(cache, *rows)[1])
    cache.lengths, cache.B = [96], 1
    cache.rows = {n: x[1:] for n, x in cache.rows.items()}
    want, _ = cache.decode64(*(x[1:] for x in rows))
    assert _rel(got[1:], want) <= TOL


def test_decode_of_values_that_are_not_finite():
    """-inf scores weigh nothing, also where a whole chunk has them; a row of them, +inf and NaN give NaN, in their own
    sequence and head alone."""
    cache = Cache([600, 600, 600, 600], 2, 64, torch.float32, seed=7)
    rows = cache.queries()
    F = cache.rows["f"]
    F[0, 0, :256] = math.inf               # a score of -inf for one whole chunk
    F[1, 1, :] = math.inf                  # and for a whole row
    F[2, 0, 300] = -math.inf               # a score of +inf
    cache.rows["k"][3, 1, 10, 0] = math.nan
    for i in range(4):
        for j0 in range(0, 600, 64):
            page, j1 = int(cache.table[i, j0 // 64]), min(600, j0 + 64)
            cache.t["f"][page, :, :j1 - j0] = F[i, :, j0:j1]
            cache.t["k"][page, :, :j1 - j0] = cache.rows["k"][i, :, j0:j1]
    w = torch.zeros(4, 2, 600, device=DEV)
    out = _decode(cache, *rows, max_len=600, weights=w)
    want, received = cache.decode64(*rows)
    lost = torch.zeros(4, 2, dtype=torch.bool, device=DEV)
    lost[1, 1] = lost[2, 0] = lost[3, 1] = True
    assert out[lost].isnan().all() and not out[~lost].isnan().any() and w[~lost].isfinite().all()
    assert w[lost].isnan().any(-1).all()
    assert _rel(out[~lost], want[~lost]) <= TOL and _rel(w[~lost], received[~lost]) <= TOL
    assert w[0, 0, :256].eq(0).all()


def test_decode_marks_lengths_and_pages_outside_the_pool():
    """Every position that these name is checked against the table's width and the pool before it is read."""
    from sisa_amd.kernels.paged import sisa_paged_decode_hip
    cache = Cache([300, 300, 300, 300, 300], 2, 64, torch.bfloat16, seed=9)
    q, c, g, f = cache.queries()
    table = cache.table.clone()
    table[1, 2], table[2, 4] = -1, cache.pool.pages          # within the sequence: NaN
    w = torch.zeros(5, 2, 310, device=DEV)
    out = sisa_paged_decode_hip(q, c, g, f, cache.lam, cache.pool, table, _ints(300, 300, 300, -3, 311), max_len=310,
                                weights=w)
    assert torch.equal(out[0], _decode(cache, q, c, g, f, max_len=310)[0])
    assert out[1:].isnan().all() and w[1:3, :, :300].isnan().all() and w[3:].eq(0).all() and w[1:3, :, 300:].eq(0).all()


def test_refusals_on_the_gpu():
    """What the calls can see from the host: shapes, dtypes, devices, gradients, expanded outputs."""
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip, sisa_paged_decode_hip, sisa_paged_write_hip
    cache = Cache([20, 30], 2, 16, torch.float16, seed=1)
    q, c, g, f = cache.queries()
    n, lam, pool, table = _ints(20, 30), cache.lam, cache.pool, cache.table
    wide = torch.zeros(2, 2, 32, device=DEV)
    for bad, kind in ((dict(q=q.float()), ValueError), (dict(q=q[:, :1]), ValueError), (dict(q=q[..., :32]), ValueError),
                      (dict(f=None), ValueError), (dict(lam=lam[:1]), ValueError), (dict(lam=lam.double()), ValueError),
                      (dict(g=g.double()), ValueError), (dict(table=table.long()), ValueError), (dict(table=table[0]), ValueError),
                      (dict(n=n[:1]), ValueError), (dict(n=n.cpu()), ValueError), (dict(max_len=0), ValueError),
                      (dict(max_len=33), ValueError), (dict(weights=wide[:, :, :20]), ValueError),
                      (dict(weights=wide.double()), ValueError), (dict(weights_out=wide), ValueError),
                      (dict(weights=wide, weights_out=wide[:, :1].expand(2, 2, 32)), ValueError),
                      (dict(table=table[:, :0]), ValueError), (dict(q=q.clone().requires_grad_(True)), RuntimeError)):
        a = dict(q=q, c=c, g=g, f=f, lam=lam, pool=pool, table=table, n=n) | bad
        args = [a.pop(x) for x in ("q", "c", "g", "f", "lam", "pool", "table", "n")]
        with pytest.raises(kind):
            sisa_paged_decode_hip(*args, **a)
    one = wide[:1, :1].expand(1, 1, 32)                         # expanded along axes of one: written like any other
    single = Cache([20], 1, 16, torch.float16, seed=2)
    sisa_paged_decode_hip(*single.queries(), single.lam, single.pool, single.table, _ints(20), max_len=32, weights=one)
    row = cache.rows
    for bad in (dict(k=row["k"].float()), dict(v=row["v"][:, :1]), dict(b=row["k"]), dict(g=row["g"][:, :, :3]), dict(f=None),
                dict(start=n.long()), dict(count=n[:1]), dict(table=table[:1])):
        a = dict(pool=pool, table=table, start=_ints(0, 0), k=row["k"], v=row["v"], b=row["b"], g=row["g"], f=row["f"],
                 count=None) | bad
        with pytest.raises(ValueError):
            sisa_paged_write_hip(*a.values())
    other = PagePool.empty(4, 3, 16, torch.float16, DEV)
    for bad in (dict(recent=0), dict(recent=9), dict(new=other), dict(w=wide[:, :, :31]), dict(max_len=33),
                dict(new_table=table[:1]), dict(new_table=table[:, :0]), dict(w=wide.clone().requires_grad_(True))):
        a = dict(pool=pool, table=table, n=n, w=wide, keep=8, recent=2, new=pool, new_table=table) | bad
        args = [a.pop(x) for x in ("pool", "table", "n", "w", "keep", "recent", "new", "new_table")]
        with pytest.raises((ValueError, RuntimeError)):
            sisa_cache_evict_hip(*args, **a)
    # nothing to do
    none = sisa_paged_decode_hip(q[:0], c[:0], g[:0], f[:0], lam, pool, table[:0], n[:0])
    assert none.shape == (0, 2, 1, 64)
    assert sisa_paged_decode_hip(q[:, :, :0], c[:, :, :0], g[:, :, :0], f[:, :, :0], lam, pool, table, n).shape == (2, 2, 0, 64)
    sisa_paged_write_hip(pool, table[:0], n[:0], *(row[x][:0] for x in ("k", "v", "b", "g", "f")))
    got = sisa_cache_evict_hip(pool, table[:0], n[:0], wide[:0], 8, 2, pool, table[:0])
    assert got.lengths.shape == (0,) and got.weights.shape == got.positions.shape == (0, 2, 8)


def test_decode_beyond_32_bit_offsets():
    """Pages whose rows start past 2^31 elements, and 2^32 bytes, of their tensor."""
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip, sisa_paged_decode_hip, sisa_paged_write_hip
    S, H, P = 1024, 8, 4200                                  # 4200 x 8 x 1024 x 64 = 2.2e9 elements
    dt, gen = torch.float16, _gen(1)
    pool = PagePool.empty(P, H, S, dt, DEV)
    table = torch.tensor([[P - 1, 3], [P - 2, 4]], device=DEV, dtype=torch.int32)
    M = 1500
    new = lambda w: torch.randn(2, H, M, w, generator=gen, device=DEV).to(dt)  # noqa: E731
    k, v, b, g, f = new(64), new(64), new(32), _gates(gen, 2, H, M), _gates(gen, 2, H, M)
    sisa_paged_write_hip(pool, table, _ints(0, 0), k, v, b, g, f)
    assert torch.equal(pool.k[P - 1], k[0, :, :S]) and torch.equal(pool.g[4, :, :M - S], g[1, :, S:])
    lam, q, c = torch.rand(H, device=DEV), new(64)[:, :, :1], new(32)[:, :, :1]
    out = sisa_paged_decode_hip(q, c, g[:, :, -1:], f[:, :, -1:], lam, pool, table, _ints(M, M))
    small = PagePool.empty(4, H, S, dt, DEV)
    near = torch.tensor([[0, 1], [2, 3]], device=DEV, dtype=torch.int32)
    sisa_paged_write_hip(small, near, _ints(0, 0), k, v, b, g, f)
    assert torch.equal(out, sisa_paged_decode_hip(q, c, g[:, :, -1:], f[:, :, -1:], lam, small, near, _ints(M, M)))
    w = torch.rand(2, H, M, generator=gen, device=DEV)
    far = torch.tensor([[P - 3], [P - 4]], device=DEV, dtype=torch.int32)
    got = sisa_cache_evict_hip(pool, table, _ints(M, M), w, 700, 100, pool, far, max_len=M)
    picked = got.positions.long()
    for i, page in enumerate((P - 3, P - 4)):
        assert torch.equal(pool.v[page, :, :700], v[i].gather(1, picked[i, :, :, None].expand(-1, -1, 64)))


# ------------------------------------------------------------------------------------------------ write
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,counts,H,S,M", [([0], [1], 1, 16, 1), ([0, 31, 32, 33], None, 3, 32, 2),
                                                 ([5, 100, 0], [40, 0, 17], 2, 16, 40), ([63], [130], 12, 64, 130)])
def test_write(starts, counts, H, S, M, dtype):
    from sisa_amd.kernels.paged import sisa_paged_write_hip
    cache = Cache(starts, H, S, dtype, seed=H, room=M)
    before = {n: x.clone() for n, x in cache.t.items()}
    B = len(starts)
    # rows with strides of a (B, M, H, .) projection, k not 16-byte aligned (copied by the call)
    new = lambda w: torch.randn(B, M, H, w, generator=cache.gen, device=DEV).to(dtype).transpose(1, 2)  # noqa: E731
    k = torch.randn(B, H, M, 65, generator=cache.gen, device=DEV).to(dtype)[..., 1:]
    v, b, g, f = new(64), new(32), _gates(cache.gen, B, H, M), _gates(cache.gen, B, M, H).transpose(1, 2)
    sisa_paged_write_hip(cache.pool, cache.table, _ints(*starts), k, v, b, g, f,
                         None if counts is None else _ints(*counts))
    for i in range(B):
        for m in range(M if counts is None else counts[i]):
            page, slot = int(cache.table[i, (starts[i] + m) // S]), (starts[i] + m) % S
            for name, x in dict(k=k, v=v, b=b, g=g, f=f).items():
                before[name][page, :, slot] = x[i, :, m]
    for name, x in before.items():
        assert torch.equal(x.nan_to_num(9.0), cache.t[name].nan_to_num(9.0)), name


# 64 rows a wave: 134,400 rows, with waves that begin within a head, and 422,400, which are 256 MB and more read and written
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,M,S", [(3, 16, 2800, 64), (4, 16, 6600, 16)])
def test_write_of_many_rows(B, H, M, S, dtype):
    from sisa_amd.kernels.paged import PagePool, sisa_paged_write_hip
    gen, starts, counts = _gen(M), [(37 * n) % 100 for n in range(B)], [M, M - 1, 1, M // 2 + 3][:B]
    W = -(-(M + 100) // S)
    pool = PagePool.empty(B * W + 5, H, S, dtype, DEV)
    held = dict(k=pool.k, v=pool.v, b=pool.b, g=pool.g, f=pool.fgate)
    for t in held.values():
        t.fill_(7)
    table = torch.randperm(pool.pages, generator=gen, device=DEV)[:B * W].view(B, W).to(torch.int32)
    new = lambda *w: torch.randn(B, M, H, *w, generator=gen, device=DEV).transpose(1, 2)  # noqa: E731
    rows = dict(k=new(64).to(dtype), v=new(64).to(dtype), b=new(32).to(dtype), g=new(), f=new())
    want = {n: x.clone() for n, x in held.items()}
    for i in range(B):
        pos = starts[i] + torch.arange(counts[i], device=DEV)
        for n, x in rows.items():
            want[n][table[i].long()[pos // S], :, pos % S] = x[i, :, :counts[i]].transpose(0, 1)
    sisa_paged_write_hip(pool, table, _ints(*starts), *rows.values(), _ints(*counts))
    assert all(torch.equal(want[n], held[n]) for n in held)


def test_write_leaves_out_what_has_no_page():
    """Rows before position 0, past the table and on pages outside the pool, and counts above M or below 0."""
    from sisa_amd.kernels.paged import sisa_paged_write_hip
    cache = Cache([20, 20, 20, 20], 2, 16, torch.bfloat16, seed=2, room=12)
    table = cache.table.clone()
    assert table.shape == (4, 2)
    table[1, 1], table[2, 1] = cache.pool.pages, -1
    before = {n: x.clone() for n, x in cache.t.items()}
    M = 3
    one = lambda *w: torch.ones(4, 2, M, *w, device=DEV, dtype=torch.bfloat16)  # noqa: E731
    gates = torch.ones(4, 2, M, device=DEV)
    sisa_paged_write_hip(cache.pool, table, _ints(-1, 15, 16, 31), one(64), one(64), one(32), gates, gates, _ints(9, 9, 9, 9))
    sisa_paged_write_hip(cache.pool, table, _ints(1, 1, 1, 1), one(64), one(64), one(32), gates, gates, _ints(-1, 0, -7, 0))
    for name, x in cache.t.items():
        before[name][int(table[0, 0]), :, :2] = 1           # positions 0 and 1, 15 and 31: the only ones with a page
        before[name][int(table[1, 0]), :, 15] = 1
        before[name][int(table[3, 1]), :, 15] = 1
        assert torch.equal(x.nan_to_num(9.0), before[name].nan_to_num(9.0)), name


# ------------------------------------------------------------------------------------------------ eviction
def _chosen(w, n, keep, recent):
    """Positions that stay, by sorting: w (N,) of one head."""
    if n <= keep:
        return list(range(n))
    w = w[:n - recent].double()
    key = [(1 if math.isnan(x) else 0, 0.0 if math.isnan(x) else x) for x in w.tolist()]
    order = sorted(range(len(key)), key=lambda i: (-key[i][0], -key[i][1], i))[:keep - recent]
    return sorted(order) + list(range(n - recent, n))


def _evict_case(lengths, H, S, keep, recent, dtype, values, seed=0, S_new=None):
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip
    cache = Cache(lengths, H, S, dtype, seed=seed)
    N, S_new = max(1, max(lengths)), S_new or S
    w = values(cache.gen, cache.B, H, N + 3)
    to = PagePool.empty(cache.B * -(-keep // S_new) + 1, H, S_new, dtype, DEV)
    for t in (to.k, to.v, to.b, to.g, to.fgate):
        t.fill_(5)
    order = torch.randperm(to.pages, generator=cache.gen, device=DEV)[1:].to(torch.int32)
    table = order.view(cache.B, -1)
    old = {n: x.clone() for n, x in cache.t.items()}
    got = sisa_cache_evict_hip(cache.pool, cache.table, _ints(*lengths), w, keep, recent, to, table, max_len=N)
    assert got.lengths.tolist() == [min(n, keep) for n in lengths]
    hits = {n: torch.full_like(x, 5) for n, x in (("k", to.k), ("v", to.v), ("b", to.b), ("g", to.g), ("f", to.fgate))}
    for i, n in enumerate(lengths):
        for h in range(H):
            stay = _chosen(w[i, h], n, keep, recent)
            assert got.positions[i, h].tolist() == stay + [-1] * (keep - len(stay)), (i, h)
            at = torch.tensor(stay, device=DEV, dtype=torch.long)
            assert torch.equal(got.weights[i, h, :len(stay)].nan_to_num(9.0), w[i, h, at].nan_to_num(9.0))
            assert got.weights[i, h, len(stay):].eq(0).all()
            new = torch.arange(len(stay), device=DEV)
            for name, x in hits.items():
                x[table[i].long()[new // S_new], h, new % S_new] = cache.rows[name][i, h, at]
    for name, x in hits.items():
        assert torch.equal(x, {"k": to.k, "v": to.v, "b": to.b, "g": to.g, "f": to.fgate}[name]), name
        assert torch.equal(old[name].nan_to_num(9.0), cache.t[name].nan_to_num(9.0)), name


def _heavy(gen, *shape):
    return torch.exp(2.0 * torch.randn(shape, generator=gen, device=DEV))


def _tied(gen, *shape):
    return torch.randint(0, 3, shape, generator=gen, device=DEV).float() - 1.0


def _odd(gen, *shape):
    """NaN of both signs, infinities, zeros of both signs, subnormals, negative values."""
    menu = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, 1.0, -1.0, 3.0], device=DEV)
    return menu[torch.randint(0, len(menu), shape, generator=gen, device=DEV)]


@pytest.mark.parametrize("values", [_heavy, _tied, _odd])
@pytest.mark.parametrize("lengths,H,S,keep,recent", [([1], 1, 16, 1, 1), ([2, 1, 0], 2, 16, 1, 1),
                                                     ([40, 17, 18], 3, 16, 17, 3), ([300, 64, 65], 2, 32, 64, 64),
                                                     ([1025, 1, 2300], 2, 64, 500, 1), ([5000], 1, 1024, 4999, 30),
                                                     ([1200, 1100], 2, 128, 1099, 1000)])
def test_evict(lengths, H, S, keep, recent, values):
    _evict_case(lengths, H, S, keep, recent, torch.bfloat16, values, seed=keep)


@pytest.mark.parametrize("dtype", DTYPES)
def test_evict_to_another_page_size(dtype):
    _evict_case([333, 90], 3, 64, 100, 20, dtype, _heavy, seed=4, S_new=16)
    _evict_case([333, 90], 3, 16, 100, 20, dtype, _heavy, seed=5, S_new=128)


# as many positions as a thread holds 8, 16 and 24 of, and the edges between
@pytest.mark.parametrize("values", [_heavy, _tied, _odd])
@pytest.mark.parametrize("lengths,keep,recent", [([4097, 8192, 30], 700, 20), ([8193, 16384], 3000, 1000),
                                                 ([24576, 16385, 0, 12000], 9000, 1)])
def test_evict_of_more_positions_a_thread(lengths, keep, recent, values):
    _evict_case(lengths, 1, 1024, keep, recent, torch.float16, values, seed=keep)


@pytest.mark.parametrize("high,low", [(1e6, 1e-6), (0.0, -math.inf), (math.nan, math.inf), (-1.0, -2.0), (1.5, 1.4999999)])
@pytest.mark.parametrize("more", [0, 1, -1])
def test_evict_where_a_digit_settles_it(high, low, more):
    """As many positions of one weight as are picked, one more, or one fewer; all others of another."""
    def values(gen, B, H, n):
        w = torch.full((B, H, n), low, device=DEV)
        w[..., 3:3 + 40 + more] = high
        return w
    _evict_case([300, 53, 51], 2, 16, 50, 10, torch.bfloat16, values)


# 64 rows a wave: 134,400 kept rows, out of caches below and above 256 MB
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,S,S_new", [(4000, 64, 16), (17500, 128, 128)])
def test_evict_of_many_rows(n, S, S_new, dtype):
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip
    B, H, keep, recent, gen = 4, 12, 2800, 333, _gen(n)
    lengths = [n, n - 1, keep - 5, n // 2 + 1000]
    W, W_new = -(-n // S), -(-keep // S_new)
    pool, to = PagePool.empty(B * W, H, S, dtype, DEV), PagePool.empty(B * W_new + 3, H, S_new, dtype, DEV)
    old, new = (dict(k=p.k, v=p.v, b=p.b, g=p.g, f=p.fgate) for p in (pool, to))
    for t in old.values():
        t.copy_(torch.randn(t.shape, generator=gen, device=DEV, dtype=torch.float32))
    for t in new.values():
        t.fill_(7)
    table = torch.randperm(pool.pages, generator=gen, device=DEV).view(B, W).to(torch.int32)
    new_table = torch.randperm(to.pages, generator=gen, device=DEV)[:B * W_new].view(B, W_new).to(torch.int32)
    w = _heavy(gen, B, H, n)
    want, i = {x: t.clone() for x, t in new.items()}, torch.arange(keep, device=DEV)
    got = sisa_cache_evict_hip(pool, table, _ints(*lengths), w, keep, recent, to, new_table, max_len=n)
    assert got.lengths.tolist() == [min(m, keep) for m in lengths]
    for m in range(B):
        N, K = lengths[m], min(lengths[m], keep)
        if N <= keep:
            stay = i[:K].expand(H, K)
        else:
            order = w[m, :, :N - recent].sort(descending=True, stable=True).indices[:, :keep - recent]
            stay = torch.cat([order.sort().values, torch.arange(N - recent, N, device=DEV).expand(H, recent)], 1)
        assert torch.equal(got.positions[m, :, :K].long(), stay) and got.positions[m, :, K:].eq(-1).all()
        assert torch.equal(got.weights[m, :, :K], w[m].gather(1, stay)) and got.weights[m, :, K:].eq(0).all()
        h = torch.arange(H, device=DEV)[:, None].expand_as(stay)
        for x in want:
            want[x][new_table[m].long()[i[:K] // S_new].expand(H, K), h, (i[:K] % S_new).expand(H, K)] = \
                old[x][table[m].long()[stay // S], h, stay % S]
    assert all(torch.equal(want[x], new[x]) for x in new)


def test_evict_of_a_long_cache():
    """More positions than a workgroup keeps at once; equal weights, of which the lowest stay, among them."""
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip
    n, keep, recent, S = 150_001, 60_000, 777, 1024
    gen = _gen(6)
    W = -(-n // S)
    pool = PagePool.empty(W, 1, S, torch.float16, DEV)
    to = PagePool.empty(-(-keep // S), 1, S, torch.float16, DEV)
    pool.g.copy_(torch.arange(W * S, device=DEV).view(W, 1, S))
    table, new = (torch.arange(p.pages, device=DEV, dtype=torch.int32)[None] for p in (pool, to))
    for w in (torch.rand(1, 1, n, generator=gen, device=DEV), torch.randint(0, 2, (1, 1, n), generator=gen, device=DEV).float(),
              torch.ones(1, 1, n, device=DEV)):
        got = sisa_cache_evict_hip(pool, table, _ints(n), w, keep, recent, to, new, max_len=n)
        order = w[0, 0, :n - recent].sort(descending=True, stable=True).indices[:keep - recent].sort().values
        want = torch.cat([order, torch.arange(n - recent, n, device=DEV)])
        assert torch.equal(got.positions[0, 0].long(), want)
        assert torch.equal(to.g.transpose(0, 1).flatten()[:keep].long(), want)


def test_evict_marks_lengths_and_pages_outside_the_pool():
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip
    cache = Cache([90] * 6, 2, 16, torch.bfloat16, seed=8)
    table = cache.table.clone()
    table[1, 5], table[2, 5] = -1, cache.pool.pages          # the page of the last, recent positions
    to = PagePool.empty(12, 2, 16, torch.bfloat16, DEV)
    new = torch.arange(12, device=DEV, dtype=torch.int32).view(6, 2)
    new[5, 1] = 12
    w = torch.rand(6, 2, 96, device=DEV)
    got = sisa_cache_evict_hip(cache.pool, table, _ints(90, 90, 90, -1, 97, 90), w, 30, 10, to, new, max_len=96)
    assert got.lengths.tolist() == [30, -1, -1, -1, -1, -1]
    short = sisa_cache_evict_hip(cache.pool, cache.table, _ints(90, 16, 15, 0, 90, 90), w, 30, 10, to, new[:, :1], max_len=96)
    assert short.lengths.tolist() == [-1, 16, 15, 0, -1, -1]                     # one new page holds 16


def test_tokens_after_an_eviction_that_could_not_be_done():
    """Negative lengths are kept as they are: NaN for every later token of their sequences, nothing in their pages."""
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip, sisa_paged_decode_hip, sisa_paged_write_hip
    cache = Cache([90] * 5, 2, 16, torch.bfloat16, seed=14)
    table, keep = cache.table.clone(), 30
    table[1, 5] = -1                                         # the page of the last, recent positions
    w = torch.rand(5, 2, 96, generator=cache.gen, device=DEV)
    w[4, :, 16:32] = -1.0                                    # none of these stays: their page is not looked at
    table[4, 1] = cache.pool.pages
    to = PagePool.empty(20, 2, 16, torch.bfloat16, DEV)
    for t in (to.k, to.v, to.b, to.g, to.fgate):
        t.zero_()
    new = torch.arange(20, device=DEV, dtype=torch.int32).view(5, 4)
    new[2, 1] = 20
    got = sisa_cache_evict_hip(cache.pool, table, _ints(90, 90, 90, 97, 90), w, keep, 10, to, new, max_len=96)
    assert got.lengths.tolist() == [keep, -1, -1, -1, keep]
    whole = sisa_cache_evict_hip(cache.pool, cache.table, _ints(90, 90, 90, 90, 90), w, keep, 10,
                                 PagePool.empty(10, 2, 16, torch.bfloat16, DEV),
                                 torch.arange(10, device=DEV, dtype=torch.int32).view(5, 2), max_len=96)
    assert torch.equal(got.positions[4], whole.positions[4]) and torch.equal(got.weights[4], whole.weights[4])
    held, kept = got.lengths, got.positions.long()
    rows = {n: x.gather(2, kept.clamp(min=0)[..., None].expand(-1, -1, -1, x.shape[3]) if x.dim() == 4 else kept.clamp(min=0))
            for n, x in cache.rows.items()}
    pages = {n: x.clone() for n, x in (("k", to.k), ("g", to.g))}
    for step in range(3):
        q, c, g, f = cache.queries()
        g, f = g - 1 - step, f - 1 - step
        k, v, b = (torch.randn(5, 2, 1, wd, generator=cache.gen, device=DEV).to(torch.bfloat16) for wd in (64, 64, 32))
        sisa_paged_write_hip(to, new, held, k, v, b, g, f)
        held = torch.where(held < 0, held, held + 1)
        out = sisa_paged_decode_hip(q, c, g, f, cache.lam, to, new, held, max_len=64)
        rows = {n: torch.cat([rows[n], x], 2) for n, x in dict(k=k, v=v, b=b, g=g, f=f).items()}
        assert out[1:4].isnan().all()
        near = Cache.__new__(Cache)
        near.__dict__.update(cache.__dict__, rows=rows, lengths=[keep + step + 1] * 5)
        want, _ = near.decode64(q, c, g, f)
        for i in (0, 4):
            assert _rel(out[i], want[i]) <= TOL
    assert torch.equal(to.k[4:16], pages["k"][4:16]) and torch.equal(to.g[4:16], pages["g"][4:16])


# ------------------------------------------------------------------------------------------------ received weights
def _weights64(q, k, c, b, g, lam, f, lengths, window):
    out = torch.zeros(g.shape, device=DEV, dtype=torch.float64)
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        first = max(0, n - (window or n))
        x = [t[i, :, :n].double() for t in (q, k, c, b, g)]
        s = x[0] @ x[1].mT / 8 + lam.double()[:, None, None] * (x[4][:, :, None] - x[4][:, None]).exp() * (x[2] @ x[3].mT)
        if f is not None:
            s = s + f[i, :, :n, None].double() - f[i, :, None, :n].double()
        hidden = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
        out[i, :, :n] = s.masked_fill(hidden, -math.inf).softmax(-1).masked_fill(hidden, 0.0)[:, first:].sum(1)
    return out


# lengths at the edges of 16-position tiles, 64-position blocks and key splits; windows of one query, within a tile, across
# blocks and longer than a sequence; ragged batches with an empty sequence, NaN behind their ends
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,L,H,window", [([1], 1, 1, None), ([15, 16, 17], 17, 2, None), ([64, 63, 65], 65, 2, None),
                                                ([200, 0, 1, 129], 200, 3, None), ([257, 90], 300, 2, 1),
                                                ([257, 9, 258], 258, 2, 16), ([600, 70, 31], 601, 2, 67),
                                                ([1500], 1500, 2, 64), ([513], 513, 5, 512), ([33, 20], 33, 2, 500)])
def test_received_weights(lengths, L, H, window, dtype):
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    gen, B = _gen(L + H), len(lengths)
    rows = lambda w: torch.randn(B, L, H, w, generator=gen, device=DEV).to(dtype).transpose(1, 2)  # noqa: E731
    x = [rows(64), rows(64), rows(32), rows(32), _gates(gen, B, H, L)]
    f = _gates(gen, B, H, L)
    lam = torch.rand(H, generator=gen, device=DEV) + 0.1
    for t in (*x, f):
        for i, n in enumerate(lengths):
            t[i, :, n:] = math.nan
    for forget in (f, None):
        want = _weights64(*x, lam, forget, lengths, window)
        got = sisa_attention_weights_hip(*x, lam, forget, lengths=_ints(*lengths), window=window)
        assert _rel(got, want) <= TOL
        assert all(got[i, :, n:].eq(0).all() for i, n in enumerate(lengths))
        # every query's weights sum to one
        count = torch.tensor([min(n, window or n) for n in lengths], device=DEV, dtype=torch.float64)
        assert (got.double().sum(-1) - count[:, None]).abs().max() <= 1e-5 * max(1.0, float(count.max()))
        assert torch.equal(got, sisa_attention_weights_hip(*x, lam, forget, lengths=_ints(*lengths), window=window))
    if B == 1:
        clamped = sisa_attention_weights_hip(*x, lam, f, lengths=_ints(10 * L), window=window)
        assert torch.equal(clamped, sisa_attention_weights_hip(*x, lam, f, window=window))
        assert sisa_attention_weights_hip(*x, lam, f, lengths=_ints(-4), window=window).eq(0).all()


# heads and sequences enough for every width of the blocks: 135 to 720 blocks of 64 rows; whole tiles, an anchor
# within a block, ends at the edges of 16 and 32
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,L,H,window", [([130, 0, 64, 95], 130, 12, None), ([530, 300, 33], 530, 9, 280),
                                                ([129, 97, 128, 32, 1, 79], 129, 20, None), ([400, 127], 400, 24, None),
                                                ([130, 33, 31, 130, 7, 96, 64, 65], 130, 30, None)])
def test_received_weights_of_many_heads(lengths, L, H, window, dtype):
    test_received_weights(lengths, L, H, window, dtype)


# windows whose first pass is split into 11, 32 and (256 blocks of 64 rows) no parts; and on either side of 256, where the
# keys are no longer split
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,L,H,window", [([2600, 50], 2600, 2, 17), ([9000], 9000, 1, 64), ([8200, 3, 4100], 8200, 2, 65),
                                                ([450, 449, 99, 300, 0, 1, 101, 400], 450, 16, 100), ([4000], 4000, 2, 256),
                                                ([4000, 700], 4000, 2, 257), ([4001], 4001, 4, 1000)])
def test_received_weights_of_windows_of_long_prompts(lengths, L, H, window, dtype):
    test_received_weights(lengths, L, H, window, dtype)


def test_received_weights_with_steep_gates():
    """Gates that fall by tens per position, and by hundreds over the sequence: the weights gather on the diagonal, and
    what underflows is 0."""
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    gen, L, H = _gen(11), 400, 3
    rows = lambda w: torch.randn(1, H, L, w, generator=gen, device=DEV).to(torch.bfloat16)  # noqa: E731
    x = [rows(64), rows(64), rows(32), rows(32)]
    for step_g, step_f in ((0.0, 40.0), (60.0, 0.01), (30.0, 30.0), (1000.0, 0.0)):
        g, f = (-(s * torch.rand(1, H, L, generator=gen, device=DEV)).cumsum(-1) for s in (step_g, step_f))
        lam = torch.tensor([0.3, 4.0, 0.0], device=DEV)
        got = sisa_attention_weights_hip(*x, g, lam, f)
        # |F| reaches 16,000 here: a difference of two is exact to 2^-24 of the larger in both, the inputs being the same
        assert _rel(got, _weights64(*x, g, lam, f, [L], None)) <= TOL


# Gates that rise again, by more than a factor of the kernels' may hold. The scores' own decays stay moderate: where keys lie
# below a query's g by `dip`, lam is e^-dip; F differences stay below 40, as the tolerance has them. A few heads (16 queries a
# block), many, a window (its queries lie below every key, whose blocks rise and fall among themselves by more than 88).
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,L,window", [(1, 3, 300, None), (2, 24, 210, None), (2, 30, 700, None), (2, 3, 700, 64),
                                          (1, 2, 1100, 300)])
def test_received_weights_with_rising_gates(B, H, L, window, dtype):
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    gen = _gen(L + H)
    rows = lambda w: torch.randn(B, L, H, w, generator=gen, device=DEV).to(dtype).transpose(1, 2)  # noqa: E731
    x = [rows(64), rows(64), rows(32), rows(32)]
    lengths = [L, 150][:B]
    at = torch.arange(L, device=DEV)
    for dip, f_dip in ((0.0, 30.0), (30.0, 0.0), (40.0, 30.0), (110.0, 0.0)):
        if dip > 88 and window is None:
            continue
        lam = torch.rand(H, generator=gen, device=DEV) * math.exp(-min(dip, 40.0) if window is None else 0.0)
        g, f = _gates(gen, B, H, L), _gates(gen, B, H, L)
        for n, i in zip(lengths, range(B)):
            low = ((at // 37) % 2 == 1) & (at < n - (window or 0))           # by turns, across every block's edges
            g[i, :, low] -= dip
            f[i, :, low] -= f_dip
            if window is not None:                                           # the queries that count lie below all keys
                g[i, :, max(0, n - window):] -= dip + 10
                f[i, :, max(0, n - window):] -= f_dip
        got = sisa_attention_weights_hip(*x, g, lam, f, lengths=_ints(*lengths), window=window)
        assert _rel(got, _weights64(*x, g, lam, f, lengths, window)) <= TOL, (dip, f_dip)
        if dip:
            got = sisa_attention_weights_hip(*x, g, lam, lengths=_ints(*lengths), window=window)
            assert _rel(got, _weights64(*x, g, lam, None, lengths, window)) <= TOL, (dip, f_dip)


@pytest.mark.parametrize("window", [40, 300])
@pytest.mark.parametrize("j", [63, 64, 127, 15, 16, 200])
def test_received_weights_of_keys_that_are_forgotten(j, window):
    """F or g of +inf at a key that no counted query is: it receives 0, the others what they would without it."""
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    gen, L, H = _gen(j), 700, 2
    rows = lambda w: torch.randn(1, H, L, w, generator=gen, device=DEV)  # noqa: E731
    x = [rows(64), rows(64), rows(32), rows(32)]
    g, f, lam = _gates(gen, 1, H, L), _gates(gen, 1, H, L), torch.rand(H, generator=gen, device=DEV) + 0.1
    f[0, 0, j] = g[0, 1, j] = math.inf
    got = sisa_attention_weights_hip(*x, g, lam, f, window=window)
    assert got.isfinite().all() and got[0, 0, j] == 0
    assert _rel(got, _weights64(*x, g, lam, f, [L], window)) <= TOL


def test_received_weights_of_other_layouts():
    """Positions far apart in memory, gates that are not neighbours, expanded ones, rows that begin off 16 bytes: copied."""
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    gen, B, H, L = _gen(17), 2, 3, 70
    x = [torch.randn(B, H, L, w, generator=gen, device=DEV).to(torch.float16) for w in (64, 64, 32, 32)]
    g, f = _gates(gen, B, H, L), _gates(gen, B, L, H).transpose(1, 2)
    lam = torch.rand(1, device=DEV).expand(H)
    off = torch.zeros(B, H, L, 65, device=DEV, dtype=torch.float16)
    off[..., 1:] = x[1]
    got = sisa_attention_weights_hip(x[0].transpose(0, 2).contiguous().transpose(0, 2), off[..., 1:], x[2], x[3], g, lam, f)
    assert torch.equal(got, sisa_attention_weights_hip(*x, g, lam.contiguous(), f.contiguous()))
    flat = torch.zeros(B, H, 1, device=DEV)                     # no decay, no forgetting: one value for every position
    got = sisa_attention_weights_hip(*x, flat.expand(B, H, L), lam, flat.expand(B, H, L))
    assert _rel(got, _weights64(*x, flat.expand(B, H, L), lam, None, [L] * B, None)) <= TOL


def test_received_weights_of_values_that_are_not_finite():
    """A query with NaN makes its own weights NaN, those of positions up to it; other heads are not touched."""
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    gen, L, H = _gen(12), 150, 2
    rows = lambda w: torch.randn(1, H, L, w, generator=gen, device=DEV)  # noqa: E731
    x = [rows(64), rows(64), rows(32), rows(32), _gates(gen, 1, H, L)]
    f, lam = _gates(gen, 1, H, L), torch.ones(H, device=DEV)
    x[0][0, 0, 70, 3] = math.nan
    got = sisa_attention_weights_hip(*x, lam, f)
    assert got[0, 0, :71].isnan().all() and not got[0, 0, 71:].isnan().any() and not got[0, 1].isnan().any()
    want = _weights64(*x, lam, f, [L], None)
    assert _rel(got[0, 0, 71:], want[0, 0, 71:]) <= TOL and _rel(got[0, 1], want[0, 1]) <= TOL


# ------------------------------------------------------------------------------------------------ together
def test_a_prompt_evicted_and_continued():
    """Prompts of unequal lengths written to pages, their received weights, the cache cut by them, then tokens written and
    attended with tracking, and cut again: against a softmax in float64 over the rows that stayed."""
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip, sisa_paged_decode_hip, sisa_paged_write_hip
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    gen, B, H, L, S, keep, recent, dt = _gen(21), 3, 4, 200, 16, 48, 12, torch.bfloat16
    lengths, T = [200, 131, 30], 230
    rows = lambda w: torch.randn(B, H, T, w, generator=gen, device=DEV).to(dt)  # noqa: E731
    q, k, v, c, b = rows(64), rows(64), rows(64), rows(32), rows(32)
    g, f, lam = _gates(gen, B, H, T), _gates(gen, B, H, T), torch.rand(H, generator=gen, device=DEV)
    pool = PagePool.empty(120, H, S, dt, DEV)
    free = list(range(120))
    take = lambda n: torch.tensor([[free.pop() for _ in range(n)] for _ in range(B)], device=DEV, dtype=torch.int32)  # noqa: E731
    cut = lambda t, n=L: t[:, :, :n]  # noqa: E731
    table, held = take(13), _ints(*lengths)
    sisa_paged_write_hip(pool, table, _ints(0, 0, 0), cut(k), cut(v), cut(b), cut(g), cut(f), held)
    w = torch.zeros(B, H, 208, device=DEV)
    w[:, :, :L] = sisa_attention_weights_hip(cut(q), cut(k), cut(c), cut(b), cut(g), lam, cut(f), lengths=held)
    stay = [[list(range(n)) for _ in range(H)] for n in lengths]           # original positions in the cache
    w64 = w.double()
    at = list(lengths)
    for round_ in range(2):
        new = take(5)
        got = sisa_cache_evict_hip(pool, table, held, w, keep, recent, pool, new, max_len=w.shape[2])
        for i in range(B):
            n = len(stay[i][0])
            for h in range(H):
                stay[i][h] = [stay[i][h][j] for j in _chosen(w[i, h], n, keep, recent)]
                picked = got.positions[i, h, :len(stay[i][h])].long()
                assert _rel(got.weights[i, h, :len(picked)], w64[i, h, picked]) <= 2 * TOL
        table, held = new, got.lengths
        w = torch.cat([got.weights, torch.zeros(B, H, 80 - keep, device=DEV)], 2)
        w64 = w.double()
        for _ in range(10):
            sel = torch.tensor(at, device=DEV)
            pick = lambda t: t[torch.arange(B, device=DEV), :, sel][:, :, None]  # noqa: E731
            sisa_paged_write_hip(pool, table, held, pick(k), pick(v), pick(b), pick(g), pick(f))
            held = held + 1
            out = sisa_paged_decode_hip(pick(q), pick(c), pick(g), pick(f), lam, pool, table, held, max_len=80, weights=w)
            for i in range(B):
                for h in range(H):
                    stay[i][h].append(at[i])
                    j = torch.tensor(stay[i][h], device=DEV)
                    s = k[i, h, j].double() @ q[i, h, at[i]].double() / 8 + lam[h].double() * (
                        g[i, h, at[i]].double() - g[i, h, j].double()).exp() * (b[i, h, j].double() @ c[i, h, at[i]].double())
                    p = (s + f[i, h, at[i]].double() - f[i, h, j].double()).softmax(0)
                    assert _rel(out[i, h, 0], p @ v[i, h, j].double()) <= TOL
                    w64[i, h, :len(j)] += p
                at[i] += 1
            assert _rel(w, w64) <= 2 * TOL


def test_captured_and_replayed_on_another_stream():
    """One graph of a step (write, attention with tracking, eviction into other pages) replayed with other lengths, tables
    and rows, with eager calls between, and a second graph beside it."""
    from sisa_amd.kernels.paged import PagePool, sisa_cache_evict_hip, sisa_paged_decode_hip, sisa_paged_write_hip
    from sisa_amd.kernels.weights import sisa_attention_weights_hip
    H, S, keep, recent = 3, 32, 64, 16
    cache = Cache([150, 37], H, S, torch.float16, seed=13, room=8)
    to = PagePool.empty(4, H, S, torch.float16, DEV)
    new = torch.arange(4, device=DEV, dtype=torch.int32).view(2, 2)
    held = _ints(150, 37)
    w, w2 = torch.rand(2, H, 160, generator=cache.gen, device=DEV), torch.zeros(2, H, 160, device=DEV)
    row = lambda wd: torch.randn(2, H, 1, wd, generator=cache.gen, device=DEV).to(torch.float16)  # noqa: E731
    q, k, v, c, b = row(64), row(64), row(64), row(32), row(32)
    g, f = (-torch.rand(2, H, 1, generator=cache.gen, device=DEV) - 4 for _ in range(2))

    def step():
        sisa_paged_write_hip(cache.pool, cache.table, held, k, v, b, g, f)
        n = held + 1
        out = sisa_paged_decode_hip(q, c, g, f, cache.lam, cache.pool, cache.table, n, max_len=160, weights=w, weights_out=w2)
        return (out, w2, *sisa_cache_evict_hip(cache.pool, cache.table, n, w2, keep, recent, to, new, max_len=160), to.k)

    px = [torch.randn(1, H, 90, wd, generator=cache.gen, device=DEV).to(torch.float16) for wd in (64, 64, 32, 32)]
    pg, pf, plen = _gates(cache.gen, 1, H, 90), _gates(cache.gen, 1, H, 90), _ints(90)

    def prompt():
        return sisa_attention_weights_hip(*px, pg, cache.lam, pf, lengths=plen, window=40)

    step(), prompt()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for fn in (step, prompt):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                res = fn()
            graphs.append((graph, res))
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        for t in (q, k, v, c, b):
            t.copy_(torch.randn(t.shape, generator=cache.gen, device=DEV))
        held.copy_(_ints(150 - 40 * turn, 37 - 3 * turn))
        plen.copy_(_ints(90 - 29 * turn))
        w.copy_(torch.rand(w.shape, generator=cache.gen, device=DEV))
        # only what the step keeps is compared: pages it does not write hold the last turn's rows on both sides
        w2.zero_(), to.k.zero_()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in graphs[0][1]], graphs[1][1].clone()
        w2.zero_(), to.k.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = [x.clone() for x in step()], prompt()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(replayed[0], eager[0])) and torch.equal(replayed[1], eager[1]), turn
