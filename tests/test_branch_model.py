"""Branches of a prompt and positions that are taken back: SISAPagedCache.branch, tentative and keep, and generate(samples=,
draft=), on the CPU in float64 against caches that hold one continuation each, on the GPU against float64 and the module path."""
import pytest
import torch

from model_utils import rel_err, tiny_model, token_ids
from sisa_amd import SISAPagedCache, generate
from sisa_amd.generation import verify_drafts
from test_branch_gpu import _want

DEV = "cuda:0"

# The gates are float32 in a float64 model, and torch rounds their functions differently in a vector's body and its tail, so
# in passes of other shapes. Here their sums are below 64 in magnitude and of at most 60 steps, each rounded by at most 2^-19
# (half a step below 64) on either side: scores differ by at most 2 * 2 * 60 * 2^-19 = 4.6e-4 in g and F together, weights by
# 9.2e-4 of themselves, logits after two layers by no more than a few of that.
GATES = 2e-3


def _model64(**kw):
    return tiny_model(seed=3, theta_scale=0.25, **kw).double().eval()


def _alone(model, prompt, tokens):
    """Logits of a prompt's last position and of the tokens behind it, one by one, from a cache of their own."""
    cache = SISAPagedCache(1, prompt.numel() + tokens.numel(), page_size=16)
    out = [model(prompt[None], cache=cache, logits_to_keep=1).logits]
    out += [model(tokens[None, t:t + 1], cache=cache).logits for t in range(tokens.numel())]
    return torch.cat(out, 1)[0]


def _branched(model, ids, lengths, n, pages=None, room=24):
    k = len(lengths)
    cache = SISAPagedCache(k * n, max(lengths) + room, page_size=16, pages=pages)
    cache[:k].expect(lengths)
    first = model(ids[:k], cache=cache[:k], logits_at=[m - 1 for m in lengths]).logits
    cache.branch(n)
    return cache, first


# a prompt that ends in a page, at its end, inside its first, and of one token
@torch.no_grad()
@pytest.mark.parametrize("lengths", [[37], [32, 16, 5], [1, 40]])
def test_branches_continue_as_each_would_alone(lengths):
    model, n, steps = _model64(), 3, 8
    ids, k = token_ids(len(lengths), max(lengths), seed=1), len(lengths)
    tokens = token_ids(k * n, steps, seed=2)
    cache, first = _branched(model, ids, lengths, n)
    assert cache.lengths == [m for m in lengths for _ in range(n)]
    shared = sum(m // 16 for m in lengths)
    assert cache._store.pages - cache.free_pages == shared + n * sum(m % 16 > 0 for m in lengths)
    got = [model(tokens[:, :3], cache=cache).logits] + [model(tokens[:, t:t + 1], cache=cache).logits for t in range(3, steps)]
    got = torch.cat(got, 1)
    for i, m in enumerate(lengths):
        for b in range(i * n, i * n + n):
            want = _alone(model, ids[i, :m], tokens[b])
            assert rel_err(got[b], want[1:]) <= GATES and rel_err(first[i, 0], want[0]) <= GATES
    # a branch that ends leaves the others theirs, and takes another prompt
    cache[1].release()
    other = token_ids(1, 20, seed=4)
    held = model(other, cache=cache[1], logits_to_keep=1).logits
    more = token_ids(k * n, 2, seed=5)
    late = torch.cat([model(more[:, t:t + 1], cache=cache).logits for t in range(2)], 1)
    assert cache.lengths == [steps + 2 + m if j != 1 else 22 for j, m in enumerate(m for m in lengths for _ in range(n))]
    for i, m in enumerate(lengths):
        for b in range(i * n, i * n + n):
            prompt, behind = (other[0], more[b]) if b == 1 else (ids[i, :m], torch.cat([tokens[b], more[b]]))
            assert rel_err(late[b], _alone(model, prompt, behind)[-2:]) <= GATES
    assert rel_err(held[0, 0], _alone(model, other[0], more[1])[0]) <= GATES
    cache.release()
    assert cache.free_pages == cache._store.pages and sorted(cache._store.free) == list(range(cache._store.pages))
    assert not cache._store.others


@torch.no_grad()
def test_branch_takes_reserved_pages_back_and_refuses():
    model, ids = _model64(), token_ids(2, 20, seed=6)
    cache = SISAPagedCache(4, 40, page_size=16, pages=6)
    cache[:2].expect([20, 20])
    model(ids, cache=cache[:2])
    cache[2].reserve(16)
    assert cache.free_pages == 1
    cache.branch(2)                                       # two copies: the free page and the reserved one
    assert cache.free_pages == 0 and cache.lengths == [20] * 4
    cache[0].release()
    assert cache.free_pages == 1                          # its copy of the page that was not full
    few = SISAPagedCache(4, 40, page_size=16, pages=4)
    model(ids[:1], cache=few[0])
    before = (few.lengths, few.free_pages)
    with pytest.raises(RuntimeError, match="3 pages are needed"):
        few.branch(4)
    assert (few.lengths, few.free_pages) == before and not few._store.others
    for bad, word in ((lambda c: c.branch(3), "prompts of n = 3"), (lambda c: c.branch(0), "n = 0"), (lambda c: c.branch(4), "empty")):
        c = SISAPagedCache(4, 40, page_size=16)
        model(ids, cache=c[:2])
        with pytest.raises(ValueError, match=word):
            bad(c)
    tracked = SISAPagedCache(4, 40, track=True)
    model(ids, cache=tracked[:2])
    with pytest.raises(ValueError, match="track=True"):
        tracked.branch(2)
    with pytest.raises(ValueError, match="track=True"):
        tracked[:2].tentative(3)
    with pytest.raises(ValueError, match="empty"):
        SISAPagedCache(2, 10).branch(2)


@torch.no_grad()
@pytest.mark.parametrize("passes", [[5], [1, 1, 1, 1, 1], [2, 3]])
def test_kept_positions_continue_as_if_the_others_had_not_been(passes):
    model, lengths = _model64(), [30, 16, 7]
    ids = token_ids(3, 30, seed=7)
    cache = SISAPagedCache(3, 64, page_size=16)
    cache.expect(lengths)
    model(ids, cache=cache)
    seen = [ids[i, :m].tolist() for i, m in enumerate(lengths)]
    for turn, counts in enumerate(([2, 0, 5], [5, 5, 5], [1, 3, 0])):
        tokens = token_ids(3, 5, seed=20 + turn)
        cache.tentative(6)
        at, got = 0, []
        for m in passes:
            got.append(model(tokens[:, at:at + m], cache=cache).logits)
            at += m
        got = torch.cat(got, 1)
        for i in range(3):
            want = _alone(model, torch.tensor(seen[i]), tokens[i])[1:]
            assert rel_err(got[i], want) <= GATES
        cache.keep(counts)
        seen = [s + tokens[i, :c].tolist() for i, (s, c) in enumerate(zip(seen, counts))]
        assert cache.lengths == [len(s) for s in seen]
    cache.tentative(2)
    cache.keep([0, 0, 0])                                 # nothing was proposed
    step = token_ids(3, 1, seed=30)
    got = model(step, cache=cache).logits
    for i in range(3):
        assert rel_err(got[i], _alone(model, torch.tensor(seen[i]), step[i])[1:]) <= GATES


@torch.no_grad()
def test_branches_and_drafts_at_once():
    model, n = _model64(), 2
    ids, tokens, more = token_ids(1, 20, seed=8), token_ids(2, 4, seed=9), token_ids(2, 1, seed=10)
    cache, _ = _branched(model, ids, [20], n)
    cache.tentative(4)
    got = model(tokens, cache=cache).logits
    cache.keep([1, 3])
    after = model(more, cache=cache).logits
    for b, c in enumerate((1, 3)):
        assert rel_err(got[b], _alone(model, ids[0], tokens[b])[1:]) <= GATES
        assert rel_err(after[b], _alone(model, ids[0], torch.cat([tokens[b, :c], more[b]]))[-1:]) <= GATES


@torch.no_grad()
def test_tentative_and_keep_refuse():
    model, ids = _model64(), token_ids(2, 10, seed=11)
    cache = SISAPagedCache(2, 20, page_size=16)
    with pytest.raises(ValueError, match="empty"):
        cache.tentative(2)
    model(ids, cache=cache)
    with pytest.raises(RuntimeError, match="comes first"):
        cache.keep([0, 0])
    with pytest.raises(ValueError, match="positive"):
        cache.tentative(0)
    cache.tentative(3)
    for call in (lambda: cache.tentative(1), lambda: cache[0].tentative(1), lambda: cache.branch(1)):
        with pytest.raises(RuntimeError, match="keep"):
            call()
    with pytest.raises(ValueError, match="all of them"):
        model(ids[:1, :1], cache=cache[0])
    with pytest.raises(ValueError, match="3 positions"):
        model(ids[:, :4], cache=cache)
    assert cache.lengths == [10, 10]
    model(ids[:, :2], cache=cache)
    for bad in ([3, 0], [0], [-1, 0]):
        with pytest.raises(ValueError, match="0 .. 2"):
            cache.keep(bad)
    with pytest.raises(RuntimeError, match="same sequences"):
        cache[0].keep([1])
    cache[0].release()                                    # what was tentative is gone with it
    with pytest.raises(RuntimeError, match="comes first"):
        cache.keep([1, 1])
    assert cache.lengths == [0, 12]


# ------------------------------------------------------------------------------------------------ generate
def test_generate_samples():
    model, ids, lengths = _model64(), token_ids(3, 24, seed=8), [24, 3, 11]
    want = generate(model, ids, 9, prompt_lengths=lengths)
    got = generate(model, ids, 9, prompt_lengths=lengths, samples=2)
    assert torch.equal(got, want.repeat_interleave(2, 0))
    assert torch.equal(generate(model, ids, 9, samples=3), generate(model, ids, 9).repeat_interleave(3, 0))
    one = generate(model, ids[0], 5, samples=4)
    assert one.shape == (4, 29) and torch.equal(one[3], generate(model, ids[0], 5))
    stop = int(want[1, 5])
    ended = generate(model, ids, 9, prompt_lengths=lengths, eos_token_id=[stop, 300], samples=2)
    assert torch.equal(ended, generate(model, ids, 9, prompt_lengths=lengths, eos_token_id=[stop, 300]).repeat_interleave(2, 0))
    gen = torch.Generator().manual_seed(1)
    drawn = generate(model, ids, 12, do_sample=True, samples=3, generator=gen)
    assert drawn.shape == (9, 36) and not torch.equal(drawn[0], drawn[1])


def test_generate_samples_holds_what_is_shared_once(monkeypatch):
    """The pool is of a prompt's whole pages once, and of each sample's own: enough for all, and all taken at the end (but for
    the last token, which is not cached)."""
    from sisa_amd import generation
    made = []
    monkeypatch.setattr(generation, "SISAPagedCache", lambda *a, **kw: made.append(SISAPagedCache(*a, **kw)) or made[-1])
    model = _model64()
    for lengths, n, new in (([300], 16, 5), ([64, 200, 1, 129], 3, 70), ([63, 128], 2, 1), ([128], 4, 65), ([130, 63], 5, 2)):
        ids = token_ids(len(lengths), max(lengths), seed=9)
        got = generate(model, ids, new, prompt_lengths=lengths, samples=n)
        assert torch.equal(got, generate(model, ids, new, prompt_lengths=lengths).repeat_interleave(n, 0))
        cache = next(c for c in made if len(c) == n * len(lengths))
        made.clear()
        most = sum(m // 64 + n * (-(-(m + new) // 64) - m // 64) for m in lengths)
        held = sum(m // 64 + n * (-(-(m + new - 1) // 64) - m // 64) for m in lengths)
        assert cache._store.pages == most and cache._store.pages - cache.free_pages == held
    generate(model, ids, 3, samples=2)
    assert made[0]._store.pages == 2 * (2 + 2 * 1)


def test_generate_with_a_draft():
    model, ids, lengths = _model64(), token_ids(3, 24, seed=8), [24, 3, 11]
    small = tiny_model(seed=5, n_layer=1).double().eval()
    for kw in ({}, dict(prompt_lengths=lengths)):
        want = generate(model, ids, 13, **kw)
        for draft in (model, small):
            for k in (1, 4):
                assert torch.equal(generate(model, ids, 13, draft=draft, draft_tokens=k, **kw), want)
    stop = int(generate(model, ids, 13, prompt_lengths=lengths)[1, 6])
    kw = dict(prompt_lengths=lengths, eos_token_id=[stop, 300])
    assert torch.equal(generate(model, ids, 13, draft=model, **kw), generate(model, ids, 13, **kw))
    assert torch.equal(generate(model, ids, 1, draft=small), generate(model, ids, 1))
    assert torch.equal(generate(model, ids, 0, draft=small), ids)
    assert torch.equal(generate(model, ids[1], 7, draft=small), generate(model, ids[1], 7))
    gen = torch.Generator().manual_seed(2)
    drawn = generate(model, ids, 20, do_sample=True, temperature=0.8, top_k=30, draft=small, generator=gen)
    assert drawn.shape == (3, 44) and int(drawn.min()) >= 0 and int(drawn.max()) < 257


def test_generate_refuses():
    model, ids = _model64(), token_ids(1, 4)
    for kw in (dict(samples=2, draft=model), dict(samples=2, cache_budget=4), dict(draft=model, cache_budget=4)):
        with pytest.raises(ValueError, match="together"):
            generate(model, ids, 2, **kw)
    for kw in (dict(samples=0), dict(draft=model, draft_tokens=0)):
        with pytest.raises(ValueError, match="positive"):
            generate(model, ids, 2, **kw)
    with pytest.raises(ValueError, match="tokens"):
        generate(model, ids, 2, draft=tiny_model(vocab_size=300))


@pytest.mark.parametrize("V", [1, 5, 300])
def test_plain_verification(V):
    gen = torch.Generator().manual_seed(V)
    p, q = (torch.randn(40, k, V, generator=gen).mul(2).softmax(-1) for k in (4, 3))
    q[3], p[4, :, 0] = p[3, :3], 0.0
    drafts = torch.multinomial(q.flatten(0, 1), 1, generator=gen).view(40, 3)
    u = torch.rand(40, 4, generator=gen)
    u[5, 3], u[6, 3] = 0.0, 1.0
    u[3, :3] = 1.0                                        # refused with nothing left of p - q
    tokens, accepted = verify_drafts(p, drafts, u, q)
    want = _want(p, drafts, u, q)
    if V > 1:
        assert torch.equal(tokens, want[0])
    assert torch.equal(accepted, want[1])


def test_plain_verification_edges():
    """What test_verify_edges asks of the kernel: weights that are 0 everywhere, sums that are not finite, values below 0, drafts
    outside the vocabulary, random numbers at the ends of their range and outside it; and no drafts at all."""
    nan, inf, V = float("nan"), float("inf"), 100
    gen = torch.Generator().manual_seed(5)
    p, q = (torch.randn(19, k, V, generator=gen).mul(3).softmax(-1) for k in (3, 2))
    drafts = torch.multinomial(q.flatten(0, 1), 1, generator=gen).view(19, 2)
    u = torch.full((19, 3), 0.99999994)
    drafts[0, 0], drafts[1, 0], drafts[2, 1] = -1, V, 1 << 40
    p[3, 0], u[3] = q[3, 0], 1.0                          # refused with nothing left of p - q
    p[4] = 0.0                                            # nothing to draw from
    for n in range(5, 9):
        p[n, 0, drafts[n, 0]] = 0.0                       # the first draft is refused
    for n, (x, y) in enumerate(((nan, 0.1), (inf, 0.1), (0.1, nan), (inf, inf)), 5):
        at = 7 if int(drafts[n, 0]) != 7 else 8
        p[n, 0, at], q[n, 0, at] = x, y
    u[9, 2], u[10, 2], u[11, 2], u[12, 2], u[13, 2] = 0.0, 1.0, -1.0, 2.0, nan
    p[9:14, :, :5] = p[9:14, :, 95:] = 0.0                # first and last tokens that cannot be
    u[14, 0] = nan
    p[15] = -0.25                                         # not probabilities: below 0 counts as 0
    p[16], u[17, :2], p[17, 2], u[18, :2] = nan, 0.0, 0.0, 0.0
    p[18, 2, 50:] = -1.0                                  # after the last draft, too
    tokens, accepted = verify_drafts(p, drafts, u, q)
    want = _want(p, drafts, u, q)
    assert accepted.tolist() == want[1].tolist() and tokens.tolist() == want[0].tolist()
    assert all(tokens[n, accepted[n]] == -1 for n in (4, 5, 6, 7, 8, 15, 16, 17)) and accepted[17] == accepted[18] == 2
    none = verify_drafts(p[:, :1], drafts[:, :0], u[:, 2:], q[:, :0])
    assert none[0].tolist() == _want(p[:, :1], drafts[:, :0], u[:, 2:], q[:, :0])[0].tolist() and not none[1].any()


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("k", [1, 3])
def test_drafted_samples_are_the_models(k, device):
    """Three tokens of 4,000 rows behind one prompt, drawn with a draft that thinks otherwise, against the model's probabilities
    of all 125 continuations. A share x of n rows has the standard deviation sqrt(x (1 - x) / n): six of them (chances of 2e-9 a
    cell), and a row for cells of next to no weight."""
    n, V = 4000, 5
    model = tiny_model(seed=3, theta_scale=0.25, vocab_size=V, attn_impl="auto").to(device).eval()
    small = tiny_model(seed=5, n_layer=1, vocab_size=V, attn_impl="auto").to(device).eval()
    prompt = torch.tensor([[1, 4, 0, 2, 2, 3, 1]], device=device)
    every = torch.cartesian_prod(*[torch.arange(V, device=device)] * 3)
    with torch.no_grad():
        behind = torch.cat([prompt.expand(len(every), -1), every], 1)
        p, other = (m(behind).logits[:, -4:-1].float().div(0.7).softmax(-1).gather(2, every[..., None])[..., 0] for m in (model, small))
    assert (p[:, 0] - other[:, 0]).abs().max() > 0.05     # else nothing would be refused
    want = p.prod(1)
    got = generate(model, prompt.expand(n, -1), 3, do_sample=True, temperature=0.7, draft=small, draft_tokens=k,
                   generator=torch.Generator(device).manual_seed(4))[:, 7:]
    share = torch.bincount((got * torch.tensor([V * V, V, 1], device=device)).sum(1), minlength=V ** 3) / n
    assert ((share - want).abs() <= 6 * (want * (1 - want) / n).sqrt() + 1 / n).all()


@pytest.mark.parametrize("first", [-1, 300, 1 << 40])
def test_ends_that_are_no_tokens(first):
    """An end that is no token of the vocabulary (a tokenizer without one says -1) pads the rows that are done, and is never read:
    neither where a draft lets some rows end before others, nor behind an end that is a token."""
    model, ids, lengths = _model64(), token_ids(3, 24, seed=8), [24, 3, 11]
    small = tiny_model(seed=5, n_layer=1).double().eval()
    plain = generate(model, ids, 13)
    for eos in (first, [first, int(plain[1, 28])]):
        want = plain.clone()
        if eos is not first:
            for row in want:
                hits = (row[24:] == eos[1]).nonzero()
                if hits.numel():
                    row[24 + int(hits[0]) + 1:] = first
        for kw in ({}, dict(samples=2), dict(draft=small), dict(draft=model, draft_tokens=3), dict(cache_budget=200)):
            got = generate(model, ids, 13, eos_token_id=eos, **kw)
            assert torch.equal(got, want.repeat_interleave(kw.get("samples", 1), 0)), kw
    ended = dict(prompt_lengths=lengths, eos_token_id=first)
    assert torch.equal(generate(model, ids, 13, draft=small, **ended), generate(model, ids, 13, **ended))


def test_generate_with_a_draft_ends_where_probabilities_are_not_finite():
    model, small, ids = _model64(), tiny_model(seed=5, n_layer=1).double().eval(), token_ids(2, 9, seed=8)
    kw = dict(do_sample=True, draft=small, draft_tokens=3, generator=torch.Generator().manual_seed(3))
    for value in (float("nan"), float("inf"), float("-inf")):
        def later(module, args, kwargs, out):             # all but the prompt's pass
            if kwargs["cache"].seq_len > 9:
                out.logits.fill_(value)
        hook = model.register_forward_hook(later, with_kwargs=True)
        with pytest.raises(RuntimeError, match="not finite"):
            generate(model, ids, 8, **kw)
        hook.remove()
    assert generate(model, ids, 8, **kw).shape == (2, 17)


# ------------------------------------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bound", [(torch.float32, 2e-5), (torch.bfloat16, 5e-2), (torch.float16, 1e-2)])
def test_branches_and_drafts_on_the_gpu(dtype, bound, monkeypatch):
    """Prompts of unequal lengths, branched, steps, drafts of which some are kept, steps, against the model's float64 copy on
    the CPU. Bounds: the contiguous cache's logits of these models are off float64 by up to half of them."""
    from sisa_amd.kernels import prefix, step
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).to(dtype).eval()
    ref = tiny_model(seed=3, theta_scale=0.25).eval()
    ref.load_state_dict({n: t.cpu() for n, t in model.state_dict().items()})
    ref = ref.double()
    used, real, whole = [], prefix.sisa_prefix_decode_hip, step.layer_step_branch
    monkeypatch.setattr(prefix, "sisa_prefix_decode_hip", lambda *a, **kw: used.append("attention") or real(*a, **kw))
    monkeypatch.setattr(step, "layer_step_branch", lambda *a: used.append("step") or whole(*a))
    lengths, n = [90, 17, 64], 3
    ids, tokens = token_ids(3, 90, seed=10), token_ids(9, 14, seed=11)
    outs = []
    for m, dev in ((model, DEV), (ref, "cpu")):
        x, y = ids.to(dev), tokens.to(dev)
        cache = SISAPagedCache(9, 128, page_size=32)
        with torch.no_grad():
            cache[:3].expect(lengths)
            m(x, cache=cache[:3])
            cache.branch(n)
            got = [m(y[:, t:t + 1], cache=cache).logits for t in range(4)]
            cache.tentative(6)
            got += [m(y[:, 4:8], cache=cache).logits, m(y[:, 8:9], cache=cache).logits]
            cache.keep([5, 0, 2, 1, 3, 4, 5, 0, 1])
            got += [m(y[:, t:t + 1], cache=cache).logits for t in range(9, 12)]
            for part in (cache[0:3], cache[4:5]):         # some of a prompt's branches, and one alone
                part.tentative(1)
                got.append(torch.zeros_like(got[0]))
                got[-1][part._lo:part._hi] = m(y[part._lo:part._hi, 12:13], cache=part).logits
                part.keep([1] * len(part))
        outs.append(torch.cat(got, 1).double().cpu())
    assert used.count("attention" if dtype == torch.float32 else "step") == 2 * 11
    assert rel_err(outs[0], outs[1]) <= bound
    for i in range(9):
        assert rel_err(outs[0][i], outs[1][i]) <= 1.5 * bound


# one and several rows a sequence, one and two column groups of the products, widths that are no multiple of 8, few heads and many
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,n,M,H,d_ff,longest", [(1, 4, 1, 2, 256, 40), (2, 3, 5, 12, 2744, 300), (5, 1, 7, 5, 329, 65), (4, 16, 1, 16, 1000, 33),
                                                  (1, 2, 32, 2, 256, 700)])
def test_step_matches_modules(k, n, M, H, d_ff, longest, dtype, monkeypatch):
    """A layer's step over branches and drafts behind one C call against the module path, which takes the same attention: both
    round the same quantities, and neither is further from the float64 model than the other by more than the spread of such
    errors."""
    from sisa_amd.kernels import step as K
    model = tiny_model(seed=k, theta_scale=0.25, attn_impl="auto", n_head=H, d_model=64 * H, d_ff=d_ff).to(DEV).to(dtype).eval()
    B, lengths = k * n, [max(1, longest * (i + 1) // k) for i in range(k)]
    ids, tokens = token_ids(k, longest, seed=H).to(DEV), token_ids(B, 3 * M, seed=H + 1).to(DEV)
    calls, real = [], K.layer_step_branch
    monkeypatch.setattr(K, "layer_step_branch", lambda *a: calls.append(1) or real(*a))
    outs, held = [], []
    for watched in (False, True):
        hooks = [blk.attn.W_Q.register_forward_hook(lambda *a: None) for blk in model.layers] if watched else []
        cache = SISAPagedCache(B, longest + 3 * M, page_size=32)
        calls.clear()
        with torch.no_grad():
            cache[:k].expect(lengths)
            model(ids, cache=cache[:k])
            cache.branch(n)
            cache.tentative(2 * M)
            got = [model(tokens[:, :M], cache=cache).logits, model(tokens[:, M:2 * M], cache=cache).logits]
            cache.keep([(M + i) % (2 * M + 1) for i in range(B)])
            cache.tentative(M)
            got.append(model(tokens[:, 2 * M:], cache=cache).logits)
            cache.keep([M] * B)
        assert len(calls) == (0 if watched else 2 * 3)
        outs.append(torch.cat(got, 1).float())
        held.append(cache)
        for h in hooks:
            h.remove()
    assert held[0].lengths == held[1].lengths
    from oracle import model64 as M64
    p64 = M64.params64(model, requires_grad=False)
    some = list(range(min(B, 5)))
    rows = [(torch.cat([ids[b // n:b // n + 1, :lengths[b // n]], tokens[b:b + 1, :2 * M]], 1),
             torch.cat([ids[b // n:b // n + 1, :lengths[b // n]], tokens[b:b + 1, :(M + b) % (2 * M + 1)], tokens[b:b + 1, 2 * M:]], 1))
            for b in some]
    ref = torch.cat([torch.cat([M64.logits64(model, p64, a)[:, -2 * M:], M64.logits64(model, p64, b)[:, -M:]], 1) for a, b in rows])
    a, b = (rel_err(o[:len(some)], ref) for o in outs)
    assert a <= 1.25 * b + 1e-3
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    for layer in range(2):
        for u, v in zip(*(c.last(layer) for c in held)):
            assert rel_err(u, v) <= 2 * eps + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_row_without_a_place_ends_its_sequence(dtype):
    """A drafted position beyond the sequence's pages: NaN from its row on and in all of its attention, and later; the other
    sequences are as they were."""
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).to(dtype).eval()
    ids, tokens = token_ids(3, 30, seed=12).to(DEV), token_ids(3, 4, seed=13).to(DEV)
    outs = []
    for cut in (False, True):
        cache = SISAPagedCache(3, 64, page_size=16)
        with torch.no_grad():
            model(ids, cache=cache)
            cache.reserve(8)
            if cut:
                cache._store.table[1, 2] = -1             # positions 32 .. 47
            cache.tentative(4)
            got = model(tokens, cache=cache).logits
            cache.keep([4, 4, 4])
            outs.append(torch.cat([got, model(tokens[:, :1], cache=cache).logits], 1))
    plain, cut = outs
    assert torch.equal(cut[0], plain[0]) and torch.equal(cut[2], plain[2]) and cut[1].isnan().all() and plain.isfinite().all()


@pytest.mark.gpu
def test_generate_on_the_gpu():
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).eval()
    small = tiny_model(seed=5, n_layer=1, attn_impl="auto").to(DEV).eval()
    ids, lengths = token_ids(3, 40, seed=11).to(DEV), [40, 9, 25]
    want = generate(model, ids, 12, prompt_lengths=lengths)
    assert torch.equal(generate(model, ids, 12, prompt_lengths=lengths, samples=3), want.repeat_interleave(3, 0))
    for draft in (model, small):
        assert torch.equal(generate(model, ids, 12, prompt_lengths=lengths, draft=draft), want)
    half, little = model.to(torch.bfloat16), small.to(torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(3)
    drawn = generate(half, ids, 20, do_sample=True, top_k=50, draft=little, draft_tokens=5, generator=gen)
    again = generate(half, ids, 20, do_sample=True, top_k=50, draft=little, draft_tokens=5,
                     generator=torch.Generator(device=DEV).manual_seed(3))
    assert drawn.shape == (3, 60) and torch.equal(drawn, again) and int(drawn.max()) < 257
    assert generate(half, ids, 20, do_sample=True, samples=4, generator=gen).shape == (12, 60)


@pytest.mark.gpu
def test_a_step_that_fails_is_taken_back(monkeypatch):
    from sisa_amd.kernels import step
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).to(torch.bfloat16).eval()
    ids, tokens = token_ids(2, 30, seed=14).to(DEV), token_ids(4, 3, seed=15).to(DEV)
    with torch.no_grad():
        caches = [_branched(model, ids, [30, 20], 2)[0] for _ in range(2)]
        want = [model(tokens[:, t:t + 1], cache=caches[0]).logits for t in range(3)]
        real = step._step_branch

        def fails(*a):
            raise RuntimeError("planted")
        monkeypatch.setattr(step, "_step_branch", fails)
        before = (caches[1].lengths, caches[1].free_pages)
        with pytest.raises(RuntimeError, match="planted"):
            model(tokens[:, :1], cache=caches[1])
        assert (caches[1].lengths, caches[1].free_pages) == before
        monkeypatch.setattr(step, "_step_branch", real)
        got = [model(tokens[:, t:t + 1], cache=caches[1]).logits for t in range(3)]
    assert torch.equal(torch.cat(got, 1), torch.cat(want, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("tentative", [False, True])
def test_many_new_positions_in_parts(tentative, monkeypatch):
    """Twenty positions behind branches of ragged prompts, and behind single sequences that can go back, three at a time, against
    the model's float64 copy; the bound as above."""
    from sisa_amd import paged
    from sisa_amd.kernels import prefix
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).eval()
    ref = tiny_model(seed=3, theta_scale=0.25).eval()
    ref.load_state_dict({n: t.cpu() for n, t in model.state_dict().items()})
    ref = ref.double()
    prompts, more, lengths, n = token_ids(2, 40, seed=11), token_ids(4, 20, seed=12), [40, 17], 1 if tentative else 2
    monkeypatch.setattr(paged, "MAX_ROWS", 3 * 2 * n * model.config.n_head + 1)
    calls, real = [], prefix.sisa_prefix_decode_hip
    monkeypatch.setattr(prefix, "sisa_prefix_decode_hip", lambda q, *a, **kw: calls.append(q.shape[2]) or real(q, *a, **kw))
    outs = []
    with torch.no_grad():
        for m, dev in ((model, DEV), (ref, "cpu")):
            cache, _ = _branched(m, prompts.to(dev), lengths, n)
            if tentative:
                cache.tentative(20)
            outs.append(m(more[:2 * n].to(dev), cache=cache).logits.cpu())
            if tentative:
                cache.keep([11, 20])
            outs.append(m(more[:2 * n, :1].to(dev), cache=cache).logits.cpu())
    assert calls[:14] == [3, 3, 3, 3, 3, 3, 2] * 2 and set(calls[14:]) <= {1}
    assert rel_err(outs[0], outs[2]) <= 2e-5 and rel_err(outs[1], outs[3]) <= 2e-5
