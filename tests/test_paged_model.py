"""SISAPagedCache and what generate() does with it: on the CPU in float64 against the contiguous cache and against dense
formulas, on the GPU (bf16, fp32) against the same model in float64."""
import math

import pytest
import torch

from model_utils import rel_err, tiny_model, token_ids
from sisa_amd import SISACache, SISAPagedCache, generate
from sisa_amd.paged import attention_weights

DEV = "cuda:0"


# The gates are float32 in a float64 model, and torch rounds their functions differently in a vector's body and its tail, so
# in passes of other shapes. Here their sums are below 64 in magnitude and of at most 50 steps, each rounded by at most 2^-19
# (half a step below 64) on either side: scores differ by at most 2 * 2 * 50 * 2^-19 = 3.9e-4 in g and F together, weights by
# 7.8e-4 of themselves, logits after two layers by no more than a few of that.
GATES = 2e-3


def _model64(**kw):
    return tiny_model(seed=3, theta_scale=0.25, **kw).double().eval()


def _logits(model, ids, cache, first, counts=None, at=None):
    """Logits of every later position, by a first pass and then one by one."""
    with torch.no_grad():
        if counts is not None:
            cache.expect(counts)
        out = [model(ids[:, :first], cache=cache).logits]
        out += [model(ids[:, t:t + 1], cache=cache).logits for t in range(first, ids.shape[1])]
    return torch.cat(out, 1)


def test_equal_lengths_continue_as_the_contiguous_cache():
    model = _model64()
    ids = token_ids(3, 70, seed=1)
    want = _logits(model, ids, SISACache(), 40)
    for page_size, kw in ((16, {}), (64, dict(track=True))):
        cache = SISAPagedCache(3, 70, page_size=page_size, **kw)
        got = _logits(model, ids, cache, 40)
        assert rel_err(got, want) <= 1e-12 and cache.lengths == [70] * 3 and cache.seq_len == 70
    # several positions at once behind a filled cache
    # (the float32 sums of the gates depend on where a pass ends: the same passes on both sides)
    cache, other = SISAPagedCache(3, 70, track=True), SISACache()
    with torch.no_grad():
        got, want = (torch.cat([model(ids[:, a:b], cache=c).logits for a, b in ((0, 33), (33, 50), (50, 70))], 1)
                     for c in (cache, other))
    assert rel_err(got, want) <= 1e-12
    # every query's weights sum to one, however they came in
    for layer in range(2):
        w = cache.weights(layer)
        assert (w.double().sum(-1) - 70).abs().max() <= 70 * 70 * 2 ** -24 and w.shape == (3, 2, 70)


def test_unequal_lengths_are_what_each_gives_alone():
    model = _model64()
    ids, counts = token_ids(4, 60, seed=2), [37, 1, 16, 40]
    cache = SISAPagedCache(4, 61, page_size=16, track=True)
    with torch.no_grad():
        cache.expect(counts)
        first = model(ids[:, :40], cache=cache, logits_at=[n - 1 for n in counts]).logits
        later = [model(ids[:, t:t + 1], cache=cache).logits for t in range(40, 45)]
    assert cache.lengths == [n + 5 for n in counts]
    for i, n in enumerate(counts):
        row = torch.cat([ids[i:i + 1, :n], ids[i:i + 1, 40:45]], 1)
        alone = SISACache()
        want = _logits(model, row, alone, n)
        got = torch.cat([first[i:i + 1], *(x[i:i + 1] for x in later)], 1)
        assert rel_err(got, want[:, n - 1:]) <= GATES
        one = SISAPagedCache(1, 50, track=True)
        _logits(model, row, one, n)
        for layer in range(2):
            held, single = cache.weights(layer)[i], one.weights(layer)[0]
            assert rel_err(held[:, :n + 5], single[:, :n + 5]) <= GATES
            assert held[:, n + 5:].eq(0).all()


def test_parts_release_and_reuse():
    model = _model64()
    ids = token_ids(3, 50, seed=4)
    cache = SISAPagedCache(3, 50, pages=8, page_size=16)
    want = [_logits(model, ids[i:i + 1], SISACache(), 20) for i in range(3)]
    with torch.no_grad():
        for i in (2, 0):                                    # one after the other, not in order
            assert rel_err(model(ids[i:i + 1, :20], cache=cache[i]).logits, want[i][:, :20]) <= GATES
        assert cache.lengths == [20, 0, 20] and cache.free_pages == 4
        with pytest.raises(ValueError, match="some of these sequences are empty"):
            model(ids[:, 20:21], cache=cache)
        assert rel_err(model(ids[1:2, :20], cache=cache[1]).logits, want[1][:, :20]) <= GATES
        step = model(ids[:, 20:21], cache=cache).logits
        assert rel_err(step, torch.cat(want)[:, 20:21]) <= GATES
        cache[0:2].release()
        assert cache.lengths == [0, 0, 21] and cache.free_pages == 6
        # the pages go to another sequence; the third is not touched
        assert rel_err(model(ids[1:2, :20], cache=cache[0]).logits, want[1][:, :20]) <= GATES
        assert rel_err(model(ids[2:, 21:22], cache=cache[-1]).logits, want[2][:, 21:22]) <= GATES
        cache[1].reserve(40)                                # before its first pass
        assert cache.free_pages == 1
        with pytest.raises(RuntimeError, match="more pages"):
            model(ids[:1, 20:49], cache=cache[0:1])         # 49 positions: two pages more
        assert cache.lengths == [20, 0, 22]
    early = SISAPagedCache(2, 50, page_size=16)             # reserved before there is a device to show the table on
    early.reserve(50)
    assert early.free_pages == 0
    assert rel_err(_logits(model, ids[:2], early, 20), torch.cat(want[:2])) <= GATES
    assert len(cache) == 3 and len(cache[1:]) == 2
    for bad in (slice(2, 1), slice(0, 3, 2)):
        with pytest.raises(ValueError):
            cache[bad]
    with pytest.raises(IndexError):
        cache[3]


def test_a_pass_without_enough_pages_takes_none():
    model = _model64()
    ids = token_ids(2, 17, seed=4)
    want = _logits(model, ids, SISACache(), 16)
    cache = SISAPagedCache(2, 40, pages=3, page_size=16)
    with torch.no_grad():
        model(ids[:, :16], cache=cache)
        for more in (lambda: model(ids[:, 16:], cache=cache), lambda: cache.reserve(1)):
            with pytest.raises(RuntimeError, match="2 more pages"):
                more()
            assert cache.free_pages == 1 and cache.lengths == [16, 16]
        cache[1].release()
        assert rel_err(model(ids[:1, 16:], cache=cache[0]).logits, want[:1, 16:]) <= GATES
        assert cache.lengths == [17, 0] and cache.free_pages == 1


def test_what_is_expected_belongs_to_the_sequences():
    model = _model64()
    ids = token_ids(3, 20, seed=5)
    want = [_logits(model, ids[i:i + 1, :n], SISACache(), n) for i, n in enumerate((7, 20, 12))]
    cache = SISAPagedCache(3, 40, page_size=16)
    with torch.no_grad():
        cache[0].expect([7])                                # another handle of the sequence than the pass is given
        assert rel_err(model(ids[:1], cache=cache[0]).logits[:, :7], want[0]) <= GATES and cache.lengths == [7, 0, 0]
        cache[1:].expect([20, 12])
        got = [model(ids[i:i + 1], cache=cache[i]).logits for i in (1, 2)]
        assert all(rel_err(y[:, :w.shape[1]], w) <= GATES for y, w in zip(got, want[1:])) and cache.lengths == [7, 20, 12]
        cache[2].release()
        cache[2].expect([5])
        cache.release()
        model(ids, cache=cache)
        assert cache.lengths == [20] * 3


def _failing(at):
    """A function that raises at its ``at``-th call, and the calls so far."""
    calls = []

    def wrap(real):
        def fn(*a, **kw):
            calls.append(1)
            if len(calls) == at:
                raise MemoryError("no room")
            return real(*a, **kw)
        return fn
    return wrap


@pytest.mark.parametrize("track", [False, True])
def test_a_pass_that_fails_before_it_is_written_is_taken_back(track, monkeypatch):
    """A first and a later pass fail in the write of the first layer, for all sequences and for some; passes of other lengths
    follow."""
    from sisa_amd import paged
    model = _model64()
    ids, counts = token_ids(3, 40, seed=12), [9, 30, 17]
    want = [_logits(model, ids[i:i + 1], SISACache(), n)[:, n - 1:] for i, n in enumerate(counts)]
    cache = SISAPagedCache(3, 60, page_size=16, track=track)
    cache[2].reserve(40)
    free = cache.free_pages

    def fails(part, x):
        before = cache.lengths, cache.free_pages
        with monkeypatch.context() as m:
            m.setattr(paged, "_write", _failing(1)(paged._write))
            with pytest.raises(MemoryError):
                model(x, cache=part)
        assert (cache.lengths, cache.free_pages) == before

    with torch.no_grad():
        cache.expect(counts)
        fails(cache, ids[:, :34])
        assert cache.free_pages == free and cache.lengths == [0, 0, 0]
        got = [model(ids[:, :30], cache=cache, logits_at=[n - 1 for n in counts]).logits]      # what was expected still is
        assert cache.lengths == counts
        for i, n in enumerate(counts):                       # from here on each at its own positions
            fails(cache[i], ids[i:i + 1, n:n + 5])
            y = model(ids[i:i + 1, n:n + 3], cache=cache[i]).logits
            assert rel_err(torch.cat([got[0][i:i + 1], y], 1), want[i][:, :4]) <= GATES
        fails(cache, ids[:, 30:31])
        fails(cache[0:2], ids[:2, 30:33])
        y = torch.cat([model(ids[i:i + 1, n + 3:n + 4], cache=cache[i]).logits for i, n in enumerate(counts)])
        assert rel_err(y, torch.cat([w[:, 4:5] for w in want])) <= GATES
    assert cache.lengths == [n + 4 for n in counts]


def test_a_pass_that_is_given_up_between_two_calls_is_taken_back():
    """Begun and never written, as by an interrupt outside of the cache's own functions: every entry finds the cache as before."""
    model = _model64()
    ids = token_ids(2, 30, seed=15)
    want = _logits(model, ids, SISACache(), 20)
    p = model.layers[0].attn._unfused_inputs(model.embed(ids[:, 20:29]).detach())
    for entry in (lambda c: model(ids[:, 20:23], cache=c), lambda c: c.reserve(3), lambda c: c[1].release(),
                  lambda c: c.evict(20, 5), lambda c: c[0].release()):
        cache = SISAPagedCache(2, 60, page_size=16, track=True, pages=20)
        with torch.no_grad():
            model(ids[:, :20], cache=cache)
            cache.begin(0, p.k, p.b, False)
            entry(cache)
            for i in range(2):
                if not cache.lengths[i]:
                    model(ids[i:i + 1, :20], cache=cache[i])
                n = cache.lengths[i]
                assert rel_err(model(ids[i:i + 1, n:n + 1], cache=cache[i]).logits, want[i:i + 1, n:n + 1]) <= GATES
    cache = SISAPagedCache(2, 60)
    cache.expect([9, 4])
    with torch.no_grad():
        cache.begin(0, p.k, p.b, False)
        cache.expect([3, 8])                                # still the first pass
        model(ids[:, :9], cache=cache)
    assert cache.lengths == [3, 8]


@pytest.mark.parametrize("n_layer,name,at", [(2, "_write", 2), (1, "paged_attention", 1), (2, "paged_attention", 1),
                                             (2, "paged_attention", 2), (1, "attention_weights", 1), (2, "attention_weights", 1)])
def test_a_pass_that_fails_later_ends_its_sequences(n_layer, name, at, monkeypatch):
    """It has reached some layers: no pass and no eviction goes on from there, others do, and release() mends it."""
    from sisa_amd import paged
    model = _model64(n_layer=n_layer)
    ids = token_ids(2, 40, seed=13)
    want = _logits(model, ids, SISACache(), 20)
    cache = SISAPagedCache(2, 60, page_size=16, track=True, pages=20)
    with torch.no_grad():
        model(ids[1:, :20], cache=cache[1])
        if name != "attention_weights":
            model(ids[:1, :20], cache=cache[0])
        with monkeypatch.context() as m:
            m.setattr(paged, name, _failing(at)(getattr(paged, name)))
            with pytest.raises(MemoryError):
                model(ids[:1, 20:21] if cache.lengths[0] else ids[:1, :20], cache=cache[0])
        for x in (ids[:1, 20:21], ids[:1, 20:24], ids[:1, :20]):
            with pytest.raises(RuntimeError, match="release"):
                model(x, cache=cache[0])
        with pytest.raises(RuntimeError):
            cache.evict(8, 2)
        assert rel_err(model(ids[1:, 20:21], cache=cache[1]).logits, want[1:, 20:21]) <= GATES
        cache[0].release()
        got = [model(ids[:1, :20], cache=cache[0]).logits, model(ids[:1, 20:21], cache=cache[0]).logits]
        assert rel_err(torch.cat(got, 1), want[:1, :21]) <= GATES and cache.lengths == [21, 21]


def _dense(model, x, layer, kept):
    """Attention of the last row of ``x`` (1, n, d), the layer's normalised input, over the rows ``kept[h]``."""
    at = model.layers[layer].attn
    p, lam, n = at._unfused_inputs(x), at.lam().double(), x.shape[1]
    heads = []
    for h, rows in enumerate(kept):
        j = torch.tensor(rows)
        s = p.k[0, h, j] @ p.q[0, h, -1] / 8 + lam[h] * (p.g[0, h, -1] - p.g[0, h, j]).exp() * (p.b[0, h, j] @ p.c[0, h, -1])
        w = (s + p.fgate[0, h, -1] - p.fgate[0, h, j]).softmax(0)
        heads.append((w @ p.v[0, h, j], w))
    return torch.cat([o for o, _ in heads]), [w for _, w in heads]


@pytest.mark.parametrize("keep,recent", [(12, 4), (12, 12), (20, 1), (1, 1)])
def test_evict_leaves_a_softmax_over_what_is_kept(keep, recent):
    """One layer, whose inputs do not depend on what it keeps: positions chosen by sorting, attention over them alone."""
    model = _model64(n_layer=1)
    block, at = model.layers[0], model.layers[0].attn
    ids = token_ids(1, 60, seed=5)
    cache = SISAPagedCache(1, 60, page_size=16, track=True, pages=8)
    with torch.no_grad():
        x = block.attn_norm(model.embed(ids))
        p = at._unfused_inputs(x[:, :40])
        w = attention_weights(p.q, p.k, p.c, p.b, p.g, at.lam(), p.fgate, torch.tensor([40]))[0]
        at(x[:, :40], cache=cache)
        kept = [list(range(40)) for _ in range(2)]
        w = [row for row in w.double()]
        for t in range(40, 60):
            if t in (40, 47, 48):
                before = cache.free_pages
                cache.evict(keep, recent)
                for h in range(2):
                    n = len(kept[h])
                    if n > keep:
                        old = sorted(range(n - recent), key=lambda i: (-float(w[h][i]), i))[:keep - recent]
                        stay = sorted(old) + list(range(n - recent, n))
                        kept[h], w[h] = [kept[h][i] for i in stay], w[h][stay]
                assert cache.lengths == [min(keep, t)] and cache.free_pages >= before
            for h in range(2):
                kept[h].append(t)
            y = at(x[:, t:t + 1], cache=cache)
            want, new = _dense(model, x[:, :t + 1], 0, kept)
            assert rel_err(y[0, 0], at.W_O(want)) <= GATES
            w = [torch.cat([a, a.new_zeros(1)]) + b for a, b in zip(w, new)]
        for h in range(2):
            assert rel_err(cache.weights(0)[0, h, :len(kept[h])], w[h]) <= GATES
            assert cache.weights(0)[0, h, len(kept[h]):].eq(0).all()


def test_evict_with_few_free_pages_goes_sequence_by_sequence():
    model = _model64()
    ids = token_ids(3, 64, seed=6)
    with torch.no_grad():
        roomy, tight = SISAPagedCache(3, 64, page_size=16, pages=30, track=True), SISAPagedCache(
            3, 64, page_size=16, pages=13, track=True)
        for c in (roomy, tight):
            model(ids[:, :63], cache=c)
            c.evict(10, 3)
        assert roomy.lengths == tight.lengths == [10] * 3 and tight.free_pages == 10
        for layer in range(2):
            assert torch.equal(roomy.weights(layer), tight.weights(layer))
        a, b = (model(ids[:, 63:], cache=c).logits for c in (roomy, tight))
        assert torch.equal(a, b)
        none = SISAPagedCache(1, 64, page_size=16, pages=4, track=True)
        model(ids[:1, :63], cache=none)
        with pytest.raises(RuntimeError, match="free pages"):
            none.evict(10, 3)
        assert none.lengths == [63] and rel_err(model(ids[:1, 63:], cache=none).logits,
                                                _logits(model, ids[:1], SISACache(), 63)[:, 63:]) <= GATES


@pytest.mark.parametrize("sequences,max_length,keep", [(1, 50, 40), (1, 16, 15), (3, 50, 49)])
def test_evict_at_the_limit_of_a_default_cache(sequences, max_length, keep):
    """Sequences of max_length positions, in as many pages as the cache comes with."""
    model = _model64()
    ids = token_ids(sequences, max_length + 1, seed=17)
    with torch.no_grad():
        cache, roomy = (SISAPagedCache(sequences, max_length, page_size=16, track=True, **kw) for kw in ({}, dict(pages=40)))
        for c in (cache, roomy):
            model(ids[:, :max_length], cache=c)
            c.evict(keep, keep // 2)
        assert cache.lengths == [keep] * sequences
        a, b = (model(ids[:, max_length:], cache=c).logits for c in (cache, roomy))
        assert torch.equal(a, b)


@pytest.mark.parametrize("at", [1, 2])
def test_an_eviction_that_fails_leaves_the_cache_as_it_was(at, monkeypatch):
    """In the first and in the second layer; lengths, pages, weights and what follows are those of a cache it never touched."""
    from sisa_amd import paged
    model = _model64()
    ids = token_ids(2, 60, seed=16)
    caches = [SISAPagedCache(2, 64, page_size=16, pages=12, track=True) for _ in range(2)]
    outs = []
    for cache, failing in zip(caches, (False, True)):
        with torch.no_grad():
            model(ids[:, :50], cache=cache)
            if failing:
                weights = [cache.weights(layer).clone() for layer in range(2)]
                with monkeypatch.context() as m:
                    m.setattr(paged, "_evict", _failing(at)(paged._evict))
                    with pytest.raises(MemoryError):
                        cache.evict(20, 5)
                assert cache.lengths == [50, 50] and cache.free_pages == 4
                assert all(torch.equal(cache.weights(layer), weights[layer]) for layer in range(2))
            got = [model(ids[:, 50:51], cache=cache).logits]
            cache.evict(20, 5)
            got += [model(ids[:, t:t + 1], cache=cache).logits for t in range(51, 60)]
        assert cache.lengths == [29, 29] and cache.free_pages == 8
        outs.append(torch.cat(got, 1))
    assert torch.equal(*outs) and all(torch.equal(*(c.weights(layer) for c in caches)) for layer in range(2))


def test_refusals():
    model = _model64()
    ids = token_ids(2, 20, seed=7)
    for kw in (dict(sequences=0), dict(max_length=0), dict(page_size=8), dict(page_size=48), dict(pages=0)):
        with pytest.raises(ValueError):
            SISAPagedCache(**(dict(sequences=1, max_length=4) | kw))
    cache = SISAPagedCache(2, 20)
    with pytest.raises(RuntimeError, match="inference"):
        model(ids, cache=cache)
    with torch.no_grad():
        with pytest.raises(ValueError, match="2 sequences"):
            model(ids[:1], cache=cache)
        with pytest.raises(ValueError, match="track=True"):
            cache.evict(4, 1)
        with pytest.raises(ValueError, match="track=True"):
            cache.weights(0)
        for counts in ([3], [0, 3], [3, 3, 3]):
            with pytest.raises(ValueError, match="expect"):
                cache.expect(counts)
        cache.expect([3, 21])
        with pytest.raises(ValueError, match="were expected"):
            model(ids, cache=cache)
        cache.expect([20, 3])
        model(ids, cache=cache)
        with pytest.raises(ValueError, match="first pass"):
            cache.expect([1, 1])
        with pytest.raises(ValueError, match="max_length"):
            model(ids[:, :1], cache=cache)
        tracked = SISAPagedCache(2, 20, track=True)
        model(ids, cache=tracked)
        for keep, recent in ((4, 0), (4, 5), (0, 0)):
            with pytest.raises(ValueError, match="recent"):
                tracked.evict(keep, recent)
        for at in ([1], [1, 20], [-1, 0]):
            with pytest.raises(ValueError, match="logits_at"):
                model(ids, logits_at=at)
        with pytest.raises(ValueError, match="labels"):
            model(ids, labels=ids, logits_at=[1, 1])


# ------------------------------------------------------------------------------------------------ generate
def test_generate_from_unequal_prompts():
    model = _model64()
    ids, lengths = token_ids(3, 24, seed=8), [24, 3, 11]
    got = generate(model, ids, 9, prompt_lengths=lengths)
    assert got.shape == (3, 33)
    for i, n in enumerate(lengths):
        want = generate(model, ids[i:i + 1, :n], 9)
        assert torch.equal(got[i, :n + 9], want[0]) and got[i, n + 9:].eq(0).all()
    assert torch.equal(generate(model, ids, 9, prompt_lengths=torch.tensor([24, 24, 24])), generate(model, ids, 9))
    # an end: the row's rest is the first stop id
    stop = int(got[1, 5])
    ended = generate(model, ids, 9, prompt_lengths=lengths, eos_token_id=[stop, 300])
    first = got[1, 3:12].tolist().index(stop)
    assert ended[1, 3 + first:].eq(stop).all() and torch.equal(ended[1, :3 + first], got[1, :3 + first])
    one = generate(model, ids[1], 4, prompt_lengths=[3])
    assert one.dim() == 1 and torch.equal(one[:7], got[1, :7])
    for bad in ([24, 3], [24, 0, 3], [25, 3, 3], [24.0, 3, 3]):
        with pytest.raises(ValueError, match="prompt_lengths"):
            generate(model, ids, 2, prompt_lengths=bad)


@pytest.mark.parametrize("pad", [-1, -100, 10 ** 6])
def test_generate_from_prompts_padded_with_no_token(pad):
    model = _model64()
    ids, lengths = token_ids(3, 24, seed=8), torch.tensor([24, 3, 11])
    padded = torch.where(torch.arange(24) < lengths[:, None], ids, pad)
    before = padded.clone()
    for kw in ({}, dict(eos_token_id=5), dict(cache_budget=8)):
        want = generate(model, ids, 9, prompt_lengths=lengths, **kw)
        assert torch.equal(generate(model, padded, 9, prompt_lengths=lengths, **kw), want)
    assert torch.equal(padded, before)


def test_generate_within_a_budget():
    model = _model64()
    ids = token_ids(2, 50, seed=9)
    free = generate(model, ids, 40)
    assert torch.equal(generate(model, ids, 40, cache_budget=90), free)            # a budget that is never reached
    cut = generate(model, ids, 40, cache_budget=16, cache_recent=8)
    assert cut.shape == (2, 90) and torch.equal(cut[:, :51], free[:, :51])         # the prompt itself is seen whole
    # by hand: cut after the prompt, and when 16 more have come
    cache = SISAPagedCache(2, 90, track=True)
    with torch.no_grad():
        token, out = model(ids, cache=cache).logits[:, -1].argmax(-1), [ids]
        cache.evict(16, 8)
        for _ in range(39):
            out.append(token[:, None])
            if cache.seq_len >= 32:
                cache.evict(16, 8)
            token = model(token[:, None], cache=cache).logits[:, -1].argmax(-1)
    assert torch.equal(cut, torch.cat([*out, token[:, None]], 1))
    assert generate(model, ids, 30, cache_budget=1, prompt_lengths=[50, 2]).shape == (2, 80)
    for kw in (dict(cache_budget=0), dict(cache_recent=3), dict(cache_budget=4, cache_recent=5), dict(cache_budget=4, cache_recent=0)):
        with pytest.raises(ValueError, match="cache_"):
            generate(model, ids, 2, **kw)


# ------------------------------------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bound", [(torch.float32, 2e-5), (torch.bfloat16, 5e-2), (torch.float16, 1e-2)])
def test_unequal_lengths_on_the_gpu(dtype, bound, monkeypatch):
    """Ragged prompts, steps, an eviction, steps, against the model's float64 copy on the CPU with the same positions kept.
    Bounds: the contiguous cache's logits of these models are off float64 by up to half of them."""
    from sisa_amd.kernels import paged as K
    from sisa_amd.kernels import step
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).to(dtype).eval()
    ref = tiny_model(seed=3, theta_scale=0.25).eval()
    ref.load_state_dict({n: t.cpu() for n, t in model.state_dict().items()})
    ref = ref.double()
    used, real = [], (K.sisa_paged_decode_hip, K.sisa_cache_evict_hip)
    monkeypatch.setattr(K, "sisa_paged_decode_hip", lambda *a, **kw: used.append("decode") or real[0](*a, **kw))
    whole = step.layer_step_paged
    monkeypatch.setattr(step, "layer_step_paged", lambda *a: used.append("step") or whole(*a))
    ids, counts = token_ids(3, 120, seed=10), [90, 17, 64]
    monkeypatch.setattr(K, "sisa_cache_evict_hip", lambda *a, **kw: used.append("evict") or real[1](*a, **kw))
    caches = [SISAPagedCache(3, 128, page_size=32, pages=20, track=True) for _ in range(2)]
    outs = []
    for m, cache, dev in ((model, caches[0], DEV), (ref, caches[1], "cpu")):
        x = ids.to(dev)
        with torch.no_grad():
            cache.expect(counts)
            got = [m(x[:, :90], cache=cache, logits_at=[n - 1 for n in counts]).logits]
            got += [m(x[:, t:t + 1], cache=cache).logits for t in range(90, 95)]
            if m is model:
                weights = [cache.weights(layer).clone() for layer in range(2)]
            else:
                for layer in range(2):
                    assert rel_err(weights[layer].cpu(), cache.weights(layer).double()) <= bound
                    # choose by the GPU's weights: near ties may fall differently
                    cache.weights(layer).copy_(weights[layer])
            cache.evict(40, 10)
            got += [m(x[:, t:t + 1], cache=cache).logits for t in range(95, 100)]
        outs.append(torch.cat(got, 1).cpu())
        assert cache.lengths == [45, 27, 45]
    assert used.count("decode" if dtype == torch.float32 else "step") == 20 and used.count("evict") >= 2
    assert rel_err(outs[0], outs[1]) <= bound
    for i in range(3):
        assert rel_err(outs[0][i], outs[1][i]) <= 1.5 * bound


@pytest.mark.gpu
def test_generate_on_the_gpu_with_lengths_and_budget():
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).eval()
    ids, lengths = token_ids(3, 40, seed=11).to(DEV), [40, 9, 25]
    got = generate(model, ids, 12, prompt_lengths=lengths)
    for i, n in enumerate(lengths):
        assert torch.equal(got[i, :n + 12], generate(model, ids[i:i + 1, :n], 12)[0])
    assert torch.equal(generate(model, ids, 12, cache_budget=64), generate(model, ids, 12))
    cut = generate(model, ids, 30, cache_budget=16, prompt_lengths=lengths)
    again = generate(model, ids, 30, cache_budget=16, prompt_lengths=lengths)
    assert cut.shape == (3, 70) and torch.equal(cut, again)
    half = model.to(torch.bfloat16)
    assert generate(half, ids, 20, cache_budget=32, cache_recent=8).shape == (3, 60)


# rows: one and two column groups of the products; a hidden width that is no multiple of 8; few and many heads; with and without
# tracking; a cache that one workgroup takes whole, and longer ones
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,d_ff,longest,track", [(1, 2, 256, 40, False), (3, 12, 2744, 300, True), (17, 5, 329, 65, True),
                                                    (64, 16, 1000, 20, False), (2, 2, 256, 1500, True)])
def test_step_matches_modules(B, H, d_ff, longest, track, dtype, monkeypatch):
    """A layer's step behind one C call against the module path: near prompts' lengths of their own, steps, an eviction in
    between. Both round the same quantities: neither is further from the float64 model than the other by more than the spread
    of such errors (the bound of the contiguous cache's step test)."""
    from sisa_amd.kernels import step as K
    steps = 6
    model = tiny_model(seed=B, theta_scale=0.25, attn_impl="auto", n_head=H, d_model=64 * H, d_ff=d_ff).to(DEV).to(dtype).eval()
    ids, counts = token_ids(B, longest + steps, seed=H).to(DEV), [max(1, longest * (i + 1) // B) for i in range(B)]
    calls, real = [], K.layer_step_paged
    monkeypatch.setattr(K, "layer_step_paged", lambda *a: calls.append(1) or real(*a))
    outs, held = [], []
    for watched in (False, True):
        hooks = [blk.attn.W_Q.register_forward_hook(lambda *a: None) for blk in model.layers] if watched else []
        cache = SISAPagedCache(B, longest + steps, page_size=32, track=track, pages=2 * B * -(-(longest + steps) // 32))
        calls.clear()
        with torch.no_grad():
            cache.expect(counts)
            model(ids[:, :longest], cache=cache)
            if not watched:
                first = cache
            got = []
            for t in range(longest, longest + steps):
                if track and t == longest + 3:
                    cache.evict(max(1, longest // 2), max(1, longest // 4))
                got.append(model(ids[:, t:t + 1], cache=cache).logits)
        assert len(calls) == (0 if watched else 2 * steps)
        outs.append(torch.cat(got, 1).float())
        held.append(cache)
        for h in hooks:
            h.remove()
    assert held[0].lengths == held[1].lengths
    # Without an eviction against float64: each row's own prompt and the steps' tokens. With one, rows that keep other
    # positions after a near tie cannot be compared: the first three steps.
    n = 3 if track else steps
    rows = [torch.cat([ids[i:i + 1, :c], ids[i:i + 1, longest:longest + n]], 1) for i, c in enumerate(counts)][:4]
    from oracle import model64 as M64
    p64 = M64.params64(model, requires_grad=False)
    ref = torch.cat([M64.logits64(model, p64, r)[:, c:] for r, c in zip(rows, counts)])
    a, b = (rel_err(o[:4, :n], ref) for o in outs)
    assert a <= 1.25 * b + 1e-3
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    if track:
        assert all(torch.isfinite(o).all() for o in outs)
        for layer in range(2):
            w = [c.weights(layer) for c in held]
            assert all(x.isfinite().all() and (x >= 0).all() for x in w)
    else:
        for layer in range(2):
            x, y = (c.last(layer) for c in held)
            for u, v in zip(x, y):
                assert rel_err(u, v) <= 2 * eps + 1e-6


@pytest.mark.gpu
def test_calls_that_keep_the_module_path_with_pages(monkeypatch):
    from sisa_amd.kernels import step as K
    calls, real = [], K.layer_step_paged
    monkeypatch.setattr(K, "layer_step_paged", lambda *a: calls.append(1) or real(*a))
    model = tiny_model(seed=1, attn_impl="auto").to(DEV).to(torch.bfloat16).eval()

    def steps_of(model, rows=3, n=1, ctx=torch.no_grad, part=None):
        ids = token_ids(rows, 12, seed=1).to(DEV)
        cache = SISAPagedCache(rows, 20)
        calls.clear()
        with torch.no_grad():
            model(ids[:, :8], cache=cache)
            with ctx():
                model(ids[:1, 8:8 + n] if part else ids[:, 8:8 + n], cache=cache[0] if part else cache)
        return len(calls)

    assert steps_of(model) == 2 and steps_of(model, part=True) == 2
    assert steps_of(model, n=2) == 0 and steps_of(model, rows=65) == 0
    assert steps_of(model, ctx=lambda: torch.autocast("cuda", dtype=torch.bfloat16)) == 0
    model.set_attn_impl("hip")
    assert steps_of(model) == 0
    ids, cache = token_ids(2, 9).to(DEV), SISAPagedCache(2, 20)
    with torch.no_grad():
        model(ids[:, :8], cache=cache)
        model.set_attn_impl("torch")
        with pytest.raises(ValueError, match="HIP implementation"):
            model(ids[:, 8:], cache=cache)
    assert steps_of(tiny_model(seed=1, attn_impl="auto").to(DEV).eval()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("track", [False, True])
def test_many_new_positions_in_parts(track, monkeypatch):
    """Twenty positions behind ragged prompts, three at a time, against the model's float64 copy; the bound as above."""
    from sisa_amd import paged
    from sisa_amd.kernels import paged as K
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).eval()
    ref = tiny_model(seed=3, theta_scale=0.25).eval()
    ref.load_state_dict({n: t.cpu() for n, t in model.state_dict().items()})
    ref = ref.double()
    ids, counts = token_ids(3, 60, seed=11), [40, 1, 17]
    monkeypatch.setattr(paged, "MAX_SCORES", 3 * 3 * model.config.n_head * 60 + 1)
    calls, real = [], K.sisa_paged_decode_hip
    monkeypatch.setattr(K, "sisa_paged_decode_hip", lambda q, *a, **kw: calls.append(q.shape[2]) or real(q, *a, **kw))
    caches = [SISAPagedCache(3, 64, page_size=16, track=track) for _ in range(2)]
    outs = []
    for m, cache, dev in ((model, caches[0], DEV), (ref, caches[1], "cpu")):
        with torch.no_grad():
            cache.expect(counts)
            m(ids[:, :40].to(dev), cache=cache)
            outs.append(m(ids[:, 40:].to(dev), cache=cache).logits.cpu())
    assert calls == [3, 3, 3, 3, 3, 3, 2] * 2 and caches[0].lengths == [60, 21, 37]
    assert rel_err(outs[0], outs[1]) <= 2e-5
    if track:
        for layer in range(2):
            assert rel_err(caches[0].weights(layer).cpu(), caches[1].weights(layer).double()) <= 2e-5


@pytest.mark.gpu
def test_a_step_or_prompt_that_fails_is_taken_back_on_the_gpu(monkeypatch):
    """The first layer's step, and a prompt's write, raise before anything is launched; then the same pass again, and one of
    another length."""
    from sisa_amd.kernels import paged as K
    from sisa_amd.kernels import step
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).to(torch.bfloat16).eval()
    ids, counts = token_ids(2, 30, seed=14).to(DEV), [20, 11]
    outs = []
    for failing in (False, True):
        cache = SISAPagedCache(2, 40, page_size=16, track=True)
        with torch.no_grad():
            cache.expect(counts)
            if failing:
                with monkeypatch.context() as m:
                    m.setattr(K, "sisa_paged_write_hip", _failing(1)(K.sisa_paged_write_hip))
                    with pytest.raises(MemoryError):
                        model(ids[:, :25], cache=cache)
                assert cache.lengths == [0, 0]
            got = [model(ids[:, :20], cache=cache, logits_at=[n - 1 for n in counts]).logits]
            for t in range(20, 24):
                if failing:
                    with monkeypatch.context() as m:
                        m.setattr(step, "_step_paged", _failing(1)(step._step_paged))
                        with pytest.raises(MemoryError):
                            model(ids[:, t:t + 1], cache=cache)
                    assert cache.lengths == [n + t - 20 for n in counts]
                got.append(model(ids[:, t:t + 1], cache=cache).logits)
            got.append(model(ids[:, 24:27], cache=cache).logits)
        outs.append(torch.cat(got, 1))
    assert torch.equal(*outs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_step_without_a_place_ends_its_sequence(dtype, monkeypatch):
    """Device tables and lengths that name no place for the new position: NaN, and NaN from then on, also where start and
    lengths are counted on to valid ones; the other sequences as beside sequences that are well."""
    from sisa_amd.kernels import step
    model = tiny_model(seed=3, theta_scale=0.25, attn_impl="auto").to(DEV).to(dtype).eval()
    ids = token_ids(6, 45, seed=18).to(DEV)
    calls, real = [], step.layer_step_paged
    monkeypatch.setattr(step, "layer_step_paged", lambda *a: calls.append(1) or real(*a))
    outs, held = [], []
    for lost in (False, True):
        cache = SISAPagedCache(6, 64, page_size=16, track=True)
        with torch.no_grad():
            model(ids[:, :40], cache=cache)
            before = [cache.weights(layer).clone() for layer in range(2)]
            st, got = cache._store, []
            if lost:                       # the answer of a failed eviction; a length far below; no page; a page outside
                st.end[1], st.end[2] = -1, -1000
                st.table[3, 2], st.table[4, 2] = -1, st.pages
            for t in range(40, 45):
                if lost and t == 41:       # a place again, as if the caller had counted on, and mended the tables
                    assert st.end.tolist()[1] == 0
                    st.end[2] = 41
                    st.table[3, 2], st.table[4, 2] = st.held[3][2], st.held[4][2]
                got.append(model(ids[:, t:t + 1], cache=cache).logits)
                if lost and t == 40:
                    for layer in range(2):
                        assert torch.equal(cache.weights(layer)[1:5], before[layer][1:5])
        outs.append(torch.cat(got, 1))
        held.append([cache.weights(layer) for layer in range(2)])
    assert len(calls) == 20 and outs[0].isfinite().all()
    assert outs[1][1:5].isnan().all()
    for i in (0, 5):
        assert torch.equal(outs[0][i], outs[1][i])
        assert all(torch.equal(a[i], b[i]) for a, b in zip(*held))
