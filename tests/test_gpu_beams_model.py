"""The decoder's beam search, forks and sliding window on the paged 8-bit cache (GPU).

The search is compared with one driven by the host: the same passes on forked sequences, and the oracle's
selection in 64 bits. Logits of the two differ by rounding (the LM head takes other numbers of rows), a
sum of n of them by no more than n 1e-4 here, and the random models' offers lie further apart."""
import numpy as np
import pytest

from lowbit_amd import model as M
from oracle import beams as B
from test_gpu_kv8_model import pool_of
from test_gpu_kv8 import check

pytestmark = pytest.mark.gpu


def model_of(backend="w4a16", seed=1, **over):
    cfg = M.tiny_config(max_position=500, **over)
    return M.Model(cfg, M.random_weights(cfg, seed=seed), backend, max_tokens=8)


def by_hand(model, prompts, n_new, W, eos, page):
    """[(tokens, sum)] of each prompt, best first, by forks and passes of the cache's public calls."""
    G, V = len(prompts), model.cfg.vocab_size
    n = G * W
    cache = model.new_cache(max(map(len, prompts)) + n_new, "e4m3", 2 * n, page)  # the beams and their parents
    y = model.forward_batch([prompts[i // W] if i < n and i % W == 0 else [] for i in range(2 * n)], cache)[:n]
    score = np.where(np.arange(n) % W == 0, 0, -np.inf).astype(np.float32)
    done, beams = np.zeros(n, int), [[] for _ in range(n)]
    for t in range(n_new):
        tok, parent, total, end = B.select(np.nan_to_num(y), score, done, W, eos)
        for i in range(n):
            cache.truncate(n + i)
        for i in range(n):
            if parent[i] >= 0 and not end[i]:
                cache.fork(n + i, parent[i])
        for i in range(n):
            cache.truncate(i)
        for i in range(n):
            if parent[i] >= 0 and not end[i]:
                cache.fork(i, n + i)
                cache.truncate(n + i)
        beams = [beams[p] + ([int(v)] if p >= 0 and not done[p] else []) if p >= 0 else None
                 for p, v in zip(parent, tok)]
        score, done = total.astype(np.float32), end
        if t + 1 < n_new:
            feed = [[int(tok[i])] if parent[i] >= 0 and not done[i] else [] for i in range(n)]
            if not any(feed):
                break
            y = model.forward_batch(feed + [[] for _ in range(n)], cache)[:n]
    return [[(beams[i], float(score[i])) for i in range(g, g + W) if beams[i] is not None] for g in range(0, n, W)]


def same(got, want, n_new):
    for a, b in zip(got, want):
        assert [t for t, _ in a] == [t for t, _ in sorted(b, key=lambda x: -x[1])]
        assert np.allclose([s for _, s in a], [s for _, s in sorted(b, key=lambda x: -x[1])], atol=1e-4 * n_new)


@pytest.mark.parametrize("backend", M.BACKENDS)
@pytest.mark.parametrize("W", [1, 3, 4])
def test_one_prompt(backend, W):
    model = model_of(backend)
    prompt = [list(np.random.default_rng(2).integers(0, 97, 21))]
    got = model.generate_beams(prompt, 14, W, length_penalty=0.0)
    assert len(got[0]) == W and all(len(t) == 14 for t, _ in got[0])
    same(got, by_hand(model, prompt, 14, W, -1, 16), 14)
    eager = model.generate_beams(prompt, 14, W, length_penalty=0.0, graph=False)
    assert got == eager
    if W == 1:
        assert got[0][0][0] == model.generate(prompt[0], 14, model.new_cache(64, kv="e4m3", page=16))


@pytest.mark.parametrize("page", [16, 32])
def test_several_prompts(page):
    """Prompts of other lengths, over page ends, on a given cache."""
    model = model_of()
    rng = np.random.default_rng(5)
    prompts = [list(rng.integers(0, 97, n)) for n in (15, 1, 32, 47)]
    cache = model.new_cache(47 + 40, "e4m3", 4 * 5, page)
    got = model.generate_beams(prompts, 40, 5, length_penalty=0.0, cache=cache)
    same(got, by_hand(model, prompts, 40, 5, -1, page), 40)
    # the sequences hold the beams, all but their last token: one pass more gives what the search would have seen
    for g in range(4):
        assert list(cache.lengths[5 * g:5 * g + 5]) == [len(prompts[g]) + 39] * 5
    assert sorted(cache._free) == list(np.flatnonzero(cache._refs == 0))
    y = model.forward_batch([[t[-1]] for g in got for t, _ in g], cache)
    for g in range(4):
        for w, (t, _) in enumerate(got[g]):
            alone = model.new_cache(200, "e4m3", page=page)
            z = model.forward(prompts[g], alone)
            for v in t:
                z = model.forward([v], alone)
            assert np.abs(y[5 * g + w] - z).max() < 1e-2 * np.abs(z).max()


@pytest.mark.parametrize("n_new", [1, 2, 3, 4, 5, 20])
def test_numbers_of_tokens(n_new):
    model = model_of()
    prompts = [list(np.random.default_rng(n).integers(0, 97, n)) for n in (16, 3)]
    cache = model.new_cache(60, "e4m3", 8, 16)
    got = model.generate_beams(prompts, n_new, 4, length_penalty=0.0, cache=cache)
    same(got, by_hand(model, prompts, n_new, 4, -1, 16), n_new)
    assert list(cache.lengths) == [16 + n_new - 1] * 4 + [3 + n_new - 1] * 4
    held = cache._table[cache._table >= 0]
    assert np.array_equal(np.bincount(held, minlength=cache.pages), cache._refs)
    assert all((cache._table[i, :h] >= 0).all() for i, h in enumerate(cache._held))


def test_beams_that_end():
    """With an end token that comes up: ended beams keep their tokens up to it, and stop early together."""
    model = model_of(seed=4)
    prompts = [list(np.random.default_rng(n).integers(0, 97, n)) for n in (9, 14)]
    free = model.generate_beams(prompts, 30, 4, length_penalty=0.0)
    eos = free[0][0][0][5]
    got = model.generate_beams(prompts, 30, 4, eos=eos, length_penalty=0.0)
    want = by_hand(model, prompts, 30, 4, eos, 16)
    same(got, want, 30)
    assert any(len(t) < 30 and t[-1] == eos for g in got for t, _ in g)
    assert all(eos not in t[:-1] for g in got for t, _ in g)
    longer = model.generate_beams(prompts, 200, 4, eos=eos, length_penalty=1.0)
    for g in longer:
        ranks = [s / len(t) for t, s in g]
        assert ranks == sorted(ranks, reverse=True)


def test_continued():
    """A search behind earlier turns whose pages are shared: the other sequence keeps what it holds."""
    model = model_of()
    rng = np.random.default_rng(8)
    head, prompt = list(rng.integers(0, 97, 37)), list(rng.integers(0, 97, 6))
    cache = model.new_cache(120, "e4m3", 3, 16, 30)
    model.forward_batch([head, [], []], cache)
    got = model.generate_beams([prompt], 12, 3, length_penalty=0.0, cache=cache)
    fresh = model.new_cache(120, "e4m3", 3, 16)
    model.forward_batch([head, [], []], fresh)
    assert got == model.generate_beams([prompt], 12, 3, length_penalty=0.0, cache=fresh)
    same(got, by_hand(model, [head + prompt], 12, 3, -1, 16), 12)


def test_refusals():
    model = model_of()
    ok = [[1, 2], [3]]
    full = model.new_cache(50, "e4m3", 4)
    model.forward_batch([[1], [2], [], []], full)
    small = model.new_cache(50, "e4m3", 4, 16, 3)
    before = len(small._free)
    for bad in (dict(prompts=[]), dict(prompts=[[1], []]), dict(beams=0), dict(beams=33), dict(eos=97), dict(eos=-2),
                dict(cache=model.new_cache(50)), dict(cache=model.new_cache(50, "e4m3", 3)), dict(cache=full),
                dict(cache=model.new_cache(10, "e4m3", 4)), dict(cache=small)):
        with pytest.raises(ValueError):
            model.generate_beams(**{**dict(prompts=ok, n_new=20, beams=2), **bad})
    with pytest.raises(IndexError):
        model.generate_beams([[97]], 3)
    assert model.generate_beams(ok, 0) == [[], []]
    assert not small.lengths.any() and len(small._free) == 3  # refused before anything was read
    # just as many pages as the search takes: the prompt's full one, and three of each beam's own
    for pages in (6, 7):
        tight = model.new_cache(60, "e4m3", 2, 16, pages)
        model.forward_batch([[5] * 20, []], tight)
        if pages == 6:
            with pytest.raises(ValueError):
                model.generate_beams([[7, 8]], 39, 2, cache=tight)
            assert list(tight.lengths) == [20, 0]
        else:
            assert len(model.generate_beams([[7, 8]], 39, 2, cache=tight)[0]) == 2
    held = small._table[small._table >= 0]
    assert np.array_equal(np.bincount(held, minlength=3), small._refs) and before == 3


# ---------------------------------------------------------------- forks

def test_forks():
    """A fork and a sequence that got the same tokens by itself are the same from then on, bit for bit; so
    they are in a compacted and in a resized pool."""
    model = model_of()
    rng = np.random.default_rng(3)
    t = lambda n: list(rng.integers(0, 97, n))  # noqa: E731
    p, q = t(21), t(30)
    a, b = (model.new_cache(100, "e4m3", 3, 16, 24) for _ in range(2))
    for c in (a, b):
        model.forward_batch([p, [], []], c)
    a.fork(1, 0)
    model.forward_batch([[], p, []], b)
    for c in (a, b):
        model.forward_batch([[], [], q], c)
    assert len(a._free) == len(b._free) + 2
    for i in range(12):
        step = [t(1), t(1), t(1) if i % 3 else []]
        x, y = model.forward_batch(step, a), model.forward_batch(step, b)
        assert np.array_equal(x, y, equal_nan=True)
        if i == 4:
            a.truncate(2)
            b.truncate(2)
            assert a.compact() == len(np.unique(a._table[a._table >= 0]))
        if i == 7:
            a.resize(13)
            a.resize(20)
    a.fork(2, 1)
    step = [[], t(1), []]
    x, y = model.forward_batch(step, a), model.forward_batch(step, b)
    assert np.array_equal(x[1], y[1])
    assert np.array_equal(model.forward_batch([[], [], step[1]], a)[2], y[1])


# ---------------------------------------------------------------- a window

@pytest.mark.parametrize("window,sinks", [(24, 4), (1, 0), (50, 16), (33, 0)])
def test_window(window, sinks):
    """One layer: the attention of its own rows over the cache, by the oracle with a window."""
    cfg = M.tiny_config(num_layers=1, max_position=400, window=window, sinks=sinks)
    model = M.Model(cfg, M.random_weights(cfg, seed=3), "w4a16")
    H, KV, D = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
    cache = model.new_cache(300, page=16, pages=16)
    assert isinstance(cache, M.KV8Cache)
    rng, past = np.random.default_rng(0), 0
    for n in (37, 1, 1, 60, 1, 90, 1):
        table = cache._table.copy()
        model.forward(rng.integers(0, 97, n), cache)
        rows = model.qkv.to_array((n, (H + 2 * KV) * D), np.float32)
        cache_now = cache._table.copy()
        # the pages as the pass saw them: those that it gave back afterwards were held
        device = cache.table.to_array(cache._table.shape, np.int32)
        assert (device[table >= 0] == table[table >= 0]).all() and (cache_now[device < 0] < 0).all()
        pool, ref = pool_of(cache), np.zeros((n, H * D))
        mags = pool.attention([0, n], [past], device, n, rows[:, :H * D], H, ref, window, sinks)
        check(model.att.to_array((n, H * D), np.float32), ref, mags, D, H)
        past += n
    assert cache.length == past
    used = (cache._table >= 0).sum()
    assert used <= -(-sinks // 16) + window // 16 + 2


def test_a_window_generates():
    """Prompt, graph, eager steps and beams with a window; a cache of few pages serves a long answer by steps."""
    model = model_of(window=20, sinks=4)
    prompt = list(np.random.default_rng(1).integers(0, 97, 50))
    a = model.generate(prompt, 40)
    assert a == model.generate(prompt, 40, model.new_cache(120, page=32), graph=False)
    cache, c = model.new_cache(120, page=16, pages=6), []
    y = model.forward(prompt, cache)
    for _ in range(40):
        c.append(int(y.argmax()))
        y = model.forward(c[-1:], cache)
    assert a == c
    with pytest.raises(ValueError):
        cache.truncate(0, 60)
    got = model.generate_beams([prompt], 25, 3, length_penalty=0.0)
    same(got, by_hand(model, [prompt], 25, 3, -1, 16), 25)
    with pytest.raises(ValueError):
        model.new_cache(50, kv="fp32")
    wide = model_of(window=400)
    assert wide.generate(prompt, 20) == model_of().generate(prompt, 20, model_of().new_cache(100, kv="e4m3"))


class Calls:
    """The library with its calls counted."""

    def __init__(self, lib):
        self.lib, self.n = lib, {}

    def __getattr__(self, name):
        self.n[name] = self.n.get(name, 0) + 1
        return getattr(self.lib, name)


@pytest.mark.parametrize("seed,chunks", [(4, 1), (5, 2)])
@pytest.mark.parametrize("graph", [True, False])
def test_all_beams_ended(seed, chunks, graph):
    """The search stops at the first look, every 32 steps behind the first two, that finds all beams ended, with
    the history up to there: tokens and sums are the host-driven search's. The end token is likely by a channel
    that all embeddings share."""
    eos, n_new, W = 11, 150, 4
    cfg = M.tiny_config(max_position=500, tie_word_embeddings=False)
    weights = M.random_weights(cfg, seed=seed)
    embed, head = weights["model.embed_tokens.weight"], weights["lm_head.weight"]
    embed[:, 0], head[eos] = 3, 0
    head[eos, 0] = 0.6
    head *= 0.3
    model = M.Model(cfg, weights, "w4a16", max_tokens=8)
    prompts = [list(np.random.default_rng(n).integers(0, 97, n)) for n in (9, 14)]
    cache = model.new_cache(14 + n_new, "e4m3", 2 * W, 16)
    model.L = Calls(model.L)
    got = model.generate_beams(prompts, n_new, W, eos=eos, length_penalty=0.0, cache=cache, graph=graph)
    calls, model.L = model.L.n, model.L.lib
    if graph:
        assert calls["lb_graph_launch"] == 16 * chunks
    else:
        assert calls["lbd_beam_select"] == 2 + 32 * chunks
    assert not cache.lengths.any() and len(cache._free) == cache.pages
    assert all(t.index(eos) == len(t) - 1 for g in got for t, _ in g)
    assert 32 * (chunks - 1) + 2 < max(len(t) for g in got for t, _ in g) <= 32 * chunks + 2
    same(got, by_hand(model, prompts, n_new, W, eos, 16), n_new)


@pytest.mark.parametrize("window,sinks,page", [(20, 4, 16), (33, 0, 16), (1, 20, 32), (70, 33, 32)])
@pytest.mark.parametrize("graph", [True, False])
def test_a_window_generates_in_few_pages(window, sinks, page, graph):
    """A pool of no more than the prompt's or a window's pages serves an answer of any length, with the tokens of
    a large one; one of a page less is refused before anything is read."""
    model = model_of(window=window, sinks=sinks)
    rng = np.random.default_rng(2)
    head, prompt, n = list(rng.integers(0, 97, 13)), list(rng.integers(0, 97, 37)), 330
    want = model.generate(head + prompt, n, model.new_cache(400, page=page))
    seen = lambda p: {j for x in range(p + 1) if p - x < window or x < sinks for j in [x // page]}  # noqa: E731
    need = max(-(-50 // page), max(len(seen(p)) for p in range(50, 50 + n - 1)))
    for extra in (0, 1, 3):
        cache = model.new_cache(400, page=page, pages=need + extra)
        model.forward(head, cache)
        assert model.generate(prompt, n, cache, graph=graph) == want
        assert cache.length == 50 + n - 1
        held = cache._table[cache._table >= 0]
        assert np.array_equal(np.bincount(held, minlength=cache.pages), cache._refs)
        assert len(cache._free) == cache.pages - len(held)
    # and goes on: the next pass sees what a large cache's would
    large = model.new_cache(400, page=page)
    model.generate(head + prompt, n, large)
    assert np.array_equal(model.forward(want[-1:], cache), model.forward(want[-1:], large))
    small = model.new_cache(400, page=page, pages=need - 1)
    model.forward(head, small)
    with pytest.raises(ValueError):
        model.generate(prompt, n, small, graph=graph)
    assert small.length == 13
    assert model.generate(head + prompt, n, graph=graph) == want
    assert model.generate_batch([head + prompt, prompt], 60)[0] == want[:60]


@pytest.mark.parametrize("window,sinks,page", [(20, 4, 16), (33, 0, 16), (1, 20, 32), (50, 33, 16)])
@pytest.mark.parametrize("graph", [True, False])
def test_a_window_searches_in_few_pages(window, sinks, page, graph):
    """A pool of the prompts' pages and those in sight serves a search of any length, with the beams of a large
    one and a sequence's earlier turns; smaller ones are refused before anything is read."""
    model = model_of(window=window, sinks=sinks)
    rng = np.random.default_rng(6)
    head, prompts = list(rng.integers(0, 97, 45)), [list(rng.integers(0, 97, n)) for n in (3, 60)]
    large = model.new_cache(360, "e4m3", 8, page)
    model.forward_batch([head] + [[]] * 7, large)
    want = model.generate_beams(prompts, 250, 4, length_penalty=0.0, cache=large)
    same(want, by_hand(model, [head + prompts[0], prompts[1]], 250, 4, -1, page), 250)
    small, taken = None, 0
    for pages in range(5, 8 * -(-350 // page)):
        cache = model.new_cache(360, "e4m3", 8, page, pages)
        try:
            model.forward_batch([head] + [[]] * 7, cache)
            free = list(cache._free)
            got = model.generate_beams(prompts, 250, 4, length_penalty=0.0, cache=cache, graph=graph)
        except ValueError:
            assert list(cache.lengths) in ([0] * 8, [45] + [0] * 7) and (not cache.lengths.any() or cache._free == free)
            continue
        taken += 1
        assert got == want
        assert list(cache.lengths) == [45 + 3 + 249] * 4 + [60 + 249] * 4
        held = cache._table[cache._table >= 0]
        assert np.array_equal(np.bincount(held, minlength=cache.pages), cache._refs)
        assert sorted(cache._free) == list(np.flatnonzero(cache._refs == 0))
        small = small or pages
        if taken == 3:
            break
    in_sight = -(-(window + 1) // page) + 1 + -(-sinks // page)
    assert small <= -(-48 // page) + -(-60 // page) + 8 * in_sight < 8 * 15
    # and on from there: the next pass sees what a large cache's would
    feed = [[t[-1]] for g in want for t, _ in g]
    assert np.array_equal(model.forward_batch(feed, cache), model.forward_batch(feed, large))
    assert model.generate_beams([head + prompts[0], prompts[1]], 250, 4, length_penalty=0.0, graph=graph) == want


def test_a_search_in_few_pages_that_ends(monkeypatch):
    """With end tokens, and with an error in the middle: the sequences are empty where pages of the prompt's have
    been given back."""
    model = model_of(seed=4, window=24, sinks=4)
    prompts = [list(np.random.default_rng(n).integers(0, 97, n)) for n in (9, 14)]
    free = model.generate_beams(prompts, 80, 4, length_penalty=0.0)
    eos = free[0][0][0][40]
    caches = [model.new_cache(120, "e4m3", 8, 16, pages) for pages in (None, 34)]
    got = [model.generate_beams(prompts, 80, 4, eos=eos, length_penalty=0.0, cache=c) for c in caches]
    assert got[0] == got[1] and any(len(t) < 80 for g in got[0] for t, _ in g)
    for c in caches:
        assert [bool(n) for n in c.lengths] == [t[-1] != eos for g in got[0] for t, _ in g]
    cache, n, room = model.new_cache(300, "e4m3", 8, 16, 34), [0], M.KV8Cache.beam_room
    model.forward_batch([prompts[1]] + [[]] * 7, cache)

    def fails(self, *a):
        n[0] += 1
        if n[0] == 3:
            raise KeyboardInterrupt
        return room(self, *a)

    monkeypatch.setattr(M.KV8Cache, "beam_room", fails)
    with pytest.raises(KeyboardInterrupt):
        model.generate_beams(prompts, 250, 4, length_penalty=0.0, cache=cache)
    assert n[0] == 3 and not cache.lengths.any() and len(cache._free) == 34
    n[0] = 2  # before the first step: the prompts, as they were read
    model.forward_batch([prompts[1]] + [[]] * 7, cache)
    with pytest.raises(KeyboardInterrupt):
        model.generate_beams(prompts, 250, 4, length_penalty=0.0, cache=cache)
    assert list(cache.lengths) == [23, 0, 0, 0, 14, 0, 0, 0]
