"""KV8Cache's shared pages on the CPU: forks, copies on the first write, pages behind a window, compaction and
resizing. Its device buffers are stand-ins; page copies are carried out on a table of what each page holds."""
import numpy as np
import pytest

from lowbit_amd import kernels as K
from lowbit_amd import model as M
from oracle import beams as B
from test_kv8_cache import Buffer


class Lib:
    def __getattr__(self, name):
        return lambda *a: 0


@pytest.fixture
def new(monkeypatch):
    monkeypatch.setattr(M, "_buf", Buffer)
    monkeypatch.setattr(K.DeviceBuffer, "from_array", classmethod(lambda cls, a: Buffer(a.nbytes)))
    monkeypatch.setattr(K, "lib", lambda: Lib())

    def make(*a, window=0, sinks=0, **k):
        cache = M.KV8Cache(M.tiny_config(window=window, sinks=sinks), *a, **k)
        cache.held = {p: {} for p in range(cache.pages)}  # page -> slot -> token

        def copy(pairs, stream):
            was = {p: dict(c) for p, c in cache.held.items()}
            assert not {d for _, d in pairs} & {x for i, (x, _) in enumerate(pairs)}
            for x, y in pairs:
                cache.held[y] = was[x]
        cache._copy = copy
        return cache

    return make


def write(cache, seq, tokens):
    """What a pass does that appends tokens: nothing is written to a page that another sequence holds."""
    at = int(cache.lengths[seq])
    cache.reserve(seq, at + len(tokens))
    cache.upload()
    for i, t in enumerate(tokens):
        p, slot = int(cache._table[seq, (at + i) // cache.page]), (at + i) % cache.page
        assert cache._refs[p] == 1
        if slot == 0:
            cache.held[p] = {}
        cache.held[p][slot] = t
    cache.commit(seq, at + len(tokens))
    cache.slide(seq)


def read(cache, seq):
    cache.upload()
    return [cache.held[int(cache._table[seq, i // cache.page])].get(i % cache.page) if
            cache._table[seq, i // cache.page] >= 0 else None for i in range(int(cache.lengths[seq]))]


def consistent(cache):
    held = cache._table[cache._table >= 0]
    assert np.array_equal(np.bincount(held, minlength=cache.pages), cache._refs)
    assert sorted(cache._free) == list(np.flatnonzero(cache._refs == 0))
    for i, n in enumerate(cache._held):
        a, b = cache._hole[i]
        assert (cache._table[i, n:] < 0).all() and (cache._table[i, a:b] < 0).all()
        assert (np.delete(cache._table[i, :n], np.arange(a, min(b, n))) >= 0).all()


def test_a_fork_shares_until_it_writes(new):
    cache = new(100, page=16, sequences=3, pages=20)
    write(cache, 0, list(range(40)))
    cache.fork(1, 0)
    assert len(cache._free) == 17 and list(cache.lengths) == [40, 40, 0]
    write(cache, 0, [100])  # the first to write takes a copy of the third page
    write(cache, 1, [200])  # and leaves it to the other
    assert len(cache._free) == 16
    assert read(cache, 0) == [*range(40), 100] and read(cache, 1) == [*range(40), 200]
    cache.fork(2, 1)
    cache.truncate(1, 10)
    write(cache, 1, [5, 6])  # into a page that two others hold
    assert read(cache, 1) == [*range(10), 5, 6] and read(cache, 2) == [*range(40), 200]
    cache.truncate(0)
    cache.truncate(2)
    consistent(cache)
    assert len(cache._free) == 19
    with pytest.raises(ValueError):
        cache.fork(1, 1)


def test_full_pages_are_shared_for_good(new):
    cache = new(64, page=16, sequences=2, pages=4)
    write(cache, 0, list(range(32)))
    cache.fork(1, 0)
    write(cache, 1, [7])  # begins a page of its own: nothing is copied
    assert not cache._copies and len(cache._free) == 1
    with pytest.raises(ValueError):  # two pages more than there are
        write(cache, 0, [1] * 20)
    write(cache, 0, [8])
    assert read(cache, 0)[-1] == 8 and read(cache, 1)[-1] == 7
    consistent(cache)


def test_no_page_for_a_copy(new):
    cache = new(64, page=16, sequences=2, pages=1)
    write(cache, 0, [1, 2])
    cache.fork(1, 0)
    with pytest.raises(ValueError):
        cache.reserve(1, 3)
    cache.reserve(1, 2)  # no new token: no copy
    consistent(cache)
    cache.truncate(0)
    write(cache, 1, [3])
    assert read(cache, 1) == [1, 2, 3]


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 0), (17, 5), (1, 0), (16, 16), (33, 40)])
def test_at_random(new, window, sinks):
    """Forks, writes, cuts, compactions and resizing in any order: every sequence keeps its tokens."""
    rng = np.random.default_rng(window + sinks)
    cache = new(90, page=16, sequences=5, pages=24, window=window, sinks=sinks)
    want, tick = [[] for _ in range(5)], 0
    for _ in range(800):
        s, what = int(rng.integers(5)), rng.random()
        try:
            if what < 0.55:
                n = int(rng.integers(1, 12))
                write(cache, s, list(range(tick, tick + n)))
                want[s] = want[s] + list(range(tick, tick + n))
                tick += n
            elif what < 0.7:
                d = (s + int(rng.integers(1, 5))) % 5
                cache.fork(d, s)
                want[d] = list(want[s])
            elif what < 0.85:
                n = int(rng.integers(0, len(want[s]) + 1)) if rng.random() < 0.7 else 0
                cache.truncate(s, n)
                want[s] = want[s][:n]
            elif what < 0.95:
                assert cache.compact() == np.count_nonzero(cache._refs)
                assert not cache._refs[np.count_nonzero(cache._refs):].any()
            else:
                n = int(rng.integers(18, 30))
                cache.resize(n)
                cache.held = {p: cache.held.get(p, {}) for p in range(n)}
                assert cache.pages == n
        except ValueError:
            for i in range(5):  # what a refused pass had reserved
                cache.commit(i, len(want[i]))
        consistent(cache)
        for i in range(5):
            n = len(want[i])
            assert cache.lengths[i] == n
            got = read(cache, i)
            for at in range(n):  # what the next token sees
                if not window or at < sinks or at > n - window:
                    assert got[at] == want[i][at]
        held = sum(len(set(range(n)) - {x for x in range(n) if window and x >= -(-sinks // 16) * 16
                                        and x // 16 < max(n - window + 1, 0) // 16}) for n in map(len, want))
        assert (cache._table >= 0).sum() * 16 - 15 * 5 <= held


def test_pages_behind_a_window(new):
    cache = new(1000, page=16, sequences=1, pages=6, window=40, sinks=4)
    for t in range(500):  # far more tokens than the pool has slots
        write(cache, 0, [t])
    assert cache.length == 500 and len(cache._free) >= 1
    assert read(cache, 0)[:4] == [0, 1, 2, 3] and read(cache, 0)[-39:] == list(range(461, 500))
    for n in (499, 470, 100, 17):
        with pytest.raises(ValueError):
            if n == 499:
                cache.truncate(0, 459)
            else:
                cache.truncate(0, n)
    cache.truncate(0, 499)  # position 499 still sees 460 .. 498
    cache.truncate(0, 10)   # only the sinks' page
    consistent(cache)
    write(cache, 0, [9] * 30)
    assert read(cache, 0)[:10] == list(range(10))


def test_resize_refuses(new):
    cache = new(64, page=16, sequences=2, pages=6)
    write(cache, 0, [1] * 40)
    for n in (0, -1, 2):
        with pytest.raises(ValueError):
            cache.resize(n)
    cache.resize(3)
    with pytest.raises(ValueError):
        write(cache, 1, [1])
    cache.resize(4)
    write(cache, 1, [1])
    consistent(cache)


def test_batches_of_copies(new):
    """A copy's page freed and taken again before the copies are made: they are made one after the other."""
    cache = new(64, page=16, sequences=4, pages=4)
    write(cache, 0, [1, 2])
    cache.fork(1, 0)
    cache.reserve(1, 3)        # copy of 0's page
    cache.fork(2, 0)
    cache.commit(1, 0)         # its page returns
    cache.reserve(2, 3)        # and is taken for another copy
    cache.fork(3, 2)
    cache.commit(0, 0)
    cache.reserve(3, 3)
    cache.upload()
    cache.commit(2, 2)
    cache.commit(3, 2)
    assert read(cache, 2) == [1, 2] and read(cache, 3) == [1, 2]
    consistent(cache)


def test_a_window_takes_the_8_bit_cache():
    with pytest.raises(ValueError):
        M.KVCache(M.tiny_config(window=8), 10)
    for bad in (dict(window=-1), dict(window=4, sinks=-1), dict(sinks=3)):
        with pytest.raises(ValueError):
            M.Model(M.tiny_config(**bad), {})


@pytest.mark.parametrize("sinks", [0, 4, 40])
def test_a_step_gives_back_only_what_it_left_behind(new, sinks):
    """Behind the window a step looks at no page that has been given back, and a step that gives none back
    leaves the table as the device has it."""
    cache = new(4000, page=16, sequences=2, pages=40, window=50, sinks=sinks)
    walked, drop = [], cache._drop
    cache._drop = lambda seq, first, last: (walked.append(last - first), drop(seq, first, last))
    for t in range(1500):
        held = cache._table.copy()
        for s in (0, 1):
            at = int(cache.lengths[s])
            cache.reserve(s, at + 1)
        cache.upload()
        assert not cache._dirty
        for s in (0, 1):
            cache.lengths[s] += 1
            cache.slide(s)
        assert cache._dirty == ((held >= 0) & (cache._table < 0)).any()
        consistent(cache)
    assert max(walked) == 1 and len(walked) <= 2 * (1500 // 16)
    # cut down to the sinks the hole is gone, and grows anew
    left = min(sinks, 3)
    cache.truncate(0, left)
    assert not cache._hole[0].any()
    write(cache, 0, [7] * 200)
    consistent(cache)
    assert cache._hole[0, 1] == (200 + left - 50 + 1) // 16


def test_many_copies_in_several_calls(new, monkeypatch):
    """A call takes 2^24 pairs; more of them are cut."""
    cache, calls = new(64, page=16), []
    del cache._copy  # the method itself
    monkeypatch.setattr(Lib, "__getattr__", lambda self, name: lambda *a: calls.append(a[4]) or 0)
    monkeypatch.setattr(K.DeviceBuffer, "from_array", classmethod(lambda cls, a: Buffer(a.nbytes)))
    cache._copy([(0, 1)] * 5, None)
    assert calls == [5]

    class Pairs:  # as long as a pool of small pages may be, without its memory
        def __len__(self):
            return (1 << 25) + 3

        def __getitem__(self, part):
            return [(part.start, 0)]

    cache._copy(Pairs(), None)
    assert calls[1:] == [1 << 24, 1 << 24, 3]


class Counted(Buffer):
    """A stand-in whose bytes are counted while it lives."""
    live, peak, room = 0, 0, 1 << 60

    def __init__(self, nbytes):
        if Counted.live + nbytes > Counted.room:
            self.nbytes = 0
            raise MemoryError
        super().__init__(nbytes)
        Counted.live += nbytes
        Counted.peak = max(Counted.peak, Counted.live)

    def __del__(self):
        Counted.live -= self.nbytes


def test_resize_does_not_need_two_pools(new, monkeypatch):
    """Peak: the larger pool and one buffer. Where even that is too much the cache is a whole one of the fewer
    pages, with what it held."""
    monkeypatch.setattr(M, "_buf", Counted)
    Counted.live, Counted.room = 0, 1 << 60
    cache = new(3200, page=16, pages=200)
    layers, code, exps = len(cache.layers), cache._kv * 16 * cache._d, cache._kv
    rest = Counted.live - layers * 200 * 2 * (code + exps)
    size = lambda pages: rest + layers * pages * 2 * (code + exps)  # noqa: E731
    write(cache, 0, list(range(100)))
    whole = lambda: [[b.nbytes for b in x] for _, x in cache.layers]  # noqa: E731
    for pages in (50, 170, 170, 169):
        top = max(size(cache.pages), size(pages))
        Counted.peak = 0
        cache.resize(pages)
        assert Counted.live == size(pages) == size(cache.pages) and Counted.peak <= top + pages * code
        assert whole() == [[pages * code] * 2 + [pages * exps] * 2] * layers
        assert read(cache, 0) == list(range(100)) and len(cache._free) == pages - 7
    for pages, room, left in ((300, size(240), 169), (20, size(169) + 10 * code, 20)):
        Counted.room = room
        with pytest.raises(MemoryError):
            cache.resize(pages)
        Counted.room = 1 << 60
        assert cache.pages == left and len(cache._refs) == left and all(p.pages == left for p in cache.pools)
        assert all(n >= left * m for b in whole() for n, m in zip(b, (code, code, exps, exps)))
        consistent(cache)
        assert read(cache, 0) == list(range(100))
    write(cache, 0, list(range(100, 320)))
    with pytest.raises(ValueError):
        write(cache, 0, [1])
    cache.resize(40)
    assert Counted.live == size(40)
    write(cache, 0, [320])
    assert read(cache, 0) == list(range(321))


def test_fork_by_negative_and_wrong_indexes(new):
    """A sequence named in two ways is one sequence; a source that is none leaves the destination as it is."""
    cache = new(64, page=16, sequences=3, pages=9)
    write(cache, 0, list(range(20)))
    write(cache, 2, [7] * 5)
    for dst, src in ((2, -1), (-1, 2), (0, -3)):
        with pytest.raises(ValueError):
            cache.fork(dst, src)
    for dst, src in ((2, 3), (2, -4), (3, 0), (-4, 0)):
        with pytest.raises(IndexError):
            cache.fork(dst, src)
    assert read(cache, 0) == list(range(20)) and read(cache, 2) == [7] * 5
    cache.fork(-2, -3)
    assert read(cache, 1) == list(range(20))
    write(cache, 1, [9])
    assert read(cache, 0) == list(range(20)) and read(cache, 1)[-1] == 9
    consistent(cache)


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 4), (1, 0), (40, 50), (33, 0), (17, 16)])
@pytest.mark.parametrize("W,prompts,steps", [(1, [5], 60), (3, [37], 100), (4, [16, 3, 50], 70), (2, [90, 32], 1), (5, [7], 0)])
def test_beams_in_as_many_pages_as_they_are_said_to_take(new, window, sinks, W, prompts, steps):
    """A search's table work by hand, on a pool of exactly the pages that beam_pages asks for: sequences of random
    parents, some ended, find their tokens again, and the pool never runs out."""
    rng = np.random.default_rng(W + steps + window)
    n, G = len(prompts) * W, len(prompts)
    for turn in range(3):  # earlier turns in the first sequences, the last of them shared with another prompt's
        cache = new(300, page=16, sequences=n, pages=400, window=window, sinks=sinks)
        for g in range(G):
            if turn == 1 or (turn == 2 and g == 0):
                write(cache, g * W, list(range(1000, 1021 + 30 * g + 20 * (turn == 2))))
            elif turn == 2:
                cache.fork(g * W, 0)
        ends = [int(cache.lengths[g * W]) + p for g, p in enumerate(prompts)]
        copies = [bool(cache.lengths[g * W] % 16 and cache._refs[cache._table[g * W, cache.lengths[g * W] // 16]] > 1)
                  for g in range(G)]
        more = sum(cache.beam_pages(g * W, ends[g], steps, W) + copies[g] for g in range(G)).max()
        read = sum(max(-(-ends[g] // 16) - int(cache._held[g * W]), 0) + copies[g] for g in range(G))
        cache.resize(int(np.count_nonzero(cache._refs) + max(more, read)))
        assert len(cache._free) == max(more, read)
        want = [[] for _ in range(n)]
        for g, p in enumerate(prompts):
            tokens = list(range(10000 * (g + 1), 10000 * (g + 1) + p))
            was = [cache.held[int(cache._table[g * W, x // 16])].get(x % 16) if cache._table[g * W, x // 16] >= 0 else None
                   for x in range(int(cache.lengths[g * W]))]
            want[g * W] = was + tokens
        for g, p in enumerate(prompts):  # all prompts' pages at once, as in a pass
            cache.reserve(g * W, ends[g])
        cache.upload()
        for g, p in enumerate(prompts):
            at = ends[g] - p
            for i, t in enumerate(want[g * W][at:]):
                page, slot = int(cache._table[g * W, (at + i) // 16]), (at + i) % 16
                cache.held[page] = {**(cache.held[page] if slot else {}), slot: t}
            cache.commit(g * W, ends[g])
        for g in range(G):
            cache.slide(g * W)
        hole = cache._hole[::W].copy()
        room, own = cache.beam_room(W, steps, 1)
        table, past, tick, left, rounds = cache._table.copy(), np.where(cache.lengths > 0, cache.lengths, -1), 0, steps, 0
        parent, add = np.arange(n) // W * W, 0
        while True:
            done = (rng.random(n) < 0.02) | (past[parent] < 0)
            past, table, moves = B.reorder(parent, done, past, table, own, W, add, 16, cache.pages)
            for a, b, k in moves:
                cache.held[b] = {s: v for s, v in cache.held[a].items() if s < k} | {
                    s: v for s, v in cache.held[b].items() if s >= k}
            want = [list(want[p]) if past[i] >= 0 else [] for i, p in enumerate(parent)]
            for i in range(n):
                for x in range(max(past[i], 0)):
                    if not window or x < sinks or x > past[i] - window:
                        assert cache.held[int(table[i, x // 16])].get(x % 16) == want[i][x]
            if not left:
                break
            if not room:
                rounds += 1
                cache.adopt(table, past)
                for i in np.flatnonzero(cache.lengths):
                    cache._hole[i] = hole[i // W]
                for i in np.flatnonzero(cache.lengths):
                    cache.slide(i)
                    hole[i // W] = cache._hole[i]
                room, own = cache.beam_room(W, left, 0)
                assert room == left or room % 2 == 0
                table = cache._table.copy()
            for i in np.flatnonzero(past >= 0):  # a step
                page, slot = int(table[i, past[i] // 16]), past[i] % 16
                assert page >= 0
                cache.held[page] = {**(cache.held[page] if slot else {}), slot: tick}
                want[i].append(tick)
                tick += 1
            left, room = left - 1, room - 1
            parent, add = np.arange(n) // W * W + rng.integers(0, W, n), 1
        assert not rounds if not window else rounds or turn or steps < 60 or sinks > 16 or window > 33 or W == 1
        cache.adopt(table, past)
        for i in np.flatnonzero(cache.lengths):
            cache._hole[i] = hole[i // W]
            cache.slide(i)
        consistent(cache)
