"""Pages of the paged 8-bit cache copied (lbd_kv8_copy_pages) and a beam search's sequences put in order
(lbd_kv8_reorder) on the GPU: bytes, compared with the oracle's."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from oracle import beams as B
from oracle import kv_cache as O
from test_gpu_kv8 import ok
from test_beam import written_once
from test_gpu_kv8_guards import Guarded

pytestmark = pytest.mark.gpu
NAMES = ("k", "v", "ke", "ve")


class Layers:
    """The pools of a decoder's layers, each array between guards."""

    def __init__(self, rng, layers, pages, page, KV, D):
        self.host = [O.Pool(rng, pages, page, KV, D) for _ in range(layers)]
        self.dev = [{n: Guarded(getattr(p, n)) for n in NAMES} for p in self.host]
        self.pools = (K.LbdKv8Pool * layers)(*(K.LbdKv8Pool(*(d[n].ptr for n in NAMES), pages, page, KV, D)
                                               for d in self.dev))

    def check(self, moves):
        """What the layers hold is what they held, after `moves`."""
        for p, d in zip(self.host, self.dev):
            B.move(p, moves)
            for n in NAMES:
                assert np.array_equal(d[n].read(), getattr(p, n)), n


SHAPES = [(1, 16, 1, 32), (3, 32, 2, 64), (2, 128, 8, 128), (65, 16, 3, 32), (5, 64, 1, 128), (1, 128, 70, 32)]


@pytest.mark.parametrize("layers,page,KV,D", SHAPES)
def test_copies(rng, layers, page, KV, D):
    """Pairs in no order, one source twice, a page onto itself, entries outside the pool."""
    pages, up = 17, K.DeviceBuffer.from_array
    L = Layers(rng, layers, pages, page, KV, D)
    order = rng.permutation(pages)
    src = np.concatenate([order[:5], [order[0], order[1], order[10], -1, order[2], 17, 2 ** 31 - 1]])
    dst = np.concatenate([order[5:10], [order[12], order[13], order[10], order[14], -5, order[15], order[16]]])
    ds, dd = up(src.astype(np.int32)), up(dst.astype(np.int32))
    ok(K.lib().lbd_kv8_copy_pages(L.pools, layers, ds.ptr, dd.ptr, len(src), None))
    ok(K.lib().lb_dev_synchronize())
    L.check([(a, b, None) for a, b in zip(src, dst) if 0 <= a < pages and 0 <= b < pages])
    ok(K.lib().lbd_kv8_copy_pages(L.pools, layers, ds.ptr, dd.ptr, 0, None))
    ok(K.lib().lbd_kv8_copy_pages(L.pools, layers, None, None, 0, None))
    ok(K.lib().lb_dev_synchronize())
    L.check([])


def test_many_copies(rng):
    pages, up = 3000, K.DeviceBuffer.from_array
    L = Layers(rng, 2, pages, 16, 2, 32)
    order = rng.permutation(pages).astype(np.int32)
    ds, dd = up(order[:1400]), up(order[1400:2800])
    ok(K.lib().lbd_kv8_copy_pages(L.pools, 2, ds.ptr, dd.ptr, 1400, None))
    ok(K.lib().lb_dev_synchronize())
    L.check([(a, b, None) for a, b in zip(order[:1400], order[1400:2800])])


@pytest.mark.parametrize("n,layers,page,KV,D", [(9 << 20, 1, 16, 1, 32), (1 << 21, 5, 16, 1, 32), (70000, 64, 128, 2, 128)])
def test_more_copies_than_a_launch_holds(rng, n, layers, page, KV, D):
    """Calls of more than 2^24 workgroups: pairs at their beginning and end and around the launches' ends, all
    others skipped."""
    pages, up = 40, K.DeviceBuffer.from_array
    L = Layers(rng, layers, pages, page, KV, D)
    parts = -(-KV * page * D // (1 << 14))
    most = (2 ** 32 - 1) // 256 // layers // (2 * parts)
    assert 2 * n * parts * layers >= 1 << 24 and most < n
    src, dst, order = np.full(n, -1, np.int32), np.full(n, 3, np.int32), rng.permutation(pages)
    at = [0, 1, most - 1, most, most + 1, n - 2, n - 1]
    src[at], dst[at] = order[:7], order[7:14]
    ds, dd = up(src), up(dst)
    ok(K.lib().lbd_kv8_copy_pages(L.pools, layers, ds.ptr, dd.ptr, n, None))
    ok(K.lib().lb_dev_synchronize())
    L.check([(a, b, None) for a, b in zip(order[:7], order[7:14])])


def test_recorded_copies(rng):
    """A replayed graph copies the pages that the arrays name by then; two graphs of other layers in turn."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    lays = [Layers(rng, n, 12, 16, 2, 32) for n in (2, 70)]
    ds, dd, s = up(np.zeros(4, np.int32)), up(np.zeros(4, np.int32)), C.c_void_p()
    ok(L.lb_stream_create(C.byref(s)))
    graphs = []
    for lay in lays:
        ex = C.c_void_p()
        ok(L.lb_stream_begin_capture(s.value))
        rc = L.lbd_kv8_copy_pages(lay.pools, len(lay.host), ds.ptr, dd.ptr, 4, s.value)
        ok(L.lb_stream_end_capture(s.value, C.byref(ex)))
        ok(rc)
        graphs.append(ex.value)
    for _ in range(4):
        order = rng.permutation(12).astype(np.int32)
        ok(L.lb_memcpy_h2d(ds.ptr, order.ctypes.data, 16))
        ok(L.lb_memcpy_h2d(dd.ptr, order[4:].copy().ctypes.data, 16))
        for g in graphs:
            ok(L.lb_graph_launch(g, s.value))
        ok(L.lb_stream_synchronize(s.value))
        for lay in lays:
            lay.check([(a, b, None) for a, b in zip(order[:4], order[4:8])])
    for g in graphs:
        ok(L.lb_graph_destroy(g))
    ok(L.lb_stream_destroy(s.value))


def test_pools_past_32_bits():
    """Pages 5 GB into a pool copied to its front and back, whole and by a beam's tokens."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    pages, page, KV, D = 40000, 128, 8, 128
    one = KV * page * D
    bufs = [K.DeviceBuffer(pages * one), K.DeviceBuffer(pages * one), K.DeviceBuffer(pages * KV), K.DeviceBuffer(pages * KV)]
    for b in bufs:
        ok(L.lb_memset_d(b.ptr, 7, b.nbytes))
    ok(L.lb_dev_synchronize())
    pool = (K.LbdKv8Pool * 1)(K.LbdKv8Pool(*(b.ptr for b in bufs), pages, page, KV, D))
    rng = np.random.default_rng(0)
    held = [rng.integers(0, 256, n, dtype=np.uint8) for n in (one, one, KV, KV)]
    far = pages - 2

    def put(p, what):
        for b, h in zip(bufs, what):
            ok(L.lb_memcpy_h2d(b.ptr + p * len(h), h.ctypes.data, len(h)))

    def get(p):
        out = [np.empty_like(h) for h in held]
        for b, h in zip(bufs, out):
            ok(L.lb_memcpy_d2h(h.ctypes.data, b.ptr + p * len(h), len(h)))
        return out

    put(far, held)
    src, dst = up(np.array([far, far], np.int32)), up(np.array([3, pages - 1], np.int32))
    ok(L.lbd_kv8_copy_pages(pool, 1, src.ptr, dst.ptr, 2, None))
    ok(L.lb_dev_synchronize())
    for p in (3, pages - 1, far):
        assert all(np.array_equal(a, b) for a, b in zip(get(p), held))
    assert all((x == 7).all() for p in (2, 4, pages - 3) for x in get(p))
    # two children of a beam whose page lies far: 70 tokens of it into another far page
    table, own = np.array([[far], [-1]], np.int32), np.array([[far], [pages - 5]], np.int32)
    a = [up(x) for x in (np.zeros(2, np.int32), np.array([69, -1], np.int32), table, own)]
    new_past, new_table = up(np.zeros(2, np.int32)), up(np.zeros((2, 1), np.int32))
    o = K.LbdKv8Order(a[0].ptr, None, a[1].ptr, a[2].ptr, a[3].ptr, new_past.ptr, new_table.ptr, 1, 2, 1, 1)
    ok(L.lbd_kv8_reorder(pool, 1, C.byref(o), None))
    ok(L.lb_dev_synchronize())
    assert list(new_table.to_array((2,), np.int32)) == [far, pages - 5]
    got = get(pages - 5)
    for x, h in zip(got[:2], held):
        x, h = x.reshape(KV, page, D), h.reshape(KV, page, D)
        assert np.array_equal(x[:, :70], h[:, :70]) and (x[:, 70:] == 7).all()
    assert np.array_equal(got[2], held[2]) and np.array_equal(got[3], held[3])


# ---------------------------------------------------------------- beams

def family(rng, prompts, W, page, wide, lengths=None):
    """A state as a search leaves it: table, own, past and the pages; in every prompt the pages being
    written are own's, in another order."""
    places = prompts * W
    top = wide * page
    past = np.repeat([int(rng.integers(0, top)) for _ in range(prompts)] if lengths is None else lengths, W)
    pages = places * wide + 4
    own = rng.permutation(pages)[:places * wide].reshape(places, wide).astype(np.int32)
    table = np.full((places, wide), -1, np.int32)
    for g in range(prompts):
        at = past[g * W] // page
        shared = own[g * W:(g + 1) * W]
        for i in range(g * W, (g + 1) * W):
            table[i, :at] = [shared[rng.integers(W), j] for j in range(at)]
            own[i, :at] = -1 if i % 2 else own[i, :at]
        table[g * W:(g + 1) * W, at] = rng.permutation(shared[:, at])
    return pages, past.astype(np.int32), table, own


def run(rng, prompts, W, page, wide, layers, KV, D, parent, done=None, add=1, state=None, check=True):
    L, up = K.lib(), K.DeviceBuffer.from_array
    pages, past, table, own = family(rng, prompts, W, page, wide) if state is None else state
    lay = Layers(rng, layers, pages, page, KV, D)
    places = prompts * W
    arrays = [up(np.asarray(x, np.int32)) for x in (parent, np.zeros(places) if done is None else done, past, table, own)]
    new_past, new_table = Guarded(np.full(places, 99, np.int32)), Guarded(np.full((places, wide), 99, np.int32))
    o = K.LbdKv8Order(arrays[0].ptr, None if done is None else arrays[1].ptr, *(a.ptr for a in arrays[2:]),
                      new_past.ptr, new_table.ptr, prompts, W, wide, add)
    ok(L.lbd_kv8_reorder(lay.pools, layers, C.byref(o), None))
    ok(L.lb_dev_synchronize())
    w_past, w_table, moves = B.reorder(np.asarray(parent), done, past, table, own, W, add, page, pages)
    assert np.array_equal(new_past.read(), w_past)
    assert np.array_equal(new_table.read(), w_table)
    lay.check(moves)
    return w_past, w_table, moves


@pytest.mark.parametrize("prompts,W,page,wide,layers,KV,D", [
    (1, 4, 16, 3, 2, 2, 64), (3, 1, 16, 4, 1, 1, 32), (5, 3, 32, 5, 3, 3, 32), (2, 32, 16, 2, 1, 1, 64),
    (2, 5, 128, 2, 2, 8, 128), (1, 7, 64, 40, 66, 1, 32), (40, 2, 16, 3, 1, 2, 32), (3, 17, 16, 300, 1, 1, 32)])
def test_families(rng, prompts, W, page, wide, layers, KV, D):
    places = prompts * W
    base = np.arange(places) // W * W
    for kind in ("any", "one", "swap", "none", "ended"):
        parent = base + rng.integers(0, W, places)
        done = None
        if kind == "one":  # a single beam's children take every place
            parent = base + rng.integers(0, W)
        if kind == "swap":
            parent = base + (np.arange(places) - base + 1) % W
        if kind == "none":
            parent[rng.random(places) < 0.4] = -1
        if kind == "ended":
            done = (rng.random(places) < 0.3).astype(int)
        for add in (0, 1, 3):
            run(rng, prompts, W, page, wide, layers, KV, D, parent, done, add)


def test_page_ends(rng):
    """A page that has just been filled is shared like the others, and the next one is each place's own."""
    W, page, wide = 4, 16, 4
    for n in (0, 1, 14, 15, 16, 17, 31, 62, 63, 64, 100, 2 ** 30, 2 ** 31 - 1):
        state = list(family(rng, 2, W, page, wide, [min(n, wide * page - 1)] * 2))
        state[1] = np.full(2 * W, n, np.int64).astype(np.int32)
        run(rng, 2, W, page, wide, 1, 1, 32, np.array([0, 0, 3, 3, 4, 5, 4, 4]), state=state)


def test_parents_that_make_no_sense(rng):
    """Places of other prompts, outside the batch, sequences that are none: no sequence."""
    W, page, wide = 3, 16, 3
    pages, past, table, own = family(rng, 3, W, page, wide, [20, 7, 40])
    past[4] = -1
    past[8] = -2 ** 31
    parent = np.array([3, -1, 1, 4, 3, 4, 2 ** 31 - 1, -2 ** 31, 8])
    w_past, _, _ = run(rng, 3, W, page, wide, 1, 2, 32, parent, state=(pages, past, table, own))
    assert list(w_past) == [-1, -1, 21, -1, 8, -1, -1, -1, -1]


def test_pages_that_are_none(rng):
    """Too few pages of one's own, entries outside the pool: places go without, nothing is written there."""
    W, page, wide = 5, 16, 3
    pages, past, table, own = family(rng, 2, W, page, wide, [20, 20])
    own[1, 1], own[2, 1], own[7, 1], own[8, 1], own[9, 1] = -1, pages, -7, 2 ** 31 - 1, -1
    table[6, 1] = -1
    run(rng, 2, W, page, wide, 2, 1, 32, np.array([0, 0, 0, 0, 0, 6, 6, 6, 6, 6]), state=(pages, past, table, own))


def test_lengths_that_differ_within_a_prompt(rng):
    W, page, wide = 4, 16, 4
    pages, past, table, own = family(rng, 1, W, page, wide, [0])
    own = rng.permutation(pages)[:W * wide].reshape(W, wide).astype(np.int32)
    past = np.array([20, 37, 20, 47], np.int32)
    for i in range(W):
        table[i] = own[i]
    run(rng, 1, W, page, wide, 2, 1, 32, np.array([1, 1, 0, 0]), state=(pages, past, table, own))
    run(rng, 1, W, page, wide, 2, 1, 32, np.array([3, 3, 1, 1]), state=(pages, past, table, own))


def test_a_search_of_many_steps(rng):
    """Over many steps of random parents every sequence keeps its own history: each place's token of each
    step, written into its page as the search would write it, is found again through the final table."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    prompts, W, page, KV, D, steps, T0 = 2, 5, 16, 1, 32, 75, 21
    places, wide = prompts * W, 7
    pages = places * wide
    own = rng.permutation(pages).reshape(places, wide).astype(np.int32)
    table = own.copy()
    for g in range(prompts):
        table[g * W:(g + 1) * W] = own[g * W]
    lay = Layers(rng, 2, pages, page, KV, D)
    dev = [up(x) for x in (np.zeros(places, np.int32), np.full(places, T0 - 1, np.int32), table, own)]
    other = [up(np.zeros(places, np.int32)), up(np.zeros((places, wide), np.int32))]
    hist = [[] for _ in range(places)]
    host = [{n: d[n].read() for n in NAMES} for d in lay.dev]
    for t in range(steps):
        parent = np.arange(places) // W * W + (rng.integers(0, W, places) if t else 0)
        ok(L.lb_memcpy_h2d(dev[0].ptr, np.ascontiguousarray(parent, np.int32).ctypes.data, 4 * places))
        o = K.LbdKv8Order(dev[0].ptr, None, dev[1].ptr, dev[2].ptr, dev[3].ptr, other[0].ptr, other[1].ptr, prompts, W,
                          wide, 1)
        ok(L.lbd_kv8_reorder(lay.pools, 2, C.byref(o), None))
        ok(L.lb_dev_synchronize())
        dev[1], other[0] = other[0], dev[1]
        dev[2], other[1] = other[1], dev[2]
        hist = [list(hist[p]) for p in parent]
        # each place writes a token of its own at its position
        tab, n = dev[2].to_array((places, wide), np.int32), T0 + t
        assert (dev[1].to_array((places,), np.int32) == n).all()
        tails = tab[:, n // page]
        assert len(set(tails)) == places
        for d, h in zip(lay.dev, host):
            h["k"] = d["k"].read()
            for i in range(places):
                mark = (7 * t + 31 * i) % 251
                h["k"][tails[i], 0, n % page] = mark
            ok(L.lb_memcpy_h2d(d["k"].ptr, np.ascontiguousarray(h["k"]).ctypes.data, h["k"].nbytes))
        for i in range(places):
            hist[i].append((7 * t + 31 * i) % 251)
    for d in lay.dev:
        k = d["k"].read()
        for i in range(places):
            held = np.concatenate([k[p, 0] for p in tab[i]])[T0:T0 + steps, 0]
            assert list(held) == hist[i]


def test_recorded(rng):
    """A replayed graph of two orders, back and forth between two tables."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    W, page, wide, KV, D = 3, 16, 3, 2, 32
    pages, past, table, own = family(rng, 2, W, page, wide, [17, 17])
    lay = Layers(rng, 3, pages, page, KV, D)
    parents = [up(np.zeros(6, np.int32)) for _ in range(2)]
    a, b = [up(past), up(table)], [up(past), up(table)]
    downs = up(own)
    s, ex = C.c_void_p(), C.c_void_p()
    ok(L.lb_stream_create(C.byref(s)))
    ok(L.lb_stream_begin_capture(s.value))
    rcs = [L.lbd_kv8_reorder(lay.pools, 3, C.byref(K.LbdKv8Order(p.ptr, None, x[0].ptr, x[1].ptr, downs.ptr, y[0].ptr,
                                                                 y[1].ptr, 2, W, wide, 1)), s.value)
           for p, x, y in ((parents[0], a, b), (parents[1], b, a))]
    ok(L.lb_stream_end_capture(s.value, C.byref(ex)))
    assert min(rcs) >= 0
    for _ in range(4):
        for p in parents:
            parent = np.arange(6) // W * W + rng.integers(0, W, 6)
            ok(L.lb_memcpy_h2d(p.ptr, np.ascontiguousarray(parent, np.int32).ctypes.data, 24))
            past, table, moves = B.reorder(parent, None, past, table, own, W, 1, page, pages)
            for q in lay.host:
                B.move(q, moves)
        ok(L.lb_graph_launch(ex.value, s.value))
        ok(L.lb_stream_synchronize(s.value))
        assert np.array_equal(a[0].to_array((6,), np.int32), past)
        assert np.array_equal(a[1].to_array((6, wide), np.int32), table)
        lay.check([])
    ok(L.lb_graph_destroy(ex.value))
    ok(L.lb_stream_destroy(s.value))


@pytest.mark.parametrize("prompts,W,page,wide,layers,KV,D", [
    (1, 2, 16, 4, 1, 1, 32), (3, 4, 16, 7, 2, 2, 64), (2, 7, 32, 5, 3, 1, 32), (1, 32, 16, 12, 1, 1, 32),
    (2, 5, 128, 3, 2, 8, 128), (4, 3, 16, 40, 1, 1, 32)])
def test_lengths_of_any_kind(rng, prompts, W, page, wide, layers, KV, D):
    """Sequences of other lengths within a prompt, over several steps from any state that a step leaves: no
    page that is written has a second owner, and the pools are the oracle's."""
    places, top = prompts * W, wide * page
    pages = places * wide + 3
    own = rng.permutation(pages)[:places * wide].reshape(places, wide).astype(np.int32)
    for kind in ("near", "far", "ended", "full"):
        table = own.copy()
        past = rng.integers(0, top - 2, places) if kind != "near" else rng.integers(0, 2 * page, places)
        if kind == "full":
            past = past // page * page
        for add in (1, 0, 3):
            parent = np.arange(places) // W * W + rng.integers(0, W, places)
            done = (rng.random(places) < 0.3).astype(int) if kind == "ended" else None
            if kind == "far":
                parent[rng.random(places) < 0.2] = -1
            past, table, moves = run(rng, prompts, W, page, wide, layers, KV, D, parent, done, add,
                                     state=(pages, past.astype(np.int32), table.astype(np.int32), own))
            written_once(past, table, moves, page)
