"""Beam search, the page copies and the windowed attention on the CPU: what their entry points refuse
before any device work."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from oracle import beams as O
from test_kv8 import P, SHAPES, structs

L = K.lib


def window(window=8, sinks=2, H=4, q=P, q_stride=256, out=2 * P, out_stride=256, work=P, work_bytes=1 << 40, **over):
    pool, batch = structs(**over)
    return L().lbd_kv8_attention_window(C.byref(pool), C.byref(batch), q, q_stride, H, window, sinks, out, out_stride,
                                        work, work_bytes, None)


@pytest.mark.parametrize("over", SHAPES + [dict(window=0), dict(window=-3), dict(sinks=-1)], ids=str)
def test_window_shapes(over):
    assert window(**over) == -1
    pool, batch = structs(**over)
    assert L().lbd_kv8_attention_window_work_bytes(C.byref(pool), C.byref(batch), over.get("H", 4),
                                                   over.get("window", 8), over.get("sinks", 2)) == 0


@pytest.mark.parametrize("over,rc", [
    (dict(q_stride=252), -1), (dict(q_stride=258), -1), (dict(out_stride=252), -1), (dict(out_stride=270), -1),
    (dict(q=None), -6), (dict(out=None), -6), (dict(q=P + 4), -6), (dict(out=P + 4), -6), (dict(work=None), -6),
    (dict(work_bytes=16), -6), (dict(work=P + 4), -6)] + [
    (dict([(n, None)]), -6) for n in ("k", "v", "ke", "ve", "q_start", "past", "table")], ids=str)
def test_window_refuses(over, rc):
    assert window(**over) == rc


def test_window_workspace():
    """Whatever the window, no more than the whole cache's; none for null structures."""
    pool, batch = structs(max_pages=2000, T=64, max_new=64)
    whole = L().lbd_kv8_attention_work_bytes(C.byref(pool), C.byref(batch), 4)
    for w, s in ((1, 0), (100, 4), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert 0 < L().lbd_kv8_attention_window_work_bytes(C.byref(pool), C.byref(batch), 4, w, s) <= whole
    assert L().lbd_kv8_attention_window_work_bytes(None, C.byref(batch), 4, 8, 0) == 0


# ---------------------------------------------------------------- pages

def copy(n_pools=2, src=P, dst=P, n=3, second=None, pools=True, **over):
    one = [structs(**over)[0] for _ in range(max(n_pools, 1))]
    if second:
        one[1] = structs(**second)[0]
    arr = (K.LbdKv8Pool * len(one))(*one)
    return L().lbd_kv8_copy_pages(arr if pools else None, n_pools, src, dst, n, None)


POOLS = [(dict(page=p), -1) for p in (0, 8, 24, 256, -16)] + [(dict(D=d), -1) for d in (0, 48, 256)] + [
    (dict(KV=0), -1), (dict(KV=1 << 17), -1), (dict(pages=0), -1), (dict(n_pools=0), -1), (dict(n_pools=-1), -1),
    (dict(pools=False), -6)] + [(dict([(n, None)]), -6) for n in ("k", "v", "ke", "ve")] + [
    (dict([(n, P + 8)]), -6) for n in ("k", "v")] + [
    (dict(second=s), -1) for s in (dict(pages=5), dict(page=32), dict(KV=1), dict(D=32))] + [
    (dict(second=dict(ve=None)), -6), (dict(n_pools=70, second=dict(k=P + 8)), -6)]


@pytest.mark.parametrize("over,rc", POOLS + [(dict(src=None), -6), (dict(dst=None), -6), (dict(n=-1), -1),
                                             (dict(n=(1 << 24) + 1), -1), (dict(n=1 << 24, KV=60000, page=128), -1)],
                         ids=str)
def test_copy_refuses(over, rc):
    assert copy(**over) == rc


def test_no_pages():
    assert copy(n=0) == 0 and copy(n=0, src=None, dst=None) == 0


def order(n_pools=2, second=None, pools=True, null=False, B=2, W=3, max_pages=4, add=1, arrays=(), **over):
    one = [structs(**over)[0] for _ in range(max(n_pools, 1))]
    if second:
        one[1] = structs(**second)[0]
    arr = (K.LbdKv8Pool * len(one))(*one)
    at = dict(parent=P, done=P, past=2 * P, table=3 * P, own=P, new_past=4 * P, new_table=5 * P)
    at.update(arrays)
    o = K.LbdKv8Order(**at, B=B, W=W, max_pages=max_pages, add=add)
    return L().lbd_kv8_reorder(arr if pools else None, n_pools, None if null else C.byref(o), None)


@pytest.mark.parametrize("over,rc", POOLS + [
    (dict(null=True), -6), (dict(B=0), -1), (dict(W=0), -1), (dict(W=33), -1), (dict(B=1 << 20, W=2), -1),
    (dict(max_pages=0), -1), (dict(max_pages=1 << 27), -1), (dict(add=-1), -1), (dict(add=2 ** 31 - 1), -1),
    (dict(B=1 << 20, W=1, KV=60000), -1), (dict(arrays=dict(new_table=3 * P)), -6), (dict(arrays=dict(new_past=2 * P)), -6)] + [
    (dict(arrays=dict([(n, None)])), -6) for n in ("parent", "past", "table", "own", "new_past", "new_table")], ids=str)
def test_reorder_refuses(over, rc):
    assert order(**over) == rc


# ---------------------------------------------------------------- selection

def select(logits=P, ld=100, work=P, work_bytes=1 << 40, null=False, **over):
    f = dict(score=P, done=P, new_score=P, new_done=P, tok=P, parent=P, hist_tok=None, hist_parent=None, step=None,
             hist_len=0, B=2, W=3, V=100, eos=-1)
    f.update(over)
    b = K.LbdBeams(**f)
    return L().lbd_beam_select(logits, ld, None if null else C.byref(b), work, work_bytes, None), b


@pytest.mark.parametrize("over", [dict(B=0), dict(W=0), dict(W=33), dict(B=1 << 20, W=2), dict(V=0),
                                  dict(V=(1 << 24) + 1), dict(V=-5)], ids=str)
def test_select_shapes(over):
    rc, b = select(**over)
    assert rc == -1 and L().lbd_beam_select_work_bytes(C.byref(b)) == 0


@pytest.mark.parametrize("over,rc", [
    (dict(ld=99), -1), (dict(logits=P + 2), -6), (dict(eos=100), -6), (dict(eos=-2), -6), (dict(logits=None), -6), (dict(null=True), -6),
    (dict(work=None), -6), (dict(work=P + 8), -6), (dict(work_bytes=16), -6), (dict(hist_tok=P), -6),
    (dict(step=P, hist_len=3), -6), (dict(hist_tok=P, hist_parent=P, step=P), -6)] + [
    (dict([(n, None)]), -6) for n in ("score", "new_score", "new_done", "tok", "parent")], ids=str)
def test_select_refuses(over, rc):
    assert select(**over)[0] == rc


# ---------------------------------------------------------------- the oracle

def test_oracle_selects():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8], [1, 1, 1], [0.2, 0.3, 0.5]], np.float64))
    tok, parent, total, done = O.select(x, np.log([0.5, 0.4, 0.9, 0.1]), [0, 0, 1, 0], 2, 2)
    assert list(parent) == [1, 0, 2, 3] and list(tok) == [2, 0, 2, 2] and list(done) == [1, 0, 1, 1]
    assert np.allclose(np.exp(total), [0.32, 0.25, 0.9, 0.05])


def test_oracle_reorders():
    """Two children of one parent: the first keeps its page, the other gets a copy in a page that is free."""
    table, own = np.array([[7, 0], [7, 1], [7, 2]]), np.array([[-1, 0], [-1, 1], [-1, 2]])
    past, new, moves = O.reorder(np.array([1, 1, 2]), None, np.array([20, 20, 20]), table, own, 3, 1, 16, 8)
    assert list(past) == [21] * 3 and new.tolist() == [[7, 1], [7, 0], [7, 2]] and moves == [(1, 0, 5)]
    _, new, moves = O.reorder(np.array([1, 1, 2]), None, np.array([15, 15, 15]), table, own, 3, 1, 16, 8)
    assert new.tolist() == [[7, 0], [7, 1], [7, 2]] and not moves


def written_once(new_past, new_table, moves, page):
    """No page that a step writes belongs to a second sequence: destinations of the copies, and the pages that
    the next tokens go to."""
    places, wide = new_table.shape
    to = [b for _, b, _ in moves]
    assert len(set(to)) == len(to) and not set(to) & {a for a, _, _ in moves}
    live = [i for i in range(places) if new_past[i] >= 0]
    full = {i: {int(new_table[i, j]) for j in range(new_past[i] // page)} for i in live}
    for i in live:
        for j in range(new_past[i] // page, wide):
            p = int(new_table[i, j])
            assert p >= 0
            for k in live:
                assert k == i or (p not in full[k] and p not in new_table[k, new_past[k] // page:])


@pytest.mark.parametrize("W", [2, 3, 4, 7])
def test_oracle_reorders_other_lengths(W):
    """Over many steps of sequences of other lengths every sequence keeps its own tokens, and no page that is
    written has two owners. Places that go without a sequence for a while come back as children."""
    rng = np.random.default_rng(W)
    page, wide, G = 16, 6, 2
    places, pages = G * W, G * W * wide
    for trial in range(30):
        own = rng.permutation(pages).reshape(places, wide)
        table, past = own.copy(), rng.integers(0, 40, places)
        held = np.full((pages, page), -1)  # the token in each slot
        hist, tick = [[] for _ in range(places)], 0
        for i in range(places):
            for x in range(past[i]):
                held[table[i, x // page], x % page] = tick
                hist[i].append(tick)
                tick += 1
        for _ in range(25):
            add = int(rng.integers(0, 4))
            for i in range(places):  # the pass appends
                for x in range(past[i], past[i] + add) if past[i] >= 0 else ():
                    held[table[i, x // page], x % page] = tick
                    hist[i].append(tick)
                    tick += 1
            parent = np.arange(places) // W * W + rng.integers(0, W, places)
            done = rng.random(places) < 0.1
            past, new_table, moves = O.reorder(parent, done, past, table, own, W, add, page, pages)
            written_once(past, new_table, moves, page)
            before = held.copy()
            for a, b, n in moves:
                held[b, :n] = before[a, :n]
            table, hist = new_table, [list(hist[p]) if past[i] >= 0 else [] for i, p in enumerate(parent)]
            for i in range(places):
                assert [held[table[i, x // page], x % page] for x in range(past[i])] == hist[i]
            if past.max() + 4 > wide * page:
                break


def test_reorder_bounds_its_places():
    """B W (2 x a page's 16 KB of K codes + 1) below 2^24: a page of 64 heads of 64 and 128 tokens has 32."""
    assert order(B=((1 << 24) - 1) // 65 + 1, W=1, KV=64, page=128) == -1
