"""Attention with a sliding window and sinks over the paged 8-bit cache (GPU) against the oracle:
lbd_kv8_attention_window. The arithmetic is lbd_kv8_attention's over fewer keys, so the tolerance is
its own (tests/test_gpu_kv8.py)."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from test_gpu_kv8 import FILL, HEADS, SEQS, Device, batch_of, cached, check, ok

pytestmark = pytest.mark.gpu


def attend(dev, q, H, out_width, window, sinks, stream=None, work=None):
    """The call on a Device's pool and batch; the workspace lies before a guard."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    dq, do = up(q), up(np.full((len(q), out_width), FILL))
    need = L.lbd_kv8_attention_window_work_bytes(C.byref(dev.pool), C.byref(dev.batch), H, window, sinks)
    assert need
    ws = up(np.full(need + 16, 0xFF, np.uint8)) if work is None else work  # needs no clearing
    ok(L.lbd_kv8_attention_window(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, q.shape[1], H, window, sinks, do.ptr,
                                  out_width, ws.ptr, need, stream))
    ok(L.lb_dev_synchronize())
    if work is None:
        assert (ws.to_array((need + 16,), np.uint8)[need:] == 0xFF).all()
    return do.to_array((len(q), out_width), np.float32)


def give_back(table, page, seqs, window, sinks):
    """The table without the pages that no new token's window or sinks reach."""
    t = table.copy()
    for b, (p, n) in enumerate(seqs):
        for j in range(t.shape[1]):
            if j * page >= sinks and (j + 1) * page <= max(p, 0) - window + 1:
                t[b, j] = -1
    return t


def run(rng, D, page, KV, H, seqs, window, sinks, pad=2, extra=1, gone=True, pool=None, table=None, max_new=None):
    pages, q_start, past, t, T = batch_of(rng, page, seqs, pad, extra)
    table = t if table is None else table
    pool = cached(rng, pages, page, KV, D, table, seqs) if pool is None else pool
    if gone:  # what they hold is anyone's
        table = give_back(table, page, seqs, window, sinks)
        free = np.setdiff1d(np.arange(pool.pages), table)
        for n in ("k", "v", "ke", "ve"):
            getattr(pool, n)[free] = 0xFF
    q = (rng.standard_normal((T, H * D + 4)) * 1.5).astype(np.float32)
    max_new = max(n for _, n in seqs) if max_new is None else max_new
    got = attend(Device(pool, q_start, past, table, max_new, T), q, H, H * D + 8, window, sinks)
    ref = np.full(got.shape, FILL, np.float64)
    mags = pool.attention(q_start, past, table, max_new, q, H, ref, window, sinks)
    check(got, ref, mags, D, H)
    return got


WINDOWS = [(1, 0), (1, 1), (5, 3), (16, 16), (17, 0), (33, 40), (64, 4), (100, 17), (1000, 4), (3, 1000)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("seqs", SEQS, ids=str)
@pytest.mark.parametrize("D,page,KV,H", [(64, 16, 2, 14), (128, 32, 1, 4), (32, 64, 3, 3), (128, 128, 1, 33)])
def test_lengths(rng, D, page, KV, H, seqs, window, sinks):
    run(rng, D, page, KV, H, SEQS[seqs], window, sinks)


@pytest.mark.parametrize("D,page,KV,H", HEADS)
def test_heads(rng, D, page, KV, H):
    run(rng, D, page, KV, H, [(200, 1), (90, 40), (0, 77), (30, 0), (7, 1)], 48, 5)


@pytest.mark.parametrize("window,sinks", [(1, 0), (15, 2), (16, 16), (300, 0), (1024, 4), (2000, 130), (4000, 1)])
@pytest.mark.parametrize("past", [255, 1000, 1039, 1040, 2047, 4100, 9000])
def test_steps(rng, past, window, sinks):
    """Long sequences, whose windows begin anywhere in a tile and a page, beside short ones."""
    for D, page, KV, H in ((64, 16, 2, 14), (128, 64, 1, 4)):
        run(rng, D, page, KV, H, [(past, 1), (past // 2 + 3, 1), (3, 1)], window, sinks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (31, 4), (128, 16), (500, 100)])
@pytest.mark.parametrize("past,new", [(0, 17), (0, 400), (500, 33), (1, 64), (900, 300)])
def test_prompts(rng, past, new, window, sinks):
    for D, page, KV, H in ((64, 16, 2, 14), (128, 64, 1, 4), (32, 128, 1, 1), (128, 32, 1, 5)):
        run(rng, D, page, KV, H, [(past, new)], window, sinks)


@pytest.mark.parametrize("D,KV,H,seqs,window", [
    (32, 1, 2, [(40000, 1)], 30000), (128, 8, 8, [(3100 - 20 * i, 1) for i in range(40)], 1500),
    (64, 1, 24, [(4000, 90)], 2000), (128, 8, 56, [(0, 500), (3000, 20)], 700),
    (32, 8, 64, [(0, 950), (2500, 80)], 300)], ids=str)
def test_slices(rng, D, KV, H, seqs, window):
    run(rng, D, 32, KV, H, seqs, window, 20)


@pytest.mark.parametrize("D,KV,H,seqs,window", [
    # row blocks of prompts taken whole, steps beside them cut into slices, and the other way round
    (64, 2, 14, [(1200, 300)] * 3 + [(3000, 1), (2500, 2)] * 4, 1800),
    (128, 1, 4, [(2500, 100), (2400, 1), (5, 1)], 500), (64, 2, 14, [(4000, 30), (3900, 1)], 2600),
    # two waves a workgroup: short windows of many row blocks, alone and beside steps
    (64, 8, 32, [(0, 1100)], 100), (32, 8, 64, [(10, 800), (700, 1), (0, 90), (300, 3)], 200),
    (128, 8, 32, [(0, 790), (900, 1)], 33), (32, 64, 256, [(3, 400)], 900)], ids=str)
def test_ways_of_cutting(rng, D, KV, H, seqs, window):
    run(rng, D, 64, KV, H, seqs, window, 6)


def test_many_sequences(rng):
    seqs = [(int(rng.integers(0, 90)), int(rng.integers(0, 3))) for _ in range(150)]
    run(rng, 64, 16, 1, 4, seqs, 20, 3)


def test_a_window_of_everything(rng):
    """A window as long as the sequences is lbd_kv8_attention: each within the tolerance of the other's
    result in 64 bits (keys may be cut into other slices)."""
    for seqs in ([(700, 1)], [(40, 90)], [(5, 1), (300, 40), (0, 3)]):
        pages, q_start, past, table, T = batch_of(rng, 32, seqs, 1, 1)
        pool = cached(rng, pages, 32, 2, 64, table, seqs)
        q = rng.standard_normal((T, 8 * 64)).astype(np.float32)
        most = max(n for _, n in seqs)
        dev, ref = Device(pool, q_start, past, table, most, T), np.full(q.shape, FILL, np.float64)
        mags = pool.attention(q_start, past, table, most, q, 8, ref)
        check(dev.attention(q, 8, 8 * 64), ref, mags, 64, 8)
        for window, sinks in ((2000, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 5000)):
            check(attend(dev, q, 8, 8 * 64, window, sinks), ref, mags, 64, 8)


def test_positions_past_the_table(rng):
    """Tokens at positions that the table does not reach see the sinks and what is left of their window."""
    D, page, KV, H = 64, 16, 1, 4
    table = np.array([[3, 1, 0]], np.int32)
    pool = cached(rng, 5, page, KV, D, table, [(0, 48)])
    for past, n in ((40, 30), (47, 3), (60, 2), (100, 40), (5000, 1)):
        for window, sinks in ((8, 3), (20, 20), (1, 0), (90, 0), (30, 48)):
            pages, q_start, pasts, _, T = batch_of(rng, page, [(past, n)], 1, 0)
            q = rng.standard_normal((T, H * D)).astype(np.float32)
            got = attend(Device(pool, q_start, pasts, table, n, T), q, H, H * D, window, sinks)
            ref = np.full(got.shape, FILL, np.float64)
            mags = pool.attention(q_start, pasts, table, n, q, H, ref, window, sinks)
            check(got, ref, mags, D, H)


@pytest.mark.parametrize("seqs", [[(150, 1)], [(100, 60)]], ids=str)
def test_without_pages(rng, seqs):
    """Pages inside the window that are gone are left out; a row with none left gets zeros."""
    D, page, KV, H = 64, 16, 2, 4
    table = np.array([[4, 3, 6, 8, -1, 5, 99, 2, -7, 1, 2 ** 31 - 1]], np.int32)
    pool = cached(rng, 9, page, KV, D, table, seqs)
    run(rng, D, page, KV, H, seqs, 70, 4, pool=pool, table=table, gone=False)
    got = run(rng, D, page, KV, H, seqs, 70, 0, pool=pool, table=np.full((1, 11), -1, np.int32), gone=False)
    assert not got[:seqs[0][1], :H * D].any()


@pytest.mark.parametrize("which", ["ke", "ve"])
@pytest.mark.parametrize("seqs", [[(150, 1)], [(100, 60)]], ids=str)
def test_nan_blocks(rng, seqs, which):
    """A NaN block reaches the rows whose window or sinks reach it, and no others."""
    D, page, KV, H = 64, 16, 2, 4
    table = np.arange(11, dtype=np.int32)[None, ::-1].copy()
    for j in (0, 1, 5, 8):
        pool = cached(rng, 11, page, KV, D, table, seqs)
        getattr(pool, which)[table[0, j], 1] = 255
        run(rng, D, page, KV, H, seqs, 40, 7, pool=pool, table=table, gone=False)


def test_values_that_the_window_left_behind(rng):
    """Blocks behind the window may be as large as they like: what the rows see decides their precision."""
    D, page, KV, H = 64, 16, 1, 2
    for seqs in ([(150, 1)], [(130, 16)]):
        pages, q_start, past, table, T = batch_of(rng, page, seqs, 0, 0)
        pool = cached(rng, pages, page, KV, D, table, seqs)
        pool.ve[table[0, :4], 0] = 230
        pool.ke[table[0, :4], 0] = 200
        got = run(rng, D, page, KV, H, seqs, 40, 0, pad=0, extra=0, pool=pool, table=table, gone=False)
        assert np.abs(got[:, :H * D]).max() < 1e4


def test_batches_that_make_no_sense(rng):
    """q_start that runs backwards or outside the rows, positions near 2^31: inside the workspace."""
    D, page, KV, H, T = 64, 16, 1, 2, 5
    from oracle import kv_cache as O
    pool = O.Pool(rng, 4, page, KV, D)
    q_start = np.array([-9, 3, 2, 2 ** 31 - 1, 2], np.int64).astype(np.int32)
    past = np.array([2 ** 31 - 1, 5, -2 ** 31, 30], np.int64).astype(np.int32)
    table = np.array([[0, 1]] * 4, np.int32)
    q = rng.standard_normal((T, H * D)).astype(np.float32)
    dev = Device(pool, q_start, past, table, T, T)
    for window, sinks in ((1, 0), (20, 3), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert attend(dev, q, H, H * D, window, sinks).shape == (T, H * D)


def test_a_recorded_call_takes_other_lengths(rng):
    """A replayed graph reads lengths, tables and rows anew; two graphs share the workspace in turn."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    D, page, KV, H, B, wide = 64, 16, 2, 8, 3, 100
    cases = [[(1500, 1), (20, 1), (800, 1)], [(3, 1), (1400, 1), (0, 1)], [(1000, 1), (1001, 1), (1002, 1)]]
    seqs0 = [(1598, 2)] * B
    pages, q_start, _, table, T = batch_of(rng, page, [(p, 1) for p, _ in seqs0], 0, 0)
    assert table.shape[1] == wide
    pool = cached(rng, pages, page, KV, D, table, seqs0)
    q = rng.standard_normal((T, H * D)).astype(np.float32)
    dev = Device(pool, q_start, [0] * B, table, 1, T)
    dq, outs = up(q), [up(np.zeros((T, H * D), np.float32)) for _ in range(2)]
    args = [(300, 4), (90, 0)]
    need = max(L.lbd_kv8_attention_window_work_bytes(C.byref(dev.pool), C.byref(dev.batch), H, *a) for a in args)
    ws, s = up(np.zeros(need, np.uint8)), C.c_void_p()
    ok(L.lb_stream_create(C.byref(s)))
    graphs = []
    for a, o in zip(args, outs):
        ok(L.lb_stream_begin_capture(s.value))
        rc = L.lbd_kv8_attention_window(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, H * D, H, *a, o.ptr, H * D,
                                        ws.ptr, need, s.value)
        ex = C.c_void_p()
        ok(L.lb_stream_end_capture(s.value, C.byref(ex)))
        ok(rc)
        graphs.append(ex.value)
    for seqs in cases + cases[:1]:
        past = np.array([p for p, _ in seqs], np.int32)
        ok(L.lb_memcpy_h2d(dev.arrays[1].ptr, past.ctypes.data, past.nbytes))
        for g in graphs:
            ok(L.lb_graph_launch(g, s.value))
        ok(L.lb_stream_synchronize(s.value))
        for a, o in zip(args, outs):
            got, ref = o.to_array((T, H * D), np.float32), np.zeros((T, H * D))
            mags = pool.attention(q_start, past, table, 1, q, H, ref, *a)
            check(got, ref, mags, D, H)
            assert np.array_equal(got, attend(dev, q, H, H * D, *a))
    for g in graphs:
        ok(L.lb_graph_destroy(g))
    ok(L.lb_stream_destroy(s.value))


@pytest.mark.parametrize("seqs", [[(200, 1)], [(150, 60)], [(200, 1), (170, 40)]], ids=str)
def test_far_positions(rng, seqs):
    """Behind 2^30 - 2^12 positions in a table of 2^30 a window reads what it reads near the beginning, bit for bit."""
    D, page, KV, H, far = 64, 128, 2, 4, (1 << 30) - (1 << 12)
    pages, q_start, past, table, T = batch_of(rng, page, seqs, 1, 0)
    pool = cached(rng, pages, page, KV, D, table, seqs)
    q, most = rng.standard_normal((T, H * D)).astype(np.float32), max(n for _, n in seqs)
    near = np.full((len(seqs), 32), -1, np.int32)
    near[:, :table.shape[1]] = table
    long = np.full((len(seqs), 1 << 23), -1, np.int32)
    long[:, far // page:far // page + table.shape[1]] = table
    for window in (1, 100, 128):  # (longer ones see positions that only one of the two has)
        want = attend(Device(pool, q_start, past, near, most, T), q, H, H * D, window, 0)
        got = attend(Device(pool, q_start, past + far, long, most, T), q, H, H * D, window, 0)
        assert np.array_equal(got, want)
        ref = np.full(got.shape, FILL, np.float64)
        check(got, ref, pool.attention(q_start, past, near, most, q, H, ref, window, 0), D, H)


def test_two_streams(rng):
    """Two calls at once on two streams, with a workspace each."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    D, page, KV, H = 128, 32, 2, 8
    runs = []
    for seqs, window in (([(3000, 1), (900, 1)], 2000), ([(40, 400)], 900)):
        pages, q_start, past, table, T = batch_of(rng, page, seqs, 0, 0)
        pool = cached(rng, pages, page, KV, D, table, seqs)
        q, most = rng.standard_normal((T, H * D)).astype(np.float32), max(n for _, n in seqs)
        dev, st = Device(pool, q_start, past, table, most, T), C.c_void_p()
        ok(L.lb_stream_create(C.byref(st)))
        need = L.lbd_kv8_attention_window_work_bytes(C.byref(dev.pool), C.byref(dev.batch), H, window, 4)
        runs.append((dev, up(q), up(np.zeros_like(q)), up(np.zeros(need, np.uint8)), need, st, window,
                     attend(dev, q, H, H * D, window, 4)))
    ok(L.lb_dev_synchronize())
    for _ in range(5):
        for dev, dq, do, ws, need, st, window, _ in runs:
            ok(L.lbd_kv8_attention_window(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, H * D, H, window, 4, do.ptr,
                                          H * D, ws.ptr, need, st.value))
    ok(L.lb_dev_synchronize())
    for dev, dq, do, ws, need, st, window, want in runs:
        assert np.array_equal(do.to_array(want.shape, np.float32), want)
        ok(L.lb_stream_destroy(st.value))


@pytest.mark.parametrize("D,page,KV,H,seqs,window,sinks", [
    # row blocks of 8 and of 16, in one slice and in many, the window's first position anywhere in a tile
    (64, 16, 2, 14, [(150, 1), (151, 1), (165, 1)], 39, 5), (64, 64, 2, 14, [(9000, 1), (80, 1)], 4001, 7),
    (128, 128, 1, 4, [(700, 1), (90, 2), (33, 1)], 50, 21), (32, 32, 3, 3, [(200, 2), (71, 1)], 17, 0),
    (128, 64, 1, 16, [(500, 1), (333, 1)], 101, 3), (64, 16, 1, 9, [(3000, 1)], 2900, 1),
    # row blocks of 32, whole and in slices
    (64, 32, 2, 14, [(150, 60)], 39, 5), (128, 64, 1, 5, [(1000, 300)], 333, 21), (32, 128, 1, 1, [(77, 400)], 21, 3),
    (128, 16, 1, 16, [(6000, 90)], 3001, 9),
    # of two waves, alone and beside steps
    (64, 64, 8, 32, [(333, 1100)], 100, 5), (32, 32, 8, 64, [(90, 800), (701, 1), (50, 90), (300, 3)], 201, 3),
    (128, 64, 8, 32, [(61, 790), (900, 1)], 33, 9)], ids=str)
def test_slots_that_no_token_sees_may_hold_anything(rng, D, page, KV, H, seqs, window, sinks):
    """NaN codes in the slots of partly visible pages that lie before the first token's window, behind the
    sinks or behind the last token reach no row."""
    pages, q_start, past, table, T = batch_of(rng, page, seqs, 2, 0)
    pool = cached(rng, pages, page, KV, D, table, seqs)
    table = give_back(table, page, seqs, window, sinks)
    q = (rng.standard_normal((T, H * D)) * 1.5).astype(np.float32)
    most = max(n for _, n in seqs)
    ref = np.full(q.shape, FILL, np.float64)
    mags = pool.attention(q_start, past, table, most, q, H, ref, window, sinks)
    held, hidden = pool.copy(), 0
    for b, (p, n) in enumerate(seqs):
        for x in range(table.shape[1] * page):
            pg = table[b, x // page]
            if pg >= 0 and not (x < p + n and (x >= p + 1 - window or x < sinks)):
                hidden += x < p + n
                held.k[pg, :, x % page] = 0xFF if x & 1 else 0x7F
                held.v[pg, :, x % page] = 0x7F if x & 1 else 0xFF
    assert hidden
    got = attend(Device(held, q_start, past, table, most, T), q, H, H * D, window, sinks)
    check(got, ref, mags, D, H)
