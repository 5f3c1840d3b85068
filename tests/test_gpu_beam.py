"""Beam search's selection (lbd_beam_select) on the GPU against the oracle in 64 bits.

A sum s + x - lse: x - lse is exact to float64's rounding but for lse, whose sum of exponentials is added
in float32: each exponential is within 2^-22 of its value (v_exp_f32 and the product with log2 e, 1 ulp
each and half an ulp of an argument of at most 126 in base 2: 2^-24 (126 / 2 + 4) < 2^-18 for the smallest
terms, which count for as little as they are small), and V of them are added by threads of at most
V / 256 + 64 one after another, then in trees. 2^-18 + (V / 256 + 80) 2^-24 bounds lse's error; float32
rounds the sum once, by 2^-24 of it."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from oracle import beams as O
from test_gpu_kv8 import ok

pytestmark = pytest.mark.gpu
MARK = -77


def call(logits, V, score, done, W, eos, ld=None, work=None, stream=None, offset=0):
    """One step on rows of ld floats, `offset` floats into their buffer."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    n = len(score)
    flat = np.concatenate([np.full(offset, np.nan, np.float32), logits.reshape(-1)])
    dx, ds = up(flat), up(score.astype(np.float32))
    dd = None if done is None else up(np.asarray(done, np.int32))
    outs = [up(np.full(n + 1, MARK, t)) for t in (np.float32, np.int32, np.int32, np.int32)]
    b = K.LbdBeams(ds.ptr, None if dd is None else dd.ptr, *(o.ptr for o in outs), None, None, None, 0, n // W, W, V,
                   eos)
    need = L.lbd_beam_select_work_bytes(C.byref(b))
    assert need
    ws = up(np.full(need + 16, 0xFF, np.uint8)) if work is None else work
    ok(L.lbd_beam_select(dx.ptr + 4 * offset, logits.shape[1], C.byref(b), ws.ptr, need, stream))
    ok(L.lb_dev_synchronize())
    if work is None:
        assert (ws.to_array((need + 16,), np.uint8)[need:] == 0xFF).all()
    got = [o.to_array((n + 1,), t) for o, t in zip(outs, (np.float32, np.int32, np.int32, np.int32))]
    assert all(g[n] == MARK for g in got)
    return [g[:n] for g in got]  # sum, done, tok, parent


def check(logits, V, score, done, W, eos=-1, **kw):
    total, end, tok, parent = call(logits, V, score, done, W, eos, **kw)
    with np.errstate(invalid="ignore"):
        w_tok, w_parent, w_total, w_end = O.select(logits[:, :V], score, done, W, eos)
    assert np.array_equal(parent, w_parent) and np.array_equal(tok, w_tok) and np.array_equal(end, w_end)
    dead = w_parent < 0
    assert (total[dead] == -np.inf).all()
    tol = 2.0 ** -18 + (V / 256 + 80) * 2.0 ** -24 + np.abs(w_total[~dead]) * 2.0 ** -24
    assert (np.abs(total[~dead] - w_total[~dead]) <= tol).all()
    return total, end, tok, parent


def random_rows(rng, n, V, ld=None):
    x = (rng.standard_normal((n, V if ld is None else ld)) * 3).astype(np.float32)
    return x, (-20 + 5 * rng.standard_normal(n)).astype(np.float32)


@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8, 13, 16, 17, 32])
@pytest.mark.parametrize("V", [1, 2, 3, 5, 31, 64, 97, 255, 256, 257, 1000, 1023, 1024, 1025, 2047, 4099, 8192, 8193,
                               20000])
def test_sizes(rng, V, W):
    x, s = random_rows(rng, 3 * W, V)
    check(x, V, s, None, W)


@pytest.mark.parametrize("B,W,V", [(1, 4, 151936), (1, 1, 151936), (5, 8, 151936), (2, 32, 200001), (40, 3, 32003),
                                   (1, 2, 1 << 20), (300, 2, 97)])
def test_vocabularies(rng, B, W, V):
    x, s = random_rows(rng, B * W, V)
    done = rng.random(B * W) < 0.2
    check(x, V, s, done, W, eos=int(rng.integers(V)))


@pytest.mark.parametrize("offset", [0, 1, 2, 3])
@pytest.mark.parametrize("slack", [0, 1, 2, 3, 5])
def test_rows_of_any_alignment(rng, offset, slack):
    """Rows that begin anywhere in 16 bytes; NaN before the first and between them is not looked at."""
    for V in (1, 6, 97, 1030, 9001):
        x, s = random_rows(rng, 6, V, V + slack)
        x[:, V:] = np.nan
        check(x, V, s, None, 3, offset=offset)


@pytest.mark.parametrize("W", [1, 3, 8, 32])
@pytest.mark.parametrize("V", [40, 5000, 70000])
def test_ties(rng, V, W):
    """Few values, so that nearly all offers tie: by place, then the lower token. Beams with the same sum
    and the same logits in another order tie between them too."""
    one = rng.integers(0, 3, V).astype(np.float32)
    x = np.stack([one] * (2 * W))
    s = np.full(2 * W, -3.0, np.float32)
    check(x, V, s, None, W)
    x[:] = 0.0
    x[::2, ::2] = -0.0  # equal to 0
    check(x, V, s, None, W)
    x[:] = -7.5
    check(x, V, s, None, W)
    # all of a row equal but one far below, so that a threshold finds nearly everything above it
    x[:, V // 2] = -100
    check(x, V, s, None, W)


@pytest.mark.parametrize("W", [2, 8, 32])
@pytest.mark.parametrize("order", ["rising", "falling", "blocks", "spikes"])
def test_orders(rng, order, W):
    """Logits sorted, so that the best lie together in one thread's or wave's part of a row."""
    V = 30011
    x = np.sort(rng.standard_normal((2 * W, V)).astype(np.float32) * 3, 1)
    if order == "falling":
        x = x[:, ::-1].copy()
    if order == "blocks":
        x = np.concatenate([x[:, 20000:], x[:, :20000]], 1)
    if order == "spikes":  # all the best in 64 neighbours
        x = (rng.standard_normal(x.shape) * 0.1).astype(np.float32)
        x[:, 7000:7064] += 50
    check(x, V, random_rows(rng, 2 * W, 1)[1], None, W)


def test_masked_tokens(rng):
    """Logits of -inf are no offers; places that none is left for are empty."""
    V = 5000
    x, s = random_rows(rng, 12, V)
    x[rng.random(x.shape) < 0.999] = -np.inf
    x[4:8] = -np.inf
    x[5, 17] = 1.0  # the second prompt has two offers
    x[6, 4999] = -3e38
    total, _, tok, parent = check(x, V, s, None, 4)
    assert list(parent[4:8] < 0) == [False, False, True, True] and (tok[6:8] == 0).all()
    total, _, tok, parent = check(x, V, s, None, 4, eos=7)
    assert (tok[6:8] == 7).all()


def test_rows_that_offer_nothing(rng):
    """NaN or +inf among the logits, no beam (-inf, NaN), ended beams: their rows are out of the race, and
    those of ended and empty places are not read."""
    V, W = 3000, 4
    for bad in (np.nan, np.inf):
        x, s = random_rows(rng, 3 * W, V)
        x[1, 2999] = bad
        x[5, 0] = bad
        s[2], s[6] = -np.inf, np.nan
        done = np.zeros(3 * W, int)
        done[[3, 7, 8]] = 1
        x[[2, 3, 6, 7, 8]] = np.nan
        total, end, tok, parent = check(x, V, s, done, W, eos=5)
        assert not np.isin([1, 2], parent).any() and 3 in parent
    x, s = random_rows(rng, W, V)
    s[:] = -np.inf
    total, end, tok, parent = check(x, V, s, None, W)
    assert (parent == -1).all() and not end.any()


def test_only_the_first_beam(rng):
    """The step behind a prompt: one beam of sum 0 and none in the other places."""
    x, s = random_rows(rng, 10, 4000)
    s[:] = -np.inf
    s[[0, 5]] = 0
    x[[1, 2, 3, 4, 6, 7, 8, 9]] = np.nan
    _, _, _, parent = check(x, 4000, s, None, 5)
    assert list(parent) == [0] * 5 + [5] * 5


@pytest.mark.parametrize("big", [1e30, 3.4e38, 80.0, 1e-30])
def test_sizes_of_logits(rng, big):
    """Logits of any size, distinct in float32: 1e30 and above leave log-probabilities of 0 and far below."""
    x = (rng.standard_normal((8, 2000)) * big / 6).astype(np.float32)
    x = np.clip(x, -3.4e38, 3.4e38)
    _, s = random_rows(rng, 8, 1)
    if big > 1:
        check(x, 2000, s, None, 4)
    else:  # sums that differ by less than float64 shows: the order within a beam is the logits'
        total, _, tok, parent = call(x, 2000, s, None, 4, -1)
        for b in (0, 4):
            best = b + int(s[b:b + 4].argmax())
            assert (parent[b:b + 4] == best).all()
            assert list(tok[b:b + 4]) == list(np.argsort(-x[best], kind="stable")[:4])


def test_ended_beams(rng):
    V, W, eos = 2000, 4, 11
    x, s = random_rows(rng, 2 * W, V)
    x[:, eos] += 12  # the likeliest token
    done = np.array([0, 1, 0, 1, 1, 1, 1, 1])
    total, end, tok, parent = check(x, V, s, done, W, eos=eos)
    assert (tok[end == 1] == eos).all() and (end[4:] == 1).all()
    order = 4 + np.argsort(-s[4:], kind="stable")
    assert list(parent[4:]) == list(order) and np.array_equal(total[4:], s[order])


@pytest.mark.parametrize("likely", [4, 14])
def test_in_place_and_recorded(rng, likely):
    """Sums and ends in place, steps recorded on the device, replayed as a graph with other logits."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    B, W, V, eos, H = 3, 4, 5003, 9, 5
    n = B * W
    s = np.where(np.arange(n) % W == 0, 0.0, -np.inf).astype(np.float32)
    ds, dd, dx = up(s), up(np.zeros(n, np.int32)), up(np.zeros((n, V), np.float32))
    tok, parent, step = (up(np.zeros(k, np.int32)) for k in (n, n, B))
    ht, hp = (up(np.full((H + 1, n), MARK, np.int32)) for _ in range(2))
    b = K.LbdBeams(ds.ptr, dd.ptr, ds.ptr, dd.ptr, tok.ptr, parent.ptr, ht.ptr, hp.ptr, step.ptr, H, B, W, V, eos)
    need = L.lbd_beam_select_work_bytes(C.byref(b))
    ws, st, ex = up(np.zeros(need, np.uint8)), C.c_void_p(), C.c_void_p()
    ok(L.lb_stream_create(C.byref(st)))
    ok(L.lb_stream_begin_capture(st.value))
    rc = L.lbd_beam_select(dx.ptr, V, C.byref(b), ws.ptr, need, st.value)
    ok(L.lb_stream_end_capture(st.value, C.byref(ex)))
    ok(rc)
    done, hist = np.zeros(n, int), []
    for t in range(H + 2):
        x = random_rows(rng, n, V)[0]
        x[:, eos] += likely
        ok(L.lb_memcpy_h2d(dx.ptr, x.ctypes.data, x.nbytes))
        ok(L.lb_graph_launch(ex.value, st.value))
        ok(L.lb_stream_synchronize(st.value))
        w_tok, w_parent, w_s, w_done = O.select(x, s, done, W, eos)
        assert np.array_equal(tok.to_array((n,), np.int32), w_tok)
        assert np.array_equal(parent.to_array((n,), np.int32), w_parent)
        s, done = ds.to_array((n,), np.float32), dd.to_array((n,), np.int32)
        assert np.array_equal(done, w_done)
        assert (np.abs(s - w_s) <= 2.0 ** -17 + np.abs(w_s) * 2.0 ** -24).all()
        hist.append((w_tok, w_parent))
    assert done.any() or likely == 4
    assert (step.to_array((B,), np.int32) == H + 2).all()
    for got, want in ((ht, 0), (hp, 1)):
        a = got.to_array((H + 1, n), np.int32)
        assert np.array_equal(a[:H], np.stack([h[want] for h in hist[:H]])) and (a[H] == MARK).all()
    ok(L.lb_graph_destroy(ex.value))
    ok(L.lb_stream_destroy(st.value))


def test_two_streams(rng):
    """Two steps at once on two streams, with a workspace each."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    B, W, V = 4, 5, 60001
    runs = []
    for _ in range(2):
        x, s = random_rows(rng, B * W, V)
        d = [up(x), up(s)] + [up(np.zeros(B * W, np.int32)) for _ in range(4)]
        b = K.LbdBeams(d[1].ptr, None, *(o.ptr for o in d[2:]), None, None, None, 0, B, W, V, -1)
        st = C.c_void_p()
        ok(L.lb_stream_create(C.byref(st)))
        runs.append((x, s, d, b, up(np.zeros(L.lbd_beam_select_work_bytes(C.byref(b)), np.uint8)), st))
    ok(L.lb_dev_synchronize())
    for _ in range(5):
        for x, s, d, b, ws, st in runs:
            ok(L.lbd_beam_select(d[0].ptr, V, C.byref(b), ws.ptr, ws.nbytes, st.value))
    ok(L.lb_dev_synchronize())
    for x, s, d, b, ws, st in runs:
        want = O.select(x, s, None, W, -1)
        assert np.array_equal(d[4].to_array((B * W,), np.int32), want[0])
        assert np.array_equal(d[5].to_array((B * W,), np.int32), want[1])
        ok(L.lb_stream_destroy(st.value))


def test_the_same_bits_every_time(rng):
    x, s = random_rows(rng, 24, 40000)
    a = call(x, 40000, s, None, 8, 3)
    for _ in range(3):
        assert all(np.array_equal(u, v) for u, v in zip(a, call(x, 40000, s, None, 8, 3)))


@pytest.mark.parametrize("B,W,V", [(70000, 1, 33), (20000, 2, 50), (1500, 32, 40)])
def test_many_rows(rng, B, W, V):
    """More rows than a grid's second dimension holds."""
    x, s = random_rows(rng, B * W, V)
    x = np.round(x * 4096).astype(np.float32) / 4096
    total, end, tok, parent = call(x, V, s, None, W, -1)
    for b in np.concatenate([[0, 1, B - 1], rng.integers(0, B, 40)]):
        rows = slice(b * W, b * W + W)
        w_tok, w_parent, w_total, _ = O.select(x[rows], s[rows], None, W, -1)
        assert np.array_equal(tok[rows], w_tok) and np.array_equal(parent[rows], w_parent + b * W)
        assert np.abs(total[rows] - w_total).max() < 1e-4


def test_logits_past_32_bits():
    """70 rows of 2^24 logits, 4.7 GB: all 0 but for a few, so that all others tie."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    W, B, V = 2, 35, 1 << 24
    n = W * B
    x = K.DeviceBuffer(4 * n * V)
    ok(L.lb_memset_d(x.ptr, 0, x.nbytes))
    ok(L.lb_dev_synchronize())
    spikes = {(0, 5): 3.0, (0, V - 1): 2.0, (69, V - 1): 4.0, (69, V // 2 + 1): 9.0, (68, 0): 1.0, (40, 1 << 23): -1.0}
    for (row, v), y in spikes.items():
        a = np.array([y], np.float32)
        ok(L.lb_memcpy_h2d(x.ptr + 4 * (row * V + v), a.ctypes.data, 4))
    s = np.where(np.arange(n) % W == 0, 0.0, -1.0).astype(np.float32)
    d = [up(s)] + [up(np.zeros(n, np.float32))] + [up(np.zeros(n, np.int32)) for _ in range(3)]
    b = K.LbdBeams(d[0].ptr, None, d[1].ptr, d[2].ptr, d[3].ptr, d[4].ptr, None, None, None, 0, B, W, V, -1)
    need = L.lbd_beam_select_work_bytes(C.byref(b))
    ws = up(np.zeros(need, np.uint8))
    ok(L.lbd_beam_select(x.ptr, V, C.byref(b), ws.ptr, need, None))
    ok(L.lb_dev_synchronize())
    tok, parent, total = d[3].to_array((n,), np.int32), d[4].to_array((n,), np.int32), d[1].to_array((n,), np.float32)
    want = [[(2 * g, 0), (2 * g, 1)] for g in range(B)]  # the first beam's lowest tokens
    want[0] = [(0, 5), (0, V - 1)]
    want[34] = [(69, V // 2 + 1), (69, V - 1)]  # 9 and 4 below log 2^24 and a sum of -1, against 1
    assert list(zip(parent, tok)) == [o for g in want for o in g]
    lse = np.log(2.0 ** 24)
    assert abs(total[2] + lse) < 2.0 ** -10  # 2^24 terms of 1: 65536 a thread and trees, exact
    assert abs(total[0] - (3 - lse)) < 2.0 ** -10
