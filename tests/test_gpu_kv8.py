"""The paged 8-bit cache on the GPU (lbd_kv8_append, lbd_kv8_attention) against the oracle.

Append: the rotation is defined in float32 with every product rounded, and a code is the
nearest E4M3 value, so rotated q, codes and exponents are compared bit for bit; against the
float64 rotation a held value may be off by half a step of E4M3 (2^-4 of it, or half the
smallest step of its block) and the rotation's own rounding, 3 x 2^-24 of |x1| + |x2|.

Attention, with A the row's largest sum |q k| / sqrt(D) and V the weighted mean of |v|:
a score is a float32 sum of D exact products (D + 16 roundings of 2^-24, the last few the
scales and the exponential's argument) of q in two float16 terms (2^-20 of A covers both
terms' rounding and the flushed tail of small elements), so weights are off by twice
((D + 16) 2^-24 + 2^-20) A; a weight's own exponential and two terms add 2^-19, and the
weighted sum at most keys / 32 + 64 float32 additions one after another (32 keys a matrix
instruction, waves and slices merged)."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from oracle import kv_cache as O

pytestmark = pytest.mark.gpu
FILL = np.float32(-7.25)


def ok(rc):
    assert rc >= 0, K.lib().lb_last_error()


class Device:
    """A pool and a batch on the device, and the calls on them."""

    def __init__(self, pool, q_start, past, table, max_new, T):
        up = K.DeviceBuffer.from_array
        self.host = pool
        self.buf = {n: up(getattr(pool, n)) for n in ("k", "v", "ke", "ve")}
        self.arrays = [up(np.asarray(a, np.int32)) for a in (q_start, past, table)]
        self.pool = K.LbdKv8Pool(*(self.buf[n].ptr for n in ("k", "v", "ke", "ve")), pool.pages, pool.page, pool.kv,
                                 pool.d)
        self.batch = K.LbdKv8Batch(*(a.ptr for a in self.arrays), len(past), np.shape(table)[1], max_new, T)

    def append(self, qkv, bias, H, cos, sin, q_out=None, in_place=False, stream=None):
        up = K.DeviceBuffer.from_array
        dq, db = up(qkv), None if bias is None else up(bias)
        do = dq if in_place else up(q_out)
        dc, ds = up(cos), up(sin)
        ok(K.lib().lbd_kv8_append(C.byref(self.pool), C.byref(self.batch), dq.ptr, qkv.shape[1],
                                  None if db is None else db.ptr, H, dc.ptr, ds.ptr, len(cos), do.ptr,
                                  (qkv if in_place else q_out).shape[1], stream))
        ok(K.lib().lb_dev_synchronize())
        return do.to_array((qkv if in_place else q_out).shape, np.float32)

    def held(self):
        p = self.host.copy()
        for n, b in self.buf.items():
            setattr(p, n, b.to_array(getattr(p, n).shape, np.uint8))
        return p

    def attention(self, q, H, out_width, stream=None):
        L, up = K.lib(), K.DeviceBuffer.from_array
        dq = up(q)
        do = up(np.full((len(q), out_width), FILL))
        need = L.lbd_kv8_attention_work_bytes(C.byref(self.pool), C.byref(self.batch), H)
        ws = up(np.full(need + 16, 0xFF, np.uint8))  # needs no clearing
        ok(L.lbd_kv8_attention(C.byref(self.pool), C.byref(self.batch), dq.ptr, q.shape[1], H, do.ptr, out_width,
                               ws.ptr if need else None, need, stream))
        ok(L.lb_dev_synchronize())
        assert (ws.to_array((need + 16,), np.uint8)[need:] == 0xFF).all()
        return do.to_array((len(q), out_width), np.float32)


def tables(rng, pages, page, seqs, extra=0):
    """Page tables of sequences (past, new): every page of its own, in no order."""
    need = [max(0, -(-(max(p, 0) + n) // page)) for p, n in seqs]
    order = rng.permutation(pages)
    t = np.full((len(seqs), max(need) + extra), -1, np.int32)
    for i, m in enumerate(need):
        t[i, :m] = order[sum(need[:i]):sum(need[:i + 1])]
    return t


def batch_of(rng, page, seqs, pad=0, extra=0):
    pages = sum(-(-(max(p, 0) + n) // page) for p, n in seqs) + 3
    q_start = np.concatenate([[0], np.cumsum([n for _, n in seqs])])
    return pages, q_start, np.array([p for p, _ in seqs]), tables(rng, pages, page, seqs, extra), int(q_start[-1]) + pad


def angles(rng, n, d):
    a = rng.uniform(0, 6.28, (n, d // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def same_pool(got, want):
    for n in ("ke", "ve", "k", "v"):
        a, b = getattr(got, n), getattr(want, n)
        if len(n) == 1:  # a NaN is a NaN, whatever its sign
            a, b = (np.where(x & 0x7F == 0x7F, 0x7F, x) for x in (a, b))
        differ = np.argwhere(a != b)
        assert not len(differ), (n, differ[:5])


SEQS = {
    "one": [(0, 1)], "step": [(37, 1)], "page end": [(15, 1), (16, 1), (31, 2)], "prompt": [(0, 83)],
    "chunk": [(21, 70)], "mixed": [(5, 1), (0, 40), (127, 3), (64, 1), (0, 1), (33, 17)],
    "idle": [(3, 0), (9, 2), (-1, 3), (40, 0), (8, 1), (7, 0)],
}


@pytest.mark.parametrize("seqs", SEQS, ids=str)
@pytest.mark.parametrize("D,page,KV,H", [(64, 16, 2, 14), (128, 32, 1, 3), (32, 64, 3, 3), (128, 128, 2, 2),
                                         (64, 64, 1, 16), (32, 16, 1, 1)])
def test_append(rng, D, page, KV, H, seqs):
    seqs = SEQS[seqs]
    pages, q_start, past, table, T = batch_of(rng, page, seqs, pad=3)
    bias = None if D == 32 else rng.standard_normal((H + 2 * KV) * D).astype(np.float32)
    pool = O.Pool(rng, pages, page, KV, D)
    pool.ke[pool.ke > 140] = 118  # earlier tokens' blocks: ordinary exponents
    pool.ve[pool.ve > 140] = 119
    qkv = rng.standard_normal((T, (H + 2 * KV) * D + 8)).astype(np.float32)
    qkv *= (2.0 ** rng.integers(-9, 10, (T, 1))).astype(np.float32)
    cos, sin = angles(rng, 400, D)
    q_out = np.full((T, H * D + 4), FILL)
    dev = Device(pool, q_start, past, table, max(n for _, n in seqs), T)
    got = dev.append(qkv, bias, H, cos, sin, q_out)
    want = pool.copy()
    want.append(q_start, past, table, max(n for _, n in seqs), qkv, bias, H, cos, sin, q_out)
    assert np.array_equal(got, q_out)
    same_pool(dev.held(), want)
    # once more: the same tokens in the same slots change nothing, q in place
    got = dev.append(qkv, bias, H, cos, sin, in_place=True)
    same_pool(dev.held(), want)
    rows = np.concatenate([np.arange(a, a + n) for a, (p, n) in zip(q_start, seqs) if p >= 0]).astype(int)
    ref = qkv.copy()
    ref[rows, :H * D] = q_out[rows, :H * D]
    assert np.array_equal(got, ref)


def test_append_against_float64(rng):
    D, page, KV, H, n = 128, 32, 2, 2, 50
    pages, q_start, past, table, T = batch_of(rng, page, [(0, n)])
    pool = O.Pool(rng, pages, page, KV, D)
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    cos, sin = angles(rng, n, D)
    dev = Device(pool, q_start, past, table, n, T)
    q = dev.append(qkv, None, H, cos, sin, np.full((T, H * D), FILL))
    held = dev.held()
    x = qkv.astype(np.float64).reshape(n, -1, D)
    y = O.rotate(x, cos.astype(np.float64), sin.astype(np.float64))
    slack = 3 * 2.0 ** -24 * (np.abs(x) + np.abs(np.roll(x, D // 2, 2)))
    assert (np.abs(q.reshape(n, H, D) - y[:, :H]) <= slack[:, :H]).all()
    for codes, exps, ref, s in ((held.k, held.ke, y[:, H:H + KV], slack[:, H:H + KV]),
                                (held.v, held.ve, x[:, H + KV:], 0)):
        val = np.moveaxis(held.values(codes[table[0]], exps[table[0]]), 1, 2).reshape(-1, KV, D)[:n]
        unit = np.repeat(2.0 ** (exps[table[0]].astype(np.float64) - 127), page, 0)[:n, :, None]
        assert (np.abs(val - ref) <= np.maximum(2.0 ** -4 * (np.abs(ref) + s), 2.0 ** -10 * unit) + s).all()


def test_append_grows_token_by_token(rng):
    """Each token larger than the ones before: the block's codes shift every time."""
    D, page, KV, H = 64, 16, 1, 1
    table, pool = np.array([[1, 2]], np.int32), O.Pool(rng, 3, page, 1, D)
    cos, sin = angles(rng, 64, D)
    want = pool.copy()
    dev = Device(pool, [0, 1], [0], table, 1, 1)
    for t in range(20):
        qkv = (rng.standard_normal((1, 3 * D)) * 3.0 ** (t - 8)).astype(np.float32)
        dev.arrays[1] = K.DeviceBuffer.from_array(np.array([t], np.int32))
        dev.batch.past = dev.arrays[1].ptr
        q = np.full((1, D), FILL)
        got = dev.append(qkv, None, H, cos, sin, q)
        want.append([0, 1], [t], table, 1, qkv, None, H, cos, sin, q)
        assert np.array_equal(got, q)
        same_pool(dev.held(), want)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_of_what_is_not_finite(rng, bad):
    """The token's own blocks become NaN and stay so; the other heads and blocks do not."""
    D, page, KV, H = 64, 16, 2, 2
    pages, q_start, past, table, T = batch_of(rng, page, [(4, 40)])
    pool = O.Pool(rng, pages, page, KV, D)
    pool.ke[:], pool.ve[:] = 120, 120
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    qkv[20, (H + 1) * D + 3] = bad        # key head 1
    qkv[30, (H + KV) * D + 60] = bad      # value head 0
    cos, sin = angles(rng, 60, D)
    dev, want, q = Device(pool, q_start, past, table, 40, T), pool.copy(), np.full((T, H * D), FILL)
    got = dev.append(qkv, None, H, cos, sin, q)
    want.append(q_start, past, table, 40, qkv, None, H, cos, sin, q)
    assert np.array_equal(got, q)
    held = dev.held()
    same_pool(held, want)
    assert (held.ke == 255).sum() == 1 and (held.ve == 255).sum() == 1
    dev2 = Device(held, [0, 1], [40], table, 1, 1)  # a later finite token of the NaN value block's page
    q1 = np.full((1, H * D), FILL)
    dev2.append(np.ones((1, (H + 2 * KV) * D), np.float32), None, H, cos, sin, q1)
    assert dev2.held().ve[table[0, 2], 0] == 255 if held.ve[table[0, 2], 0] == 255 else True


def test_append_extremes(rng):
    """Blocks of zeros, of subnormals, of the largest floats, and one after the other."""
    D, page, KV, H = 32, 16, 1, 1
    sizes = [0.0, 1e-45, 1e-38, 3.4028234e38, 0.0, 1e-30, 448.0, 448.00003, 0.21875, 1.0]
    table = np.arange(len(sizes), dtype=np.int32)[None]
    pool = O.Pool(rng, len(sizes), page, KV, D)
    T = page * len(sizes)
    qkv = np.zeros((T, 3 * D), np.float32)
    for i, s in enumerate(sizes):
        qkv[i * page:(i + 1) * page, 2 * D:] = np.float32(s) * rng.choice([-1, 0, 1], (page, D)).astype(np.float32)
        qkv[i * page + 3, 2 * D + 5] = s
    cos, sin = np.ones((4, D // 2), np.float32), np.zeros((4, D // 2), np.float32)  # positions past the table
    q = np.full((T, D), FILL)
    dev, want = Device(pool, [0, T], [0], table, T, T), pool.copy()
    dev.append(qkv, None, H, cos, sin, q)
    want.append([0, T], [0], table, T, qkv, None, H, cos, sin, q)
    same_pool(dev.held(), want)


@pytest.mark.parametrize("page", [16, 128])
def test_append_drops_what_has_no_page(rng, page):
    """Entries outside the pool, positions past the table, and tokens past max_new."""
    D, KV, H = 64, 2, 4
    pool = O.Pool(rng, 6, page, KV, D)
    pool.ke[:], pool.ve[:] = 121, 122
    table = np.array([[0, -1, 1], [6, 2, 2 ** 31 - 1], [3, -2 ** 31, 4]], np.int32)
    seqs = [(page - 3, page + 9), (page - 2, 5), (3 * page - 2, 6)]
    q_start = np.concatenate([[0], np.cumsum([n for _, n in seqs])])
    past, T, max_new = np.array([p for p, _ in seqs]), int(q_start[-1]) + 2, page + 7
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    cos, sin = angles(rng, 3 * page, D)
    q = np.full((T, H * D), FILL)
    dev, want = Device(pool, q_start, past, table, max_new, T), pool.copy()
    got = dev.append(qkv, None, H, cos, sin, q)
    want.append(q_start, past, table, max_new, qkv, None, H, cos, sin, q)
    assert np.array_equal(got, q)
    same_pool(dev.held(), want)


def test_batches_that_make_no_sense(rng):
    """q_start that runs backwards or outside the rows, positions near 2^31: nothing outside the
    buffers is touched (the guards around them stay)."""
    D, page, KV, H, T = 64, 16, 1, 2, 5
    pool = O.Pool(rng, 4, page, KV, D)
    q_start = np.array([-9, 3, 2, 2 ** 31 - 1, 2], np.int64).astype(np.int32)
    past = np.array([2 ** 31 - 1, 5, -2 ** 31, 30], np.int64).astype(np.int32)
    table = np.array([[0, 1]] * 4, np.int32)
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    cos, sin = angles(rng, 8, D)
    dev = Device(pool, q_start, past, table, T, T)
    dev.append(qkv, None, H, cos, sin, np.full((T, H * D), FILL))
    got = dev.attention(qkv[:, :H * D].copy(), H, H * D)
    assert got.shape == (T, H * D)


@pytest.mark.parametrize("rows,G", [(1, 8), (2000, 1)])
def test_rows_of_several_sequences_at_once(rng, rows, G):
    """q_start that goes back and forth, so that far more rows take part than there are: the long
    sequence's slices, which lie about the workspace's end, stay inside it (its guard stays)."""
    D, page, B, past = 64, 128, 2001 if rows > 1 else 3000, 20000
    pool = O.Pool(rng, 2, page, 1, D)
    q_start = np.arange(B + 1) % 2 * rows
    pasts = np.zeros(B, np.int64)
    pasts[96 if rows > 1 else 1000:][:8] = past
    table = rng.integers(0, 2, (B, -(-(past + rows) // page))).astype(np.int32)
    q = rng.standard_normal((rows, G * D)).astype(np.float32)
    got = Device(pool, q_start, pasts, table, rows, rows).attention(q, G, G * D)
    assert got.shape == q.shape


# ---------------------------------------------------------------- attention

def cached(rng, pages, page, KV, D, table, seqs, spread=2):
    """A pool as append leaves it: finite codes in held slots, any byte elsewhere."""
    pool = O.Pool(rng, pages, page, KV, D)
    pool.ke[:] = rng.integers(119, 119 + spread, pool.ke.shape)
    pool.ve[:] = rng.integers(118, 118 + 2 * spread, pool.ve.shape)
    x = np.clip(rng.standard_normal(pool.k.shape) * 130, -448, 448)
    y = np.clip(rng.standard_normal(pool.v.shape) * 130, -448, 448)
    kc, vc = O.e4m3_round(x), O.e4m3_round(y)
    for b, (p, n) in enumerate(seqs):
        for pos0 in range(0, max(p, 0) + n, page):
            pg, m = table[b, pos0 // page], min(page, max(p, 0) + n - pos0)
            if 0 <= pg < pages:
                pool.k[pg, :, :m], pool.v[pg, :, :m] = kc[pg, :, :m], vc[pg, :, :m]
    return pool


def check(got, ref, mags, D, H):
    a, v, keys = np.moveaxis(np.repeat(mags, D, 1), 2, 0)  # [T, H D] each
    tol = (2 * ((D + 16) * 2.0 ** -24 + 2.0 ** -20) * a + 2.0 ** -19 + (keys / 32 + 64) * 2.0 ** -24) * v
    g, r = got[:, :H * D], ref[:, :H * D]
    nan = np.isnan(r)
    assert np.array_equal(np.isnan(g), nan)
    err = np.where(nan, 0, np.abs(np.where(nan, 0, g) - np.where(nan, 0, r)))
    over = np.argwhere(~nan & (err > tol))
    assert not len(over), (over[:4], np.nanmax(np.where(nan, 0, err / np.maximum(tol, 1e-300))))
    assert np.array_equal(got[:, H * D:], ref[:, H * D:])


def run_attention(rng, D, page, KV, H, seqs, pad=2, extra=1, pool=None, table=None, q=None, max_new=None):
    pages, q_start, past, t, T = batch_of(rng, page, seqs, pad, extra)
    table = t if table is None else table
    pool = cached(rng, pages, page, KV, D, table, seqs) if pool is None else pool
    q = (rng.standard_normal((T, H * D + 4)) * 1.5).astype(np.float32) if q is None else q
    max_new = max(n for _, n in seqs) if max_new is None else max_new
    got = Device(pool, q_start, past, table, max_new, T).attention(q, H, H * D + 8)
    ref = np.full(got.shape, FILL, np.float64)
    mags = pool.attention(q_start, past, table, max_new, q, H, ref)
    check(got, ref, mags, D, H)
    return got


HEADS = [(64, 16, 2, 14), (128, 32, 1, 4), (32, 64, 3, 3), (128, 128, 1, 16), (64, 64, 1, 9), (32, 16, 1, 1),
         (128, 16, 1, 33), (64, 32, 2, 16)]


@pytest.mark.parametrize("seqs", SEQS, ids=str)
@pytest.mark.parametrize("D,page,KV,H", HEADS)
def test_attention(rng, D, page, KV, H, seqs):
    run_attention(rng, D, page, KV, H, SEQS[seqs])


@pytest.mark.parametrize("D,page,KV,H", [(64, 16, 2, 14), (128, 64, 1, 4), (32, 128, 1, 2), (128, 32, 1, 16)])
@pytest.mark.parametrize("past", [62, 63, 64, 127, 255, 256, 257, 1000, 2047, 4100])
def test_attention_step_lengths(rng, D, page, KV, H, past):
    """One long sequence cut into slices, beside a short one."""
    run_attention(rng, D, page, KV, H, [(past, 1), (3, 1)])


@pytest.mark.parametrize("D,page,KV,H", [(64, 16, 2, 14), (128, 64, 1, 4), (32, 128, 1, 1), (128, 32, 1, 5)])
@pytest.mark.parametrize("past,new", [(0, 15), (0, 16), (0, 17), (0, 129), (500, 33), (1, 64), (63, 65), (900, 100)])
def test_attention_prompts(rng, D, page, KV, H, past, new):
    run_attention(rng, D, page, KV, H, [(past, new)])


def test_attention_many_sequences(rng):
    """More sequences than lanes, most of them short, some idle."""
    seqs = [(int(rng.integers(0, 40)), int(rng.integers(0, 3))) for _ in range(150)]
    run_attention(rng, 64, 16, 1, 4, seqs)
    run_attention(rng, 32, 16, 2, 4, [(p, min(n, 1)) for p, n in seqs])


@pytest.mark.parametrize("D,KV,H,seqs", [
    # few rows: 157 slices of a row, merged a workgroup a row (more slices than lanes)
    (32, 1, 2, [(40000, 1)]), (128, 1, 5, [(40000, 1)]),
    # and 40 sequences of several slices, merged a row to D / 4 lanes
    (32, 8, 16, [(300 + 27 * i, 1) for i in range(40)]), (64, 8, 8, [(300 + 27 * i, 1) for i in range(40)]),
    (128, 8, 8, [(1100 - 20 * i, 1) for i in range(40)]),
    # many rows: 68 row blocks in 9 and more slices; row blocks enough for workgroups of two waves,
    # with a sequence long enough to be cut beside them
    (64, 1, 24, [(4000, 90)]), (32, 1, 24, [(4000, 90)]),
    (128, 8, 56, [(0, 500), (3000, 20)]), (64, 8, 64, [(0, 700), (2500, 20), (5, 90)]),
    (32, 8, 64, [(0, 950), (2500, 80)])], ids=str)
def test_attention_slices(rng, D, KV, H, seqs):
    run_attention(rng, D, 32, KV, H, seqs)


def test_attention_more_row_blocks_than_slots(rng):
    """Many row blocks of short prompts, and a sequence longer than twice the mean whose own row blocks
    outnumber the slices that a call may add."""
    run_attention(rng, 32, 64, 32, 32, [(0, 320)] * 20 + [(0, 3200)], pad=0)


def test_attention_prompts_and_steps(rng):
    run_attention(rng, 64, 32, 2, 8, [(700, 1), (0, 90), (1300, 1), (33, 2), (0, 1), (250, 40), (64, 0)])


@pytest.mark.parametrize("seqs", [[(70, 1)], [(20, 60)]], ids=str)
def test_attention_without_pages(rng, seqs):
    """Positions whose page is gone are left out; a row with none left gets zeros."""
    D, page, KV, H = 64, 16, 2, 4
    table = np.array([[4, -1, 5, 99, 2, 1]], np.int32)
    pool = cached(rng, 6, page, KV, D, table, seqs)
    run_attention(rng, D, page, KV, H, seqs, pool=pool, table=table)
    gone = np.array([[-1, -5, 6, 99, -1, 2 ** 31 - 1]], np.int32)
    got = run_attention(rng, D, page, KV, H, seqs, pool=pool, table=gone)
    assert not got[:seqs[0][1], :H * D].any()


@pytest.mark.parametrize("seqs", [[(70, 1)], [(20, 60)]], ids=str)
def test_attention_over_nan_blocks(rng, seqs):
    """A NaN block reaches the rows that see one of its positions, and no others."""
    D, page, KV, H = 64, 16, 2, 4
    table = np.array([[3, 0, 5, 4, 2]], np.int32)
    for which in ("ke", "ve"):
        pool = cached(rng, 6, page, KV, D, table, seqs)
        getattr(pool, which)[2, 1] = 255  # positions 64 .. 79 of head 1
        got = run_attention(rng, D, page, KV, H, seqs, pool=pool, table=table)
        nan = np.isnan(got[:seqs[0][1], :H * D]).reshape(-1, H, D)
        assert nan.any() and not nan[:, :2].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("n", [1, 60])
def test_attention_of_a_query_that_is_not_finite(rng, bad, n):
    D, H = 64, 4
    q = (rng.standard_normal((n + 2, H * D + 4)) * 1.5).astype(np.float32)
    q[n // 2, D + 5] = bad
    clean = np.where(np.isfinite(q), q, 0).astype(np.float32)
    pages, q_start, past, table, T = batch_of(rng, 16, [(20, n)], 2, 1)
    pool = cached(rng, pages, 16, 2, D, table, [(20, n)])
    dev = Device(pool, q_start, past, table, n, T)
    got, ref = dev.attention(q, H, H * D), dev.attention(clean, H, H * D)
    hit = np.zeros(got.shape, bool)
    hit[n // 2, D:2 * D] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], ref[~hit])


@pytest.mark.parametrize("n", [1, 50])
def test_attention_of_very_different_blocks(rng, n):
    """Value blocks of sizes 2^-30 .. 2^30 apart and keys that pick one of them: each row as exact
    as its own blocks allow."""
    D, page, KV, H = 64, 16, 1, 2
    seqs = [(150, n)]
    pages, q_start, past, table, T = batch_of(rng, page, seqs, 0, 0)
    pool = cached(rng, pages, page, KV, D, table, seqs)
    pool.ve[table[0], 0] = 119 + np.resize([-30, 0, 30, -10, 10], table.shape[1])
    pool.k[:, :, :, 0] = O.e4m3_round(np.array(0.0))
    pool.k[table[0, 0], :, :, 0] = O.e4m3_round(np.array(448.0))  # the small block's keys
    q = (rng.standard_normal((T, H * D)) * 0.1).astype(np.float32)
    q[:, 0] = 400.0
    got = run_attention(rng, D, page, KV, H, seqs, pad=0, pool=pool, table=table, q=q)
    assert np.abs(got[:n, :D]).max() < 2.0 ** -20  # head 0 picks them


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e4, 1e30])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_query_sizes(rng, scale, n):
    """Rows of any size: the two float16 terms are taken relative to the row. Scores of 1e34 leave
    one key its weight, scores of 1e-26 give the mean."""
    D, H = 128, 4
    q = (rng.standard_normal((n, H * D)) * scale).astype(np.float32)
    pages, q_start, past, table, T = batch_of(rng, 32, [(77, n)])
    pool = cached(rng, pages, 32, 2, D, table, [(77, n)])
    got = Device(pool, q_start, past, table, n, T).attention(q, H, H * D)
    ref = np.full(got.shape, 0.0)
    mags = pool.attention(q_start, past, table, n, q, H, ref)
    if scale < 1e5:
        mags[..., 0] = np.minimum(mags[..., 0], 1e5)
        check(got, ref, mags, D, H)
    else:
        assert np.abs(got - ref).max() <= 2.0 ** -19 * np.abs(ref).max()


@pytest.mark.parametrize("n", [1, 20, 100])
def test_attention_of_zeros(rng, n):
    """Rows of zeros over blocks of the least exponent: every key counts alike, those behind a row not."""
    D, page, KV, H, seqs = 64, 16, 1, 3, [(37, n), (0, n)]
    pages, q_start, past, table, T = batch_of(rng, page, seqs)
    pool = cached(rng, pages, page, KV, D, table, seqs)
    pool.ke[:] = 0
    q = np.zeros((T, H * D + 4), np.float32)
    q[::3] = 1e-30
    run_attention(rng, D, page, KV, H, seqs, pad=0, extra=0, pool=pool, table=table, q=q)


def test_rows_before_the_first_sequence_and_positions_past_the_table(rng):
    """q_start may begin behind row 0; a token past the table's last position is not written and
    attends over all of it."""
    D, page, KV, H = 64, 16, 2, 6
    q_start, past, T = np.array([3, 8, 8, 30]), np.array([44, 3, 40]), 33
    table = np.array([[5, 1, 7], [2, -1, -1], [0, 3, 6]], np.int32)
    pool = cached(rng, 8, page, KV, D, table, [(44, 4), (3, 0), (40, 8)])
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    cos, sin = angles(rng, 50, D)
    dev, want, q = Device(pool, q_start, past, table, 22, T), pool.copy(), np.full((T, H * D), FILL)
    got = dev.append(qkv, None, H, cos, sin, q)
    want.append(q_start, past, table, 22, qkv, None, H, cos, sin, q)
    assert np.array_equal(got, q)
    same_pool(dev.held(), want)
    out, ref = dev.attention(got, H, H * D), np.full((T, H * D), FILL, np.float64)
    mags = want.attention(q_start, past, table, 22, got, H, ref)
    check(out, ref, mags, D, H)


def test_pool_past_four_gib(rng):
    """Pages whose codes lie past 2^32 bytes: the same as in a small pool."""
    D, page, KV, H, far = 128, 128, 8, 16, 33000  # 131072 code bytes a page
    L, up = K.lib(), K.DeviceBuffer.from_array
    seqs = [(0, 140), (0, 3)]
    small = np.array([[1, 3], [0, -1]], np.int32)
    big = np.where(small >= 0, far - 4 + small, -1).astype(np.int32)
    q_start, past, T = np.array([0, 140, 143]), np.array([0, 0]), 143
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    cos, sin = angles(rng, 140, D)
    pool = O.Pool(rng, 4, page, KV, D)
    near = Device(pool, q_start, past, small, 140, T)
    q = near.append(qkv, None, H, cos, sin, np.full((T, H * D), FILL))
    want = near.attention(q, H, H * D)
    buf = [K.DeviceBuffer(far * KV * n) for n in (page * D, page * D, 1, 1)]
    assert buf[0].nbytes > 1 << 32
    dev = Device(pool, q_start, past, big, 140, T)
    dev.pool = K.LbdKv8Pool(*(b.ptr for b in buf), far, page, KV, D)
    assert np.array_equal(dev.append(qkv, None, H, cos, sin, np.full((T, H * D), FILL)), q)
    assert np.array_equal(dev.attention(q, H, H * D), want)
    # one more token each, few rows
    for d in (near, dev):
        d.arrays[:2] = [up(np.array(a, np.int32)) for a in ([0, 1, 2], [140, 3])]
        d.batch = K.LbdKv8Batch(*(a.ptr for a in d.arrays), 2, 2, 1, 2)
    step = qkv[:2].copy()
    q1, q2 = (d.append(step, None, H, cos, sin, np.full((2, H * D), FILL)) for d in (near, dev))
    assert np.array_equal(q1, q2) and np.array_equal(near.attention(q1, H, H * D), dev.attention(q1, H, H * D))
    ok(L.lb_dev_synchronize())


def test_one_workspace_for_calls_of_all_sizes(rng):
    """Calls in stream order share a workspace that is the largest of theirs."""
    D, page, KV, H = 64, 32, 2, 8
    L, up = K.lib(), K.DeviceBuffer.from_array
    runs = []
    for seqs in ([(3000, 1), (5, 1)], [(700, 90), (0, 40)], [(1200, 1)] * 9, [(4000, 3)]):
        pages, q_start, past, table, T = batch_of(rng, page, seqs)
        pool = cached(rng, pages, page, KV, D, table, seqs)
        q = rng.standard_normal((T, H * D)).astype(np.float32)
        dev = Device(pool, q_start, past, table, max(n for _, n in seqs), T)
        runs.append((dev, up(q), up(np.full((T, H * D), FILL)), dev.attention(q, H, H * D), T))
    need = max(L.lbd_kv8_attention_work_bytes(C.byref(d.pool), C.byref(d.batch), H) for d, *_ in runs)
    ws = K.DeviceBuffer(need)
    for _ in range(2):
        for dev, dq, do, _, T in runs:
            ok(L.lbd_kv8_attention(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, H * D, H, do.ptr, H * D, ws.ptr, need,
                                   None))
    ok(L.lb_dev_synchronize())
    for _, _, do, want, T in runs:
        assert np.array_equal(do.to_array((T, H * D), np.float32), want)


def test_runs_of_append_and_attention(rng):
    """A prompt in two chunks and single tokens for three sequences in one pool, as a serving
    program calls them, against the oracle's own cache."""
    D, page, KV, H = 64, 16, 2, 6
    total = [90, 37, 150]
    table = tables(rng, 24, page, [(0, n) for n in total], 1)
    pool = O.Pool(rng, 24, page, KV, D)
    want, length = pool.copy(), np.zeros(3, np.int64)
    cos, sin = angles(rng, 160, D)
    dev = Device(pool, [0] * 4, [0] * 3, table, 1, 1)
    for news in ((60, 0, 17), (25, 30, 1), (1, 1, 120), (1, 0, 1), (1, 1, 1), (1, 1, 1)):
        q_start, T = np.concatenate([[0], np.cumsum(news)]), sum(news) + 1
        qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
        dev.arrays[:2] = [K.DeviceBuffer.from_array(np.asarray(a, np.int32)) for a in (q_start, length)]
        dev.batch = K.LbdKv8Batch(*(a.ptr for a in dev.arrays), 3, table.shape[1], max(news), T)
        q = np.full((T, H * D), FILL)
        got = dev.append(qkv, None, H, cos, sin, q)
        want.append(q_start, length, table, max(news), qkv, None, H, cos, sin, q)
        same_pool(dev.held(), want)
        out, ref = dev.attention(got, H, H * D), np.full((T, H * D), FILL, np.float64)
        mags = want.attention(q_start, length, table, max(news), got, H, ref)
        check(out, ref, mags, D, H)
        length += news


def test_replayed_graph_on_a_stream_of_its_own(rng):
    """One recorded step of both calls, replayed with other lengths, equals the eager calls."""
    D, page, KV, H, B = 64, 16, 2, 6, 3
    L, up = K.lib(), K.DeviceBuffer.from_array
    start = np.array([30, 100, 7])
    table = tables(rng, 30, page, [(int(p), 12) for p in start], 0)
    pool = cached(rng, 30, page, KV, D, table, [(int(p), 0) for p in start])
    cos, sin = angles(rng, 160, D)
    rows = [rng.standard_normal((B, (H + 2 * KV) * D)).astype(np.float32) for _ in range(5)]
    q_start = np.arange(B + 1)

    s, ex = C.c_void_p(), C.c_void_p()
    ok(L.lb_stream_create(C.byref(s)))
    dev = Device(pool, q_start, start, table, 1, B)
    dq, dc, ds, do = up(rows[0]), up(cos), up(sin), up(np.full((B, H * D), FILL))
    dqo = up(np.zeros((B, H * D), np.float32))
    need = L.lbd_kv8_attention_work_bytes(C.byref(dev.pool), C.byref(dev.batch), H)
    ws = K.DeviceBuffer(max(need, 16))

    def step(stream):
        ok(L.lbd_kv8_append(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, rows[0].shape[1], None, H, dc.ptr, ds.ptr,
                            len(cos), dqo.ptr, H * D, stream))
        ok(L.lbd_kv8_attention(C.byref(dev.pool), C.byref(dev.batch), dqo.ptr, H * D, H, do.ptr, H * D, ws.ptr, need,
                               stream))

    ok(L.lb_stream_begin_capture(s.value))
    step(s.value)
    ok(L.lb_stream_end_capture(s.value, C.byref(ex)))
    eager = Device(pool, q_start, start, table, 1, B)
    for t, x in enumerate(rows):
        past = (start + t).astype(np.int32)
        ok(L.lb_memcpy_h2d(dq.ptr, x.ctypes.data, x.nbytes))
        ok(L.lb_memcpy_h2d(dev.arrays[1].ptr, past.ctypes.data, past.nbytes))
        ok(L.lb_graph_launch(ex.value, s.value))
        ok(L.lb_stream_synchronize(s.value))
        eager.arrays[1] = up(past)
        eager.batch.past = eager.arrays[1].ptr
        q = eager.append(x, None, H, cos, sin, np.full((B, H * D), FILL))
        out = eager.attention(q, H, H * D)
        assert np.array_equal(do.to_array((B, H * D), np.float32), out)
        same_pool(dev.held(), eager.held())
    ok(L.lb_graph_destroy(ex.value))
    ok(L.lb_stream_destroy(s.value))


def test_same_bits_twice(rng):
    D, page, KV, H, seqs = 64, 16, 2, 14, [(3000, 1), (5, 1), (1200, 1)]
    pages, q_start, past, table, T = batch_of(rng, page, seqs)
    pool = cached(rng, pages, page, KV, D, table, seqs)
    q = rng.standard_normal((T, H * D)).astype(np.float32)
    dev = Device(pool, q_start, past, table, 1, T)
    assert np.array_equal(dev.attention(q, H, H * D), dev.attention(q, H, H * D))


def test_two_streams_at_once(rng):
    """Calls on two streams, each with a workspace of its own, over one pool."""
    D, page, KV, H = 64, 32, 2, 8
    L, up = K.lib(), K.DeviceBuffer.from_array
    runs = []
    for seqs in ([(3000, 1)] * 6, [(700, 90), (0, 200), (2000, 1)]):
        pages, q_start, past, table, T = batch_of(rng, page, seqs)
        pool = cached(rng, pages, page, KV, D, table, seqs)
        q = rng.standard_normal((T, H * D)).astype(np.float32)
        dev = Device(pool, q_start, past, table, max(n for _, n in seqs), T)
        need = L.lbd_kv8_attention_work_bytes(C.byref(dev.pool), C.byref(dev.batch), H)
        s = C.c_void_p()
        ok(L.lb_stream_create(C.byref(s)))
        runs.append((dev, up(q), up(np.full((T, H * D), FILL)), K.DeviceBuffer(need), need, s,
                     dev.attention(q, H, H * D)))
    for _ in range(20):
        for dev, dq, do, ws, need, s, _ in runs:
            ok(L.lbd_kv8_attention(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, H * D, H, do.ptr, H * D, ws.ptr, need,
                                   s.value))
    ok(L.lb_dev_synchronize())
    for _, _, do, _, _, s, want in runs:
        assert np.array_equal(do.to_array(want.shape, np.float32), want)
        ok(L.lb_stream_destroy(s.value))
