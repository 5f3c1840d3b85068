"""What the paged 8-bit cache's calls leave alone (GPU): every buffer that they may write lies between
guards, and the bytes that no token and no row of the batch owns are compared with those before."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from oracle import kv_cache as O
from test_gpu_kv8 import FILL, Device, angles, batch_of, ok

pytestmark = pytest.mark.gpu
GUARD, MARK = 4096, 0xA5


class Guarded:
    """A device array between GUARD bytes of MARK on either side."""

    def __init__(self, a):
        self.shape, self.dtype, self.n = a.shape, a.dtype, a.nbytes
        edge = np.full(GUARD, MARK, np.uint8)
        self.buf = K.DeviceBuffer.from_array(np.concatenate([edge, np.ascontiguousarray(a).view(np.uint8).reshape(-1),
                                                             edge]))
        self.ptr = self.buf.ptr + GUARD

    def read(self):
        b = self.buf.to_array((self.n + 2 * GUARD,), np.uint8)
        assert (b[:GUARD] == MARK).all() and (b[-GUARD:] == MARK).all()
        return b[GUARD:-GUARD].copy().view(self.dtype).reshape(self.shape)


def run(pool, q_start, past, table, max_new, T, qkv, H, cos, sin):
    """Append of qkv and the attention of its rotated rows, everything that they write guarded: the pool,
    q_out and out as they come back."""
    L, up = K.lib(), K.DeviceBuffer.from_array
    names, width = ("k", "v", "ke", "ve"), H * pool.d
    held = {n: Guarded(getattr(pool, n)) for n in names}
    arrays = [up(np.asarray(a, np.int32)) for a in (q_start, past, table)]
    p = K.LbdKv8Pool(*(held[n].ptr for n in names), pool.pages, pool.page, pool.kv, pool.d)
    b = K.LbdKv8Batch(*(a.ptr for a in arrays), len(past), np.shape(table)[1], max_new, T)
    dq, dc, ds = up(qkv), up(cos), up(sin)
    q, out = Guarded(np.full((T, width), FILL)), Guarded(np.full((T, width), FILL))
    need = L.lbd_kv8_attention_work_bytes(C.byref(p), C.byref(b), H)
    assert need
    ws = Guarded(np.zeros(need, np.uint8))
    ok(L.lbd_kv8_append(C.byref(p), C.byref(b), dq.ptr, qkv.shape[1], None, H, dc.ptr, ds.ptr, len(cos), q.ptr, width,
                        None))
    ok(L.lbd_kv8_attention(C.byref(p), C.byref(b), q.ptr, width, H, out.ptr, width, ws.ptr, need, None))
    ok(L.lb_dev_synchronize())
    ws.read()
    return {n: held[n].read() for n in names}, q.read(), out.read()


@pytest.mark.parametrize("D,H", [(64, 2), (128, 1), (32, 20)])
def test_batches_that_make_no_sense_stay_inside(rng, D, H):
    """q_start that runs backwards or outside the rows, positions near 2^31: pages that no table entry
    names and rows that no sequence claims keep their bytes."""
    page, KV, T = 16, 1, 9
    pool = O.Pool(rng, 4, page, KV, D)
    q_start = np.array([-9, 3, 2, 2 ** 31 - 1, 2], np.int64).astype(np.int32)  # rows 0 .. 2, none, 2 .. 8, none
    past = np.array([2 ** 31 - 1, 5, -2 ** 31, 30], np.int64).astype(np.int32)
    table = np.array([[0, 1]] * 4, np.int32)
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    cos, sin = angles(rng, 8, D)
    held, q, out = run(pool, q_start, past, table, T, T, qkv, H, cos, sin)
    for n, a in held.items():
        assert np.array_equal(a[2:], getattr(pool, n)[2:]), n
        assert np.array_equal(a[:2], getattr(pool, n)[:2]), n  # nor is there a position below the table's 32 to write
    # sequence 0's rows lie past every position, sequence 2 has no new tokens (past < 0)
    assert (q[3:] == FILL).all() and (out[3:] == FILL).all() and (q[:3] != FILL).any()


def test_ordinary_batches_touch_only_their_own(rng):
    """Idle places, rows before and behind the sequences, pages of nobody, slots behind the last token."""
    D, page, KV, H = 64, 16, 2, 6
    seqs = [(5, 1), (0, 40), (40, 0), (33, 17), (-1, 2)]
    pages, q_start, past, table, T = batch_of(rng, page, seqs, pad=5, extra=1)
    q_start, T = q_start + 3, T + 3
    pool = O.Pool(rng, pages, page, KV, D)
    pool.ke[:], pool.ve[:] = 121, 122
    for n in ("k", "v"):
        setattr(pool, n, O.e4m3_round(rng.uniform(-300, 300, pool.k.shape)))
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    cos, sin = angles(rng, 80, D)
    held, q, out = run(pool, q_start, past, table, 40, T, qkv, H, cos, sin)
    own, rows = np.zeros((pages, page), bool), np.zeros(T, bool)
    touched = np.zeros(pages, bool)
    for b, (p, n) in enumerate(seqs):
        if p < 0:
            continue
        rows[q_start[b]:q_start[b + 1]] = True
        for x in range(p, p + n):
            own[table[b, x // page], x % page] = touched[table[b, x // page]] = True
    assert (q[~rows] == FILL).all() and (out[~rows] == FILL).all()
    assert (q[rows] != FILL).all() and (out[rows] != FILL).all()
    for n, e in (("k", "ke"), ("v", "ve")):
        assert np.array_equal(held[e][~touched], getattr(pool, e)[~touched])
        # earlier tokens of a touched page: as they were where its exponent stayed
        same = ~own[:, None, :] & (held[e] == getattr(pool, e))[:, :, None]
        same |= ~touched[:, None, None]
        assert np.array_equal(held[n][same], getattr(pool, n)[same])
    # slots behind the last token of a page, whatever became of its exponent
    for b, (p, n) in enumerate(seqs):
        if p >= 0 and n and (p + n) % page:
            pg, lo = table[b, (p + n) // page], (p + n) % page
            assert np.array_equal(held["k"][pg, :, lo:], pool.k[pg, :, lo:])
            assert np.array_equal(held["v"][pg, :, lo:], pool.v[pg, :, lo:])


@pytest.mark.parametrize("which,bad", [("K", np.nan), ("K", np.inf), ("V", np.nan), ("V", -np.inf)])
def test_a_nan_block_stays_until_its_page_is_begun_again(rng, which, bad):
    D, page, KV, H = 64, 16, 2, 2
    pages, q_start, past, table, T = batch_of(rng, page, [(4, 40)], extra=1)
    pool = O.Pool(rng, pages, page, KV, D)
    pool.ke[:], pool.ve[:] = 120, 120
    qkv = rng.standard_normal((T, (H + 2 * KV) * D)).astype(np.float32)
    qkv[30, (H + (KV if which == "V" else 0)) * D + 5] = bad  # head 0 of position 34: page table[0, 2]
    cos, sin = angles(rng, 60, D)
    dev, hit = Device(pool, q_start, past, table, 40, T), table[0, 2]
    dev.append(qkv, None, H, cos, sin, np.full((T, H * D), FILL))
    held = dev.held()
    exps = lambda p: p.ve if which == "V" else p.ke  # noqa: E731
    assert exps(held)[hit, 0] == 255 and (exps(held) == 255).sum() == 1 and (held.ke == 255).sum() + \
        (held.ve == 255).sum() == 1
    one = np.ones((1, (H + 2 * KV) * D), np.float32)

    def later(pool, at):
        d = Device(pool, [0, 1], [at], table, 1, 1)
        d.append(one, None, H, cos, sin, np.full((1, H * D), FILL))
        return d.held()

    held = later(held, 44)  # a finite token behind it
    assert exps(held)[hit, 0] == 255 and exps(held)[hit, 1] != 255
    codes = held.v if which == "V" else held.k
    assert not codes[hit, 0, 12].any()  # its codes are zeros
    held = later(held, 32)  # slot 0 begins the page
    assert exps(held)[hit, 0] != 255
