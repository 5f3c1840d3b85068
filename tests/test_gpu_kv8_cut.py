"""How the paged 8-bit cache's attention is cut (GPU): the first launch's slices are the ones that the merge
adds."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from test_gpu_kv8 import FILL, Device, batch_of, cached, ok

pytestmark = pytest.mark.gpu
HEAD = 64  # words before the sums


@pytest.mark.parametrize("D,KV,H,seqs,R", [
    (64, 1, 4, [(3000, 1)], 8), (128, 2, 8, [(5000, 1)], 8), (32, 1, 16, [(9000, 1)], 16), (64, 2, 4, [(2500, 70)], 32),
    (128, 1, 2, [(6000, 16)], 32)], ids=str)
def test_the_cut_stands_in_the_workspace(rng, D, KV, H, seqs, R):
    """One sequence's workspace: 256 bytes that begin with a slice's keys, then for every slice of every row
    block and KV head the rows' sums, then their scalars (reference, unit, its mid, denominator). The
    slices that the first word tells, added in 64 bits, are the output."""
    (past, n), G = seqs[0], H // KV
    pages, q_start, pasts, table, T = batch_of(rng, 32, seqs, 0)
    pool = cached(rng, pages, 32, KV, D, table, seqs)
    q = rng.standard_normal((T, H * D)).astype(np.float32)
    dev, L, up = Device(pool, q_start, pasts, table, n, T), K.lib(), K.DeviceBuffer.from_array
    need = L.lbd_kv8_attention_work_bytes(C.byref(dev.pool), C.byref(dev.batch), H)
    dq, do, ws = up(q), up(np.full(q.shape, FILL)), up(np.full(need, 0xFF, np.uint8))
    ok(L.lbd_kv8_attention(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, H * D, H, do.ptr, H * D, ws.ptr, need, None))
    ok(L.lb_dev_synchronize())
    words = ws.to_array((need // 4,), np.float32)
    units = (need // 4 - HEAD) // (KV * R * (D + 4))
    assert HEAD + units * KV * R * (D + 4) == need // 4
    keys, cut = past + n, int(words[:1].view(np.int32)[0])
    blocks, slices = -(-n * G // R), -(-keys // cut)
    assert cut % 128 == 0 and 1 < slices and blocks * slices <= units
    sums = words[HEAD:HEAD + units * KV * R * D].reshape(units, KV, R, D).astype(np.float64)
    m, um, mid, den = np.moveaxis(words[HEAD + units * KV * R * D:].reshape(units, KV, R, 4).astype(np.float64), 3, 0)
    got = do.to_array(q.shape, np.float32).reshape(n, KV, G, D)
    for r in range(n * G):
        at = slice(r // R * slices, r // R * slices + slices)
        for h in range(KV):
            M, u = m[at, h, r % R], (um - mid)[at, h, r % R]
            top, unit = M.max(), u.max()
            num = (sums[at, h, r % R] * np.exp2(M - top)[:, None]).sum(0)
            want = num * np.exp2(top - unit) / (den[at, h, r % R] * np.exp2(u - unit)).sum()
            have = got[r // G, h, r % G]
            # float32: a factor, a division, and one addition a slice of sums that may be larger than theirs
            size = (np.abs(sums[at, h, r % R]) * np.exp2(M - top)[:, None]).sum(0) * np.abs(want / num)
            assert (np.abs(have - want) <= (slices + 16) * 2.0 ** -24 * size).all()


def test_graphs_that_share_a_workspace(rng):
    """Three recorded calls that are cut differently, replayed in turn on one stream with one workspace (on the
    16 bytes that it has to be aligned to), eager calls on another between them."""
    D, page, KV, H = 64, 32, 2, 8
    L, up = K.lib(), K.DeviceBuffer.from_array
    s = C.c_void_p()
    ok(L.lb_stream_create(C.byref(s)))
    runs = []
    for seqs in ([(3000, 1), (5, 1)], [(700, 90), (0, 40), (2000, 1)], [(9000, 20)]):
        pages, q_start, past, table, T = batch_of(rng, page, seqs)
        pool = cached(rng, pages, page, KV, D, table, seqs)
        q = rng.standard_normal((T, H * D)).astype(np.float32)
        dev = Device(pool, q_start, past, table, max(n for _, n in seqs), T)
        runs.append((dev, q, up(q), up(np.full(q.shape, FILL)), dev.attention(q, H, H * D)))
    need = max(L.lbd_kv8_attention_work_bytes(C.byref(d.pool), C.byref(d.batch), H) for d, *_ in runs)
    ws, graphs = K.DeviceBuffer(need + 16), []
    for dev, q, dq, do, _ in runs:
        ex = C.c_void_p()
        ok(L.lb_stream_begin_capture(s.value))
        ok(L.lbd_kv8_attention(C.byref(dev.pool), C.byref(dev.batch), dq.ptr, H * D, H, do.ptr, H * D, ws.ptr + 16,
                               need, s.value))
        ok(L.lb_stream_end_capture(s.value, C.byref(ex)))
        graphs.append(ex)
    fill = np.full(max(q.size for _, q, *_ in runs), FILL)
    for turn in range(4):
        for _, q, _, do, _ in runs:
            ok(L.lb_memcpy_h2d(do.ptr, fill.ctypes.data, q.nbytes))
        for i in (0, 1, 2, 1, 0, 2):
            ok(L.lb_graph_launch(graphs[i].value, s.value))
        for dev, q, _, _, want in runs:
            assert np.array_equal(dev.attention(q, H, H * D), want)
        ok(L.lb_stream_synchronize(s.value))
        for _, q, _, do, want in runs:
            assert np.array_equal(do.to_array(q.shape, np.float32), want)
    for ex in graphs:
        ok(L.lb_graph_destroy(ex.value))
    ok(L.lb_stream_destroy(s.value))
