"""The paged 8-bit cache on the CPU: what its entry points refuse before any device work, and
the oracle that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from lowbit_amd import kernels as K
from oracle import kv_cache as O

P = 0x1000  # a pointer that is never followed


def structs(**over):
    pool = dict(k=P, v=P, ke=P, ve=P, pages=4, page=16, KV=2, D=64)
    batch = dict(q_start=P, past=P, table=P, B=2, max_pages=3, max_new=5, T=7)
    pool.update({n: v for n, v in over.items() if n in pool})
    batch.update({n: v for n, v in over.items() if n in batch})
    return K.LbdKv8Pool(**pool), K.LbdKv8Batch(**batch)


def append(H=4, stride=512, max_pos=64, qkv=P, cos=P, sin=P, q_out=2 * P, q_stride=256, bias=None, **over):
    pool, batch = structs(**over)
    return K.lib().lbd_kv8_append(C.byref(pool), C.byref(batch), qkv, stride, bias, H, cos, sin, max_pos, q_out,
                                  q_stride, None)


def attention(H=4, q=P, q_stride=256, out=2 * P, out_stride=256, work=P, work_bytes=1 << 40, **over):
    pool, batch = structs(**over)
    return K.lib().lbd_kv8_attention(C.byref(pool), C.byref(batch), q, q_stride, H, out, out_stride, work, work_bytes,
                                     None)


SHAPES = [dict(page=p) for p in (0, 8, 24, 256, -16)] + [dict(D=d) for d in (0, 48, 256)] + [
    dict(KV=0), dict(KV=3), dict(H=0), dict(H=-4), dict(pages=0), dict(B=0), dict(max_pages=0), dict(max_new=0),
    dict(T=0), dict(T=-1), dict(max_pages=1 << 27), dict(B=(1 << 24) + 1), dict(T=(1 << 24) + 1), dict(H=1 << 17)]


@pytest.mark.parametrize("over", SHAPES, ids=str)
def test_bad_shapes(over):
    assert append(**over) == -1 and attention(**over) == -1
    pool, batch = structs(**over)
    assert K.lib().lbd_kv8_attention_work_bytes(C.byref(pool), C.byref(batch), over.get("H", 4)) == 0


@pytest.mark.parametrize("over,rc", [
    (dict(stride=508), -1), (dict(stride=514), -1), (dict(q_stride=252), -1), (dict(q_stride=258), -1),
    (dict(max_pos=0), -1), (dict(qkv=None), -6), (dict(cos=None), -6), (dict(sin=None), -6), (dict(q_out=None), -6),
    (dict(qkv=P + 4), -6), (dict(cos=P + 8), -6), (dict(sin=P + 4), -6), (dict(q_out=P + 12), -6),
    (dict(bias=P + 4), -6), (dict(q_out=P, q_stride=256), -6)] + [
    (dict([(n, None)]), -6) for n in ("k", "v", "ke", "ve", "q_start", "past", "table")] + [
    (dict([(n, P + 8)]), -6) for n in ("k", "v")], ids=str)
def test_append_refuses(over, rc):
    assert append(**over) == rc


@pytest.mark.parametrize("over,rc", [
    (dict(q_stride=252), -1), (dict(q_stride=258), -1), (dict(out_stride=252), -1), (dict(out_stride=270), -1),
    (dict(q=None), -6), (dict(out=None), -6), (dict(q=P + 4), -6), (dict(out=P + 4), -6)] + [
    (dict([(n, None)]), -6) for n in ("k", "v", "ke", "ve", "q_start", "past", "table")], ids=str)
def test_attention_refuses(over, rc):
    assert attention(**over) == rc


def test_too_many_rows_for_a_launch():
    over = dict(B=1 << 24, T=1 << 24, H=16, KV=16)
    assert attention(**over, q_stride=1024, out_stride=1024) == -1
    pool, batch = structs(**over)
    assert K.lib().lbd_kv8_attention_work_bytes(C.byref(pool), C.byref(batch), 16) == 0
    assert append(**over, stride=3200, q_stride=1024) == -1


def test_null_structures():
    pool, batch = structs()
    L = K.lib()
    assert L.lbd_kv8_append(None, C.byref(batch), P, 512, None, 4, P, P, 64, P, 512, None) == -6
    assert L.lbd_kv8_attention(C.byref(pool), None, P, 256, 4, P, 256, P, 1 << 40, None) == -6
    assert L.lbd_kv8_attention_work_bytes(None, C.byref(batch), 4) == 0


# ---------------------------------------------------------------- the oracle

def test_e4m3_values_and_rounding():
    assert O.E4M3[0x7E] == 448 and O.E4M3[0x08] == 2.0 ** -6 and O.E4M3[0x01] == 2.0 ** -9 and O.E4M3[0xB8] == -1
    codes = np.array([c for c in range(256) if c & 0x7F != 0x7F], np.uint8)
    assert np.array_equal(O.e4m3_round(O.E4M3[codes]), codes)
    mid = (O.E4M3[:126] + O.E4M3[1:127]) / 2  # ties go to the even code
    assert np.array_equal(O.e4m3_round(mid) % 2, np.zeros(126))
    x = np.random.default_rng(0).uniform(-448, 448, 4000) * 2.0 ** np.random.default_rng(1).integers(-20, 1, 4000)
    best = np.abs(x[:, None] - O.E4M3[codes][None]).min(1)
    assert np.array_equal(np.abs(x - O.E4M3[O.e4m3_round(x)]), best)


@pytest.mark.parametrize("big,e", [(448.0, 127), (np.nextafter(np.float32(448), np.float32(500)), 128), (0.0, 0),
                                   (1.75, 119), (1.0, 119), (3.4e38, 247), (1e-45, 0), (np.inf, 255), (np.nan, 255)])
def test_block_exponent(big, e):
    assert O.e8m0_for(np.array([0.0, big], np.float32)) == e


def test_appending_token_by_token_is_appending_at_once():
    """A block's exponent and its codes above the subnormals do not depend on the calls."""
    rng = np.random.default_rng(3)
    page, d, n = 16, 32, 23
    cos, sin = (f(rng.uniform(0, 6, (40, d // 2))).astype(np.float32) for f in (np.cos, np.sin))
    qkv = (rng.standard_normal((n, 3 * d)) * 2.0 ** rng.integers(-3, 4, (n, 1))).astype(np.float32)
    table = np.array([[2, 0]], np.int32)
    one = O.Pool(rng, 3, page, 1, d)
    many = one.copy()
    out = np.zeros((n, d), np.float32)
    one.append([0, n], [0], table, n, qkv, None, 1, cos, sin, out)
    for t in range(n):
        many.append([0, 1], [t], table, 1, qkv[t:t + 1], None, 1, cos, sin, out[:1])
    for a, b, ea, eb in ((one.k, many.k, one.ke, many.ke), (one.v, many.v, one.ve, many.ve)):
        assert np.array_equal(ea[[2, 0]], eb[[2, 0]])
        x, y = (p[[2, 0]].reshape(-1, d)[:n] for p in (a, b))
        normal = np.abs(O.E4M3[x]) >= 2.0 ** -6
        assert np.array_equal(x[normal], y[normal])
        assert np.abs(O.E4M3[x] - O.E4M3[y]).max() <= 2.0 ** -9


def test_attention_without_rounding():
    """Two keys with known scores: weights 1/3 and 2/3; a row whose pages are gone: zeros."""
    p = O.Pool(np.random.default_rng(0), 1, 16, 1, 32)
    p.k[:], p.v[:], p.ke[:], p.ve[:] = 0, 0, 127, 127
    p.v[0, 0, 0], p.v[0, 0, 1] = 0x38, 0x40  # 1 and 2
    p.k[0, 0, 1, 0] = 0x38
    q = np.zeros((2, 32))
    q[:, 0] = np.log(2) * np.sqrt(32)
    out = np.full((2, 32), 7.0)
    p.attention([0, 1, 2], [1, 0], np.array([[0], [-1]], np.int32), 1, q, 1, out)
    assert np.allclose(out[0], 5 / 3) and not out[1].any()
