"""The paged 8-bit cache on the GPU where its numbers lie far apart: weights far below a row's
largest, query elements far below a row's largest, blocks of the least and the greatest exponents."""
import numpy as np
import pytest

from oracle import kv_cache as O
from test_gpu_kv8 import FILL, Device, batch_of, same_pool

pytestmark = pytest.mark.gpu

# steps of 8, 16 and 32 query rows a row block, prompts, and both in one call; whole and in slices
CALLS = {"step 4 on 1": (128, 1, 4, [(99, 1)]), "step 12 on 1": (64, 1, 12, [(99, 1)]),
         "step 24 on 1": (32, 1, 24, [(99, 1)]), "prompt": (128, 1, 4, [(60, 40)]), "long step": (64, 1, 4, [(5000, 1)]),
         "long steps": (128, 1, 12, [(3000, 1), (4000, 1)]), "chunk": (64, 2, 4, [(2500, 70)]),
         "mixed": (64, 1, 6, [(70, 30), (1500, 1), (4, 1)])}


def sinks(rng, D, KV, seqs, at, nats, page=32):
    """Keys that see two channels: channel 0 is 0 but at positions `at`, whose V is 0, where it lifts a
    key `nats` above the ones whose channel 1 is 0. Scores are sums of two products."""
    pages, q_start, past, table, T = batch_of(rng, page, seqs, 2, 1)
    pool = O.Pool(rng, pages, page, KV, D)
    pool.ke[:], pool.ve[:] = 119, 120
    pool.k[:] = 0
    pool.k[..., 1] = O.e4m3_round(rng.uniform(-300, 300, pool.k.shape[:3]))
    pool.v[:] = O.e4m3_round(np.clip(rng.standard_normal(pool.v.shape) * 130 + 60, -448, 448))
    for b, (p, n) in enumerate(seqs):
        for x in at:
            if x < p + n:
                pool.k[table[b, x // page], :, x % page, :2] = O.e4m3_round(np.array([448.0, 0.0]))
                pool.v[table[b, x // page], :, x % page] = 0
    return pool, q_start, past, table, T


@pytest.mark.parametrize("at", [(0,), (3, 40, 70, 97)], ids=["one", "one a wave"])
@pytest.mark.parametrize("nats", [4, 8, 11, 15, 17, 22, 30, 45])
@pytest.mark.parametrize("call", CALLS)
def test_keys_far_below_the_largest(rng, call, nats, at):
    """A key that takes nearly all of the weight and holds a V of zeros: what a row gets is the sum of the
    others, each weight e^-nats and less.

    Tolerance, relative to the weighted mean of |v|: a score is off by 9 x 2^-24 of itself at most (q's two
    terms 2^-22, five roundings of 2^-24: the sum, the scale and the exponential's argument), once in the
    key's weight and once in the denominator's; a weight's exponential and terms 2^-19, and keys / 32 + 64
    additions one after another."""
    D, KV, H, seqs = CALLS[call]
    pool, q_start, past, table, T = sinks(rng, D, KV, seqs, at, nats)
    q = np.zeros((T, H * D), np.float32)
    q[:, 0::D] = nats * np.sqrt(D) / (448 * 2.0 ** (119 - 127))
    q[:, 1::D] = rng.uniform(-1, 1, (T, H)) * np.sqrt(D)
    most = max(n for _, n in seqs)
    got = Device(pool, q_start, past, table, most, T).attention(q, H, H * D)
    ref = np.full(got.shape, FILL, np.float64)
    a, v, keys = np.moveaxis(np.repeat(pool.attention(q_start, past, table, most, q, H, ref), D, 1), 2, 0)
    tol = (18 * 2.0 ** -24 * a + 2.0 ** -19 + (keys / 32 + 64) * 2.0 ** -24) * v
    err = np.abs(got - ref)
    assert (err <= tol).all(), (np.nanmax(err / np.maximum(v, 1e-300)), np.nanmax(tol / np.maximum(v, 1e-300)))


@pytest.mark.parametrize("bits", [4, 10, 16, 20, 26])
@pytest.mark.parametrize("call", CALLS)
def test_query_elements_far_below_the_largest(rng, call, bits):
    """A query row with one element 2^bits above the others, where every key is 0: the scores are the
    others'.

    Tolerance: as for random rows (tests/test_gpu_kv8.py), with q's terms off by 2^-20 of the sum of
    |q k| and by 2^-38 of the row's largest element a key's element."""
    D, KV, H, seqs = CALLS[call]
    pages, q_start, past, table, T = batch_of(rng, 32, seqs, 2, 1)
    pool = O.Pool(rng, pages, 32, KV, D)
    pool.ke[:], pool.ve[:] = 120, 120
    pool.k[:] = O.e4m3_round(np.clip(rng.standard_normal(pool.k.shape) * 130, -448, 448))
    pool.v[:] = O.e4m3_round(np.clip(rng.standard_normal(pool.v.shape) * 130, -448, 448))
    pool.k[..., 5] = 0
    q = (rng.standard_normal((T, H * D)) * 2).astype(np.float32)
    q[:, 5::D] = 3 * 2.0 ** bits
    most = max(n for _, n in seqs)
    got = Device(pool, q_start, past, table, most, T).attention(q, H, H * D)
    ref = np.full(got.shape, FILL, np.float64)
    a, v, keys = np.moveaxis(np.repeat(pool.attention(q_start, past, table, most, q, H, ref), D, 1), 2, 0)
    floor = 2.0 ** -38 * 3 * 2.0 ** bits * D * 448 * 2.0 ** -7 / np.sqrt(D)
    tol = (2 * (((D + 16) * 2.0 ** -24 + 2.0 ** -20) * a + floor) + 2.0 ** -19 + (keys / 32 + 64) * 2.0 ** -24) * v
    err = np.abs(got - ref)
    assert (err <= tol).all(), (np.nanmax(err / np.maximum(v, 1e-300)), np.nanmax(tol / np.maximum(v, 1e-300)))


@pytest.mark.parametrize("old", [100, 200, 247, 253, 254])
@pytest.mark.parametrize("D,n", [(64, 1), (128, 3)])
def test_append_to_blocks_of_great_exponents(rng, D, n, old):
    """Pages written by other means may hold any exponent: a later token's codes are in its unit."""
    page, KV, H = 16, 2, 2
    pages, q_start, past, table, T = batch_of(rng, page, [(5, n)])
    pool = O.Pool(rng, pages, page, KV, D)
    pool.k[:], pool.v[:] = O.e4m3_round(rng.uniform(-400, 400, (2,) + pool.k.shape))
    pool.ke[:], pool.ve[:] = old, old
    # values up to the unit times 256, or 2^126
    qkv = (rng.uniform(-1, 1, (T, (H + 2 * KV) * D)) * 2.0 ** min(old - 119, 126)).astype(np.float32)
    cos, sin = np.ones((40, D // 2), np.float32), np.zeros((40, D // 2), np.float32)
    q = np.full((T, H * D), FILL)
    dev, want = Device(pool, q_start, past, table, n, T), pool.copy()
    got = dev.append(qkv, None, H, cos, sin, q)
    want.append(q_start, past, table, n, qkv, None, H, cos, sin, q)
    assert np.array_equal(got, q)
    held = dev.held()
    assert (held.ve[table[0, 0]] == old).all()
    same_pool(held, want)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("low,high", [(0, 0), (0, 60), (1, 90), (154, 254)])
def test_value_blocks_of_extreme_exponents(rng, call, low, high):
    """V's exponents from the least, 2^-127, to the greatest: blocks within 2^100 of the sequence's
    largest count in full, alone and beside each other. Keys are zeros: each counts alike. Outputs below 2^-126 are
    float32 subnormals, off by 2^-149."""
    D, KV, H, seqs = CALLS[call]
    pages, q_start, past, table, T = batch_of(rng, 32, seqs, 2, 1)
    pool = O.Pool(rng, pages, 32, KV, D)
    pool.k[:], pool.ke[:] = 0, 120
    pool.v[:] = O.e4m3_round(np.clip(rng.standard_normal(pool.v.shape) * 130, -448, 448) / (64 if high == 254 else 1))
    pool.ve[:] = low
    for b in range(len(seqs)):  # every third block of a sequence
        pool.ve[table[b, 2::3]] = high
    q = rng.standard_normal((T, H * D)).astype(np.float32)
    most = max(n for _, n in seqs)
    got = Device(pool, q_start, past, table, most, T).attention(q, H, H * D)
    ref = np.full(got.shape, FILL, np.float64)
    _, v, keys = np.moveaxis(np.repeat(pool.attention(q_start, past, table, most, q, H, ref), D, 1), 2, 0)
    tol = (2.0 ** -19 + (keys / 32 + 64) * 2.0 ** -24) * v + 2.0 ** -149
    err = np.abs(got - ref)
    assert (err <= tol).all(), (np.nanmax(err / np.maximum(v, 1e-300)), np.nanmax(tol / np.maximum(v, 1e-300)))


@pytest.mark.parametrize("nats", [0, 12, 30, 55, 75])
@pytest.mark.parametrize("call", CALLS)
def test_pages_of_zero_values_that_take_the_weight(rng, call, nats):
    """As append leaves a page whose values are zeros: exponent 0, 120 below the others'. Every fourth page is
    one, its keys `nats` above the rest.

    Tolerance as in test_keys_far_below_the_largest."""
    D, KV, H, seqs = CALLS[call]
    pool, q_start, past, table, T = sinks(rng, D, KV, seqs, (), 0)
    for b in range(len(seqs)):
        pg = table[b, 0::4]
        pool.k[pg[pg >= 0], :, :, 0] = 0x7E
        pool.v[pg[pg >= 0]], pool.ve[pg[pg >= 0]] = 0, 0
    q = np.zeros((T, H * D), np.float32)
    q[:, 0::D] = nats * np.sqrt(D) / (448 * 2.0 ** (119 - 127))
    q[:, 1::D] = rng.uniform(-1, 1, (T, H)) * np.sqrt(D)
    most = max(n for _, n in seqs)
    got = Device(pool, q_start, past, table, most, T).attention(q, H, H * D)
    ref = np.full(got.shape, FILL, np.float64)
    a, v, keys = np.moveaxis(np.repeat(pool.attention(q_start, past, table, most, q, H, ref), D, 1), 2, 0)
    tol = (18 * 2.0 ** -24 * a + 2.0 ** -19 + (keys / 32 + 64) * 2.0 ** -24) * v
    err = np.abs(got - ref)
    assert (err <= tol).all(), (np.nanmax(err / np.maximum(v, 1e-300)), np.nanmax(tol / np.maximum(v, 1e-300)))
