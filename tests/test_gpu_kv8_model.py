"""The decoder on the paged 8-bit cache (GPU): that the model hands the cache's two calls what they
need, in prompts, steps, replayed graphs and batches of sequences.

What a layer did is checked from its own buffers: with one layer, the rows that the q/k/v projection
made are still in the model's buffer (k and v untouched, q rotated in place), so the oracle's append
of those rows gives the cache's bytes exactly, and the oracle's attention over them the layer's
attention to the kernel's tolerance (tests/test_gpu_kv8.py)."""
import numpy as np
import pytest

from lowbit_amd import model as M
from oracle import kv_cache as O
from test_gpu_kv8 import check

pytestmark = pytest.mark.gpu


def small(**over):
    cfg = M.tiny_config(num_layers=1, max_position=400, **over)
    return cfg, M.random_weights(cfg, seed=3)


def pool_of(cache, layer=0):
    """The cache's pages as the oracle holds them."""
    p = object.__new__(O.Pool)
    s, b = cache.layers[layer]
    p.pages, p.page, p.kv, p.d = s.pages, s.page, s.KV, s.D
    p.k, p.v = (x.to_array((p.pages, p.page * p.kv * p.d), np.uint8).reshape(p.pages, p.kv, p.page, p.d)
                for x in b[:2])
    p.ke, p.ve = (x.to_array((p.pages, p.kv), np.uint8) for x in b[2:])
    return p


def check_layer(model, cache, before, news, past, bias):
    """The last pass's append and attention, from the model's buffers."""
    cfg, T = model.cfg, int(sum(news))
    H, KV, D = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
    rows = model.qkv.to_array((T, (H + 2 * KV) * D), np.float32)
    q_start, table, most = np.concatenate([[0], np.cumsum(news)]), cache._table, int(max(news))
    cos, sin = M.rope_tables(D, cfg.max_position, cfg.rope_theta)
    want, got = before, pool_of(cache)
    want.append(q_start, past, table, most, rows, bias, H, cos, sin, np.zeros((T, H * D), np.float32))
    held = np.zeros(want.pages, bool)
    for s, n in enumerate(news):
        held[table[s, :-(-(past[s] + n) // cache.page)]] = True
    for name in ("k", "v", "ke", "ve"):
        assert np.array_equal(getattr(got, name)[held], getattr(want, name)[held]), name
    ref = np.zeros((T, H * D))
    mags = want.attention(q_start, past, table, most, rows[:, :H * D], H, ref)
    check(model.att.to_array((T, H * D), np.float32), ref, mags, D, H)


@pytest.mark.parametrize("backend", M.BACKENDS)
@pytest.mark.parametrize("qkv_bias", [True, False])
def test_prompts_and_steps(backend, qkv_bias):
    cfg, W = small(qkv_bias=qkv_bias)
    model = M.Model(cfg, W, backend)
    cache = model.new_cache(150, kv="e4m3", page=16)
    a = "model.layers.0.self_attn."
    bias = np.concatenate([W[a + f"{n}_proj.bias"] for n in "qkv"]) if qkv_bias else None
    rng, past = np.random.default_rng(0), 0
    for n in (37, 1, 1, 60, 1):
        before = pool_of(cache)
        model.forward(rng.integers(0, 97, n), cache)
        # a one-token step adds the bias in the projection's epilogue
        check_layer(model, cache, before, [n], [past], None if n == 1 and model.fused else bias)
        past += n
    assert cache.length == past == 100
    with pytest.raises(ValueError):
        model.forward(rng.integers(0, 97, 51), cache)


@pytest.mark.parametrize("backend", M.BACKENDS)
def test_graph_is_the_steps(backend):
    """generate's replayed graph, its eager steps and forward's tokens one by one."""
    cfg = M.tiny_config(max_position=400)
    model = M.Model(cfg, M.random_weights(cfg, seed=1), backend)
    prompt = list(np.random.default_rng(1).integers(0, 97, 50))
    a = model.generate(prompt, 40, model.new_cache(120, kv="e4m3", page=16))
    b = model.generate(prompt, 40, model.new_cache(90, kv="e4m3", page=64), graph=False)
    cache, c = model.new_cache(120, kv="e4m3", page=16), []
    y = model.forward(prompt, cache)
    for _ in range(40):
        c.append(int(y.argmax()))
        y = model.forward(c[-1:], cache)
    assert a == c and len(b) == 40
    # the same answer again behind the first, on the cache that has just been truncated
    cache.length = 0
    assert model.generate(prompt, 40, cache) == a


def test_batches():
    """Ragged batches over one pool: prompts, chunks, steps and idle sequences together."""
    cfg, W = small()
    model = M.Model(cfg, W, "w4a16")
    a = "model.layers.0.self_attn."
    bias = np.concatenate([W[a + f"{n}_proj.bias"] for n in "qkv"])
    cache = model.new_cache(120, kv="e4m3", sequences=4, page=16)
    rng, past = np.random.default_rng(5), np.zeros(4, np.int64)
    for news in ([40, 0, 7, 1], [1, 25, 30, 1], [1, 1, 1, 1], [0, 0, 50, 0], [1, 2, 0, 17]):
        before = pool_of(cache)
        y = model.forward_batch([rng.integers(0, 97, n) for n in news], cache)
        check_layer(model, cache, before, news, past, bias)
        assert y.shape == (4, 97) and np.array_equal(np.isnan(y).all(1), np.array(news) == 0)
        assert np.isfinite(y[np.array(news) > 0]).all()
        past += news
    assert np.array_equal(cache.lengths, past)


def test_a_batch_of_one_is_forward():
    cfg = M.tiny_config(max_position=400)
    model = M.Model(cfg, M.random_weights(cfg, seed=1), "w4a8")
    prompt = np.random.default_rng(3).integers(0, 97, 33)
    one, many = model.new_cache(64, kv="e4m3"), model.new_cache(64, kv="e4m3")
    assert np.array_equal(model.forward(prompt, one), model.forward_batch([prompt], many)[0])


def test_generate_batch():
    cfg = M.tiny_config(max_position=400)
    model = M.Model(cfg, M.random_weights(cfg, seed=1), "w4a16", max_tokens=8)
    rng = np.random.default_rng(4)
    prompts = [list(rng.integers(0, 97, n)) for n in (12, 1, 40)]
    out = model.generate_batch(prompts, 9)
    assert [len(o) for o in out] == [9, 9, 9]
    assert model.generate_batch(prompts, 9) == out and model.generate_batch(prompts, 0) == [[], [], []]
    with pytest.raises(ValueError):
        model.generate_batch([[1], []], 3)


def test_pages_come_and_go():
    cfg, W = small()
    model = M.Model(cfg, W, "w4a16")
    cache = model.new_cache(64, kv="e4m3", sequences=3, page=16, pages=6)
    rng = np.random.default_rng(6)
    t = lambda n: rng.integers(0, 97, n)  # noqa: E731
    model.forward_batch([t(30), t(30), t(16)], cache)  # 2 + 2 + 1 pages
    with pytest.raises(ValueError):
        model.forward_batch([t(10), t(10), t(1)], cache)  # 1 + 1 + 1 more
    assert list(cache.lengths) == [30, 30, 16] and len(cache._free) == 1
    cache.truncate(1)
    assert len(cache._free) == 3 and list(cache.lengths) == [30, 0, 16]
    y = model.forward_batch([t(10), [], t(1)], cache)
    assert np.isfinite(y[[0, 2]]).all() and len(cache._free) == 1
    assert len(set(cache._table[cache._table >= 0])) == 5
    for bad in (lambda: cache.truncate(1, 5), lambda: cache.truncate(0, -1), lambda: cache.length,
                lambda: model.forward(t(3), cache), lambda: model.forward_batch([t(1)], cache),
                lambda: model.forward_batch([[], [], []], cache), lambda: model.new_cache(10, kv="int8"),
                lambda: model.new_cache(10, sequences=2), lambda: model.new_cache(10, kv="e4m3", page=20),
                lambda: model.new_cache(0, kv="e4m3")):
        with pytest.raises(ValueError):
            bad()


def test_batches_take_an_8_bit_cache():
    cfg, W = small()
    model = M.Model(cfg, W, "w4a16")
    with pytest.raises(ValueError):
        model.forward_batch([[1]], model.new_cache(10))
