"""KV8Cache's pages and lengths on the CPU: what it holds, takes from its pool and gives back. Its device
buffers are stand-ins."""
import numpy as np
import pytest

from lowbit_amd import kernels as K
from lowbit_amd import model as M


class Buffer:
    ptr = 0x1000

    def __init__(self, nbytes):
        self.nbytes = nbytes


@pytest.fixture
def new(monkeypatch):
    monkeypatch.setattr(M, "_buf", Buffer)
    monkeypatch.setattr(K.DeviceBuffer, "from_array", classmethod(lambda cls, a: Buffer(a.nbytes)))
    return lambda *a, **k: M.KV8Cache(M.tiny_config(), *a, **k)


def write(cache, seq, n):
    """What a pass does that brings the sequence to n tokens."""
    cache.reserve(seq, n)
    cache.commit(seq, n)


def test_truncate_takes_no_more_than_the_tokens_held(new):
    """Slots of a held page that no token was written to are not tokens."""
    cache = new(100, page=16)
    write(cache, 0, 3)
    for n in (4, 10, 16, 17, 100, -1):
        with pytest.raises(ValueError):
            cache.truncate(0, n)
        with pytest.raises(ValueError):
            cache.length = n
        assert cache.length == 3
    cache.reserve(0, 60)  # pages taken ahead of a pass are no tokens either
    for n in (4, 60):
        with pytest.raises(ValueError):
            cache.truncate(0, n)
    cache.truncate(0, 3)
    assert cache.length == 3 and len(cache._free) == cache.pages - 1
    cache.length = 2
    cache.length = 0
    assert cache.length == 0 and len(cache._free) == cache.pages
    with pytest.raises(ValueError):
        cache.truncate(0, 1)


def test_commit_takes_no_more_than_the_pages_held(new):
    cache = new(100, page=16, sequences=2)
    cache.reserve(1, 20)
    for seq, n in ((0, 1), (1, 33), (1, -1)):
        with pytest.raises(ValueError):
            cache.commit(seq, n)
    cache.commit(1, 20)
    assert list(cache.lengths) == [0, 20]
    cache.commit(1, 4)  # a pass that reserved more than it wrote
    assert len(cache._free) == cache.pages - 1


def test_pages_are_one_sequences_each(new):
    rng = np.random.default_rng(0)
    cache = new(90, page=16, sequences=5, pages=17)
    length = [0] * 5
    for _ in range(300):
        s = int(rng.integers(5))
        if rng.random() < 0.5:
            n = int(rng.integers(0, length[s] + 1))
            cache.truncate(s, n)
        else:
            n = int(rng.integers(length[s], 91))
            if -(-n // 16) - int(cache._held[s]) > len(cache._free):
                with pytest.raises(ValueError):
                    cache.reserve(s, n)
                continue
            write(cache, s, n)
        length[s] = n
        assert list(cache.lengths) == length and [-(-n // 16) for n in length] == list(cache._held)
        held = cache._table[cache._table >= 0]
        assert sorted([*held, *cache._free]) == list(range(17))
        assert all((cache._table[i, :h] >= 0).all() and (cache._table[i, h:] < 0).all()
                   for i, h in enumerate(cache._held))
