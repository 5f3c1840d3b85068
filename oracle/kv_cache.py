"""The paged 8-bit key / value cache, restated in numpy (lbd_kv8_* of include/lowbit_hip.h).

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). OCP E4M3 codes and E8M0 exponents are
decoded and rounded here from their definitions; the attention is float64. The rotation
before rounding to a code is evaluated as the library documents it (float32, every product
rounded), so that codes can be compared exactly; `rotated64` is the float64 value.
No counterpart in the reference (its cache is float32, src/lowbit/model.py:264-297).
"""
from __future__ import annotations

import numpy as np

# value of every E4M3 byte: 4 exponent bits (bias 7), 3 mantissa bits, no infinity, 0x7f NaN
_C = np.arange(256)
_EX, _MAN = (_C >> 3) & 15, (_C & 7).astype(np.float64)
E4M3 = np.where(_EX > 0, (8 + _MAN) * 2.0 ** (_EX - 10.0), _MAN * 2.0 ** -9)
E4M3 = np.where(_C > 127, -E4M3, E4M3)
E4M3[[0x7F, 0xFF]] = np.nan
_POS = E4M3[:127]  # 0 .. 448, increasing


def e4m3_round(x: np.ndarray) -> np.ndarray:
    """Codes nearest to x (|x| <= 448), ties to the even code; the sign of zero kept, NaN is 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isnan(x), 0, np.abs(x))
    hi = np.searchsorted(_POS, a).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    up = (dh < dl) | ((dh == dl) & (hi % 2 == 0))
    codes = np.where(up, hi, lo) | np.where(np.signbit(x), 128, 0)
    return np.where(np.isnan(x), 0x7F, codes).astype(np.uint8)


def e8m0_for(x: np.ndarray) -> int:
    """The smallest exponent byte with |x| <= 448 2^(e - 127); 255 where x is not finite."""
    if not np.isfinite(x).all():
        return 255
    big = float(np.abs(x.astype(np.float64)).max(initial=0.0))
    e = 0
    while big > 448 * 2.0 ** (e - 127):
        e += 1
    return e


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """x [n, heads, D] rotated by cos / sin [n, D/2] in x's type, each operation rounded."""
    h = x.shape[2] // 2
    a, b, c, s = x[:, :, :h], x[:, :, h:], cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s], 2)


class Pool:
    """Codes and exponents of `pages` pages; bytes as the device holds them."""

    def __init__(self, rng, pages: int, page: int, kv: int, d: int):
        r = lambda *s: rng.integers(0, 256, s, dtype=np.uint8)  # noqa: E731
        # stale content: any byte, NaN codes and NaN exponents among them
        self.k, self.v, self.ke, self.ve = (r(pages, kv, page, d), r(pages, kv, page, d), r(pages, kv), r(pages, kv))
        self.pages, self.page, self.kv, self.d = pages, page, kv, d

    def copy(self):
        p = object.__new__(Pool)
        p.__dict__ = {n: v.copy() if isinstance(v, np.ndarray) else v for n, v in self.__dict__.items()}
        return p

    def _put(self, codes, exps, pg, h, lo, y):
        """y [n, D] float32 into slots lo .. of block (pg, h)."""
        was = int(exps[pg, h]) if lo else 0
        e = max(was, e8m0_for(y))
        if e < 255:
            if lo and e != was:
                codes[pg, h, :lo] = e4m3_round(E4M3[codes[pg, h, :lo]] * 2.0 ** (was - e))
            codes[pg, h, lo:lo + len(y)] = e4m3_round(y.astype(np.float64) * 2.0 ** (127 - e))
        else:
            codes[pg, h, lo:lo + len(y)] = 0
        exps[pg, h] = e

    def append(self, q_start, past, table, max_new, qkv, bias, heads, cos, sin, q_out):
        """lbd_kv8_append on rows qkv [T, >= (heads + 2 kv) d]; q_out [T, >= heads d] edited."""
        kv, d, page = self.kv, self.d, self.page
        cap = table.shape[1] * page
        for b in range(len(past)):
            n = min(int(q_start[b + 1]) - int(q_start[b]), max_new)
            if n <= 0 or past[b] < 0:
                continue
            rows = slice(int(q_start[b]), int(q_start[b]) + n)
            x = qkv[rows, :(heads + 2 * kv) * d]
            x = (x if bias is None else x + bias).reshape(n, heads + 2 * kv, d)
            pos = past[b] + np.arange(n)
            at = np.minimum(pos, len(cos) - 1)
            with np.errstate(invalid="ignore", over="ignore"):
                y = rotate(x[:, :heads + kv], cos[at], sin[at])
            q_out[rows, :heads * d] = y[:, :heads].reshape(n, -1)
            for pi in sorted({int(p) // page for p in pos if p < cap}):
                pg, own = int(table[b, pi]), (pos // page == pi) & (pos < cap)
                if not 0 <= pg < self.pages:
                    continue
                lo = int(pos[own][0]) % page
                for h in range(kv):
                    self._put(self.k, self.ke, pg, h, lo, y[own, heads + h])
                    self._put(self.v, self.ve, pg, h, lo, x[own, heads + kv + h])

    def values(self, codes, exps):
        """float64 of blocks: codes [.., page, d], exps [..]."""
        s = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
        return E4M3[codes] * s[..., None, None]

    def attention(self, q_start, past, table, max_new, q, heads, out, window=None, sinks=0):
        """lbd_kv8_attention (lbd_kv8_attention_window with a window) of rows q [T, >= heads d] in
        float64; `out` edited. Also returns, per element of out, the scale of its rounding errors:
        (largest sum |q k| / sqrt(d), weighted mean of |v|, keys)."""
        kv, d, page = self.kv, self.d, self.page
        cap, g = table.shape[1] * page, heads // kv
        mags = np.zeros((len(q), heads, 3))
        for b in range(len(past)):
            n = min(int(q_start[b + 1]) - int(q_start[b]), max_new)
            if n <= 0 or past[b] < 0:
                continue
            last = min(int(past[b]) + n, cap)
            pgs = table[b, :-(-last // page)]
            held = np.repeat((pgs >= 0) & (pgs < self.pages), page)[:last]
            safe = np.where((pgs >= 0) & (pgs < self.pages), pgs, 0)
            k, v = (np.moveaxis(self.values(c[safe], e[safe]), 1, 0).reshape(kv, -1, d)[:, :last]
                    for c, e in ((self.k, self.ke), (self.v, self.ve)))
            rows = slice(int(q_start[b]), int(q_start[b]) + n)
            key, at = np.arange(last), past[b] + np.arange(n)[:, None]
            see = held & (key <= at)
            if window is not None:
                see &= (at - key < window) | (key < sinks)
            some = see.any(1)
            for h in range(heads):
                x = q[rows, h * d:(h + 1) * d].astype(np.float64)
                kk, vv = k[h // g], v[h // g]
                # what no row of the sequence sees, or one of them only, must not reach the others
                kk, vv = (np.where(see.any(0)[:, None], a, 0) for a in (kk, vv))
                bad = np.isnan(vv).any(1)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = np.where(see, x @ kk.T / np.sqrt(d), -np.inf)
                    p = np.exp(s - np.where(some, np.where(np.isnan(s), -np.inf, s).max(1), 0)[:, None])
                    p /= np.where(some, p.sum(1), 1)[:, None]
                    w = p @ np.where(bad[:, None], 0, vv)
                    w[(see & bad).any(1)] = np.nan
                    size = np.where(see, np.abs(x) @ np.abs(np.where(np.isnan(kk), 0, kk)).T, 0).max(1) / np.sqrt(d)
                    mean = (p @ np.abs(np.where(bad[:, None], 0, vv))).max(1)
                out[rows, h * d:(h + 1) * d] = np.where(some[:, None], w, 0)
                mags[rows, h] = np.stack([size, mean, see.sum(1)], 1)
        return mags
