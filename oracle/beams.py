"""Beam search's step and the pages of its beams, restated in numpy (lbd_beam_select, lbd_kv8_reorder
and lbd_kv8_copy_pages of include/lowbit_hip.h).

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). No counterpart in the reference, which decodes
greedily (src/lowbit/model.py:437-458).
"""
from __future__ import annotations

import numpy as np


def select(logits, score, done, beams, eos):
    """(tok, parent, sum in float64, done) of every place: logits [places, V], `beams` a prompt."""
    V = logits.shape[1]
    none = max(eos, 0)
    out = []
    for base in range(0, len(score), beams):
        offers = []  # (-sum, place, place among the beam's, token or -1 for the beam itself)
        for i in range(base, base + beams):
            s = float(score[i])
            if not s > -np.inf:
                continue
            if done is not None and done[i]:
                offers.append((-s, i, 0, -1))
                continue
            x = logits[i].astype(np.float64)
            if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
                continue
            m = x.max()
            lse = m + np.log(np.exp(x - m).sum())
            # larger logits first, of equals the lower token
            best = sorted(np.argsort(-x, kind="stable")[:beams], key=lambda v: (-x[v], v))
            offers += [(-(s + (x[v] - lse)), i, n, int(v)) for n, v in enumerate(best) if x[v] > -np.inf]
        offers.sort()
        for w in range(beams):
            if w < len(offers):
                neg, i, _, v = offers[w]
                out.append((none if v < 0 else v, i, -neg, int(v < 0 or v == eos)))
            else:
                out.append((none, -1, -np.inf, 0))
    assert V > 0
    tok, parent, total, end = zip(*out)
    return np.array(tok), np.array(parent), np.array(total), np.array(end)


def reorder(parent, done, past, table, own, beams, add, page, pages):
    """(new_past, new_table, [(from, to, tokens)]) of lbd_kv8_reorder."""
    places, wide = table.shape
    new_past, new_table, moves = np.full(places, -1), np.full((places, wide), -1), []
    for base in range(0, places, beams):
        here = range(base, base + beams)
        goes = {i: int(parent[i]) for i in here
                if base <= parent[i] < base + beams and not (done is not None and done[i]) and past[parent[i]] >= 0}
        length = {i: min(int(past[p]) + add, 1 << 30) for i, p in goes.items()}
        tail = {i: min(n, wide * page) // page for i, n in length.items()}
        used = {i: n % page if n < wide * page else 0 for i, n in length.items()}
        heir = {}
        for i, p in goes.items():
            if used[i]:
                heir.setdefault(p, i)

        def holds(i, j):
            return tail[i] > j or (tail[i] == j and used[i] > 0 and heir[goes[i]] == i)

        def page_at(i, j):
            """Of a place that holds none at index j."""
            held = {int(table[goes[k], j]) for k in goes if holds(k, j)}
            if not any(holds(k, j) for k in goes):
                return int(own[i, j])
            free = [int(own[k, j]) for k in here if 0 <= own[k, j] < pages and own[k, j] not in held]
            n = sum(k < i and not holds(k, j) for k in goes)
            return free[n] if n < len(free) else -1

        for i, p in goes.items():
            new_past[i] = length[i]
            for j in range(wide):
                new_table[i, j] = table[p, j] if holds(i, j) else page_at(i, j)
            if used[i] and heir[p] != i:
                a, b = int(table[p, tail[i]]), int(new_table[i, tail[i]])
                if b >= 0 and 0 <= a < pages:
                    moves.append((a, b, used[i]))
    return new_past, new_table, moves


def move(pool, moves):
    """The copies (from, to, tokens) in a pool of oracle.kv_cache; tokens None: the page whole."""
    was = pool.copy()
    for a, b, n in moves:
        for x in ("k", "v"):
            getattr(pool, x)[b, :, :n] = getattr(was, x)[a, :, :n]
        for x in ("ke", "ve"):
            getattr(pool, x)[b] = getattr(was, x)[a]
