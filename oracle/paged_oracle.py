"""Numpy restatement of the paged cache operators in 64 bits, one token at a time (test infrastructure only).

State: kv [2, P, H, page, Dh] float64, weights [P, H, page] float64, positions [P, H, page], table [S, M],
lens [S, H], next_pos [S, H].
"""
import math

import numpy as np


def slot(table, s, i, page):
    return int(table[s, i // page]), i % page


def named(table, s, b, pages):
    """Whether the table names a page of the pool for block b of session s."""
    return 0 <= int(table[s, b]) < pages


def with_a_page(table, s, first, want, page, pages):
    """How many of `want` tokens from slot `first` on can be held: up to the first one without a page."""
    t = 0
    while t < want and (first + t) // page < table.shape[1] and named(table, s, (first + t) // page, pages):
        t += 1
    return t


def attend(q, kv, table, lens, scale=None):
    """q [S, Hq, Dh] -> out [S, Hq, Dh], lse [S, Hq], given[s][h] [n] (the weight each held token gets), and
    spread [S, Hq, Dh] = sum_j p_j |v_j|, what errors of the weights are measured against."""
    S, Hq, Dh = q.shape
    H, page = kv.shape[2], kv.shape[3]
    G = Hq // H
    scale = 1.0 / math.sqrt(Dh) if scale is None else scale
    out, spread = np.zeros((S, Hq, Dh)), np.zeros((S, Hq, Dh))
    lse = np.full((S, Hq), -np.inf)
    given = [[np.zeros(0) for _ in range(H)] for _ in range(S)]
    for s in range(S):
        for h in range(H):
            n = int(lens[s, h])
            if n == 0:
                continue
            i = np.arange(n)
            pg, row = table[s, i // page], i % page
            k, v = kv[0, pg, h, row], kv[1, pg, h, row]
            with np.errstate(invalid="ignore", over="ignore"):
                x = (q[s, h * G:(h + 1) * G] @ k.T) * scale
                top = x.max(axis=1, keepdims=True)
                e = np.exp(x - top)
                p = e / e.sum(axis=1, keepdims=True)
                out[s, h * G:(h + 1) * G] = p @ v
                spread[s, h * G:(h + 1) * G] = p @ np.abs(v)
                lse[s, h * G:(h + 1) * G] = top[:, 0] + np.log(e.sum(axis=1))
            given[s][h] = p.sum(axis=0)
    return out, lse, given, spread


def add_given(weights, table, given, page):
    for s, row in enumerate(given):
        for h, p in enumerate(row):
            for i, x in enumerate(p):
                pg, r = slot(table, s, i, page)
                weights[pg, h, r] += x


def append(kv, table, lens, next_pos, k_new, v_new, n_new, weights, positions, w_new=None):
    S, H, T, _ = k_new.shape
    pages, page = kv.shape[1], kv.shape[3]
    for s in range(S):
        n = T if n_new is None else int(n_new[s])
        for h in range(H):
            take = with_a_page(table, s, int(lens[s, h]), n, page, pages)
            for t in range(take):
                i = int(lens[s, h]) + t
                pg, r = slot(table, s, i, page)
                kv[0, pg, h, r], kv[1, pg, h, r] = k_new[s, h, t], v_new[s, h, t]
                weights[pg, h, r] = 0.0 if w_new is None else w_new[s, h, t]
                positions[pg, h, r] = next_pos[s, h] + t
            lens[s, h] += take
            next_pos[s, h] += n


def append_evict(kv, table, lens, next_pos, k_new, v_new, n_new, weights, positions, keep, sink, recent, w_new=None):
    S, H, T, _ = k_new.shape
    pages, page = kv.shape[1], kv.shape[3]
    for s in range(S):
        for h in range(H):
            n = T if n_new is None else int(n_new[s])
            held, end = int(lens[s, h]), int(next_pos[s, h]) + n
            below = max(0, min(n, keep - held))                  # new tokens whose slot lies below the budget
            if with_a_page(table, s, held, below, page, pages) < below:
                n = with_a_page(table, s, held, below, page, pages)
            where = [slot(table, s, i, page) for i in range(held)]
            rows = [(kv[0, a, h, r].copy(), kv[1, a, h, r].copy(), weights[a, h, r], int(positions[a, h, r]))
                    if 0 <= a < pages else None for a, r in where]
            rows += [(k_new[s, h, t], v_new[s, h, t], 0.0 if w_new is None else w_new[s, h, t], int(next_pos[s, h]) + t)
                     for t in range(n)]

            def order(i):
                if i < held and rows[i] is None:   # a slot without a page: it can neither move nor be filled
                    return (-1 if i < keep else 2, False, 0.0, i)
                w, pos = rows[i][2], rows[i][3]
                if pos < sink or pos >= end - recent:
                    return (0, False, 0.0, i)
                return (1, not np.isnan(w), 0.0 if np.isnan(w) else -w, i)
            kept = sorted(range(len(rows)), key=order)[:keep]
            stay = set(kept)
            holes = [i for i in range(min(keep, len(rows))) if i not in stay]
            movers = sorted(i for i in kept if i >= keep)
            assert len(holes) == len(movers)
            for src, dst in list(zip(movers, holes)) + [(i, i) for i in kept if held <= i < keep]:
                pg, r = slot(table, s, dst, page)
                kv[0, pg, h, r], kv[1, pg, h, r], weights[pg, h, r], positions[pg, h, r] = rows[src]
            lens[s, h] = min(len(rows), keep)
            next_pos[s, h] = end
