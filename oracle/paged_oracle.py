"""Numpy restatement of the paged cache operators in 64 bits, one token at a time (test infrastructure only).

State: kv [2, P, H, page, Dh] float64, weights [P, H, page] float64, positions [P, H, page], table [S, M],
lens [S, H], next_pos [S, H].
"""
import math

import numpy as np


def slot(table, s, i, page):
    return int(table[s, i // page]), i % page


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
    page = kv.shape[3]
    cap = table.shape[1] * page
    for s in range(S):
        n = T if n_new is None else int(n_new[s])
        for h in range(H):
            for t in range(n):
                i = int(lens[s, h]) + t
                if i >= cap:
                    break
                pg, r = slot(table, s, i, page)
                kv[0, pg, h, r], kv[1, pg, h, r] = k_new[s, h, t], v_new[s, h, t]
                weights[pg, h, r] = 0.0 if w_new is None else w_new[s, h, t]
                positions[pg, h, r] = next_pos[s, h] + t
            lens[s, h] = min(lens[s, h] + n, cap)
            next_pos[s, h] += n


def append_evict(kv, table, lens, next_pos, k_new, v_new, n_new, weights, positions, keep, sink, recent, w_new=None):
    S, H, T, _ = k_new.shape
    page = kv.shape[3]
    for s in range(S):
        n = T if n_new is None else int(n_new[s])
        for h in range(H):
            held = int(lens[s, h])
            where = [slot(table, s, i, page) for i in range(held)]
            rows = [(kv[0, a, h, r].copy(), kv[1, a, h, r].copy(), weights[a, h, r], int(positions[a, h, r])) for a, r in where]
            rows += [(k_new[s, h, t], v_new[s, h, t], 0.0 if w_new is None else w_new[s, h, t], int(next_pos[s, h]) + t)
                     for t in range(n)]
            end = int(next_pos[s, h]) + n

            def order(i):
                w, pos = rows[i][2], rows[i][3]
                return (not (pos < sink or pos >= end - recent), not np.isnan(w), 0.0 if np.isnan(w) else -w, i)
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
