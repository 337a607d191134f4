"""Oracles of a serving step with a bounded cache (``include/rpa_bounded.h``, ``rpa_trim_pages``): plain numpy loops,
whole numbers or 64-bit floats, from the definitions.  Test infrastructure only.
"""

from __future__ import annotations

import numpy as np


def rotate_heads(x, positions, turns, *, interleaved=False, magnitude=1.0, weight=None, eps=1e-6):
    """(result, size) of one of the two tensors, float64 [T, H, D]: size is the sum of the magnitudes that a result is made of."""
    x = np.asarray(x, np.float64).copy()
    if weight is not None:
        x = x / np.sqrt((x**2).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    half = len(turns)
    size = np.abs(x).copy()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    # the fraction of a turn, exactly: whole numbers mod 2^64
    part = np.array([[(int(p) * int(f)) % (1 << 64) for f in turns] for p in positions], np.float64).reshape(len(positions), half)
    angle = (2 * np.pi * part / 2.0**64)[:, None, :]
    a, b = x[..., first].copy(), x[..., second].copy()
    with np.errstate(invalid="ignore"):
        x[..., first] = (a * np.cos(angle) - b * np.sin(angle)) * magnitude
        x[..., second] = (b * np.cos(angle) + a * np.sin(angle)) * magnitude
    size[..., first] = size[..., second] = (np.abs(a) + np.abs(b)) * magnitude
    return x, size


def weighed_attention(q, keys, values, weights, positions, kv_lens, table, cu, num_seqs, sm_scale, *, soft_cap=None, decay=1.0,
                      dropped=None):
    """keys, values [pages, page_size, Hkv, D] as the pool stands for them, ledger [pages, Hkv, page_size].  Returns float64 out
    [T, Hq, D], weights, int positions, and bounds of what 32-bit scores and sums may add to out and to weights."""
    q = np.asarray(q, np.float64)
    tokens, hq, dim = q.shape
    page_size, hkv = keys.shape[1], keys.shape[2]
    group = hq // hkv
    out, slack = np.zeros((tokens, hq, dim)), np.zeros((tokens, hq, dim))
    weights, positions = np.array(weights, np.float64), np.array(positions, np.int64)
    loose = np.zeros_like(weights)
    for i in range(num_seqs):
        begin, end = int(cu[i]), min(int(cu[i + 1]), tokens)
        n = min(int(kv_lens[i]), table.shape[1] * page_size)
        if end <= begin or n <= 0:
            continue
        row = np.arange(n)
        page, off = np.asarray(table[i], np.int64)[row // page_size], row % page_size
        old = n - (end - begin)
        for h in range(hkv):
            k, v = keys[page, off, h].astype(np.float64), values[page, off, h].astype(np.float64)
            x = q[begin:end, h * group:(h + 1) * group]
            s = x @ k.T * sm_scale
            # a score's error: dim products and sums in 32 bits, the scale; times 2 for the row's sum of them
            d = (dim + 8) * 2.0**-24 * (np.abs(x) @ np.abs(k).T) * abs(sm_scale)
            if soft_cap:
                s = soft_cap * np.tanh(s / soft_cap)
                d = d + 2.0**-20 * np.abs(soft_cap)
            d = 2 * d.max(-1, initial=0.0) + (n + 16) * 2.0**-24 + 2.0**-22 * np.abs(s).max(-1, initial=0.0)
            late = row > old + np.arange(end - begin)[:, None, None]
            s = np.where(late, -np.inf, s)
            top = s.max(-1, keepdims=True)
            p = np.where(np.isfinite(top) & ~late, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = p.sum(-1, keepdims=True)
            p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
            # a masked key's values count for nothing, whatever they are
            out[begin:end, h * group:(h + 1) * group] = np.einsum("tgn,nd->tgd", p, np.where(np.isfinite(v), v, 0.0))
            slack[begin:end, h * group:(h + 1) * group] = np.einsum("tgn,nd->tgd", p, np.abs(np.where(np.isfinite(v), v, 0.0))) * d[..., None]
            before = np.where(row < old, decay * weights[page, h, off] if decay else 0.0, 0.0)
            got = p.sum((0, 1))
            weights[page, h, off] = before + got
            loose[page, h, off] = (p * d[..., None]).sum((0, 1)) + ((end - begin) * group + 2) * 2.0**-24 * got + 2.0**-22 * before
            fresh = row >= max(old, 0)
            positions[page[fresh], h, off[fresh]] = row[fresh] + (int(dropped[i]) if dropped is not None else 0)
    return out, weights, positions, slack, loose


def choose_moves(weights, positions, kv_lens, table, num_seqs, *, budget, recent, sinks=0, limit=None, dropped=None, max_moves=None):
    limit, max_moves = budget if limit is None else limit, budget if max_moves is None else max_moves
    hkv, page_size = weights.shape[1], weights.shape[2]
    moves = np.full((len(kv_lens), hkv, max_moves, 2), -1, np.int64)
    for i in range(num_seqs):
        n = int(kv_lens[i])
        end = n + (int(dropped[i]) if dropped is not None else 0)
        n = min(n, table.shape[1] * page_size)
        if n <= limit:
            continue
        page, off = np.asarray(table[i], np.int64)[np.arange(n) // page_size], np.arange(n) % page_size
        slot = page * page_size + off
        for h in range(hkv):
            w, p = weights[page, h, off].astype(np.float64), positions[page, h, off]
            forced = (p < sinks) | (p >= end - recent)
            # forced rows are all alike: of too many the lowest stay
            w = np.where(forced, 0.0, w)
            order = sorted(range(n), key=lambda r: (not forced[r], bool(np.isnan(w[r])), -w[r] if not np.isnan(w[r]) else 0.0, r))
            kept = np.zeros(n, bool)
            kept[order[:budget]] = True
            late, holes = np.nonzero(kept[budget:])[0] + budget, np.nonzero(~kept[:budget])[0]
            for m, (a, b) in enumerate(zip(holes, late)):
                if m < max_moves:
                    moves[i, h, m] = slot[a], slot[b]
    return moves


def move_rows(pool, weights, positions, moves, requantise=None):
    """pool [pages, page_size, 2 * Hkv, D] of any type; requantise(rows, head, from slots, to slots) for rows that change pages."""
    pool, weights, positions = pool.copy(), weights.copy(), positions.copy()
    hkv, page_size = weights.shape[1], weights.shape[2]
    rows = pool.reshape(pool.shape[0] * page_size, hkv, 2, pool.shape[3])
    for h in range(hkv):
        for to, origin in moves[:, h].reshape(-1, 2):
            if to < 0 or origin < 0:
                continue
            x = rows[origin, h]
            rows[to, h] = requantise(x, h, origin // page_size, to // page_size) if requantise else x
            for ledger in (weights, positions):
                ledger[to // page_size, h, to % page_size] = ledger[origin // page_size, h, origin % page_size]
    return pool, weights, positions


def trim_pages(cached, dropped, table, free, count, page_size, budget, limit=None):
    """(lengths, dropped, free stack, count)."""
    cached, dropped, free, count = np.array(cached, np.int64), np.array(dropped, np.int64), np.array(free, np.int64), int(count)
    capacity = table.shape[1] * page_size
    for i in range(len(cached)):
        if cached[i] <= (budget if limit is None else limit):
            continue
        for page in table[i, -(-budget // page_size):-(-min(int(cached[i]), capacity) // page_size)]:
            if count < len(free):
                free[count] = page
                count += 1
        dropped[i] += cached[i] - budget
        cached[i] = budget
    return cached, dropped, free, count
