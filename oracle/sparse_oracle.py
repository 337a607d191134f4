"""Oracles of the page allocator, the K/V append with its page index, the choice of pages and the
attention over them (``include/rpa_sparse.h``): plain numpy loops, whole numbers or 64-bit floats,
from the definitions.  Test infrastructure only.
"""

from __future__ import annotations

import math

import numpy as np

FP8_MAX = 448.0
EXP_MIN, EXP_MAX = -100, 100


def assign_pages(cached, new, table, free, count, page_size, max_tokens):
    """(kv_lens, cu_q_lens, slot_mapping, positions, table, count), with pages taken from the top of the stack."""
    cached, table = np.array(cached, np.int64), np.array(table, np.int64)
    capacity, left = table.shape[1] * page_size, int(count)
    pages_so_far = tokens_so_far = 0
    kv, cu, slots, pos = [], [0], [], []
    for i, (c, m) in enumerate(zip(cached.tolist(), np.asarray(new).tolist())):
        ok = c >= 0 and m >= 0 and c + m <= capacity
        if ok:
            have, want = -(-c // page_size), -(-(c + m) // page_size)
            pages_so_far += want - have
            tokens_so_far += m
            ok = tokens_so_far <= max_tokens and (want == have or pages_so_far <= count)
        if ok:
            for j in range(have, want):
                left -= 1
                table[i, j] = free[left]
            for p in range(c, c + m):
                slots.append(int(table[i, p // page_size]) * page_size + p % page_size)
                pos.append(p)
        kv.append(max(c, 0) + (m if ok else 0))
        cu.append(len(slots))
    pad = max_tokens - len(slots)
    return (np.array(kv), np.array(cu), np.array(slots + [-1] * pad, np.int64), np.array(pos + [0] * pad, np.int64), table, left)


def release_pages(cached, finished, table, free, count, page_size):
    """(lengths, free stack, count)."""
    cached, free, count = np.array(cached, np.int64), np.array(free, np.int64), int(count)
    for i in np.nonzero(finished)[0]:
        for page in table[i, :-(-min(max(int(cached[i]), 0), table.shape[1] * page_size) // page_size)]:
            if count < len(free):
                free[count] = page
                count += 1
        cached[i] = 0
    return cached, free, count


# ------------------------------------------------------------------------------- index and append
def grid_exponent(amax: float) -> int:
    e = EXP_MIN
    while e < EXP_MAX and 127.0 * 2.0**e < amax:
        e += 1
    return e


def page_bounds(keys):
    """(int8 bounds [2, D], exponent) of one page's keys of one head, [n, D] floats, n >= 1."""
    keys = np.where(np.isnan(keys), 0.0, np.asarray(keys, np.float64))
    hi, lo = keys.max(0), keys.min(0)
    e = grid_exponent(max(np.abs(hi).max(), np.abs(lo).max()))
    with np.errstate(over="ignore"):
        return np.stack([np.clip(np.ceil(hi * 2.0**-e), -127, 127), np.clip(np.floor(lo * 2.0**-e), -127, 127)]), e


def e4m3(x):
    """The e4m3 value nearest to each |x| <= 448 (ties to even), as floats."""
    x = np.asarray(x, np.float64)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-30))), -6) - 3)
    return np.clip(np.rint(x / step) * step, -FP8_MAX, FP8_MAX)


# ------------------------------------------------------------------------------- choice, attention
def positions(kv_lens, cu, num_seqs, tokens):
    """(sequence, position) of each token; (-1, -1) past the last."""
    got = [(-1, -1)] * tokens
    for i in range(num_seqs):
        for t in range(int(cu[i]), min(int(cu[i + 1]), tokens)):
            got[t] = (i, int(kv_lens[i]) - (int(cu[i + 1]) - t))
    return got


def select_pages(q, bounds, exponents, kv_lens, table, cu, num_seqs, page_size, num_pages, sink=1, recent=1):
    q = np.asarray(q, np.float64)
    tokens, hq, _ = q.shape
    hkv = bounds.shape[1]
    group = hq // hkv
    out = np.full((tokens, hkv, num_pages), -1, np.int64)
    for t, (i, pos) in enumerate(positions(kv_lens, cu, num_seqs, tokens)):
        if pos < 0:
            continue
        n = min(pos // page_size, table.shape[1] - 1) + 1
        ids = np.asarray(table[i, :n], np.int64)
        for h in range(hkv):
            x = q[t, h * group:(h + 1) * group]
            x = np.where(np.isnan(x), 0.0, x)
            f = grid_exponent(np.abs(x).max())
            x = np.clip(np.rint(x * 2.0**-f), -127, 127).astype(np.int64)
            b = bounds[ids, h].astype(np.int64)
            s = np.maximum(x, 0) @ b[:, 0].T + np.minimum(x, 0) @ b[:, 1].T  # [group, n]
            s = s.max(0) * 2.0 ** exponents[ids, h].astype(np.float64)
            at = np.arange(n)
            s[(at < sink) | (at >= n - recent)] = np.inf
            best = np.sort(np.argsort(-s, kind="stable")[:num_pages])
            out[t, h, :len(best)] = best
    return out


def sparse_attention(q, keys, values, picked, kv_lens, table, cu, num_seqs, sm_scale, soft_cap=None):
    """keys, values [pages, page_size, Hkv, D] as the pool stands for them; float64 [T, Hq, D]."""
    q = np.asarray(q, np.float64)
    tokens, hq, dim = q.shape
    page_size, hkv = keys.shape[1], keys.shape[2]
    group = hq // hkv
    out = np.zeros((tokens, hq, dim))
    for t, (i, pos) in enumerate(positions(kv_lens, cu, num_seqs, tokens)):
        if pos < 0:
            continue
        for h in range(hkv):
            ks, vs = [], []
            for page in np.asarray(picked[t, h]).tolist():
                seen = min(page_size, pos + 1 - page * page_size)
                if 0 <= page < table.shape[1] and seen > 0:
                    ks.append(keys[table[i, page], :seen, h])
                    vs.append(values[table[i, page], :seen, h])
            if not ks:
                continue
            k, v = np.concatenate(ks).astype(np.float64), np.concatenate(vs).astype(np.float64)
            s = q[t, h * group:(h + 1) * group] @ k.T * sm_scale
            if soft_cap:
                s = soft_cap * np.tanh(s / soft_cap)
            w = np.exp(s - s.max(1, keepdims=True))
            out[t, h * group:(h + 1) * group] = w @ v / w.sum(1, keepdims=True)
    return out
