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
