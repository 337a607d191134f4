"""Ragged batches for the tests of the sparse entry points (not collected)."""

import numpy as np
import torch

from oracle import sparse_oracle as orc


def i32(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda")


class Batch:
    """Sequences of kv_lens keys whose last q_lens tokens are this step's, over a pool of shuffled pages;
    ``spare``: rows of the metadata past num_seqs, ``pad``: tokens past the last."""

    def __init__(self, seed, kv_lens, q_lens, page_size, hq, hkv, dim, *, spare=0, pad=0, extra_columns=2):
        self.rng = rng = np.random.default_rng(seed)
        self.page_size, self.hq, self.hkv, self.dim = page_size, hq, hkv, dim
        self.n = len(kv_lens)
        self.lens = np.array(list(kv_lens) + [0] * spare)
        pages = -(-np.array(kv_lens) // page_size)
        self.total = int(pages.sum()) + 3
        order = rng.permutation(self.total)
        width = int(pages.max(initial=0)) + extra_columns
        self.table = np.zeros((self.n + spare, width), np.int64)
        at = 0
        for i, p in enumerate(pages):
            self.table[i, :p] = order[at:at + p]
            at += p
        self.cu = np.concatenate([[0], np.cumsum(q_lens), np.full(spare, int(np.sum(q_lens)) + 7)])
        self.tokens = int(np.sum(q_lens)) + pad
        self.q = torch.from_numpy(rng.standard_normal((self.tokens, hq, dim), np.float32)).to(torch.bfloat16)

    def meta(self):
        return i32(self.lens), i32(self.table), i32(self.cu), i32([self.n])

    def pool(self, kind="bf16"):
        """(pool, scales, keys, values): the last two as float64 [pages, page_size, Hkv, D]."""
        shape = (self.total, self.page_size, self.hkv, 2, self.dim)
        x = self.rng.standard_normal(shape, np.float32)
        flat = (self.total, self.page_size, 2 * self.hkv, self.dim)
        if kind == "bf16":
            pool, scales = torch.from_numpy(x).to(torch.bfloat16), None
            held = pool.double().numpy()
        else:
            scales = self.rng.uniform(0.005, 0.02, (self.total, self.hkv, 2)).astype(np.float32)
            pool = torch.from_numpy(np.clip(x * 100, -448, 448)).to(torch.float8_e4m3fn)
            held = pool.double().numpy() * scales.astype(np.float64)[:, None, :, :, None]
        return pool.view(flat), scales, held[:, :, :, 0], held[:, :, :, 1]

    def index(self, spread=(-7, -3)):
        bounds = self.rng.integers(-127, 128, (self.total, self.hkv, 2, self.dim)).astype(np.int8)
        bounds[:, :, 0], bounds[:, :, 1] = bounds.max(2), bounds.min(2)
        return bounds, self.rng.integers(*spread, (self.total, self.hkv)).astype(np.int8)

    def lists(self, num_pages, hole=0.1):
        """For every token and head: pages of its own in random order, some entries that list nothing."""
        got = np.full((self.tokens, self.hkv, num_pages), -1)
        for t, (i, pos) in enumerate(orc.positions(self.lens, self.cu, self.n, self.tokens)):
            if pos < 0:
                continue
            n = pos // self.page_size + 1
            for h in range(self.hkv):
                pages = self.rng.permutation(n)[:num_pages]
                got[t, h, :len(pages)] = pages
                empty = self.rng.random(num_pages) < hole
                got[t, h, empty] = self.rng.choice([-1, -5, n, 10**6, 2**31 - 1], int(empty.sum()))
        return got
