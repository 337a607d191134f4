"""Offsets and lengths that are none: calls stay within their tensors, in rows and in tiles of a chunk."""

import numpy as np
import pytest
import torch

from sparse_cases import i32
from tpu_cake_amd import sparse

pytestmark = pytest.mark.gpu

MOST, LEAST = 2**31 - 1, -2**31
GUARD = 1 << 16


def _offsets(kind, n, tokens, rng):
    if kind == "most":
        return np.full(n + 1, MOST)
    if kind == "least":
        return np.full(n + 1, LEAST)
    if kind == "alternating":
        return np.where(np.arange(n + 1) % 2, MOST, 0)
    if kind == "full span":
        return np.where(np.arange(n + 1) % 2, MOST, LEAST)
    if kind == "falling":
        return tokens - np.arange(n + 1)
    if kind == "past the tokens":
        return np.arange(n + 1) * 7 + tokens - 3
    return rng.integers(LEAST, MOST, n + 1)


@pytest.mark.parametrize("n,tokens", [(400, 1000), (3, 100), (70, 500), (500, 400), (3, 5)])  # tiles, and rows
@pytest.mark.parametrize("kind", ["most", "least", "alternating", "full span", "falling", "past the tokens", "any"])
@pytest.mark.parametrize("length", [50, MOST, LEAST])
def test_any_offsets_stay_inside(cuda, n, tokens, kind, length):
    rng = np.random.default_rng(n)
    heads, dim, page, columns, top = 2, 64, 16, 8, 3
    cu, lens = i32(_offsets(kind, n, tokens, rng)), i32(np.full(n, length))
    table, num = i32(rng.integers(0, 20, (n, columns))), i32([n])
    q = torch.randn((tokens, 4 * heads, dim), device="cuda").to(torch.bfloat16)
    pool = torch.randn((20, page, 2 * heads, dim), device="cuda").to(torch.bfloat16)
    index = sparse.make_page_index(pool)
    count = tokens * heads * top
    held = torch.full((count + 2 * GUARD,), 77, dtype=torch.int32, device="cuda")
    picked = held[GUARD:GUARD + count].view(tokens, heads, top)
    sparse.select_pages(q, index, lens, table, cu, num, page_size=page, num_pages=top, out=picked)
    assert (held[:GUARD] == 77).all() and (held[GUARD + count:] == 77).all()
    assert (((picked >= -1) & (picked < columns)) | (picked == 77)).all()
    listed = i32(rng.integers(-1, columns, (tokens, heads, top)))
    held = torch.full((q.numel() + 2 * GUARD,), 77.0, dtype=torch.bfloat16, device="cuda")
    out = held[GUARD:GUARD + q.numel()].view(q.shape)
    sparse.sparse_paged_attention(q, pool, listed, lens, table, cu, num, sm_scale=0.1, out=out)
    assert (held[:GUARD] == 77).all() and (held[GUARD + q.numel():] == 77).all()
    assert torch.isfinite(out).all()
    if length == LEAST or kind in ("most", "least"):  # no token sees a key
        assert (picked[(picked != 77).all(-1)] == -1).all() and (out[(out != 77).all(-1)] == 0).all()
    assert sparse.read_error_word(clear=True) in (0, sparse._sparse_lib.ERR_LEN)
