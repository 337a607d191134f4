"""sparse_paged_attention against the 64-bit oracle, at tolerances that count its roundings:

* the output's own rounding: half a step, 2^-8 of its value;
* scores: D products and sums in fp32, at most (D + 4) 2^-24 sum|q k| sm_scale; twice that on a weight
  relative to the row's sum;
* P in two bf16 parts: 2^-16; exp2 and the running rescale: 2^-20; n keys summed in fp32, n 2^-24.
"""

import numpy as np
import pytest
import torch

from oracle import sparse_oracle as orc
from sparse_cases import Batch, i32
from tpu_cake_amd import ops, sparse

pytestmark = pytest.mark.gpu


def _tolerance(want, q, keys, values, n, sm_scale):
    finite = np.abs(np.where(np.isfinite(keys), keys, 0)).max()
    products = np.abs(q.double().numpy()).sum(-1).max() * finite * abs(sm_scale)
    score = (q.shape[-1] + 4) * 2.0**-24 * products
    return 2.0**-8 * np.abs(want) + np.abs(values).max() * (2 * score + 2.0**-16 + 2.0**-20 + n * 2.0**-24)


def _check(b, num_pages, kind="bf16", *, sm_scale=None, soft_cap=None, hole=0.1, picked=None):
    pool, scales, keys, values = b.pool(kind)
    sm_scale = b.dim ** -0.5 if sm_scale is None else sm_scale
    picked = b.lists(num_pages, hole) if picked is None else picked
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32(picked), *b.meta(), sm_scale=sm_scale, soft_cap=soft_cap,
                                        kv_scales=None if scales is None else torch.from_numpy(scales).cuda())
    want = orc.sparse_attention(b.q.double().numpy(), keys, values, picked, b.lens, b.table, b.cu, b.n, sm_scale, soft_cap)
    off = np.abs(got.double().cpu().numpy() - want)
    tol = _tolerance(want, b.q, keys, values, num_pages * b.page_size, sm_scale)
    worst = (off / tol).max()
    assert worst <= 1, f"{worst} times the tolerance, off by {off.max()}"
    return got, want


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("bf16", 64), ("bf16", 256), ("bf16", 32), ("bf16", 40), ("bf16", 96),
                                      ("fp8", 128), ("fp8", 64), ("fp8", 256), ("fp8", 80)])
@pytest.mark.parametrize("page", [1, 7, 16, 64, 100, 256])
def test_dims_and_pages(cuda, kind, dim, page):
    b = Batch(dim + page, [1, 30, 1000, 64, 0, 257], [1, 1, 1, 1, 0, 1], page, 8, 2, dim, spare=1, pad=1)
    _check(b, 9, kind)


@pytest.mark.parametrize("group,hkv", [(1, 8), (2, 3), (4, 2), (7, 1), (8, 8), (16, 1), (17, 2), (40, 1)])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_groups(cuda, group, hkv, kind):
    _check(Batch(group, [500, 77, 3], [1, 9, 3], 16, group * hkv, hkv, 128), 8, kind)


@pytest.mark.parametrize("num_pages,page", [(1, 1), (1, 16), (3, 32), (300, 16), (1500, 1), (40, 64), (5, 1024)])
def test_lists_long_and_short(cuda, num_pages, page):
    """One key to thousands; few rows, so their lists are split over workgroups."""
    _check(Batch(num_pages, [5000, 1234], [1, 1], page, 8, 2, 128), num_pages)


def test_many_rows_are_not_split(cuda):
    _check(Batch(3, [300] * 200, [1] * 200, 16, 16, 8, 64), 6)


def test_chunk_tokens_see_their_own_keys_only(cuda):
    b = Batch(8, [200, 64], [120, 64], 16, 8, 2, 128)
    _check(b, 13, hole=0.0)  # all pages: causal attention


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("bf16", 64), ("bf16", 256), ("bf16", 32), ("bf16", 40), ("bf16", 96),
                                      ("fp8", 128), ("fp8", 64), ("fp8", 256), ("fp8", 80)])
@pytest.mark.parametrize("page", [1, 7, 16, 64, 100, 256])
def test_chunks_of_dims_and_pages(cuda, kind, dim, page):
    b = Batch(dim + page, [90, 30, 1000, 64, 0, 257, 5], [33, 1, 70, 64, 0, 16, 2], page, 8, 2, dim, spare=1, pad=5)
    _check(b, 6, kind)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 9, 16, 17])
def test_chunks_of_groups(cuda, group):
    _check(Batch(group, [400, 77, 3], [50, 9, 3], 16, group * 2, 2, 64, pad=1), 8, soft_cap=30.0)


def test_chunk_with_long_lists(cuda):
    """Unions of more pages than a workgroup holds, and lists of their own that long."""
    _check(Batch(31, [4000], [12], 1, 4, 1, 64), 1500)
    _check(Batch(32, [1900, 3000], [9, 8], 1, 8, 1, 64), 300)


def test_chunk_over_a_table_past_the_bitmaps(cuda):
    _check(Batch(33, [33000], [9], 1, 4, 1, 32), 20)


def test_chunk_over_huge_pages(cuda):
    """Pages of more parts than a tile indexes."""
    _check(Batch(34, [140000, 90], [3, 5], 131072, 2, 1, 32), 2)


def test_chunk_pages_listed_twice_count_twice(cuda):
    b = Batch(35, [200, 300], [20, 40], 16, 8, 2, 64)
    picked = b.lists(7)
    picked[3, 0, 5] = picked[3, 0, 1]
    picked[33, 1] = picked[33, 1, 0]
    _check(b, 7, picked=picked)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_chunk_nan_that_other_tokens_see(cuda, kind):
    """A key that one token lists, or is far enough to see, holds NaN or infinities: only that token's rows show it."""
    b = Batch(36, [80, 70], [40, 30], 16, 8, 2, 128)
    pool, scales, keys, values = b.pool(kind)
    picked = b.lists(5, hole=0.0)
    picked[:40][picked[:40] == 1] = -1
    picked[7, 0, 0] = 1  # token 7 of the first sequence alone lists its page 1, for kv head 0
    held = pool.view(torch.uint8) if kind == "fp8" else pool
    held[b.table[0, 1], 3, :2] = 0x7F if kind == "fp8" else float("nan")
    held[b.table[1, 4], 1, 2:] = 0x7F if kind == "fp8" else float("inf")  # position 65 of 70, kv head 1
    pool = held.view(pool.dtype)
    kw = dict(sm_scale=0.1, kv_scales=None if scales is None else torch.from_numpy(scales).cuda())
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32(picked), *b.meta(), **kw).double().cpu().numpy()
    bad = np.zeros((70, 8), bool)
    bad[7, :4] = True
    for t, (i, pos) in enumerate(orc.positions(b.lens, b.cu, b.n, 70)):
        if i == 1 and pos >= 65 and (picked[t, 1] == 4).any():
            bad[t, 4:] = True
    assert bad.sum() > 8 and (~np.isfinite(got).all(-1) == bad).all()
    want = orc.sparse_attention(b.q.double().numpy(), keys, values, picked, b.lens, b.table, b.cu, b.n, 0.1)
    tol = _tolerance(want, b.q, keys, values, 80, 0.1)
    assert (np.abs(got - want) <= tol)[~bad].all()


@pytest.mark.parametrize("kind,dim,group", [("bf16", 128, 4), ("bf16", 64, 8), ("bf16", 256, 16), ("bf16", 40, 3), ("fp8", 128, 1),
                                            ("fp8", 256, 4), ("fp8", 80, 5)])
@pytest.mark.parametrize("page,num_pages", [(64, 12), (256, 12), (24, 70), (1, 1100)])
def test_short_chunks_split_their_lists(cuda, kind, dim, group, page, num_pages):
    """Three and more workgroups a tile; parts without keys, a decode row and rows past the last token."""
    b = Batch(dim + page, [1500, 700, 20, 3000], [20, 9, 2, 1], page, group * 2, 2, dim, pad=6)
    _check(b, num_pages, kind, hole=0.2)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_split_chunks_with_pages_listed_twice_and_nan(cuda, kind):
    """Each part falls back by itself: twice in one token's list, and NaN that one token lists, in different parts."""
    b = Batch(21, [4000, 900], [30, 8], 64, 8, 2, 128)
    pool, scales, keys, values = b.pool(kind)
    picked = b.lists(24, hole=0.0)
    picked[4, 0, :3] = 2  # three times
    picked[picked == 40] = -1
    picked[9, 1, 0] = 40
    held = pool.view(torch.uint8) if kind == "fp8" else pool
    held[b.table[0, 40], 3, 2:] = 0x7F if kind == "fp8" else float("nan")  # kv head 1
    pool = held.view(pool.dtype)
    kw = dict(sm_scale=0.1, kv_scales=None if scales is None else torch.from_numpy(scales).cuda())
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32(picked), *b.meta(), **kw).double().cpu().numpy()
    bad = np.zeros((b.tokens, 8), bool)
    bad[9, 4:] = True
    assert (~np.isfinite(got).all(-1) == bad).all()
    want = orc.sparse_attention(b.q.double().numpy(), keys, values, picked, b.lens, b.table, b.cu, b.n, 0.1)
    tol = _tolerance(want, b.q, keys, values, 24 * 64, 0.1)
    assert (np.abs(got - want) <= tol)[~bad].all()


@pytest.mark.parametrize("part,value", [(1, float("nan")), (1, float("inf")), (0, float("nan"))])
@pytest.mark.parametrize("page,lens,num_pages", [(7, (90, 120), 20), (16, (200, 300), 21), (24, (200, 300), 14), (16, (1500, 1300), 70)])
@pytest.mark.parametrize("repeated", [False, True])
def test_chunk_scales_that_other_tokens_list(cuda, part, value, page, lens, num_pages, repeated):
    """One token lists a page whose scale is not finite, at an entry where the others list nothing, past the
    union's size too: only its row shows it.  The longest lists are split."""
    b = Batch(page + num_pages, lens, (20, 40), page, 8, 2, 128)
    pool, scales, keys, values = b.pool("fp8")
    picked = b.lists(num_pages, hole=0.3)
    entry = num_pages - 1
    picked[:, :, entry] = -1
    picked[:20][picked[:20] == 1] = -1
    picked[:, :, 2] = -1
    picked[3, 0, entry] = 1  # page 1 of the first sequence: token 3 alone lists it, for kv head 0
    picked[18, 1, 2] = 1     # and token 18, for kv head 1
    if repeated:
        picked[5, 0, :2], picked[19, 1, :2] = 2, 0  # twice
    dirty = scales.copy()
    dirty[b.table[0, 1], :, part] = value
    kw = dict(sm_scale=0.1, kv_scales=torch.from_numpy(dirty).cuda())
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32(picked), *b.meta(), **kw).double().cpu().numpy()
    bad = np.zeros((b.tokens, 8), bool)
    bad[3, :4], bad[18, 4:] = True, True
    assert (~np.isfinite(got).all(-1) == bad).all()
    want = orc.sparse_attention(b.q.double().numpy(), keys, values, picked, b.lens, b.table, b.cu, b.n, 0.1)
    tol = _tolerance(want, b.q, keys, values, num_pages * page, 0.1)
    assert (np.abs(got - want) <= tol)[~bad].all()


@pytest.mark.parametrize("page", [7, 16, 24])
@pytest.mark.parametrize("num_pages", [9, 80])
def test_fp8_chunk_pages_listed_twice_beside_holes(cuda, page, num_pages):
    b = Batch(page, [1400, 1000], [20, 40], page, 8, 2, 64)
    picked = b.lists(num_pages, hole=0.4)
    for t in range(0, 60, 3):
        picked[t, t % 2, [1, 6, 8]] = 2, -1, 2
    _check(b, num_pages, "fp8", picked=picked)


@pytest.mark.parametrize("soft_cap", [None, 20.0, -20.0])
@pytest.mark.parametrize("sm_scale", [1.0, -0.3, 0.0])
def test_scales_and_caps(cuda, soft_cap, sm_scale):
    b = Batch(12, [300, 50], [1, 5], 16, 8, 2, 64)
    _check(b, 10, sm_scale=sm_scale, soft_cap=soft_cap)


def test_scalar_scales(cuda):
    b = Batch(13, [300, 50], [1, 5], 16, 8, 2, 128)
    picked = b.lists(6)
    for kind in ("bf16", "fp8"):
        pool, _, _, _ = b.pool(kind)
        x = pool.double().numpy().reshape(b.total, 16, 2, 2, 128)
        factor = 0.5 if kind == "bf16" else 0.01
        got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32(picked), *b.meta(), sm_scale=0.1, k_scale=factor, v_scale=2.0)
        keys, values = x[:, :, :, 0] * factor, x[:, :, :, 1] * 2.0
        want = orc.sparse_attention(b.q.double().numpy(), keys, values, picked, b.lens, b.table, b.cu, b.n, 0.1)
        assert (np.abs(got.double().cpu().numpy() - want) <= _tolerance(want, b.q, keys, values, 96, 0.1)).all()


def test_rows_without_keys_are_zero(cuda):
    b = Batch(14, [100, 40], [1, 1], 16, 8, 2, 128, spare=1, pad=3)
    picked = b.lists(4)
    picked[0, 1] = -1
    got, _ = _check(b, 4, picked=picked)
    assert (got[0, 4:] == 0).all() and (got[2:] == 0).all()


def test_a_page_listed_twice_counts_twice(cuda):
    b = Batch(15, [100], [1], 16, 4, 1, 64)
    _check(b, 4, picked=np.array([[[2, 5, 2, -1]]]))


def test_nan_and_infinity_outside_the_seen_keys(cuda):
    """Rows past a sequence's end, unlisted pages and the pool's first row hold NaN and infinities."""
    for kind in ("bf16", "fp8"):
        b = Batch(16, [100, 37, 16], [1, 1, 1], 16, 8, 2, 128, pad=1)
        pool, scales, keys, values = b.pool(kind)
        picked = np.full((4, 2, 5), -1)
        picked[0], picked[1, :, :2], picked[2, 0, 0] = [0, 2, -1, 6, 9], [2, 0], 0
        seen = np.zeros((b.total, 16), bool)
        for t, n in enumerate((100, 37, 16)):
            for page in {int(x) for x in picked[t].ravel() if 0 <= x < -(-n // 16)}:
                seen[b.table[t, page], :min(16, n - 16 * page)] = True
        dirty = pool.clone()
        held = dirty.view(torch.uint8) if kind == "fp8" else dirty
        unseen = torch.from_numpy(~seen)
        held[unseen] = 0x7F if kind == "fp8" else float("nan")
        if kind == "bf16":
            held[unseen.nonzero()[::2, 0], unseen.nonzero()[::2, 1]] = float("inf")
        dirty = held.view(pool.dtype)
        args = (i32(picked), *b.meta())
        kw = dict(sm_scale=0.1, kv_scales=None if scales is None else torch.from_numpy(scales).cuda())
        clean = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), *args, **kw)
        got = sparse.sparse_paged_attention(b.q.cuda(), dirty.cuda(), *args, **kw)
        assert torch.isfinite(got).all() and torch.equal(got, clean)


def test_scores_at_the_ends_of_the_range(cuda):
    """Scores of -1e37 alone, of both signs, and ties: the running maximum starts below all of them."""
    b = Batch(17, [64], [1], 16, 2, 1, 64)
    pool, _, keys, values = b.pool()
    held = pool.view(b.total, 16, 1, 2, 64)
    held[:, :, :, 0] = 0
    held[:, :, :, 0, 0] = -1.0
    b.q[:] = 0
    b.q[0, :, 0] = 1e37
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32([[[0, 1, 2, 3]]]), *b.meta(), sm_scale=1.0)
    x = held.double().numpy()
    want = orc.sparse_attention(b.q.double().numpy(), x[:, :, :, 0], x[:, :, :, 1], np.array([[[0, 1, 2, 3]]]), b.lens, b.table,
                                b.cu, b.n, 1.0)
    assert (np.abs(got.double().cpu().numpy() - want) <= 2.0**-8 * np.abs(want) + 5 * 2.0**-15).all()


@pytest.mark.parametrize("size", [1e37, 3e9, -3e9, -1e37])
@pytest.mark.parametrize("scale", [1.0, 0.7])
def test_large_scores_in_chunks(cuda, size, scale):
    """Tied scores of any size and scale: the mean of the values, in tiles of a chunk's tokens too."""
    b = Batch(20, [96], [32], 16, 2, 1, 64)
    pool, _, _, _ = b.pool()
    held = pool.view(b.total, 16, 1, 2, 64)
    held[:, :, :, 0] = 0
    held[:, :, :, 0, 0] = 1.0
    b.q[:] = 0
    b.q[:, :, 0] = size
    picked = np.tile(np.arange(6), (b.tokens, 1, 1))
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32(picked), *b.meta(), sm_scale=scale)
    x = held.double().numpy()
    want = orc.sparse_attention(b.q.double().numpy(), x[:, :, :, 0], x[:, :, :, 1], picked, b.lens, b.table, b.cu, b.n, scale)
    # half a step of the result, and two parts of 2^-17 of each value's weight
    assert (np.abs(got.double().cpu().numpy() - want) <= 2.0**-8 * np.abs(want) + 2.0**-16 * np.abs(x[:, :, :, 1]).max()).all()


def test_whole_lists_equal_the_dense_operator(cuda):
    """With every page listed the dense operator's result, within both operators' roundings."""
    b = Batch(18, [300, 90, 1, 600], [1, 40, 1, 1], 16, 8, 2, 128)
    pool, _, _, _ = b.pool()
    picked = np.tile(np.arange(b.table.shape[1]), (b.tokens, 2, 1))
    lens, table, cu, num = b.meta()
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32(picked), lens, table, cu, num, sm_scale=128**-0.5)
    dense = ops.ragged_paged_attention(b.q.cuda(), pool.cuda(), lens, table, cu, num, sm_scale=128**-0.5)
    assert (got.float() - dense.float()).abs().max().item() <= 2e-2


def test_strided_queries_and_out(cuda):
    b = Batch(19, [500, 64], [1, 20], 16, 8, 2, 128)
    pool, _, _, _ = b.pool()
    pool, picked, meta = pool.cuda(), i32(b.lists(6)), b.meta()
    want = sparse.sparse_paged_attention(b.q.cuda(), pool, picked, *meta, sm_scale=0.1)
    wide = torch.zeros((b.tokens, 12, 160), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:10, 32:] = b.q.cuda()
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = sparse.sparse_paged_attention(wide[:, 2:10, 32:], pool, picked, *meta, sm_scale=0.1, out=out)
    stream.synchronize()
    assert got is out and torch.equal(out, want)


def test_pages_outside_the_pool_are_flagged(cuda):
    sparse.read_error_word(clear=True)
    b = Batch(20, [100], [1], 16, 4, 1, 64)
    pool, _, _, _ = b.pool()
    lens, table, cu, num = b.meta()
    bad = table.clone()
    bad[0, 1], bad[0, 2] = -1, b.total
    got = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32([[[0, 1, 2, 3]]]), lens, bad, cu, num)
    assert sparse.read_error_word(clear=True) == sparse._sparse_lib.ERR_PAGE
    want = sparse.sparse_paged_attention(b.q.cuda(), pool.cuda(), i32([[[0, -1, -1, 3]]]), lens, table, cu, num)
    assert torch.equal(got, want)


def test_same_bits_every_time(cuda):
    b = Batch(21, [3000, 900], [1, 1], 16, 8, 2, 128)
    pool, _, _, _ = b.pool()
    args = (b.q.cuda(), pool.cuda(), i32(b.lists(100)), *b.meta())
    first = sparse.sparse_paged_attention(*args, sm_scale=0.1)
    for _ in range(5):
        assert torch.equal(sparse.sparse_paged_attention(*args, sm_scale=0.1), first)


def test_pools_past_32_bit_byte_offsets(cuda):
    pages, page = 4200, 256
    pool = torch.zeros((pages, page, 16, 128), dtype=torch.bfloat16, device="cuda")  # 4.4 GB
    pool[-1] = torch.randn((page, 16, 128), device="cuda").to(torch.bfloat16)
    q = torch.randn((1, 8, 128), device="cuda").to(torch.bfloat16)
    got = sparse.sparse_paged_attention(q, pool, i32(np.zeros((1, 8, 1))), i32([200]), i32([[pages - 1]]), i32([0, 1]), i32([1]),
                                        sm_scale=0.1)
    kv = pool[-1].double().cpu().numpy().reshape(1, page, 8, 2, 128)
    want = orc.sparse_attention(q.double().cpu().numpy(), kv[:, :, :, 0], kv[:, :, :, 1], np.zeros((1, 8, 1), int), [200],
                                np.array([[0]]), [0, 1], 1, 0.1)
    tol = _tolerance(want, q.cpu(), kv[:, :, :, 0], kv[:, :, :, 1], 256, 0.1)
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
