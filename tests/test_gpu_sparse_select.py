"""select_pages: the chosen pages equal the oracle's, in every form of the launch."""

import numpy as np
import pytest
import torch

from oracle import sparse_oracle as orc
from sparse_cases import Batch, i32
from tpu_cake_amd import sparse

pytestmark = pytest.mark.gpu


def _check(b, num_pages, *, sink=1, recent=1, index=None):
    bounds, exps = index or b.index()
    got = sparse.select_pages(b.q.cuda(), sparse.PageIndex(torch.from_numpy(bounds).cuda(), torch.from_numpy(exps).cuda()),
                              *b.meta(), page_size=b.page_size, num_pages=num_pages, sink_pages=sink, recent_pages=recent)
    want = orc.select_pages(b.q.double().numpy(), bounds, exps, b.lens, b.table, b.cu, b.n, b.page_size, num_pages, sink, recent)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    return got


@pytest.mark.parametrize("group,hkv", [(1, 8), (2, 1), (3, 2), (5, 1), (8, 4), (16, 2), (17, 1), (40, 2)])
@pytest.mark.parametrize("dim", [128, 64, 256, 32, 40, 96])
def test_decode_rows(cuda, group, hkv, dim):
    b = Batch(group + dim, [1, 15, 16, 17, 900, 0, 3000], [1, 1, 1, 1, 1, 0, 1], 16, group * hkv, hkv, dim, spare=2, pad=2)
    _check(b, 5)


@pytest.mark.parametrize("group,hkv", [(1, 2), (3, 1), (4, 2), (8, 1), (16, 1), (20, 1)])
@pytest.mark.parametrize("num_pages,sink,recent", [(1, 0, 1), (1, 0, 0), (7, 2, 3), (16, 1, 1), (64, 64, 0)])
def test_chunks(cuda, group, hkv, num_pages, sink, recent):
    b = Batch(group, [40, 700, 5, 33, 640], [40, 90, 1, 1, 17], 8, group * hkv, hkv, 128, pad=5)
    _check(b, num_pages, sink=sink, recent=recent)


@pytest.mark.parametrize("dim,group", [(64, 4), (256, 8), (96, 2)])
def test_chunks_of_other_dims(cuda, dim, group):
    _check(Batch(dim, [300, 1000], [100, 33], 4, group * 2, 2, dim), 12)


@pytest.mark.parametrize("pages,decode", [(513, True), (2049, True), (8193, True), (15000, True), (600, False), (2049, False),
                                          (33000, True), (70001, True)])
def test_long_rows(cuda, pages, decode):
    """Every number of keys a thread holds, the split form, and rows past its registers."""
    q_lens = [1, 1, 1] if decode else [3, 9, 6]
    b = Batch(pages, [pages, pages // 2, 300], q_lens, 1, 4, 2, 32)
    _check(b, 40)


def test_many_rows_of_long_tables(cuda):
    """Decode batches wide enough to keep the keys on chip."""
    b = Batch(2, [1500] * 130, [1] * 130, 1, 2, 2, 32)
    _check(b, 9)


def test_split_form_in_turns(cuda):
    """More rows than the workspace holds at once: 256 MiB, 512 kB a token and its 2 heads."""
    b = Batch(4, [65000], [600], 1, 2, 2, 32)
    bounds, exps = b.index()
    got = sparse.select_pages(b.q.cuda(), sparse.PageIndex(torch.from_numpy(bounds).cuda(), torch.from_numpy(exps).cuda()),
                              *b.meta(), page_size=1, num_pages=6).cpu().numpy()
    rows = [0, 15, 16, 300, 511, 512, 513, 599]  # the oracle's time
    for t in rows:
        want = orc.select_pages(b.q[t:t + 1].double().numpy(), bounds, exps, np.array([65000 - 599 + t]), b.table, np.array([0, 1]),
                                1, 1, 6)
        np.testing.assert_array_equal(got[t], want[0], err_msg=str(t))


def test_ties_go_to_the_earlier_page(cuda):
    b = Batch(1, [4000, 90], [1, 30], 2, 8, 2, 64)
    bounds, exps = b.index()
    bounds[:] = bounds[0]
    exps[:] = -5
    got = _check(b, 20, index=(bounds, exps))
    assert got[0, 0].tolist() == list(range(19)) + [1999]
    bounds[:, :, :, :] = 0  # scores of zero, and of both signs
    bounds[::3] = 1
    bounds[1::3] = -1
    _check(b, 20, index=(bounds, exps))


@pytest.mark.parametrize("num_pages", [34, 35, 64, 100, 193, 194, 250, 700])
@pytest.mark.parametrize("tied", [False, True])
def test_wide_lists(cuda, num_pages, tied):
    """Lists of every way that a wave or a workgroup bounds its candidates, also where all of them tie."""
    b = Batch(num_pages, [1200, 400, 380, 1400, 130], [20, 9, 1, 1, 30], 2, 4, 2, 64)
    decode = Batch(num_pages, [2000, 1100, 700, 380], [1] * 4, 2, 4, 2, 64)
    for rows in (b, decode):
        bounds, exps = rows.index()
        if tied:
            bounds[:, :, :, 2:] = 0  # scores of few different values
            bounds //= 50
            exps[:] = -5
        _check(rows, num_pages, index=(bounds, exps))


def test_exponents_at_their_ends(cuda):
    b = Batch(3, [800, 500], [1, 40], 4, 4, 2, 128)
    bounds, exps = b.index(spread=(-100, 101))
    exps[::5], exps[1::5] = -128, 127  # nothing append_kv writes: taken as -100 and 100
    clipped = np.clip(exps, -100, 100)
    got = sparse.select_pages(b.q.cuda(), sparse.PageIndex(torch.from_numpy(bounds).cuda(), torch.from_numpy(exps).cuda()),
                              *b.meta(), page_size=4, num_pages=10)
    want = orc.select_pages(b.q.double().numpy(), bounds, clipped, b.lens, b.table, b.cu, b.n, 4, 10)
    np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_extreme_queries(cuda):
    b = Batch(7, [600, 700, 200, 300, 400], [1, 1, 1, 1, 1], 4, 8, 2, 64)
    b.q[0] = 0
    b.q[1, 2, 5], b.q[1, 6, 1] = float("inf"), float("-inf")
    b.q[2, 0, :9] = float("nan")
    b.q[3] *= 1e-30
    b.q[4] *= 1e30
    _check(b, 11)


def test_strided_queries_out_and_stream(cuda):
    b = Batch(9, [500, 64, 2000], [1, 20, 1], 16, 8, 2, 128)
    bounds, exps = b.index()
    index = sparse.PageIndex(torch.from_numpy(bounds).cuda(), torch.from_numpy(exps).cuda())
    wide = torch.zeros((b.tokens, 12, 160), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:10, 32:] = b.q.cuda()
    want = orc.select_pages(b.q.double().numpy(), bounds, exps, b.lens, b.table, b.cu, b.n, 16, 6)
    out = torch.empty((b.tokens, 2, 6), dtype=torch.int32, device="cuda")
    meta = b.meta()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = sparse.select_pages(wide[:, 2:10, 32:], index, *meta, page_size=16, num_pages=6, out=out)
    stream.synchronize()
    assert got is out
    np.testing.assert_array_equal(out.cpu().numpy(), want)


def test_bad_pages_and_lengths_are_flagged(cuda):
    sparse.read_error_word(clear=True)
    b = Batch(11, [400], [1], 4, 4, 2, 64)
    bounds, exps = b.index()
    index = sparse.PageIndex(torch.from_numpy(bounds).cuda(), torch.from_numpy(exps).cuda())
    lens, table, cu, num = b.meta()
    bad = table.clone()
    bad[0, 7], bad[0, 9] = -3, b.total
    got = sparse.select_pages(b.q.cuda(), index, lens, bad, cu, num, page_size=4, num_pages=8)
    assert sparse.read_error_word(clear=True) == sparse._sparse_lib.ERR_PAGE
    assert ((got >= 0) & (got < 100)).all()
    got = sparse.select_pages(b.q.cuda(), index, lens + 10**6, table, cu, num, page_size=4, num_pages=8)
    assert sparse.read_error_word(clear=True) == sparse._sparse_lib.ERR_LEN
    assert int(got.max()) == table.shape[1] - 1
    got = sparse.select_pages(b.q.cuda(), index, lens - 400, table, cu, num, page_size=4, num_pages=8)  # q_len > kv_len
    assert (got == -1).all() and sparse.read_error_word() == 0


def test_many_sequences_find_their_tokens(cuda):
    rng = np.random.default_rng(5)
    q_lens = rng.integers(0, 4, 5000)
    lens = q_lens + rng.integers(0, 30, 5000)
    b = Batch(6, lens, q_lens, 4, 2, 1, 32, pad=3)
    _check(b, 3)
