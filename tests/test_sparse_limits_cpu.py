"""The largest sizes that the sparse entry points and the paging calls refuse before any launch: no GPU needed."""

import ctypes

import pytest

from tpu_cake_amd import _sparse_lib

FAKE = [ctypes.c_void_p((i + 1) << 44) for i in range(16)]  # far apart and never dereferenced: every call here is refused
MOST = 2**31 - 2**16 - 1


@pytest.fixture(scope="module")
def lib():
    if not _sparse_lib.library_path().exists():
        from tpu_cake_amd import build
        build.build()
    return _sparse_lib.load()


def _sparse(**kw):
    return _sparse_lib.RpaSparseShape(**{**dict(num_tokens=4, num_q_heads=8, num_kv_heads=2, head_dim=128, total_pages=64, page_size=1,
                                                max_num_seqs=4, pages_per_seq=8, kv_dtype=0, num_pages=6, q_token_stride=1024,
                                                q_head_stride=128), **kw})


def _paging(**kw):
    return _sparse_lib.RpaPagingShape(**{**dict(num_requests=4, pages_per_seq=8, page_size=1, free_capacity=9, max_tokens=16), **kw})


OPTIONS = _sparse_lib.RpaSparseOptions(1.0, 0.0, 1.0, 1.0)


def _select(lib, shape, need=1 << 60):
    return lib.rpa_select_pages(ctypes.byref(shape), 1, 1, *FAKE[:9], need, None)


def _attend(lib, shape, need=1 << 60):
    return lib.rpa_sparse_paged_attention(ctypes.byref(shape), ctypes.byref(OPTIONS), *FAKE[:2], None, *FAKE[3:10], need, None)


@pytest.mark.parametrize("field", ["pages_per_seq", "num_pages"])
def test_lists_and_tables_that_an_index_would_pass(lib, field):
    """Loops over a row step by up to 2^15 entries: at the ends of 32 bits the index would wrap below the row."""
    for count in (MOST + 1, 2**31 - 1):
        shape = _sparse(**{field: count})
        assert _select(lib, shape) == -2 and b"2^31 - 2^16 - 1" in lib.rpa_sparse_last_error()
        assert _attend(lib, shape) == -2 and b"2^31 - 2^16 - 1" in lib.rpa_sparse_last_error()
        assert lib.rpa_select_workspace_size(ctypes.byref(shape)) == 0
    assert lib.rpa_select_workspace_size(ctypes.byref(_sparse(pages_per_seq=MOST))) > 0


def test_launches_of_2_to_the_32_threads(lib):
    """HIP takes fewer along a dimension; calls that would need more say so."""
    rows = _sparse(num_tokens=1 << 22, max_num_seqs=1 << 22, num_kv_heads=1, num_q_heads=1)  # a workgroup a row
    assert _select(lib, rows) == -2 and b"one launch" in lib.rpa_sparse_last_error()
    rows = _sparse(num_tokens=1 << 24, max_num_seqs=1 << 24, num_kv_heads=1, num_q_heads=1)
    assert _attend(lib, rows) == -2 and b"one launch" in lib.rpa_sparse_last_error()
    tiles = _sparse(num_tokens=1 << 26, num_kv_heads=2, num_q_heads=2)
    assert _select(lib, tiles) == -2 and b"one launch" in lib.rpa_sparse_last_error()
    assert _attend(lib, tiles) == -2 and b"one launch" in lib.rpa_sparse_last_error()
    tokens = _sparse_lib.RpaAppendShape((1 << 30) - 1, 8, 128, 64, 16, 0, 1024, 128, 1024, 128)
    assert lib.rpa_append_kv(ctypes.byref(tokens), *FAKE[:4], None, 1.0, 1.0, *FAKE[5:7], None) == -2
    assert b"one launch" in lib.rpa_sparse_last_error()
    assert lib.rpa_release_pages(ctypes.byref(_paging(num_requests=1 << 28)), *FAKE[:7], None) == -2
    assert b"one launch" in lib.rpa_sparse_last_error()


def test_split_choices_stay_below_them_in_turns(lib):
    """Tiny rows whose queries pass the LDS, so that the workspace alone would take 2^22 of them at once."""
    shape = _sparse(num_tokens=20000, max_num_seqs=20000, num_kv_heads=1024, num_q_heads=1024 * 256, head_dim=256)
    rows = lib.rpa_select_workspace_size(ctypes.byref(shape)) // 64  # 16 keys of 4 bytes each
    assert 0 < rows * 1024 < 2**32 and rows % 1024 == 0


@pytest.mark.parametrize("field", ["num_requests", "pages_per_seq"])
def test_requests_that_an_index_would_pass(lib, field):
    for count in (MOST + 1, 2**31 - 1):
        shape = ctypes.byref(_paging(**{field: count}))
        assert lib.rpa_assign_pages(shape, *FAKE[:11], None) == -2 and b"2^31 - 2^16 - 1" in lib.rpa_sparse_last_error()
        assert lib.rpa_release_pages(shape, *FAKE[:7], None) == -2 and b"2^31 - 2^16 - 1" in lib.rpa_sparse_last_error()
