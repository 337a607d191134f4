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


@pytest.mark.parametrize("field", ["num_requests", "pages_per_seq"])
def test_requests_that_an_index_would_pass(lib, field):
    for count in (MOST + 1, 2**31 - 1):
        shape = ctypes.byref(_paging(**{field: count}))
        assert lib.rpa_assign_pages(shape, *FAKE[:11], None) == -2 and b"2^31 - 2^16 - 1" in lib.rpa_sparse_last_error()
        assert lib.rpa_release_pages(shape, *FAKE[:7], None) == -2 and b"2^31 - 2^16 - 1" in lib.rpa_sparse_last_error()
