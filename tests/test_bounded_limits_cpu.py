"""Sizes near the ends of 32 bits, which the calls over a bounded cache and its neighbours refuse before any launch: no GPU needed."""

import ctypes

import pytest

from tpu_cake_amd import _bounded_lib, _sparse_lib

FAKE = [ctypes.c_void_p((i + 1) << 44) for i in range(16)]  # far apart and never dereferenced: every call here is refused


@pytest.fixture(scope="module", params=["bounded", "sparse"])
def libs(request):
    binding = {"bounded": _bounded_lib, "sparse": _sparse_lib}[request.param]
    if not binding.library_path().exists():
        from tpu_cake_amd import build
        build.build()
    return request.param, binding.load()


@pytest.mark.parametrize("pages", [1 << 27, 1 << 28, (1 << 29) + 5, 2**31 - 1])
def test_outputs_in_the_scales_of_many_pages(libs, pages):
    """The scales' bytes pass 32 bits from 2^28 pages on: an output within them is refused all the same."""
    name, lib = libs
    inside = ctypes.c_void_p(FAKE[2].value + 16 * pages - 256)  # 8 bytes a page and kv head, two heads: their end
    if name == "bounded":
        shape = _bounded_lib.RpaWeighShape(4, 8, 2, 128, pages, 1, 4, 8, _bounded_lib.RPA_KV_FP8_E4M3, 0, 1024, 128)
        options = _bounded_lib.RpaWeighOptions(1.0, 0.0, 1.0, 1.0, 1.0)
        rc = lib.rpa_weighed_attention(ctypes.byref(shape), ctypes.byref(options), *FAKE[:10], inside, FAKE[11], 1 << 42, None)
        error = lib.rpa_bounded_last_error()
    else:
        shape = _sparse_lib.RpaSparseShape(4, 8, 2, 128, pages, 1, 4, 8, _sparse_lib.RPA_KV_FP8_E4M3, 6, 1024, 128)
        options = _sparse_lib.RpaSparseOptions(1.0, 0.0, 1.0, 1.0)
        rc = lib.rpa_sparse_paged_attention(ctypes.byref(shape), ctypes.byref(options), *FAKE[:8], inside, FAKE[9], 1 << 42, None)
        error = lib.rpa_sparse_last_error()
    assert rc == -1 and b"out overlaps kv_scales" in error, (rc, error)


@pytest.mark.parametrize("entries", [(1 << 30, 1, 1), (1 << 15, 1 << 15, 1), (1 << 14, 1 << 14, 4), (2**31 - 1, 1, 1), ((1 << 30) - 63, 1, 1)])
def test_moves_of_2_to_the_32_threads(entries):
    """Four threads an entry: HIP takes fewer than 2^32 along a dimension, and the call says so itself."""
    lists, moves, heads = entries
    shape = _bounded_lib.RpaMoveShape(lists, moves, heads, 128, 64, 16, 0)
    lib = _bounded_lib.load()
    assert lib.rpa_move_rows(ctypes.byref(shape), FAKE[0], None, *FAKE[2:5], None) == -2
    assert b"one launch" in lib.rpa_bounded_last_error()


@pytest.mark.parametrize("seqs,heads,page,pages,width", [(256, 8, 16, 40000, 8192), (64, 8, 16, 8500, 8192), (4096, 1, 64, 1 << 14, 1 << 14),
                                                         (3, 8, 16, 50000, 7700), (1, 1, 1, 32769, 40000), (2000, 2, 16, 64, 1 << 17)])
def test_choose_workspaces_follow_the_pool(seqs, heads, page, pages, width):
    """Keys of long sequences: 10 bytes a row and kv head and what a list's last block rounds up (4095 of 32769 rows at most),
    of as many rows as the pool has, and 16 bytes a list; the table's width counts for nothing."""
    shape = _bounded_lib.RpaChooseShape(seqs, width, heads, pages, page, 2048, 2111, 4, 256, 64)
    size = _bounded_lib.load().rpa_choose_workspace_size(ctypes.byref(shape))
    assert 0 < size <= 41000 / 4096 * 1.125 * pages * page * heads + 16 * seqs * heads + 64
