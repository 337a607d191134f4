"""Refusals of the page allocator, before any launch: no GPU needed."""

import ctypes

import pytest
import torch

from tpu_cake_amd import _sparse_lib, paging


@pytest.fixture(scope="module")
def lib():
    if not _sparse_lib.library_path().exists():
        from tpu_cake_amd import build
        build.build()
    return _sparse_lib.load()


def _shape(**kw):
    return _sparse_lib.RpaPagingShape(**{**dict(num_requests=4, pages_per_seq=8, page_size=16, free_capacity=9, max_tokens=4), **kw})


@pytest.mark.parametrize("bad,message", [
    (dict(num_requests=0), b"non-positive"), (dict(pages_per_seq=0), b"non-positive"), (dict(page_size=-1), b"non-positive"),
    (dict(free_capacity=1 << 30), b"2^30"), (dict(max_tokens=1 << 30), b"2^30"), (dict(max_tokens=-1), b"2^30"),
    (dict(pages_per_seq=1 << 20, page_size=1 << 12), b"int32"), ({}, b"NULL")])
def test_c_entries_refuse(lib, bad, message):
    # distinct fake pointers are never dereferenced; without them the NULL check is the last
    ptrs = [ctypes.c_void_p(256 * (i + 1)) if bad else None for i in range(11)]
    assert lib.rpa_assign_pages(ctypes.byref(_shape(**bad)), *ptrs, None) == -1
    assert message in lib.rpa_sparse_last_error()
    if "max_tokens" not in bad or bad["max_tokens"] != -1:
        assert lib.rpa_release_pages(ctypes.byref(_shape(**bad)), *ptrs[:7], None) == -1
        assert message in lib.rpa_sparse_last_error()


def test_c_entries_refuse_overlap(lib):
    ptrs = [ctypes.c_void_p(256 * (i + 1)) for i in range(11)]
    ptrs[5] = ptrs[0]
    assert lib.rpa_assign_pages(ctypes.byref(_shape()), *ptrs, None) == -1 and b"overlap" in lib.rpa_sparse_last_error()
    assert lib.rpa_assign_pages(None, *ptrs, None) == -1 and b"NULL" in lib.rpa_sparse_last_error()


def _cpu_args():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return [i(4), i(4), i(4, 8), i(9), i(1)]


def test_python_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="GPU device"):
        paging.assign_pages(*_cpu_args(), page_size=16, max_tokens=4)
    a = _cpu_args()
    a[1] = torch.zeros(4, dtype=torch.bool)
    with pytest.raises(ValueError, match="GPU device"):
        paging.release_pages(*a, page_size=16)


def test_separate_refuses_overlapping_outputs():
    a = torch.zeros(10, dtype=torch.int32)
    paging._separate({"x": a[:4]}, {"y": a[4:]})
    with pytest.raises(ValueError, match="x overlaps y"):
        paging._separate({"x": a[:5]}, {"y": a[4:]})
    with pytest.raises(ValueError, match="x overlaps z"):
        paging._separate({"x": a[:5], "z": a[4:]}, {})


@pytest.mark.parametrize("change,message", [
    (dict(cached=torch.zeros(5, dtype=torch.int32)), "expected"), (dict(cached=torch.zeros(4, dtype=torch.int64)), "dtype"),
    (dict(count=torch.zeros(2, dtype=torch.int32)), "expected"), (dict(page_size=0), "page_size"),
    (dict(page_size=1.5), "page_size"), (dict(page_size=1 << 29), "int32")])
def test_check_refuses(monkeypatch, change, message):
    monkeypatch.setattr(paging, "_require_cuda", lambda name, t: None)
    table = torch.zeros((4, 8), dtype=torch.int32)
    named = {"page_table": (table, (None, None), torch.int32),
             "cached_lens": (change.get("cached", torch.zeros(4, dtype=torch.int32)), (4,), torch.int32),
             "free_count": (change.get("count", torch.zeros(1, dtype=torch.int32)), (1,), torch.int32)}
    with pytest.raises(ValueError, match=message):
        paging._check(named, table, 4, change.get("page_size", 16))
