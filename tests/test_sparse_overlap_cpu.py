"""Outputs that lie in what a call reads, or in another output, are refused: no GPU needed."""

import ctypes

import pytest
import torch

from tpu_cake_amd import _sparse_lib, sparse

# T 6, Hq 8, Hkv 2, D 128, pools of 64 pages of 16, 4 sequences of 8 pages, lists of 6
T, HQ, HKV, D, P, S, N, PPS, K = 6, 8, 2, 128, 64, 16, 4, 8, 6


@pytest.fixture(scope="module")
def lib():
    if not _sparse_lib.library_path().exists():
        from tpu_cake_amd import build
        build.build()
    return _sparse_lib.load()


def _far(count):
    return [(i + 1) << 40 for i in range(count)]  # never dereferenced: every call here is refused


def _refused(lib, call, text):
    assert call == -1 and text in lib.rpa_sparse_last_error(), lib.rpa_sparse_last_error()


def _shape(token=HQ * D, head=D, kv_dtype=0):
    return ctypes.byref(_sparse_lib.RpaSparseShape(T, HQ, HKV, D, P, S, N, PPS, kv_dtype, K, token, head))


def _select(lib, ptrs, shape, out):
    p = [ctypes.c_void_p(x) for x in ptrs]
    return lib.rpa_select_pages(shape, 1, 1, *p[:7], ctypes.c_void_p(out), p[8], 1 << 30, None)


def _attend(lib, ptrs, shape, out):
    p = [ctypes.c_void_p(x) for x in ptrs]
    options = _sparse_lib.RpaSparseOptions(1.0, 0.0, 1.0, 1.0)
    return lib.rpa_sparse_paged_attention(shape, ctypes.byref(options), *p[:8], ctypes.c_void_p(out), p[9], 1 << 30, None)


@pytest.mark.parametrize("which,name,size", [(0, b"q", T * HQ * D * 2), (1, b"bounds", P * HKV * 2 * D), (2, b"exponents", P * HKV),
                                             (3, b"kv_lens", 4 * N), (4, b"page_indices", 4 * N * PPS), (5, b"cu_q_lens", 4 * (N + 1)),
                                             (6, b"num_seqs", 4)])
def test_select(lib, which, name, size):
    ptrs, own = _far(10), T * HKV * K * 4
    for out in (ptrs[which], ptrs[which] + size - 1 & ~3, ptrs[which] - own + 4):
        _refused(lib, _select(lib, ptrs, _shape(), out), b"selected_pages overlaps " + name)


@pytest.mark.parametrize("which,name,size", [(0, b"q", T * HQ * D * 2), (1, b"kv_pages", P * S * 2 * HKV * D), (2, b"kv_scales", P * HKV * 8),
                                             (3, b"selected_pages", T * HKV * K * 4), (4, b"kv_lens", 4 * N),
                                             (5, b"page_indices", 4 * N * PPS), (6, b"cu_q_lens", 4 * (N + 1)), (7, b"num_seqs", 4)])
def test_attention(lib, which, name, size):
    ptrs, own = _far(10), T * HQ * D * 2
    for out in (ptrs[which], ptrs[which] + size - 1 & ~15, ptrs[which] - own + 16):
        _refused(lib, _attend(lib, ptrs, _shape(kv_dtype=1), out), b"out overlaps " + name)


def test_paging(lib):
    shape = ctypes.byref(_sparse_lib.RpaPagingShape(4, 8, 16, 9, 12))
    sizes = [16, 16, 128, 36, 4, 16, 20, 4, 48, 48, 4]  # inputs 0 to 4, outputs 5 to 10
    call = lambda p: lib.rpa_assign_pages(shape, *[ctypes.c_void_p(x) for x in p], None)  # noqa: E731
    for out in range(5, 11):
        for other in (x for x in range(11) if x != out):
            for at in (sizes[other] - 4, 4 - sizes[out]):
                p = _far(11)
                p[out] = p[other] + at
                _refused(lib, call(p), b" overlaps ")
    sizes = [16, 4, 128, 36, 4, 16, 4]  # outputs 5 and 6
    call = lambda p: lib.rpa_release_pages(shape, *[ctypes.c_void_p(x) for x in p], None)  # noqa: E731
    for out in (5, 6):
        for other in (x for x in range(7) if x != out):
            for at in ((sizes[other] - 1) & ~3, 4 - sizes[out]):
                p = _far(7)
                p[out] = p[other] + at
                _refused(lib, call(p), b" overlaps ")


def _view(*shape, at=0, stride=None, of):
    got = of.view(torch.bfloat16)[at:]
    return got.as_strided(shape, stride or torch.empty(shape, device="meta").stride())


@pytest.mark.parametrize("q,out,refused", [
    (dict(at=0), 0, True), (dict(at=0), 8, True), (dict(at=0), T * HQ * D - 1, True), (dict(at=0), T * HQ * D, False),
    (dict(at=T * HQ * D), 0, False), (dict(at=T * HQ * D - 8), 0, True),
    # slices of a projection's rows: behind the last token's slice and before the first
    (dict(at=0, stride=(12 * D * HQ, D, 1)), 5 * 12 * D * HQ + HQ * D, False), (dict(at=0, stride=(12 * D * HQ, D, 1)), HQ * D, False),
    (dict(at=0, stride=(12 * D * HQ, D, 1)), HQ * D - 8, True), (dict(at=0, stride=(12 * D * HQ, D, 1)), 6 * D * HQ + 8, True),
    # heads before tokens
    (dict(at=0, stride=(D, T * D, 1)), 8, True), (dict(at=0, stride=(D, T * D, 1)), T * HQ * D, False),
    (dict(at=0, stride=(D, 0, 1)), T * D, False), (dict(at=0, stride=(D, 0, 1)), T * D - 8, True)])
def test_strided_queries(lib, q, out, refused):
    """The binding's check and the library's agree."""
    memory = torch.zeros(100 * T * HQ * D, dtype=torch.bfloat16)
    rows, out = _view(T, HQ, D, of=memory, **q), _view(T, HQ, D, at=out, of=memory)
    try:
        sparse._separate("out", out, {"q": rows})
        assert not refused
    except ValueError as e:
        assert refused and "out overlaps q" in str(e)
    if refused and out.data_ptr() % 16 == 0 and rows.stride(1) % 8 == 0:
        ptrs = _far(10)
        ptrs[0] = rows.data_ptr()
        _refused(lib, _attend(lib, ptrs, _shape(rows.stride(0), rows.stride(1), 1), out.data_ptr()), b"out overlaps q")


def test_entry_points_refuse(monkeypatch):
    monkeypatch.setattr(sparse, "_require_cuda", lambda name, t: None)
    real = sparse._tensor
    monkeypatch.setattr(sparse, "_tensor", lambda *a, **kw: real(*a))
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    memory = torch.zeros(64 * HQ * D, dtype=torch.bfloat16)
    q, pool = _view(T, HQ, D, of=memory), torch.zeros((P, S, 2 * HKV, D), dtype=torch.bfloat16)
    meta = (i(N), i(N, PPS), i(N + 1), i(1))
    with pytest.raises(ValueError, match="out overlaps q"):
        sparse.sparse_paged_attention(q, pool, i(T, HKV, K), *meta, out=_view(T, HQ, D, at=8, of=memory))
    with pytest.raises(ValueError, match="out overlaps kv_pages"):
        sparse.sparse_paged_attention(q, pool, i(T, HKV, K), *meta, out=pool.view(-1)[256:256 + q.numel()].view(q.shape))
    lists = i(2 * T, HKV, K)
    with pytest.raises(ValueError, match="out overlaps kv_lens"):
        sparse.select_pages(q, sparse.make_page_index(pool), lists.view(-1)[9:9 + N], *meta[1:], page_size=S, num_pages=K, out=lists[:T])
