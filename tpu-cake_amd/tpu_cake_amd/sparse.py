"""Sparse attention over a paged K/V pool: append, choice of pages, attention over the chosen ones.

Beside ``ops.ragged_paged_attention`` and over its tensors (``kv_pages``, ``kv_lens``,
``page_indices``, ``cu_q_lens``, ``num_seqs``): where the dense operator reads every key of a
sequence, here each token and kv head reads the keys of ``num_pages`` pages.

* ``append_kv`` writes a step's new keys and values to the slots that ``paging.assign_pages`` gave
  them, and keeps the pool's **page index**: for each page and kv head the largest and smallest
  value of every dimension of the page's keys, 2 * head_dim bytes.
* ``select_pages`` estimates the highest score that a page's keys can have for a token, from the index
  alone, and chooses the pages with the highest estimates; the first and the newest pages are always
  among them.
* ``sparse_paged_attention`` attends to the keys of the listed pages, up to the token's position.

Decode rows (one token a sequence), prompt chunks and mixes of them are one call each.  All tensors
are torch tensors on one GPU; ``q``, ``k`` and ``v`` may be slices of a larger tensor (any token and
head strides that keep rows 16-byte aligned), the others are contiguous.  Calls run on torch's
current stream, take what scratch they need from torch's allocator, and may be captured into graphs.
"""

from __future__ import annotations

import ctypes
import typing

import torch

from . import _sparse_lib
from ._sparse_lib import read_error_word  # noqa: F401
from .ops import _KV_DTYPES, _current_stream, _get_device, _require_cuda


class PageIndex(typing.NamedTuple):
    """What the choice of pages reads of a pool: a bound ``b`` of a page stands for ``b * 2**exponent``."""

    bounds: torch.Tensor     # i8[pages, Hkv, 2, D]: of every dimension the largest, then the smallest value
    exponents: torch.Tensor  # i8[pages, Hkv]


def make_page_index(kv_pages: torch.Tensor) -> PageIndex:
    """An index for ``kv_pages``, to be filled by ``append_kv`` from the pool's first row on."""
    pages, _, combined, dim = kv_pages.shape
    return PageIndex(torch.zeros((pages, combined // 2, 2, dim), dtype=torch.int8, device=kv_pages.device),
                     torch.zeros((pages, combined // 2), dtype=torch.int8, device=kv_pages.device))


# what passed the checks -> the call's structs; signatures of different entry points differ in length
_plans: dict[tuple, tuple] = {}


def _keep(sig: tuple, plan: tuple) -> tuple:
    if len(_plans) > 256:
        _plans.clear()
    _plans[sig] = plan
    return plan


def _tensor(name: str, t, dtype, shape, device, *, rows: bool = False) -> None:
    """Checks a tensor; ``rows``: any strides whose rows stay 16-byte aligned."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if rows:
        if t.device.type != "cuda":
            raise ValueError(f"{name} must be on a GPU device, got {t.device}")
    else:
        _require_cuda(name, t)
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} dtype {t.dtype} must be {dtype}")
    if t.dim() != len(shape) or any(want is not None and want != got for want, got in zip(shape, t.shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if rows and t.numel() and (t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.stride(0) < 0 or t.stride(1) < 0):
        raise ValueError(f"{name} must have contiguous rows and strides of a multiple of 8 values, got {t.stride()}")


def _pool(kv_pages) -> tuple[int, int, int, int, int]:
    """(pages, page size, kv heads, head dim, kv dtype code) of a pool."""
    if not isinstance(kv_pages, torch.Tensor):
        raise TypeError("kv_pages must be a torch.Tensor")
    if kv_pages.dim() != 4 or kv_pages.shape[2] % 2 or kv_pages.shape[2] == 0:
        raise ValueError(f"kv_pages must be [pages, page_size, 2 * kv heads, head_dim], got {tuple(kv_pages.shape)}")
    code = _KV_DTYPES.get(kv_pages.dtype)
    if code is None:
        raise ValueError(f"kv_pages dtype {kv_pages.dtype} is not bf16 or fp8-e4m3")
    _require_cuda("kv_pages", kv_pages)
    return kv_pages.shape[0], kv_pages.shape[1], kv_pages.shape[2] // 2, kv_pages.shape[3], code


def _scales(kv_scales, k_scale, v_scale, pages: int, heads: int, code: int, device) -> None:
    for name, x in (("k_scale", k_scale), ("v_scale", v_scale)):
        if not (x is None or isinstance(x, float)):
            raise ValueError(f"{name}={x!r} must be a float or None")
    if kv_scales is None:
        return
    if code != _sparse_lib.RPA_KV_FP8_E4M3:
        raise ValueError("kv_scales requires fp8 kv_pages")
    _tensor("kv_scales", kv_scales, torch.float32, (pages, heads, 2), device)
    if k_scale is not None or v_scale is not None:
        raise ValueError("pass either per-page kv_scales or scalar k_scale/v_scale, not both")


def _index(index, pages, heads, dim, device) -> PageIndex:
    if not (isinstance(index, tuple) and len(index) == 2):
        raise TypeError("index must be a PageIndex")
    _tensor("index.bounds", index[0], torch.int8, (pages, heads, 2, dim), device)
    _tensor("index.exponents", index[1], torch.int8, (index[0].shape[0], index[0].shape[1]), index[0].device)
    return index


def _blocks(t: torch.Tensor) -> tuple[int, int, int, int]:
    """A tensor's memory as (first byte, bytes of a block, blocks, bytes from one to the next): one block if contiguous,
    else (rows [T, H, D]) what lies within the larger stride."""
    size = t.element_size()
    if t.is_contiguous():
        return t.data_ptr(), t.numel() * size, 1, 0
    (inner, count), (outer, blocks) = sorted(((t.stride(0), t.shape[0]), (t.stride(1), t.shape[1])))
    return t.data_ptr(), ((count - 1) * inner + t.shape[2]) * size, blocks, outer * size


def _separate(name: str, out: torch.Tensor, ins: dict) -> None:
    """Refuses an output whose memory an input has a part of: workgroups run in no order."""
    for other, t in ins.items():
        if t is None or not t.numel() or not out.numel():
            continue
        first, size, blocks, step = _blocks(t)
        start = out.data_ptr() - first
        behind = 0 if start < size else (start - size) // step + 1 if step else blocks  # the first that ends after out begins
        if behind < blocks and behind * step < start + out.numel() * out.element_size():
            raise ValueError(f"{name} overlaps {other}: outputs need memory of their own")


def preflight_append(slot_mapping: torch.Tensor, kv_pages: torch.Tensor) -> None:
    """Host check of what ``append_kv`` takes for granted: every slot is -1 or a row of the pool, no row
    is written twice, and the new rows of a page are consecutive tokens at consecutive slots.  Reads
    ``slot_mapping`` on the host; slots of ``paging.assign_pages`` over distinct pages pass."""
    page_size, rows = kv_pages.shape[1], kv_pages.shape[0] * kv_pages.shape[1]
    slots = slot_mapping.detach().cpu().to(torch.int64)
    if bool(((slots < -1) | (slots >= rows)).any()):
        raise ValueError(f"slot_mapping holds slots outside [-1, {rows})")
    live = slots >= 0
    used = slots[live]
    if used.numel() != torch.unique(used).numel():
        raise ValueError("slot_mapping writes a row twice")
    follows = torch.zeros_like(live)
    follows[1:] = live[1:] & live[:-1] & (slots[1:] == slots[:-1] + 1)
    first = slots[live & ~(follows & (slots % page_size != 0))] // page_size
    if first.numel() != torch.unique(first).numel():
        raise ValueError("the new rows of a page must be consecutive tokens at consecutive slots")


def append_kv(
    k: torch.Tensor,             # bf16 [T, Hkv, D]
    v: torch.Tensor,             # bf16 [T, Hkv, D]
    kv_pages: torch.Tensor,      # bf16 | float8_e4m3fn | uint8 (e4m3 codes) [pages, page_size, 2*Hkv, D], written
    slot_mapping: torch.Tensor,  # i32[T]: page * page_size + row, -1: no row
    *,
    kv_scales: torch.Tensor | None = None,  # f32 [pages, Hkv, 2]: the fp8 pool's K and V scales, as they stand
    k_scale: float | None = None,           # or the whole fp8 pool's
    v_scale: float | None = None,
    index: PageIndex | None = None,         # the pool's page index, updated
) -> None:
    """Writes each token's key and value rows to its slot, and the page index with them.

    fp8 pools hold e4m3(x / scale), saturated at +-448, with the scale that ``kv_scales`` already holds
    for the slot's page and head.  Bounds are of the keys as the pool then holds them.  A page whose row
    0 is written starts its bounds anew and other pages' widen, so the index stays that of the page's
    keys while pages are filled from row 0 on; rows written again without their page's row 0 (a
    sequence that was cut back) leave bounds that are still bounds, but wider than they need be.

    Slots outside the pool are skipped and set ``ERR_SLOT`` in the error word.  The other slots have to
    differ and the new rows of one page have to be consecutive tokens, as ``paging.assign_pages`` lays
    them out; ``preflight_append`` checks it on the host.
    """
    # what the checks go by: written out, as a call costs less than a helper's calls would
    sig = (k.shape, k.dtype, k.get_device(), k.stride(), v.shape, v.dtype, v.get_device(), v.stride(),
           kv_pages.shape, kv_pages.dtype, kv_pages.get_device(), kv_pages.is_contiguous(),
           slot_mapping.shape, slot_mapping.dtype, slot_mapping.get_device(), slot_mapping.is_contiguous(),
           None if kv_scales is None else (kv_scales.shape, kv_scales.dtype, kv_scales.get_device(), kv_scales.is_contiguous()),
           k_scale, v_scale,
           None if index is None else (index[0].shape, index[0].dtype, index[0].get_device(), index[0].is_contiguous(),
                                       index[1].shape, index[1].dtype, index[1].get_device(), index[1].is_contiguous()))
    plan = _plans.get(sig)
    if plan is None:
        pages, page_size, heads, dim, code = _pool(kv_pages)
        device = kv_pages.device
        _tensor("k", k, torch.bfloat16, (None, heads, dim), device, rows=True)
        _tensor("v", v, torch.bfloat16, (k.shape[0], heads, dim), device, rows=True)
        _tensor("slot_mapping", slot_mapping, torch.int32, (k.shape[0],), device)
        _scales(kv_scales, k_scale, v_scale, pages, heads, code, device)
        if code != _sparse_lib.RPA_KV_FP8_E4M3 and (k_scale is not None or v_scale is not None):
            raise ValueError("k_scale and v_scale require fp8 kv_pages")
        for name, x in (("k_scale", k_scale), ("v_scale", v_scale)):
            if x is not None and not 0.0 < x < float("inf"):
                raise ValueError(f"{name}={x!r} must be positive and finite")
        if index is not None:
            _index(index, pages, heads, dim, device)
        shape = _sparse_lib.RpaAppendShape(k.shape[0], heads, dim, pages, page_size, code, k.stride(0), k.stride(1),
                                           v.stride(0), v.stride(1))
        plan = _keep(sig, (shape, 1.0 if k_scale is None else k_scale, 1.0 if v_scale is None else v_scale,
                           _sparse_lib.load().rpa_append_kv))
    shape, ks, vs, fn = plan
    dev = kv_pages.get_device()
    if dev != _get_device():
        with torch.cuda.device(dev):
            return append_kv(k, v, kv_pages, slot_mapping, kv_scales=kv_scales, k_scale=k_scale, v_scale=v_scale, index=index)
    rc = fn(shape, k.data_ptr(), v.data_ptr(), slot_mapping.data_ptr(), kv_pages.data_ptr(),
            None if kv_scales is None else kv_scales.data_ptr(), ks, vs, None if index is None else index[0].data_ptr(),
            None if index is None else index[1].data_ptr(), _current_stream(dev))
    if rc:
        _sparse_lib.check(rc)


def _metadata(kv_lens, page_indices, cu_q_lens, num_seqs, device) -> tuple[int, int]:
    _tensor("page_indices", page_indices, torch.int32, (None, None), device)
    n = page_indices.shape[0]
    _tensor("kv_lens", kv_lens, torch.int32, (n,), device)
    _tensor("cu_q_lens", cu_q_lens, torch.int32, (n + 1,), device)
    _tensor("num_seqs", num_seqs, torch.int32, (1,), device)
    return n, page_indices.shape[1]


def _workspace_bytes(query, shape) -> int:
    """What the call needs; the library's own refusal of the shape, if that is why it says 0."""
    return int(query(ctypes.byref(shape)))


def select_pages(
    q: torch.Tensor,             # bf16 [T, Hq, D]
    index: PageIndex,
    kv_lens: torch.Tensor,       # i32[max_num_seqs]
    page_indices: torch.Tensor,  # i32[max_num_seqs, pages_per_seq]
    cu_q_lens: torch.Tensor,     # i32[max_num_seqs + 1]
    num_seqs: torch.Tensor,      # i32[1]
    *,
    page_size: int,
    num_pages: int,
    sink_pages: int = 1,
    recent_pages: int = 1,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The pages each token and kv head should attend to: i32 [T, Hkv, num_pages], logical pages
    (columns of the sequence's ``page_indices`` row), ascending, -1 past the last.

    A token sees the pages up to its own (position // page_size).  The first ``sink_pages`` and the last
    ``recent_pages`` of them are always chosen; the others by an estimate of their highest score, of
    the index's bounds and the group's queries, rounded to int8 on one grid,

        score(p) = 2**exponent(p) * max_g sum_d max(q_gd * hi_d, q_gd * lo_d),

    the highest first and of equal scores the earlier page.  Scores are whole numbers times a power of
    two: the choice does not depend on an order of summation.  A head whose queries are all below 1/254 of
    the group's largest counts as 0, and the head with the largest scores decides.  Tokens at or past
    ``cu_q_lens[num_seqs]`` get no page.
    """
    bounds, exponents = index
    sig = (q.shape, q.dtype, q.get_device(), q.stride(), bounds.shape, bounds.dtype, bounds.get_device(), bounds.is_contiguous(),
           exponents.shape, exponents.dtype, exponents.get_device(), exponents.is_contiguous(),
           kv_lens.shape, kv_lens.dtype, kv_lens.get_device(), kv_lens.is_contiguous(),
           page_indices.shape, page_indices.dtype, page_indices.get_device(), page_indices.is_contiguous(),
           cu_q_lens.shape, cu_q_lens.dtype, cu_q_lens.get_device(), cu_q_lens.is_contiguous(),
           num_seqs.shape, num_seqs.dtype, num_seqs.get_device(), num_seqs.is_contiguous(),
           page_size, num_pages, sink_pages, recent_pages)
    plan = _plans.get(sig)
    if plan is None:
        _index(index, None, None, None, None)
        pages, heads, _, dim = index[0].shape
        device = index[0].device
        _tensor("q", q, torch.bfloat16, (None, None, dim), device, rows=True)
        n, width = _metadata(kv_lens, page_indices, cu_q_lens, num_seqs, device)
        for name, x, least in (("page_size", page_size, 1), ("num_pages", num_pages, 1), ("sink_pages", sink_pages, 0),
                               ("recent_pages", recent_pages, 0)):
            if not (isinstance(x, int) and least <= x < 1 << 31):
                raise ValueError(f"{name}={x!r} must be an int of at least {least}")
        if sink_pages + recent_pages > num_pages:
            raise ValueError(f"sink_pages={sink_pages} and recent_pages={recent_pages} exceed num_pages={num_pages}")
        if q.shape[1] == 0 or heads == 0 or q.shape[1] % heads:
            raise ValueError(f"num_q_heads={q.shape[1]} must be divisible by num_kv_heads={heads}")
        lib = _sparse_lib.load()
        shape = _sparse_lib.RpaSparseShape(q.shape[0], q.shape[1], heads, dim, pages, page_size, n, width,
                                           _sparse_lib.RPA_KV_BF16, num_pages, q.stride(0), q.stride(1))
        plan = _keep(sig, (shape, (q.shape[0], heads, num_pages), _workspace_bytes(lib.rpa_select_workspace_size, shape),
                           lib.rpa_select_pages))
    shape, out_shape, need, fn = plan
    dev = q.get_device()
    if out is None:
        out = kv_lens.new_empty(out_shape)
    else:
        _tensor("out", out, torch.int32, out_shape, q.device)
        _separate("out", out, {"q": q, "index.bounds": bounds, "index.exponents": exponents, "kv_lens": kv_lens,
                               "page_indices": page_indices, "cu_q_lens": cu_q_lens, "num_seqs": num_seqs})
    if dev != _get_device():
        with torch.cuda.device(dev):
            return select_pages(q, index, kv_lens, page_indices, cu_q_lens, num_seqs, page_size=page_size, num_pages=num_pages,
                                sink_pages=sink_pages, recent_pages=recent_pages, out=out)
    scratch = bounds.new_empty(need) if need else None  # bytes
    rc = fn(shape, sink_pages, recent_pages, q.data_ptr(), bounds.data_ptr(), exponents.data_ptr(), kv_lens.data_ptr(),
            page_indices.data_ptr(), cu_q_lens.data_ptr(), num_seqs.data_ptr(), out.data_ptr(),
            scratch.data_ptr() if need else None, need, _current_stream(dev))
    if rc:
        _sparse_lib.check(rc)
    return out


def sparse_paged_attention(
    q: torch.Tensor,               # bf16 [T, Hq, D]
    kv_pages: torch.Tensor,        # bf16 | float8_e4m3fn | uint8 (e4m3 codes) [pages, page_size, 2*Hkv, D]
    selected_pages: torch.Tensor,  # i32 [T, Hkv, num_pages]
    kv_lens: torch.Tensor,         # i32[max_num_seqs]
    page_indices: torch.Tensor,    # i32[max_num_seqs, pages_per_seq]
    cu_q_lens: torch.Tensor,       # i32[max_num_seqs + 1]
    num_seqs: torch.Tensor,        # i32[1]
    *,
    sm_scale: float = 1.0,
    soft_cap: float | None = None,
    k_scale: float | None = None,
    v_scale: float | None = None,
    kv_scales: torch.Tensor | None = None,  # f32 [pages, Hkv, 2] per-(page, kv head) K/V scales of an fp8 pool
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention over listed pages: ``ops.ragged_paged_attention`` restricted, for each token and kv
    head, to the keys of ``selected_pages`` (``select_pages``' list, or any other: logical pages of the
    token's sequence in any order, -1 or other entries outside its pages list nothing, a page listed
    twice counts twice).

    Returns bf16 [T, Hq, D] (or fills ``out``); rows without a key or without a score above -infinity,
    and rows at or past ``cu_q_lens[num_seqs]``, are zero.  Scores, softmax, probabilities and sums are fp32; scaled keys
    and values are not rounded (the dense operator rounds them, and its probabilities, to bf16).
    """
    sig = (q.shape, q.dtype, q.get_device(), q.stride(),
           kv_pages.shape, kv_pages.dtype, kv_pages.get_device(), kv_pages.is_contiguous(), selected_pages.shape,
           selected_pages.dtype, selected_pages.get_device(), selected_pages.is_contiguous(),
           kv_lens.shape, kv_lens.dtype, kv_lens.get_device(), kv_lens.is_contiguous(),
           page_indices.shape, page_indices.dtype, page_indices.get_device(), page_indices.is_contiguous(),
           cu_q_lens.shape, cu_q_lens.dtype, cu_q_lens.get_device(), cu_q_lens.is_contiguous(),
           num_seqs.shape, num_seqs.dtype, num_seqs.get_device(), num_seqs.is_contiguous(),
           sm_scale, soft_cap, k_scale, v_scale,
           None if kv_scales is None else (kv_scales.shape, kv_scales.dtype, kv_scales.get_device(), kv_scales.is_contiguous()))
    plan = _plans.get(sig)
    if plan is None:
        pages, page_size, heads, dim, code = _pool(kv_pages)
        device = kv_pages.device
        _tensor("q", q, torch.bfloat16, (None, None, dim), device, rows=True)
        _tensor("selected_pages", selected_pages, torch.int32, (q.shape[0], heads, None), device)
        n, width = _metadata(kv_lens, page_indices, cu_q_lens, num_seqs, device)
        _scales(kv_scales, k_scale, v_scale, pages, heads, code, device)
        if soft_cap is not None and soft_cap == 0.0:
            raise ValueError(f"soft_cap={soft_cap} must not be 0.0.")
        if q.shape[1] == 0 or q.shape[1] % heads:
            raise ValueError(f"num_q_heads={q.shape[1]} must be divisible by num_kv_heads={heads}")
        if selected_pages.shape[2] == 0:
            raise ValueError("selected_pages must have room for a page")
        lib = _sparse_lib.load()
        shape = _sparse_lib.RpaSparseShape(q.shape[0], q.shape[1], heads, dim, pages, page_size, n, width, code,
                                           selected_pages.shape[2], q.stride(0), q.stride(1))
        options = _sparse_lib.RpaSparseOptions(float(sm_scale), float(soft_cap or 0.0), 1.0 if k_scale is None else k_scale,
                                               1.0 if v_scale is None else v_scale)
        plan = _keep(sig, (shape, options, _workspace_bytes(lib.rpa_sparse_workspace_size, shape),
                           lib.rpa_sparse_paged_attention))
    shape, options, need, fn = plan
    dev = q.get_device()
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _tensor("out", out, torch.bfloat16, q.shape, q.device)
        _separate("out", out, {"q": q, "kv_pages": kv_pages, "selected_pages": selected_pages, "kv_lens": kv_lens,
                               "page_indices": page_indices, "cu_q_lens": cu_q_lens, "num_seqs": num_seqs, "kv_scales": kv_scales})
    if dev != _get_device():
        with torch.cuda.device(dev):
            return sparse_paged_attention(q, kv_pages, selected_pages, kv_lens, page_indices, cu_q_lens, num_seqs,
                                          sm_scale=sm_scale, soft_cap=soft_cap, k_scale=k_scale, v_scale=v_scale,
                                          kv_scales=kv_scales, out=out)
    scratch = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    rc = fn(shape, options, q.data_ptr(), kv_pages.data_ptr(), None if kv_scales is None else kv_scales.data_ptr(),
            selected_pages.data_ptr(), kv_lens.data_ptr(), page_indices.data_ptr(), cu_q_lens.data_ptr(),
            num_seqs.data_ptr(), out.data_ptr(), scratch.data_ptr() if need else None, need, _current_stream(dev))
    if rc:
        _sparse_lib.check(rc)
    return out
