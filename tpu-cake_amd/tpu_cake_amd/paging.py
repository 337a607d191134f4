"""Page allocation and step metadata on the GPU.

The pool's free pages are a stack (``free_pages[:free_count]``); a request holds the first
``ceil(len / page_size)`` entries of its ``page_table`` row.  ``assign_pages`` gives each request the
pages of its new tokens and writes what ``ops.ragged_paged_attention`` and the entry points of
``sparse`` take: lengths, cumulative query lengths, the slot of every new token (``sparse.append_kv``)
and its position.  ``release_pages`` takes the pages of finished requests back.  Nothing is read on
the host, so a serving loop's step needs no synchronisation and can be captured into a graph.

All tensors are contiguous int32 tensors on one GPU.  What a call reads is never written by it,
except new entries of ``page_table`` (``assign_pages``) and of ``free_pages`` above its count
(``release_pages``): lengths and counts come back in tensors of their own, the caller's next inputs.
"""

from __future__ import annotations

import typing

import torch

from . import _sparse_lib
from ._sparse_lib import read_error_word  # noqa: F401
from .ops import _current_stream, _get_device, _require_cuda


class StepMetadata(typing.NamedTuple):
    """What ``assign_pages`` writes (N requests)."""

    kv_lens: torch.Tensor       # i32[N]: cached and new tokens
    cu_q_lens: torch.Tensor     # i32[N + 1]
    num_seqs: torch.Tensor      # i32[1]: N
    slot_mapping: torch.Tensor  # i32[max_tokens]: page * page_size + row, -1 past the last token
    positions: torch.Tensor     # i32[max_tokens]: position in its sequence, 0 past the last token
    free_count: torch.Tensor    # i32[1]


def _check(named: dict, page_table, n: int, page_size: int) -> None:
    """Types, devices and shapes; ``named`` holds (tensor, expected shape or None, dtype)."""
    device = page_table.device
    for name, (t, shape, dtype) in named.items():
        _require_cuda(name, t)
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, page_table on {device}")
        if t.dtype != dtype:
            raise ValueError(f"{name} dtype {t.dtype} must be {dtype}")
        if t.dim() != len(shape) or any(want is not None and want != got for want, got in zip(shape, t.shape)):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if n == 0 or page_table.shape[1] == 0:
        raise ValueError("page_table must have rows and columns")
    if not (isinstance(page_size, int) and page_size > 0):
        raise ValueError(f"page_size={page_size!r} must be a positive int")
    if page_table.shape[1] * page_size > 0x7FFFFFFF:
        raise ValueError("pages_per_seq * page_size overflows int32")


def _separate(outs: dict, ins: dict) -> None:
    """Refuses an output whose memory overlaps an input's or another output's."""
    spans = [(name, t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for name, t in {**outs, **ins}.items()]
    for i, (a, lo, hi) in enumerate(spans[:len(outs)]):
        for b, lo2, hi2 in spans[i + 1:]:
            if lo < hi2 and lo2 < hi:
                raise ValueError(f"{a} overlaps {b}: outputs need memory of their own")


# one allocation for a call's outputs: views of it, without the bookkeeping that gradients would need
_parts = torch.unsafe_split_with_sizes

# shapes that passed the checks -> the call's shape struct
_plans: dict[tuple, object] = {}


def _keep(sig: tuple, plan):
    if len(_plans) > 256:
        _plans.clear()
    _plans[sig] = plan
    return plan


def assign_pages(
    cached_lens: torch.Tensor,  # i32[N]: tokens of each request already in the pool
    new_tokens: torch.Tensor,   # i32[N]: tokens it brings in this step (0: none)
    page_table: torch.Tensor,   # i32[N, pages_per_seq], new entries written in place
    free_pages: torch.Tensor,   # i32[F]
    free_count: torch.Tensor,   # i32[1]
    *,
    page_size: int,
    max_tokens: int,            # rows of slot_mapping and positions: the batch's capacity
    out: StepMetadata | None = None,
) -> StepMetadata:
    """Pages and metadata of one step, requests in order.

    A request is admitted if its lengths are not negative and fit ``page_table``, the new tokens of
    the requests up to and including it are at most ``max_tokens``, and it needs no new page or the
    pages needed up to and including it are at most ``free_count``; both sums run over all requests
    with valid lengths, admitted or not.  One that is not admitted keeps its length and has no token
    (``cu_q_lens`` does not grow): bring it again in a later step.  Its j-th new page is the next from
    the top of the stack.  Invalid lengths set ``ERR_LEN`` in the error word (``read_error_word``).
    """
    # what the checks go by: written out, as a call costs less than a helper's calls would
    sig = (page_table.shape, page_table.dtype, page_table.get_device(), page_table.is_contiguous(),
           cached_lens.shape, cached_lens.dtype, cached_lens.get_device(), cached_lens.is_contiguous(),
           new_tokens.shape, new_tokens.dtype, new_tokens.get_device(), new_tokens.is_contiguous(),
           free_pages.shape, free_pages.dtype, free_pages.get_device(), free_pages.is_contiguous(),
           free_count.shape, free_count.dtype, free_count.get_device(), free_count.is_contiguous(), page_size, max_tokens)
    plan = _plans.get(sig)
    if plan is None:
        n = page_table.shape[0]
        i32 = torch.int32
        _check({"page_table": (page_table, (None, None), i32), "cached_lens": (cached_lens, (n,), i32),
                "new_tokens": (new_tokens, (n,), i32), "free_pages": (free_pages, (None,), i32),
                "free_count": (free_count, (1,), i32)}, page_table, n, page_size)
        if not (isinstance(max_tokens, int) and 0 <= max_tokens < 1 << 30):
            raise ValueError(f"max_tokens={max_tokens!r} must be an int in [0, 2^30)")
        if free_pages.numel() >= 1 << 30:
            raise ValueError("free_pages must have fewer than 2^30 entries")
        plan = _keep(sig, (_sparse_lib.RpaPagingShape(n, page_table.shape[1], page_size, free_pages.numel(), max_tokens),
                           [n, n + 1, 1, max_tokens, max_tokens, 1], 2 * n + 3 + 2 * max_tokens,
                           _sparse_lib.load().rpa_assign_pages))
    shape, sizes, total, fn = plan
    dev = page_table.get_device()
    if out is None:
        out = StepMetadata(*_parts(page_table.new_empty(total), sizes))
    else:
        names = dict(zip(StepMetadata._fields, out))
        _check({k: (t, (n,), torch.int32) for (k, t), n in zip(names.items(), sizes)}, page_table, 1, page_size)
        _separate({"out." + k: t for k, t in names.items() if t.numel()},
                  {"cached_lens": cached_lens, "new_tokens": new_tokens, "page_table": page_table,
                   "free_pages": free_pages, "free_count input": free_count})
    if dev != _get_device():
        with torch.cuda.device(dev):
            return assign_pages(cached_lens, new_tokens, page_table, free_pages, free_count, page_size=page_size,
                                max_tokens=max_tokens, out=out)
    rc = fn(shape, cached_lens.data_ptr(), new_tokens.data_ptr(), page_table.data_ptr(), free_pages.data_ptr(),
            free_count.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(),
            out[4].data_ptr(), out[5].data_ptr(), _current_stream(dev))
    if rc:
        _sparse_lib.check(rc)
    return out


def release_pages(
    cached_lens: torch.Tensor,  # i32[N]
    finished: torch.Tensor,     # bool[N]
    page_table: torch.Tensor,   # i32[N, pages_per_seq]
    free_pages: torch.Tensor,   # i32[F], entries above the count written in place
    free_count: torch.Tensor,   # i32[1]
    *,
    page_size: int,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Pushes the pages of finished requests on the free stack, in order; returns (lengths, with 0 for
    the finished ones, and the new count).  Pages past ``free_pages``' capacity are dropped and set
    ``ERR_FREE`` in the error word."""
    sig = (page_table.shape, page_table.dtype, page_table.get_device(), page_table.is_contiguous(),
           cached_lens.shape, cached_lens.dtype, cached_lens.get_device(), cached_lens.is_contiguous(),
           finished.shape, finished.dtype, finished.get_device(), finished.is_contiguous(),
           free_pages.shape, free_pages.dtype, free_pages.get_device(), free_pages.is_contiguous(),
           free_count.shape, free_count.dtype, free_count.get_device(), free_count.is_contiguous(), page_size)
    plan = _plans.get(sig)
    if plan is None:
        n = page_table.shape[0]
        i32 = torch.int32
        _check({"page_table": (page_table, (None, None), i32), "cached_lens": (cached_lens, (n,), i32),
                "finished": (finished, (n,), torch.bool), "free_pages": (free_pages, (None,), i32),
                "free_count": (free_count, (1,), i32)}, page_table, n, page_size)
        if free_pages.numel() >= 1 << 30:
            raise ValueError("free_pages must have fewer than 2^30 entries")
        plan = _keep(sig, (_sparse_lib.RpaPagingShape(n, page_table.shape[1], page_size, free_pages.numel(), 0), [n, 1],
                           _sparse_lib.load().rpa_release_pages))
    shape, sizes, fn = plan
    dev = page_table.get_device()
    if out is None:
        out = _parts(page_table.new_empty(sizes[0] + 1), sizes)
    else:
        names = {"out lengths": out[0], "out count": out[1]}
        _check({k: (t, (n,), torch.int32) for (k, t), n in zip(names.items(), sizes)}, page_table, 1, page_size)
        _separate(names, {"cached_lens": cached_lens, "finished": finished, "page_table": page_table,
                          "free_pages": free_pages, "free_count": free_count})
    if dev != _get_device():
        with torch.cuda.device(dev):
            return release_pages(cached_lens, finished, page_table, free_pages, free_count, page_size=page_size, out=out)
    rc = fn(shape, cached_lens.data_ptr(), finished.data_ptr(), page_table.data_ptr(), free_pages.data_ptr(),
            free_count.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), _current_stream(dev))
    if rc:
        _sparse_lib.check(rc)
    return tuple(out)
