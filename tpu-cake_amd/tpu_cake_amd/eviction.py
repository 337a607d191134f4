"""A cache of bounded size: attention that accounts for the weight each key got, and the eviction of the keys
that got least.

Beside ``ops.ragged_paged_attention`` and over its tensors, with a **ledger** of the pool: for each slot and kv
head the weight that the key there got so far, and the position of its token.

* ``weighed_attention`` is causal attention over the paged cache that adds each key's probabilities to the ledger.
* ``choose_moves`` finds, for each sequence longer than ``limit`` and each kv head, the ``budget`` rows to keep -- the
  first positions, the most recent ones, and those of the highest weight -- and how they come into the first
  ``budget`` rows; ``move_rows`` moves them.  Heads keep rows of their own; which row a key stands in says nothing about
  its position any more, the ledger does.
* ``paging.trim_pages`` then cuts the sequences and takes their pages back, once for all the layers of a page table,
  and counts the tokens that each sequence lost (``dropped``), which ``rotary.rotate_heads`` adds to later positions.

The pages of different sequences have to differ: a shared prefix would be accounted and moved for all its readers.
A pool's ``sparse.PageIndex`` does not follow moved rows: a pool takes ``sparse.select_pages`` or eviction, not both.
All tensors are torch tensors on one GPU; ``q`` may be a slice of a larger tensor, the others are contiguous.  Calls run
on torch's current stream, take what scratch they need from torch's allocator, and may be captured into graphs.
"""

from __future__ import annotations

import ctypes
import typing

import torch

from . import _bounded_lib
from ._bounded_lib import read_error_word  # noqa: F401
from .ops import _current_stream, _get_device
from .sparse import _metadata, _pool, _scales, _separate, _tensor


class Ledger(typing.NamedTuple):
    """What eviction knows of a pool's keys."""

    weights: torch.Tensor    # f32[pages, Hkv, page_size]: what attention gave the key so far
    positions: torch.Tensor  # i32[pages, Hkv, page_size]: its token's position in the sequence


def make_ledger(kv_pages: torch.Tensor) -> Ledger:
    """A ledger for ``kv_pages``, to be kept by ``weighed_attention``, which starts the entries of new keys itself."""
    pages, page_size, combined, _ = kv_pages.shape
    return Ledger(torch.zeros((pages, combined // 2, page_size), dtype=torch.float32, device=kv_pages.device),
                  torch.zeros((pages, combined // 2, page_size), dtype=torch.int32, device=kv_pages.device))


# what passed the checks -> the call's structs; signatures of different entry points differ in length
_plans: dict[tuple, tuple] = {}


def _keep(sig: tuple, plan: tuple) -> tuple:
    if len(_plans) > 256:
        _plans.clear()
    _plans[sig] = plan
    return plan


def _ledger(ledger, shape, device) -> None:
    if not (isinstance(ledger, tuple) and len(ledger) == 2):
        raise TypeError("ledger must be a Ledger")
    _tensor("ledger.weights", ledger[0], torch.float32, shape, device)
    _tensor("ledger.positions", ledger[1], torch.int32, tuple(ledger[0].shape), ledger[0].device)


def preflight_pages(kv_lens: torch.Tensor, page_indices: torch.Tensor, page_size: int) -> None:
    """Host check of what the ledger takes for granted: no page is held twice.  Reads its arguments on the host."""
    table, lens = page_indices.detach().cpu(), kv_lens.detach().cpu().tolist()
    held = torch.cat([table[i, :-(-max(n, 0) // page_size)] for i, n in enumerate(lens)] + [table.new_zeros(0)])
    if held.numel() != torch.unique(held).numel():
        raise ValueError("page_indices holds a page twice")


def weighed_attention(
    q: torch.Tensor,             # bf16 [T, Hq, D]
    kv_pages: torch.Tensor,      # bf16 | float8_e4m3fn | uint8 (e4m3 codes) [pages, page_size, 2*Hkv, D]
    ledger: Ledger,              # updated
    kv_lens: torch.Tensor,       # i32[max_num_seqs]
    page_indices: torch.Tensor,  # i32[max_num_seqs, pages_per_seq]
    cu_q_lens: torch.Tensor,     # i32[max_num_seqs + 1]
    num_seqs: torch.Tensor,      # i32[1]
    *,
    sm_scale: float = 1.0,
    soft_cap: float | None = None,
    decay: float = 1.0,
    dropped: torch.Tensor | None = None,    # i32[max_num_seqs]: tokens that each sequence's cache has lost
    k_scale: float | None = None,
    v_scale: float | None = None,
    kv_scales: torch.Tensor | None = None,  # f32 [pages, Hkv, 2] per-(page, kv head) K/V scales of an fp8 pool
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal attention over the paged cache, as ``ops.ragged_paged_attention``; returns bf16 [T, Hq, D] (or fills
    ``out``).  Rows without a key or without a score above -infinity, and rows at or past ``cu_q_lens[num_seqs]``, are zero.

    For each sequence with tokens in the step, of every key and kv head,

        weights = decay * weights + sum over the step's tokens and the group's heads of the key's probability.

    The step's own keys (the last q_len of the sequence) are new: their weight starts at 0 whatever the ledger holds,
    and their position is noted, ``dropped`` plus the key's row.  ``decay`` 1 accumulates, 0 keeps the last step's weights
    (earlier ones are not read), and between them earlier steps fade.

    Scores, softmax, probabilities and sums are fp32; scaled keys and values are not rounded.  The pages of different
    sequences have to differ (``preflight_pages`` checks it on the host).
    """
    # what the checks go by: written out, as a call costs less than a helper's calls would
    weights, positions = ledger
    sig = (q.shape, q.dtype, q.get_device(), q.stride(),
           kv_pages.shape, kv_pages.dtype, kv_pages.get_device(), kv_pages.is_contiguous(),
           weights.shape, weights.dtype, weights.get_device(), weights.is_contiguous(),
           positions.shape, positions.dtype, positions.get_device(), positions.is_contiguous(),
           kv_lens.shape, kv_lens.dtype, kv_lens.get_device(), kv_lens.is_contiguous(),
           page_indices.shape, page_indices.dtype, page_indices.get_device(), page_indices.is_contiguous(),
           cu_q_lens.shape, cu_q_lens.dtype, cu_q_lens.get_device(), cu_q_lens.is_contiguous(),
           num_seqs.shape, num_seqs.dtype, num_seqs.get_device(), num_seqs.is_contiguous(),
           None if dropped is None else (dropped.shape, dropped.dtype, dropped.get_device(), dropped.is_contiguous()),
           None if kv_scales is None else (kv_scales.shape, kv_scales.dtype, kv_scales.get_device(), kv_scales.is_contiguous()),
           sm_scale, soft_cap, decay, k_scale, v_scale)
    plan = _plans.get(sig)
    if plan is None:
        pages, page_size, heads, dim, code = _pool(kv_pages)
        device = kv_pages.device
        _tensor("q", q, torch.bfloat16, (None, None, dim), device, rows=True)
        _ledger(ledger, (pages, heads, page_size), device)
        n, width = _metadata(kv_lens, page_indices, cu_q_lens, num_seqs, device)
        if dropped is not None:
            _tensor("dropped", dropped, torch.int32, (n,), device)
        _scales(kv_scales, k_scale, v_scale, pages, heads, code, device)
        for name, x in (("sm_scale", sm_scale), ("soft_cap", 1.0 if soft_cap is None else soft_cap)):
            if not isinstance(x, (int, float)):
                raise ValueError(f"{name}={x!r} must be a float")
        if soft_cap is not None and soft_cap == 0.0:
            raise ValueError(f"soft_cap={soft_cap} must not be 0.0.")
        if not (isinstance(decay, (int, float)) and 0.0 <= decay < float("inf")):
            raise ValueError(f"decay={decay!r} must be a finite float, not negative")
        if q.shape[1] == 0 or q.shape[1] % heads:
            raise ValueError(f"num_q_heads={q.shape[1]} must be divisible by num_kv_heads={heads}")
        lib = _bounded_lib.load()
        shape = _bounded_lib.RpaWeighShape(q.shape[0], q.shape[1], heads, dim, pages, page_size, n, width, code, 0, q.stride(0),
                                           q.stride(1))
        options = _bounded_lib.RpaWeighOptions(float(sm_scale), float(soft_cap or 0.0), 1.0 if k_scale is None else k_scale,
                                               1.0 if v_scale is None else v_scale, float(decay))
        plan = _keep(sig, (shape, options, int(lib.rpa_weigh_workspace_size(ctypes.byref(shape))), lib.rpa_weighed_attention))
    shape, options, need, fn = plan
    dev = q.get_device()
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _tensor("out", out, torch.bfloat16, q.shape, q.device)
        _separate("out", out, {"q": q, "kv_pages": kv_pages, "ledger.weights": ledger[0], "ledger.positions": ledger[1],
                               "kv_lens": kv_lens, "page_indices": page_indices, "cu_q_lens": cu_q_lens, "num_seqs": num_seqs,
                               "dropped": dropped, "kv_scales": kv_scales})
    if dev != _get_device():
        with torch.cuda.device(dev):
            return weighed_attention(q, kv_pages, ledger, kv_lens, page_indices, cu_q_lens, num_seqs, sm_scale=sm_scale,
                                     soft_cap=soft_cap, decay=decay, dropped=dropped, k_scale=k_scale, v_scale=v_scale,
                                     kv_scales=kv_scales, out=out)
    scratch = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    rc = fn(shape, options, q.data_ptr(), kv_pages.data_ptr(), None if kv_scales is None else kv_scales.data_ptr(),
            kv_lens.data_ptr(), page_indices.data_ptr(), cu_q_lens.data_ptr(), num_seqs.data_ptr(),
            None if dropped is None else dropped.data_ptr(), weights.data_ptr(), positions.data_ptr(), out.data_ptr(),
            scratch.data_ptr() if need else None, need, _current_stream(dev))
    if rc:
        _bounded_lib.check(rc)
    return out


def choose_moves(
    ledger: Ledger,
    kv_lens: torch.Tensor,       # i32[max_num_seqs]
    page_indices: torch.Tensor,  # i32[max_num_seqs, pages_per_seq]
    num_seqs: torch.Tensor,      # i32[1]
    *,
    budget: int,
    recent: int,
    sinks: int = 0,
    limit: int | None = None,     # budget where it is None
    dropped: torch.Tensor | None = None,  # i32[max_num_seqs]: tokens that each sequence's cache has lost
    max_moves: int | None = None,         # budget where it is None, which always suffices
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """How each kv head's rows to keep come into a sequence's first ``budget`` rows: i32 [max_num_seqs, Hkv, max_moves, 2],
    slots (page * page_size + row) to and from, -1 past the last.  Sequences of at most ``limit`` keys have no moves.

    Of a longer sequence each head keeps ``budget`` rows: those at positions below ``sinks`` or among the last
    ``recent`` positions, then those of the highest weight (NaN below all others), and of equal ones the lower rows.
    The kept rows past ``budget``, in order, take the places of the rows before it that go, in order.

    ``max_moves`` may be less where sequences grow by few tokens between two evictions: a sequence of n keys needs
    at most n - budget moves.  A list that needs more is cut short and sets ``ERR_LEN`` in the error word.
    """
    weights, positions = ledger
    sig = (weights.shape, weights.dtype, weights.get_device(), weights.is_contiguous(),
           positions.shape, positions.dtype, positions.get_device(), positions.is_contiguous(),
           kv_lens.shape, kv_lens.dtype, kv_lens.get_device(), kv_lens.is_contiguous(),
           page_indices.shape, page_indices.dtype, page_indices.get_device(), page_indices.is_contiguous(),
           num_seqs.shape, num_seqs.dtype, num_seqs.get_device(), num_seqs.is_contiguous(),
           None if dropped is None else (dropped.shape, dropped.dtype, dropped.get_device(), dropped.is_contiguous()),
           budget, recent, sinks, limit, max_moves)
    plan = _plans.get(sig)
    if plan is None:
        _ledger(ledger, (None, None, None), None)
        pages, heads, page_size = ledger[0].shape
        device = ledger[0].device
        _tensor("page_indices", page_indices, torch.int32, (None, None), device)
        n, width = page_indices.shape
        _tensor("kv_lens", kv_lens, torch.int32, (n,), device)
        _tensor("num_seqs", num_seqs, torch.int32, (1,), device)
        if dropped is not None:
            _tensor("dropped", dropped, torch.int32, (n,), device)
        most, room = budget if limit is None else limit, budget if max_moves is None else max_moves
        for name, x, least in (("budget", budget, 1), ("limit", most, budget), ("max_moves", room, 1), ("sinks", sinks, 0),
                               ("recent", recent, 0)):
            if not (isinstance(x, int) and least <= x < 1 << 31):
                raise ValueError(f"{name}={x!r} must be an int of at least {least}")
        if sinks + recent > budget:
            raise ValueError(f"sinks={sinks} and recent={recent} exceed budget={budget}")
        shape = _bounded_lib.RpaChooseShape(n, width, heads, pages, page_size, budget, most, sinks, recent, room)
        lib = _bounded_lib.load()
        plan = _keep(sig, (shape, (n, heads, room, 2), int(lib.rpa_choose_workspace_size(ctypes.byref(shape))), lib.rpa_choose_moves))
    shape, out_shape, need, fn = plan
    dev = kv_lens.get_device()
    if out is None:
        out = kv_lens.new_empty(out_shape)
    else:
        _tensor("out", out, torch.int32, out_shape, kv_lens.device)
        _separate("out", out, {"ledger.weights": ledger[0], "ledger.positions": ledger[1], "kv_lens": kv_lens,
                               "page_indices": page_indices, "num_seqs": num_seqs, "dropped": dropped})
    if dev != _get_device():
        with torch.cuda.device(dev):
            return choose_moves(ledger, kv_lens, page_indices, num_seqs, budget=budget, recent=recent, sinks=sinks, limit=limit,
                                dropped=dropped, max_moves=max_moves, out=out)
    scratch = torch.empty(need, dtype=torch.uint8, device=kv_lens.device) if need else None
    rc = fn(shape, weights.data_ptr(), positions.data_ptr(), kv_lens.data_ptr(), page_indices.data_ptr(), num_seqs.data_ptr(),
            None if dropped is None else dropped.data_ptr(), out.data_ptr(), scratch.data_ptr() if need else None, need,
            _current_stream(dev))
    if rc:
        _bounded_lib.check(rc)
    return out


def move_rows(
    kv_pages: torch.Tensor,  # bf16 | float8_e4m3fn | uint8 (e4m3 codes) [pages, page_size, 2*Hkv, D], rows moved
    ledger: Ledger,          # moved with them
    moves: torch.Tensor,     # i32 [lists, Hkv, max_moves, 2]
    *,
    kv_scales: torch.Tensor | None = None,  # f32 [pages, Hkv, 2]: the fp8 pool's K and V scales, as they stand
) -> None:
    """Copies, for each entry of ``choose_moves``' lists, a kv head's key and value rows and its ledger entries from one slot
    to another; entries with a negative slot are none.

    Rows of an fp8 pool that come to a page of another scale are rounded anew, e4m3(code * scale there / scale
    here), saturated at +-448.  Slots outside the pool are skipped and set ``ERR_SLOT`` in the error word.  No slot that is
    written may be another entry's of the same head, as those of ``choose_moves`` are not.
    """
    weights, positions = ledger
    sig = (kv_pages.shape, kv_pages.dtype, kv_pages.get_device(), kv_pages.is_contiguous(),
           weights.shape, weights.dtype, weights.get_device(), weights.is_contiguous(),
           positions.shape, positions.dtype, positions.get_device(), positions.is_contiguous(),
           moves.shape, moves.dtype, moves.get_device(), moves.is_contiguous(),
           None if kv_scales is None else (kv_scales.shape, kv_scales.dtype, kv_scales.get_device(), kv_scales.is_contiguous()))
    plan = _plans.get(sig)
    if plan is None:
        pages, page_size, heads, dim, code = _pool(kv_pages)
        device = kv_pages.device
        _ledger(ledger, (pages, heads, page_size), device)
        _tensor("moves", moves, torch.int32, (None, heads, None, 2), device)
        _scales(kv_scales, None, None, pages, heads, code, device)
        if moves.shape[2] == 0:
            raise ValueError("moves must have room for an entry")
        shape = _bounded_lib.RpaMoveShape(moves.shape[0], moves.shape[2], heads, dim, pages, page_size, code)
        plan = _keep(sig, (shape, _bounded_lib.load().rpa_move_rows))
    shape, fn = plan
    dev = kv_pages.get_device()
    if dev != _get_device():
        with torch.cuda.device(dev):
            return move_rows(kv_pages, ledger, moves, kv_scales=kv_scales)
    rc = fn(shape, moves.data_ptr(), None if kv_scales is None else kv_scales.data_ptr(), kv_pages.data_ptr(),
            weights.data_ptr(), positions.data_ptr(), _current_stream(dev))
    if rc:
        _bounded_lib.check(rc)
