"""Norms and position rotation of a step's queries and keys: what stands between the projections and
``sparse.append_kv`` and attention.

``rotate_heads`` does both in one pass over the step's tokens: the root-mean-square norm of each head, where it
is given a weight, and the rotation of the head's first dims by angles that grow with the token's position.
Positions are those of ``paging.assign_pages``; a cache that lost tokens (``eviction``) gives them as ``dropped``.

A pair's frequency is held in **turns**, the whole number of 2^-64 of a full turn that it turns by from one
position to the next (``turns_of``): the kernels multiply it with the position in 64-bit whole numbers, from
which whole turns fall away, so angles are as exact at position 2^30 as at 1, and no table of sines is kept.
"""

from __future__ import annotations

import math

import torch

from . import _bounded_lib
from ._bounded_lib import read_error_word  # noqa: F401
from .ops import _current_stream, _get_device, _require_cuda
from .sparse import _separate, _tensor


def frequencies(rotated: int, base: float = 10000.0, *, factor: float = 1.0, trained: int | None = None,
                slow: float = 1.0, fast: float = 32.0) -> torch.Tensor:
    """Radians a position for each of ``rotated / 2`` pairs, base^(-2 i / rotated), float64 on the CPU.

    ``factor`` stretches positions for contexts longer than ``trained``: all of them alike if ``trained`` is None (a
    position n then counts as n / factor); else a pair that makes at most ``slow`` turns in ``trained`` positions is
    stretched by ``factor``, one that makes at least ``fast`` not at all, and those between in proportion.
    """
    if not (isinstance(rotated, int) and rotated >= 0 and rotated % 2 == 0):
        raise ValueError(f"rotated={rotated!r} must be an even int, not negative")
    if not (base > 0 and factor > 0):
        raise ValueError(f"base={base!r} and factor={factor!r} must be positive")
    f = base ** (-2.0 * torch.arange(rotated // 2, dtype=torch.float64) / max(rotated, 1))
    if trained is None:
        return f / factor
    if not (trained > 0 and fast > slow):
        raise ValueError(f"trained={trained!r} must be positive and fast={fast!r} more than slow={slow!r}")
    keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
    return f * keep + f / factor * (1 - keep)


def turns_of(frequencies, device=None) -> torch.Tensor:
    """``rotate_heads``' turns for frequencies in radians a position (a float64 tensor or floats): int64, the unsigned
    number's 64 bits, on ``device`` (default: the current GPU)."""
    values = frequencies.double().tolist() if isinstance(frequencies, torch.Tensor) else [float(f) for f in frequencies]
    if not all(math.isfinite(f) for f in values):
        raise ValueError("frequencies must be finite")
    whole = [round(f / (2 * math.pi) * 2.0**64) % (1 << 64) for f in values]
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in whole], dtype=torch.int64, device="cuda" if device is None else device)


# what passed the checks -> the call's structs
_plans: dict[tuple, tuple] = {}


def _weight(name: str, w, heads: int, dim: int, device):
    """A norm's weight: (dtype, stride from head to head), or None."""
    if w is None:
        return None
    _require_cuda(name, w)
    if w.device != device:
        raise ValueError(f"{name} is on {w.device}, expected {device}")
    if w.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{name} dtype {w.dtype} must be torch.bfloat16 or torch.float32")
    if tuple(w.shape) not in ((dim,), (heads, dim)):
        raise ValueError(f"{name} has shape {tuple(w.shape)}, expected ({dim},) or ({heads}, {dim})")
    return w.dtype, dim if w.dim() == 2 else 0


def rotate_heads(
    q: torch.Tensor,          # bf16 [T, Hq, D]
    k: torch.Tensor,          # bf16 [T, Hkv, D]
    positions: torch.Tensor,  # i32[T]
    turns: torch.Tensor,      # i64[rotated / 2] (turns_of)
    *,
    interleaved: bool = False,
    magnitude: float = 1.0,
    q_weight: torch.Tensor | None = None,  # bf16 | f32 [D] or [Hq, D]
    k_weight: torch.Tensor | None = None,  # bf16 | f32 [D] or [Hkv, D]
    eps: float = 1e-6,
    cu_q_lens: torch.Tensor | None = None,  # i32[max_num_seqs + 1]
    num_seqs: torch.Tensor | None = None,   # i32[1]
    dropped: torch.Tensor | None = None,    # i32[max_num_seqs]: tokens that each sequence's cache has lost
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys with their heads normed (``x * rsqrt(mean(x^2) + eps) * weight``, where a weight is
    given) and the first ``rotated = 2 * len(turns)`` dims of each head turned by the token's position plus its
    sequence's ``dropped``: pairs ``(x_i, x_{i + rotated/2})``, or ``(x_2i, x_{2i+1})`` if ``interleaved``,

        (a cos - b sin, b cos + a sin) * magnitude,

    the other dims as they are.  All in fp32, rounded once.

    ``out=(q, k)`` works in place; other tensors need memory of their own.  With ``cu_q_lens`` and ``num_seqs``, rows at
    or past ``cu_q_lens[num_seqs]`` are zero, and left as they are in place; without them every row is done.
    ``rotated`` is a multiple of 8 (``interleaved``: of 2); head dims and strides are those of ``sparse``.
    """
    # what the checks go by: written out, as a call costs less than a helper's calls would
    sig = (q.shape, q.dtype, q.get_device(), q.stride(), k.shape, k.dtype, k.get_device(), k.stride(),
           positions.shape, positions.dtype, positions.get_device(), positions.is_contiguous(),
           turns.shape, turns.dtype, turns.get_device(), turns.is_contiguous(), interleaved, magnitude, eps,
           None if q_weight is None else (q_weight.shape, q_weight.dtype, q_weight.get_device(), q_weight.is_contiguous()),
           None if k_weight is None else (k_weight.shape, k_weight.dtype, k_weight.get_device(), k_weight.is_contiguous()),
           None if cu_q_lens is None else (cu_q_lens.shape, cu_q_lens.dtype, cu_q_lens.get_device(), cu_q_lens.is_contiguous()),
           None if num_seqs is None else (num_seqs.shape, num_seqs.dtype, num_seqs.get_device(), num_seqs.is_contiguous()),
           None if dropped is None else (dropped.shape, dropped.dtype, dropped.get_device(), dropped.is_contiguous()),
           None if out is None else (out[0].shape, out[0].dtype, out[0].get_device(), out[0].stride(),
                                     out[1].shape, out[1].dtype, out[1].get_device(), out[1].stride()))
    plan = _plans.get(sig)
    if plan is None:
        i32 = torch.int32
        if q.dim() != 3:
            raise ValueError(f"q must be [tokens, heads, head_dim], got {tuple(q.shape)}")
        device, tokens, dim = q.device, q.shape[0], q.shape[2]
        _tensor("q", q, torch.bfloat16, (tokens, None, dim), None, rows=True)
        _tensor("k", k, torch.bfloat16, (tokens, None, dim), device, rows=True)
        _tensor("positions", positions, i32, (tokens,), device)
        _tensor("turns", turns, torch.int64, (None,), device)
        weights = [_weight("q_weight", q_weight, q.shape[1], dim, device), _weight("k_weight", k_weight, k.shape[1], dim, device)]
        if weights[0] and weights[1] and weights[0][0] != weights[1][0]:
            raise ValueError(f"q_weight dtype {weights[0][0]} and k_weight dtype {weights[1][0]} must be the same")
        if (cu_q_lens is None) != (num_seqs is None):
            raise ValueError("cu_q_lens and num_seqs come together")
        if dropped is not None and cu_q_lens is None:
            raise ValueError("dropped needs cu_q_lens and num_seqs")
        n = 0
        if cu_q_lens is not None:
            _tensor("cu_q_lens", cu_q_lens, i32, (None,), device)
            n = cu_q_lens.shape[0] - 1
            if n < 1:
                raise ValueError("cu_q_lens must have at least two entries")
            _tensor("num_seqs", num_seqs, i32, (1,), device)
            if dropped is not None:
                _tensor("dropped", dropped, i32, (n,), device)
        if not (isinstance(interleaved, bool) and isinstance(magnitude, float) and isinstance(eps, float)):
            raise ValueError("interleaved must be a bool, magnitude and eps floats")
        if 2 * turns.shape[0] > dim or 2 * turns.shape[0] % (2 if interleaved else 8):
            raise ValueError(f"{turns.shape[0]} turns for pairs of {dim} dims: twice as many must be a multiple of "
                             f"{2 if interleaved else 8} of at most {dim}")
        if out is not None:
            for name, t, like in (("out q", out[0], q), ("out k", out[1], k)):
                _tensor(name, t, torch.bfloat16, like.shape, device, rows=True)
        q_out, k_out = (q.new_empty(q.shape), k.new_empty(k.shape)) if out is None else out
        dtype = next((w[0] for w in weights if w), torch.bfloat16)
        shape = _bounded_lib.RpaRotateShape(
            tokens, q.shape[1], k.shape[1], dim, 2 * turns.shape[0], int(interleaved), n, dtype.itemsize, q.stride(0), q.stride(1),
            k.stride(0), k.stride(1), q_out.stride(0), q_out.stride(1), k_out.stride(0), k_out.stride(1),
            weights[0][1] if weights[0] else 0, weights[1][1] if weights[1] else 0)
        if len(_plans) > 256:
            _plans.clear()
        plan = _plans[sig] = (shape, _bounded_lib.load().rpa_rotate_heads)
    shape, fn = plan
    dev = q.get_device()
    if out is None:
        out = q.new_empty(q.shape), k.new_empty(k.shape)
    else:
        ins = {"q": q, "k": k, "positions": positions, "turns": turns, "q_weight": q_weight, "k_weight": k_weight,
               "cu_q_lens": cu_q_lens, "num_seqs": num_seqs, "dropped": dropped}
        for name, t in (("out q", out[0]), ("out k", out[1])):
            if t.is_contiguous() and not any(t.data_ptr() == x.data_ptr() for x in (q, k)):  # in place: the library's checks
                _separate(name, t, ins)
    if dev != _get_device():
        with torch.cuda.device(dev):
            return rotate_heads(q, k, positions, turns, interleaved=interleaved, magnitude=magnitude, q_weight=q_weight,
                                k_weight=k_weight, eps=eps, cu_q_lens=cu_q_lens, num_seqs=num_seqs, dropped=dropped, out=out)
    rc = fn(shape, eps, magnitude, q.data_ptr(), k.data_ptr(), positions.data_ptr(), turns.data_ptr(),
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
            None if cu_q_lens is None else cu_q_lens.data_ptr(), None if num_seqs is None else num_seqs.data_ptr(),
            None if dropped is None else dropped.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), _current_stream(dev))
    if rc:
        _bounded_lib.check(rc)
    return tuple(out)
