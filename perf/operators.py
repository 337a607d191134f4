"""Long-context serving over a paged K/V pool, as measured cases: the page allocator and its step
metadata (``paging``), the write of new keys and values with the page index, the choice of pages for
each query and the attention over the chosen pages (``sparse``).

``run`` computes them in plain torch operations, or (``own``) with the package's entry points.  A
case fixes every size (lengths come from ``len_seed``); values and page orders come from the seed
given to ``prepare``.

The page index keeps, for each page and kv head, the largest and smallest value of every dimension
of the page's keys on a grid of 2^e: e is the smallest whole number in [-100, 100] with
127 * 2^e >= the largest magnitude, the largest values are rounded up and the smallest down, both
clamped to +-127.  Rounding to power-of-two grids is exact, and so is a score from them: the index
and the chosen pages are whole numbers that do not depend on an order of summation.
"""

import functools
import math
import pathlib
import sys

import numpy as np
import torch

own = False

FP8_MAX = 448.0
EXP_MIN, EXP_MAX = -100, 100

# the most one pass of a listed case reads and computes, and gathers in its plain form: drawn cases stay below
MAX_BYTES = 540e6
MAX_FLOPS = 17.5e9
MAX_GATHER = 1.1e9


@functools.lru_cache(None)
def _package():
    path = str(pathlib.Path(__file__).resolve().parent.parent / "tpu-cake_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tpu_cake_amd import paging, sparse
    return paging, sparse


# ------------------------------------------------------------------------------------------ cases
def _paging(name, **sizes):
    """One step of the allocator: finished requests give their pages back, the others get theirs."""
    case = dict(kind="paging", requests=64, page=64, pages_per_seq=128, chunk_share=0.0, chunk_hi=1, finished_share=0.1,
                spare_tokens=0, len_seed=211)
    case.update(sizes)
    return dict(case, name=name) if name else case


def _append(name, **sizes):
    """New keys and values of ``decode`` sequences of one token and ``chunks`` sequences of chunk_lo..chunk_hi."""
    case = dict(kind="append", decode=0, chunks=0, chunk_lo=1, chunk_hi=1, len_hi=4096, hq=32, hkv=8, dim=128, page=64,
                dtype="bf16", pad=0, len_seed=212)
    case.update(sizes)
    return dict(case, name=name) if name else case


def _reads(kind, name, **sizes):
    """Queries of ``decode`` sequences of one token, then ``chunks`` sequences of ``chunk`` tokens, over len_lo..len_hi
    keys, and ``top`` pages for each of them."""
    case = dict(kind=kind, decode=0, chunks=0, chunk=1, len_lo=1, len_hi=512, hq=32, hkv=8, dim=128, page=64, top=32,
                dtype="bf16", soft_cap=0.0, len_seed=213)
    case.update(sizes)
    return dict(case, name=name) if name else case


def listed():
    return [
        # a decode step's metadata: one token a request, a new page now and then; latency is all
        _paging("step_decode"),
        # thousands of requests, hundreds of them with prompt chunks, pages of 16
        _paging("step_burst", requests=4096, page=16, pages_per_seq=2048, chunk_share=0.06, chunk_hi=512, spare_tokens=999),
        # a decode step's keys and values, slices of one projection's output, into a bf16 pool
        _append("append_decode", decode=64),
        # prompt chunks of odd lengths beside decode rows into an fp8 pool, the batch padded to its bucket
        _append("append_prompt_fp8", decode=24, chunks=12, chunk_lo=333, chunk_hi=1000, dtype="fp8", pad=29, len_seed=214),
        # the smallest choice: four short sequences on a model shard, page 16
        _reads("select", "select_short", decode=4, hq=8, hkv=2, page=16, top=8),
        # decode over long contexts
        _reads("select", "select_decode", decode=64, len_lo=4096, len_hi=65536, hq=64),
        # two users with half a million keys each, pages of 16: few rows, a long axis
        _reads("select", "select_long", decode=2, len_lo=480000, len_hi=500000, page=16, top=128),
        # a prompt's chunk over its earlier keys: every token chooses for itself
        _reads("select", "select_chunk", decode=5, chunks=1, chunk=1000, len_lo=20000, len_hi=32768),
        # the smallest attention: four short sequences on a model shard, page 16
        _reads("attend", "attend_short", decode=4, hq=8, hkv=2, page=16, top=8),
        # decode over long contexts, 2048 keys for each row
        _reads("attend", "attend_decode", decode=64, len_lo=4096, len_hi=16384, hq=64),
        # two users, an fp8 pool with pages of 16: few rows, split over their keys
        _reads("attend", "attend_long_fp8", decode=2, len_lo=480000, len_hi=500000, page=16, top=128, dtype="fp8"),
        # a prompt's chunk: neighbouring tokens mostly choose the same pages
        _reads("attend", "attend_chunk", decode=5, chunks=1, chunk=500, len_lo=20000, len_hi=32768),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS and _gathered(case) <= MAX_GATHER:
            return case


def _draw(rng):
    seed = rng.randrange(1 << 30)
    kind = rng.choice(["paging", "append", "append", "select", "select", "attend", "attend", "attend"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 24])
    hkv = rng.choice([1, 2, 4, 8, 8])
    hq = hkv * rng.choice([1, 4, 4, 8, 8, 16])
    dim = rng.choice([64, 128, 128, 128, 256, 96])
    dtype = rng.choice(["bf16", "bf16", "fp8"])
    if kind == "paging":
        return _paging(None, requests=_log(rng, 1, 4096), page=page, pages_per_seq=_log(rng, 64, 2048),
                       chunk_share=rng.choice([0.0, 0.0, 0.05, 0.3]), chunk_hi=_log(rng, 2, 512),
                       finished_share=rng.choice([0.0, 0.1, 0.3]), spare_tokens=rng.randrange(100), len_seed=seed)
    if kind == "append":
        chunks = rng.choice([0, _log(rng, 1, 12)])
        return _append(None, decode=_log(rng, 1, 256) if not chunks else rng.randrange(32), chunks=chunks, chunk_lo=1,
                       chunk_hi=_log(rng, 2, 1000), len_hi=_log(rng, 256, 8192), hq=hq, hkv=hkv, dim=dim, page=page,
                       dtype=dtype, pad=rng.choice([0, rng.randrange(40)]), len_seed=seed)
    hi = _log(rng, 200, 200000)
    chunks = rng.choice([0, 0, 1, 2])
    sizes = dict(decode=_log(rng, 1, 96) if not chunks else rng.randrange(8), chunks=chunks, chunk=_log(rng, 2, 500),
                 len_lo=max(1, int(hi * rng.choice([0.01, 0.3, 0.9]))), len_hi=hi, hq=hq, hkv=hkv, dim=dim, page=page,
                 top=_log(rng, 4, 128), len_seed=seed)
    if kind == "attend":
        sizes.update(dtype=dtype, soft_cap=rng.choice([0.0, 0.0, 0.0, 30.0]))
    return _reads(kind, None, **sizes)


def _lengths(case):
    """(kv_lens, q_lens) of the case's sequences, kv_lens with the step's new tokens in them."""
    r = np.random.RandomState(case["len_seed"])
    if case["kind"] == "append":
        q = np.concatenate([np.ones(case["decode"], np.int64),
                            r.randint(case["chunk_lo"], case["chunk_hi"] + 1, case["chunks"])]).astype(np.int64)
        return q + r.randint(0, case["len_hi"], len(q)), q
    n = case["decode"] + case["chunks"]
    q = np.concatenate([np.ones(case["decode"], np.int64), np.full(case["chunks"], case["chunk"], np.int64)])
    lens = np.exp(r.uniform(math.log(case["len_lo"]), math.log(case["len_hi"]), n)).astype(np.int64)
    return np.maximum(lens, q), q


def _requests(case):
    """(cached lengths, new tokens, finished) of the allocator's requests: finished ones get no token in this step."""
    r = np.random.RandomState(case["len_seed"])
    n, cap = case["requests"], case["pages_per_seq"] * case["page"]
    chunk = r.rand(n) < case["chunk_share"]
    new = np.where(chunk, r.randint(1, case["chunk_hi"] + 1, n), 1)
    new[r.rand(n) < 0.02] = 0
    cached = r.randint(0, max(1, min(cap // 2, 40 * case["page"])), n)
    finished = r.rand(n) < case["finished_share"]
    new[finished] = 0
    new = np.minimum(new, cap - cached)
    return cached.astype(np.int64), new.astype(np.int64), finished


def _gathered(case):
    """Values that the plain form of a choice or an attention gathers."""
    if case["kind"] not in ("select", "attend"):
        return 0
    kv, q = _lengths(case)
    pages = -(-int(kv.max()) // case["page"])
    if case["kind"] == "select":
        return int(q.sum()) * pages * case["hkv"] * 2 * case["dim"]
    return int(q.sum()) * min(case["top"], pages) * case["page"] * case["hkv"] * case["dim"]


def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "paging":
        cached, new, finished = _requests(case)
        freed = int((-(-cached // page))[finished].sum())
        got = int((-(-(cached + new) // page) - -(-cached // page))[~finished].sum())
        tokens = int(new.sum()) + case["spare_tokens"]
        return {"bytes": 4 * (2 * len(new) + 2) + len(new) + 8 * freed + 8 * got + 8 * (len(new) + 1) + 8 * tokens, "flops": 0}
    d, hkv, hq = case["dim"], case["hkv"], case["hq"]
    elem = 1 if case["dtype"] == "fp8" else 2
    kv, q = _lengths(case)
    if kind == "append":
        touched = int((-(-kv // page) - (kv - q) // page).sum())
        opened = int((-(-kv // page) - -(-(kv - q) // page)).sum())
        tokens = int(q.sum())
        return {"bytes": tokens * hkv * 2 * d * (2 + elem) + (2 * touched - opened) * hkv * (2 * d + 1) + 4 * tokens
                + (8 * touched * hkv if elem == 1 else 0), "flops": 0}
    tokens, pages = int(q.sum()), -(-kv // page)
    if kind == "select":
        rows = sum(int((np.arange(k - n, k) // page + 1).sum()) for k, n in zip(kv.tolist(), q.tolist()))
        return {"bytes": int(pages.sum()) * (hkv * (2 * d + 1) + 4) + tokens * (hq * d * 2 + hkv * case["top"] * 4),
                "flops": 4 * d * hq * rows}
    seen = sum(int(np.minimum(np.arange(k - n, k) // page + 1, case["top"]).sum()) for k, n in zip(kv.tolist(), q.tolist()))
    read = sum(min(int(p), case["top"] if n == 1 else 2 * case["top"]) for p, n in zip(pages, q.tolist()))
    return {"bytes": read * page * hkv * 2 * d * elem + tokens * (2 * hq * d * 2 + hkv * case["top"] * 4)
            + (8 * read * hkv if elem == 1 else 0), "flops": 4 * d * hq * seen * page}


# ----------------------------------------------------------------------------------------- inputs
def _int(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda")


def _table(r, pages, width, total):
    """Rows of distinct random pages out of ``total``, zero past each row's own."""
    order = r.permutation(total)[:int(pages.sum())]
    table = np.zeros((len(pages), width), np.int64)
    table[np.arange(width)[None, :] < pages[:, None]] = order
    return table


def _batch(case, r):
    """The step's metadata: kv_lens, page_indices, cu_q_lens, num_seqs, and the pages of the pool."""
    kv, q = _lengths(case)
    pages = -(-kv // case["page"])
    total = int(pages.sum() * 1.25) + 1
    table = _table(r, pages, int(pages.max()), total)
    cu = np.concatenate([[0], np.cumsum(q)])
    return kv, q, table, cu, total


def _pool(case, total, g):
    """A pool of normal values: bf16, or fp8 codes with a scale for each page, head and of K and V."""
    shape = (total, case["page"], 2 * case["hkv"], case["dim"])
    if case["dtype"] == "bf16":
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g), None
    scales = torch.empty((total, case["hkv"], 2), device="cuda").uniform_(0.008, 0.012, generator=g)
    codes = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0.0, 100.0, generator=g)
    return codes.clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scales


def _index(page_dims, g):
    """A page index as the keys' statistics leave it: largest values around +2.4, smallest around -2.4."""
    total, hkv, dim = page_dims
    exps = torch.randint(-6, -4, (total, hkv), device="cuda", dtype=torch.int8, generator=g)
    mid = torch.randint(40, 110, (total, hkv, 2, dim), device="cuda", dtype=torch.int8, generator=g)
    mid[:, :, 1] *= -1
    return mid, exps


def prepare(case, seed):
    r = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, page = case["kind"], case["page"]
    if kind == "paging":
        cached, new, finished = _requests(case)
        pages = -(-cached // page)
        got = int((-(-(cached + new) // page) - pages).sum())
        spare = got + len(cached)
        total = int(pages.sum()) + spare
        table = _table(r, pages, case["pages_per_seq"], total)
        free = np.setdiff1d(np.arange(total), table[np.arange(table.shape[1])[None, :] < pages[:, None]])
        stack = np.zeros(total, np.int64)
        stack[:len(free)] = r.permutation(free)
        return dict(case=case, cached=_int(cached), new=_int(new), finished=torch.as_tensor(finished, device="cuda"),
                    table=_int(table), free=_int(stack), count=_int([len(free)]),
                    max_tokens=int(new.sum()) + case["spare_tokens"])
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    kv, q, table, cu, total = _batch(case, r)
    if kind == "append":
        tokens = int(q.sum())
        at = np.concatenate([np.arange(k - n, k) for k, n in zip(kv, q)])
        seq = np.repeat(np.arange(len(q)), q)
        slots = np.concatenate([table[seq, at // page] * page + at % page, np.full(case["pad"], -1)])
        pool, scales = _pool(case, total, g)
        bounds, exps = _index((total, hkv, dim), g)
        qkv = torch.empty((tokens + case["pad"], hq + 2 * hkv, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        return dict(case=case, k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], pool=pool, scales=scales, slots=_int(slots),
                    bounds=bounds, exps=exps)
    queries = torch.empty((int(cu[-1]), hq, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    state = dict(case=case, q=queries, lens=_int(kv), table=_int(table), cu=_int(cu), num=_int([len(kv)]))
    if kind == "select":
        state["bounds"], state["exps"] = _index((total, hkv, dim), g)
        return state
    state["pool"], state["scales"] = _pool(case, total, g)
    # the pages of a choice: mostly the sequence's own favourites, some of the token's, and the newest
    seq = torch.as_tensor(np.repeat(np.arange(len(q)), q), device="cuda")
    last = torch.as_tensor(np.concatenate([np.arange(k - n, k) for k, n in zip(kv, q)]) // page, device="cuda")[:, None, None]
    liked = torch.empty((len(kv), hkv, table.shape[1]), device="cuda").uniform_(generator=g)[seq]
    liked += 0.05 * torch.empty_like(liked).uniform_(generator=g)
    at = torch.arange(table.shape[1], device="cuda")[None, None, :]
    liked = torch.where(at > last, -1.0, torch.where(at == last, 2.0, liked))
    best = torch.topk(liked, min(case["top"], table.shape[1]), dim=-1)
    picked = torch.where(best.values >= 0, best.indices, 1 << 30).sort(dim=-1).values
    picked = torch.where(picked == 1 << 30, -1, picked)
    state["picked"] = torch.nn.functional.pad(picked, (0, case["top"] - picked.shape[-1]), value=-1).to(torch.int32).contiguous()
    return state


# ------------------------------------------------------------------------------------ plain forms
def _plain_paging(s):
    page, device = s["case"]["page"], "cuda"
    cached, table, count = s["cached"].long(), s["table"].long(), s["count"].long()
    n, width = table.shape
    # finished requests give their pages back, in order
    pages = (cached + page - 1) // page
    back = torch.where(s["finished"], pages, 0)
    ends = torch.cumsum(back, 0)
    place = torch.arange(s["free"].numel(), device=device) - count
    owner = torch.searchsorted(ends, place, right=True).clamp(max=n - 1)
    given = table[owner, (place - (ends - back)[owner]).clamp(0, width - 1)]
    free = torch.where((place >= 0) & (place < ends[-1]), given, s["free"].long())
    count = count + ends[-1]
    cached = torch.where(s["finished"], 0, cached)
    # the others' new tokens, in order, as far as pages and tokens go
    new = s["new"].long()
    pages = (cached + page - 1) // page
    valid = (cached >= 0) & (new >= 0) & (cached + new <= width * page)
    need = torch.where(valid, (cached + new + page - 1) // page - pages, 0)
    new = torch.where(valid, new, 0)
    taken = torch.cumsum(need, 0)
    admitted = valid & (torch.cumsum(new, 0) <= s["max_tokens"]) & ((need == 0) | (taken <= count))
    need, first = torch.where(admitted, need, 0), taken - need
    tokens = torch.where(admitted, new, 0)
    cu = torch.nn.functional.pad(torch.cumsum(tokens, 0), (1, 0))
    column = torch.arange(width, device=device)[None, :] - pages[:, None]
    source = (count - 1 - first[:, None] - column).clamp(0, free.numel() - 1)
    table = torch.where((column >= 0) & (column < need[:, None]), free[source], table)
    token = torch.arange(s["max_tokens"], device=device)
    owner = torch.searchsorted(cu[1:], token, right=True).clamp(max=n - 1)
    at = cached[owner] + token - cu[owner]
    inside = token < cu[-1]
    at = torch.where(inside, at, 0)
    slots = torch.where(inside, table[owner, at // page] * page + at % page, -1)
    whole = lambda x: x.to(torch.int32)  # noqa: E731
    return dict(kv_lens=whole(cached + tokens), cu_q_lens=whole(cu), slots=whole(slots), positions=whole(at), table=whole(table),
                free=whole(free), count=whole(count - need.sum(0, keepdim=True)))


def _exponent(amax):
    """The smallest e in [-100, 100] with 127 * 2^e >= amax."""
    mantissa, e = torch.frexp(amax)  # amax = mantissa * 2^e, mantissa in [0.5, 1)
    e = torch.where(mantissa * 128 > 127, e - 6, e - 7)
    return torch.where(amax > 0, e.clamp(EXP_MIN, EXP_MAX), EXP_MIN)


def _on_grid(x, e):
    return torch.ldexp(x, -e)


def _plain_append(s):
    page, hkv = s["case"]["page"], s["case"]["hkv"]
    pool, slots = s["pool"], s["slots"].long()
    total, dim = pool.shape[0], pool.shape[3]
    kept = (slots >= 0)[:, None, None]
    rows = torch.where(slots >= 0, slots, slots[0])  # padding repeats the first token
    k, v = torch.where(kept, s["k"], s["k"][:1]).float(), torch.where(kept, s["v"], s["v"][:1]).float()
    at = rows // page
    if s["scales"] is not None:
        scale = s["scales"][at]
        k = (k / scale[:, :, :1]).clamp(-FP8_MAX, FP8_MAX)
        v = (v / scale[:, :, 1:]).clamp(-FP8_MAX, FP8_MAX)
    new = torch.stack([k, v], 2).reshape(len(rows), 2 * hkv, dim).to(pool.dtype)
    held = torch.uint8 if pool.element_size() == 1 else torch.bfloat16
    pool.view(held).view(total * page, 2 * hkv, dim)[rows] = new.view(held)
    keys = new.view(-1, hkv, 2, dim)[:, :, 0].float()
    if s["scales"] is not None:
        keys = keys * scale[:, :, :1]
    # a page whose first row is written starts anew; the others widen
    fresh = torch.zeros(total, dtype=torch.int32, device="cuda").index_reduce(0, at, (rows % page == 0).int(), "amax")[:, None] > 0
    old = torch.where(fresh, EXP_MIN, s["exps"].int())
    exps = old.index_reduce(0, at, _exponent(keys.abs().amax(-1)), "amax")
    grid = exps[at][:, :, None]
    high, low = (torch.ceil(_on_grid(keys, grid)).clamp(-127, 127), torch.floor(_on_grid(keys, grid)).clamp(-127, 127))
    step = (old - exps)[:, :, None].clamp(min=-30)
    was = torch.where(fresh[:, :, None, None], torch.tensor([-127.0, 127.0], device="cuda")[:, None], s["bounds"].float())
    was = torch.where(fresh[:, :, None, None], was, torch.stack([torch.ceil(torch.ldexp(was[:, :, 0], step)),
                                                                torch.floor(torch.ldexp(was[:, :, 1], step))], 2))
    bounds = torch.stack([was[:, :, 0].index_reduce(0, at, high, "amax"), was[:, :, 1].index_reduce(0, at, low, "amin")], 2)
    return dict(pool=pool, bounds=bounds.to(torch.int8), exps=exps.to(torch.int8))


def _tokens(s):
    """Each token's sequence and position."""
    cu = s["cu"].long()
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], token, right=True).clamp(max=cu.numel() - 2)
    return seq, s["lens"].long()[seq] - (cu[seq + 1] - token)


def _plain_select(s):
    case = s["case"]
    hkv, top = case["hkv"], case["top"]
    seq, at = _tokens(s)
    tokens, hq, dim = s["q"].shape
    q = s["q"].float().view(tokens, hkv, hq // hkv, dim)
    f = _exponent(q.abs().amax((2, 3)))[:, :, None, None]
    q = torch.round(_on_grid(q, f)).clamp(-127, 127)
    q = torch.cat([q.clamp(min=0), q.clamp(max=0)], -1)
    pages = s["table"].long()[seq]                                       # [T, width]
    bounds = s["bounds"][pages].permute(0, 2, 1, 3, 4).reshape(tokens, hkv, -1, 2 * dim).float()
    score = torch.matmul(bounds, q.transpose(2, 3).contiguous()).amax(-1)  # whole numbers below 2^24
    score = torch.ldexp(score, s["exps"][pages].permute(0, 2, 1).int())
    column = torch.arange(pages.shape[1], device="cuda")[None, :]
    last = (at // case["page"])[:, None]
    forced = (column == 0) | (column == last)
    score = torch.where(forced[:, None, :], float("inf"), score)
    score = torch.where((column > last)[:, None, :], float("-inf"), score)
    best = torch.sort(score, dim=-1, descending=True, stable=True)
    far = pages.shape[1]
    picked = torch.where(best.values[..., :top] > float("-inf"), best.indices[..., :top], far).sort(dim=-1).values
    picked = torch.where(picked == far, -1, picked)
    return torch.nn.functional.pad(picked, (0, top - picked.shape[-1]), value=-1).to(torch.int32)


def _plain_attend(s):
    case = s["case"]
    hkv, page, top = case["hkv"], case["page"], case["top"]
    seq, at = _tokens(s)
    tokens, hq, dim = s["q"].shape
    picked = s["picked"].long()
    pages = s["table"].long()[seq[:, None, None], picked.clamp(min=0)]
    head = torch.arange(hkv, device="cuda")[:, None]
    held = s["pool"].view(torch.uint8) if s["scales"] is not None else s["pool"]
    kv = held.view(-1, page, hkv, 2, dim)[pages, :, head].view(s["pool"].dtype)  # [T, Hkv, top, page, 2, D]
    k, v = kv[..., 0, :].float(), kv[..., 1, :].float()
    if s["scales"] is not None:
        scale = s["scales"][pages, head][..., None, None, :]
        k, v = k * scale[..., 0], v * scale[..., 1]
    k, v = k.view(tokens, hkv, top * page, dim), v.view(tokens, hkv, top * page, dim)
    q = s["q"].float().view(tokens, hkv, hq // hkv, dim).transpose(2, 3).contiguous()
    score = torch.matmul(k, q).transpose(2, 3) * dim ** -0.5
    if case["soft_cap"]:
        score = case["soft_cap"] * torch.tanh(score / case["soft_cap"])
    where = (picked[..., None] * page + torch.arange(page, device="cuda")).view(tokens, hkv, 1, top * page)
    seen = (picked >= 0)[..., None].expand(-1, -1, -1, page).reshape(tokens, hkv, 1, top * page) & (where <= at[:, None, None, None])
    score = torch.where(seen, score, float("-inf"))
    weight = torch.where(seen, torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30)), 0.0).contiguous()
    out = torch.matmul(weight, v) / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.view(tokens, hq, dim).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------- one pass
def _own(s):
    paging, sparse = _package()
    case = s["case"]
    if case["kind"] == "paging":
        cached, count = paging.release_pages(s["cached"], s["finished"], s["table"], s["free"], s["count"], page_size=case["page"])
        step = paging.assign_pages(cached, s["new"], s["table"], s["free"], count, page_size=case["page"],
                                   max_tokens=s["max_tokens"])
        return dict(kv_lens=step.kv_lens, cu_q_lens=step.cu_q_lens, slots=step.slot_mapping, positions=step.positions,
                    table=s["table"], free=s["free"], count=step.free_count)
    if case["kind"] == "append":
        index = sparse.PageIndex(s["bounds"], s["exps"])
        sparse.append_kv(s["k"], s["v"], s["pool"], s["slots"], kv_scales=s["scales"], index=index)
        return dict(pool=s["pool"], bounds=s["bounds"], exps=s["exps"])
    if case["kind"] == "select":
        return sparse.select_pages(s["q"], sparse.PageIndex(s["bounds"], s["exps"]), s["lens"], s["table"], s["cu"], s["num"],
                                   page_size=case["page"], num_pages=case["top"])
    return sparse.sparse_paged_attention(s["q"], s["pool"], s["picked"], s["lens"], s["table"], s["cu"], s["num"],
                                         sm_scale=case["dim"] ** -0.5, soft_cap=case["soft_cap"] or None,
                                         kv_scales=s["scales"])


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "paging":
        return _plain_paging(state)
    if kind == "append":
        return _plain_append(state)
    return _plain_select(state) if kind == "select" else _plain_attend(state)


# --------------------------------------------------------------------------- in 64 bits, on the host
def _exact_paging(s):
    page, top = s["case"]["page"], s["max_tokens"]
    cached, new, fin, table, free = (s[k].cpu().numpy().copy() for k in ("cached", "new", "finished", "table", "free"))
    count = int(s["count"])
    for i in np.nonzero(fin)[0]:
        for page_id in table[i, :-(-int(cached[i]) // page)]:
            free[count], count = page_id, count + 1
        cached[i] = 0
    left, pages_seen, tokens_seen = count, 0, 0
    slots, positions, cu = [], [], [0]
    for i, (c, m) in enumerate(zip(cached.tolist(), new.tolist())):
        have, want = -(-c // page), -(-(c + m) // page)
        fits = min(c, m) >= 0 and c + m <= table.shape[1] * page
        if fits:
            pages_seen, tokens_seen = pages_seen + want - have, tokens_seen + m
            fits = tokens_seen <= top and (want == have or pages_seen <= count)
        if fits:
            for j in range(have, want):
                left -= 1
                table[i, j] = free[left]
            for p in range(c, c + m):
                slots.append(int(table[i, p // page]) * page + p % page)
                positions.append(p)
            cached[i] = c + m
        cu.append(len(slots))
    rest = top - len(slots)
    return dict(kv_lens=cached, cu_q_lens=np.array(cu, np.int32), slots=np.array(slots + [-1] * rest, np.int32),
                positions=np.array(positions + [0] * rest, np.int32), table=table, free=free, count=np.array([left], np.int32))


def _exact_append(s):
    """The pool's values before their rounding; the index is whole numbers, compared as such."""
    page, hkv, dim = s["case"]["page"], s["case"]["hkv"], s["case"]["dim"]
    pool = s["pool"].double()
    rows = pool.view(-1, hkv, 2, dim)
    slots = s["slots"].long()
    slots = slots[slots >= 0]
    for part, x in enumerate((s["k"], s["v"])):
        x = x[:len(slots)].double()
        if s["scales"] is not None:
            x = (x / s["scales"].double()[slots // page, :, part][..., None]).clamp(-FP8_MAX, FP8_MAX)
        rows[slots, :, part] = x
    return dict(pool=pool, bounds=None, exps=None)


def _exact_select(s):
    case = s["case"]
    page, hkv, top = case["page"], case["hkv"], case["top"]
    lens, table, cu = (s[k].cpu().numpy().astype(np.int64) for k in ("lens", "table", "cu"))
    tokens, hq, dim = s["q"].shape
    if tokens * hq * table.shape[1] > 2e8:
        return None
    exps, queries = s["exps"].double().cpu().numpy(), s["q"].double().cpu().numpy()
    got = np.full((tokens, hkv, top), -1, np.int32)
    for i in range(len(lens)):
        ids = table[i, :-(-int(lens[i]) // page)]
        large, small = s["bounds"][torch.as_tensor(ids, device="cuda")].double().unbind(2)
        for t in range(int(cu[i]), int(cu[i + 1])):
            visible = (int(lens[i]) - int(cu[i + 1]) + t) // page + 1
            for h in range(hkv):
                x = queries[t, h * (hq // hkv):(h + 1) * (hq // hkv)]
                f = EXP_MIN
                while 127.0 * 2.0 ** f < np.abs(x).max() and f < EXP_MAX:
                    f += 1
                x = torch.as_tensor(np.clip(np.rint(x * 2.0 ** -f), -127, 127), device="cuda")
                s1 = (x.clamp(min=0) @ large[:visible, h].T + x.clamp(max=0) @ small[:visible, h].T).amax(0).cpu().numpy()
                s1 = s1 * 2.0 ** exps[ids[:visible], h]
                s1[0] = s1[visible - 1] = np.inf
                best = np.sort(np.argsort(-s1, kind="stable")[:top])
                got[t, h, :len(best)] = best
    return got


def _exact_attend(s):
    case = s["case"]
    page, hkv = case["page"], case["hkv"]
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    tokens, hq, dim = s["q"].shape
    if tokens > 600:
        return None
    group = hq // hkv
    out = torch.zeros((tokens, hq, dim), dtype=torch.float64, device="cuda")
    pool = s["pool"].view(torch.uint8) if s["scales"] is not None else s["pool"]
    for i, n in enumerate(lens):
        for t in range(cu[i], cu[i + 1]):
            at = n - cu[i + 1] + t
            for h in range(hkv):
                chosen = s["picked"][t, h].long()
                chosen = chosen[chosen >= 0]
                ids = s["table"][i].long()[chosen]
                rows = pool[ids][:, :, 2 * h:2 * h + 2].contiguous().view(s["pool"].dtype).double()
                if s["scales"] is not None:
                    rows = rows * s["scales"][ids, h].double()[:, None, :, None]
                seen = (chosen[:, None] * page + torch.arange(page, device="cuda") <= at).reshape(-1)
                k, v = rows.permute(2, 0, 1, 3).reshape(2, -1, dim)[:, seen]
                score = s["q"][t, h * group:(h + 1) * group].double() @ k.T.contiguous() / math.sqrt(dim)
                if case["soft_cap"]:
                    score = case["soft_cap"] * torch.tanh(score / case["soft_cap"])
                out[t, h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"paging": _exact_paging, "append": _exact_append, "select": _exact_select, "attend": _exact_attend}[case["kind"]](s)
