"""A serving step with a bounded cache, as measured cases: norms and position rotation of a step's queries and keys
(``rotary``), attention that keeps account of the weight each cached key got, the choice of the keys that go when a
sequence outgrows its budget, the moves that close the gaps (``eviction``), and the pages that become free (``paging``).

``run`` computes them in plain torch operations, or (``own``) with the package's entry points.  A case fixes every size
(lengths come from ``len_seed``); values and page orders come from the seed given to ``prepare``.

The ledger of a pool holds, for each slot and kv head, the weight that attention gave the key there so far and the
position of its token: float32 and int32 [pages, kv heads, page size].
"""

import functools
import math
import pathlib
import sys

import numpy as np
import torch

own = False

FP8_MAX = 448.0

# the most one pass of a listed case reads, computes, and holds in its plain form: drawn cases stay below
MAX_BYTES = 1.6e9
MAX_FLOPS = 320e9
MAX_HELD = 3.3e9


@functools.lru_cache(None)
def _package():
    path = str(pathlib.Path(__file__).resolve().parent.parent / "tpu-cake_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tpu_cake_amd import eviction, paging, rotary
    return rotary, eviction, paging


# ------------------------------------------------------------------------------------------ cases
def _rotate(name, **sizes):
    """Queries and keys of ``decode`` sequences of one token, then ``chunks`` of 1..chunk_hi, slices of one projection's output."""
    case = dict(kind="rotate", decode=0, chunks=0, chunk_hi=1, len_hi=1 << 20, dropped_hi=0, hq=32, hkv=8, dim=128, rotated=128,
                interleaved=False, norm=True, factor=1.0, magnitude=1.0, pad=0, len_seed=311)
    case.update(sizes)
    return dict(case, name=name) if name else case


def _weigh(name, **sizes):
    """Queries of ``decode`` sequences of one token, then ``chunks`` sequences of ``chunk`` tokens, over len_lo..len_hi keys."""
    case = dict(kind="weigh", decode=0, chunks=0, chunk=1, len_lo=1, len_hi=512, dropped_hi=0, hq=32, hkv=8, dim=128, page=64,
                dtype="bf16", soft_cap=0.0, decay=1.0, len_seed=312)
    case.update(sizes)
    return dict(case, name=name) if name else case


def _evict(kind, name, **sizes):
    """``requests`` sequences of len_lo..len_hi keys, those longer than ``limit`` cut to ``budget``."""
    case = dict(kind=kind, requests=64, len_lo=1, len_hi=2112, budget=2048, limit=2048, sinks=4, recent=256, max_moves=64,
                dropped_hi=100000, hkv=8, dim=128, page=64, dtype="bf16", len_seed=313)
    case.update(sizes)
    return dict(case, name=name) if name else case


def listed():
    return [
        # a decode step's 64 tokens far into long contexts, 32 query heads on 8 kv heads, every head normed
        _rotate("rotate_decode", decode=64, dropped_hi=200000),
        # prompt chunks of odd lengths beside decode rows, half of each head rotated, in pairs, angles scaled for long
        # contexts, the batch padded to its bucket
        _rotate("rotate_prompt", decode=24, chunks=12, chunk_hi=1400, hq=64, rotated=64, interleaved=True, norm=False, factor=8.0,
                magnitude=1.2, pad=29, len_seed=314),
        # the smallest attention: four short sequences on a model shard, page 16
        _weigh("weigh_short", decode=4, hq=8, hkv=2, page=16),
        # decode over contexts of uneven length, weights accumulated
        _weigh("weigh_decode", decode=64, len_lo=1024, len_hi=8192, dropped_hi=30000, hq=64),
        # two users with a quarter of a million keys each in an fp8 pool, pages of 16: few rows, a long axis, weights that fade
        _weigh("weigh_long_fp8", decode=2, len_lo=240000, len_hi=250000, page=16, dtype="fp8", decay=0.9),
        # two prompts' chunks over their earlier keys beside decode rows: every chunk's tokens weigh the whole prompt
        _weigh("weigh_chunk", decode=5, chunks=2, chunk=777, len_lo=6000, len_hi=16384, decay=0.0, len_seed=315),
        # the steady state of decode: requests a page past their budget give up 64 keys of each head
        _evict("choose", "choose_decode", len_lo=2000),
        # long prompts cut to a budget, each head its own keys
        _evict("choose", "choose_long", requests=3, len_lo=100000, len_hi=131072, budget=4096, limit=4096, max_moves=4096, page=16,
               dropped_hi=1),
        # decode's moves: at most 64 rows of each head
        _evict("move", "move_decode", len_lo=2000),
        # a prompt's moves in an fp8 pool: most of the budget, between pages of other scales
        _evict("move", "move_prompt_fp8", requests=6, len_lo=20000, len_hi=32768, max_moves=2048, dropped_hi=1, dtype="fp8"),
        # a decode step's pages: latency is all
        _evict("trim", "trim_decode", len_lo=2000),
        # thousands of requests, some hundred prompts cut at once, pages of 16
        _evict("trim", "trim_burst", requests=4096, len_hi=20000, budget=1024, limit=1040, page=16),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread evenly over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS and _held(case) <= MAX_HELD:
            return case


def _draw(rng):
    seed = rng.randrange(1 << 30)
    kind = rng.choice(["rotate", "rotate", "weigh", "weigh", "weigh", "choose", "move", "trim"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 24])
    hkv = rng.choice([1, 2, 4, 8, 8])
    hq = hkv * rng.choice([1, 4, 4, 8, 8, 16])
    dim = rng.choice([64, 128, 128, 128, 256, 96])
    dtype = rng.choice(["bf16", "bf16", "fp8"])
    chunks = rng.choice([0, 0, 1, 2, 5])
    if kind == "rotate":
        return _rotate(None, decode=_log(rng, 1, 512) if not chunks else rng.randrange(32), chunks=chunks,
                       chunk_hi=_log(rng, 2, 3000), len_hi=_log(rng, 1000, 1 << 20), dropped_hi=rng.choice([0, 1 << 16]), hq=hq,
                       hkv=hkv, dim=dim, rotated=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.4,
                       norm=rng.random() < 0.6, factor=rng.choice([1.0, 1.0, 8.0]), magnitude=rng.choice([1.0, 1.0, 1.2]),
                       pad=rng.choice([0, rng.randrange(40)]), len_seed=seed)
    if kind == "weigh":
        hi = _log(rng, 200, 100000)
        return _weigh(None, decode=_log(rng, 1, 96) if not chunks else rng.randrange(8), chunks=chunks, chunk=_log(rng, 2, 1000),
                      len_lo=max(1, int(hi * rng.choice([0.01, 0.3, 0.9]))), len_hi=hi, dropped_hi=rng.choice([0, 1 << 16]), hq=hq,
                      hkv=hkv, dim=dim, page=page, dtype=dtype, soft_cap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                      decay=rng.choice([0.0, 0.9, 1.0, 1.0]), len_seed=seed)
    budget = _log(rng, 64, 4096)
    over = rng.choice([1, page, _log(rng, 1, 30000)])
    limit = budget + rng.choice([0, 0, page // 2])
    requests = _log(rng, 1, 4096 if kind == "trim" else 64)
    return _evict(kind, None, requests=requests, len_lo=rng.choice([1, budget // 2 + 1, budget + 1]), len_hi=budget + over,
                  budget=budget, limit=limit, sinks=rng.choice([0, 4, 16]), recent=rng.choice([0, 1, budget // 8, budget // 2]),
                  max_moves=min(budget, over), dropped_hi=rng.choice([1, 1, 100000]), hkv=hkv, dim=dim, page=page, dtype=dtype,
                  len_seed=seed)


def _lengths(case):
    """(kv_lens, q_lens) of the case's sequences, kv_lens with the step's new tokens in them."""
    r = np.random.RandomState(case["len_seed"])
    if case["kind"] == "rotate":
        q = np.concatenate([np.ones(case["decode"], np.int64), r.randint(1, case["chunk_hi"] + 1, case["chunks"])]).astype(np.int64)
        return q + r.randint(0, case["len_hi"], len(q)), q
    n = case["requests"] if "requests" in case else case["decode"] + case["chunks"]
    q = np.ones(n, np.int64)
    if case["kind"] == "weigh":
        q[case["decode"]:] = case["chunk"]
    lens = np.exp(r.uniform(math.log(case["len_lo"]), math.log(case["len_hi"]), n)).astype(np.int64)
    return np.maximum(lens, q), q


def _dropped(case):
    """How many earlier tokens of each sequence are gone."""
    r = np.random.RandomState(case["len_seed"] + 1)
    return r.randint(0, max(1, case["dropped_hi"]), len(_lengths(case)[0]))


def _held(case):
    """Values that the plain form of a call holds at once."""
    if case["kind"] == "rotate":
        return 0
    kv, q = _lengths(case)
    if case["kind"] == "trim":
        return len(kv) * int(kv.max()) // case["page"]
    if case["kind"] != "weigh":
        return len(kv) * int(kv.max()) * case["hkv"]
    return len(kv) * int(kv.max()) * max(int(q.max()) * case["hq"], 2 * case["hkv"] * case["dim"])


def work(case):
    kind = case["kind"]
    kv, q = _lengths(case)
    if kind == "rotate":
        tokens, heads = int(q.sum()), case["hq"] + case["hkv"]
        return {"bytes": 4 * tokens * heads * case["dim"] + 4 * tokens + 4 * case["rotated"] + (8 * case["dim"] if case["norm"] else 0)
                + 12 * len(kv), "flops": tokens * heads * (3 * case["rotated"] + (4 * case["dim"] if case["norm"] else 0))}
    page, hkv = case["page"], case["hkv"]
    elem = 1 if case["dtype"] == "fp8" else 2
    if kind == "weigh":
        hq, dim = case["hq"], case["dim"]
        keys, tokens, pages = int(kv.sum()), int(q.sum()), int((-(-kv // page)).sum())
        pairs = sum(int(n) * (2 * int(k) - int(n) + 1) // 2 for k, n in zip(kv, q))
        return {"bytes": keys * hkv * (2 * dim * elem + (8 if case["decay"] else 4)) + tokens * (4 * hq * dim + 4 * hkv) + 4 * pages
                + (8 * pages * hkv if elem == 1 else 0), "flops": 4 * dim * hq * pairs}
    cut = kv > case["limit"]
    if kind == "choose":
        return {"bytes": 8 * hkv * (int(kv[cut].sum()) + len(kv) * case["max_moves"]) + 4 * int((-(-kv // page))[cut].sum()), "flops": 0}
    if kind == "move":
        # of the keys that are neither first nor last any may go: the share of a budget's rows that are filled from behind it
        free = np.maximum(kv - case["sinks"] - case["recent"], 1)
        moves = int(np.minimum((kv - case["budget"]) * (case["budget"] - case["sinks"]) / free, case["max_moves"])[cut].sum()) * hkv
        return {"bytes": moves * (4 * case["dim"] * elem + 16) + 8 * len(kv) * hkv * case["max_moves"], "flops": 0}
    freed = int((-(-kv // page) - -(-case["budget"] // page))[cut].sum())
    return {"bytes": 16 * len(kv) + 8 * freed + 8, "flops": 0}


# ----------------------------------------------------------------------------------------- inputs
def _int(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda")


def _table(r, pages, total):
    """Rows of distinct random pages out of ``total``, zero past each row's own."""
    order = r.permutation(total)[:int(pages.sum())]
    width = int(pages.max())
    table = np.zeros((len(pages), width), np.int64)
    table[np.arange(width)[None, :] < pages[:, None]] = order
    return table


def _pool(case, total, g):
    """A pool of normal values: bf16, or fp8 codes with a scale for each page, head and of K and V."""
    shape = (total, case["page"], 2 * case["hkv"], case["dim"])
    if case["dtype"] == "bf16":
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g), None
    scales = torch.empty((total, case["hkv"], 2), device="cuda").uniform_(0.008, 0.012, generator=g)
    codes = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0.0, 100.0, generator=g)
    return codes.clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scales


def _frequencies(case):
    """Radians a position for each rotated pair; the slow ones stretched for long contexts, the fast ones as they are."""
    half = case["rotated"] // 2
    f = 10000.0 ** (-np.arange(half, dtype=np.float64) / half)
    keep = np.clip((8192 * f / (2 * math.pi) - 1) / (32 - 1), 0.0, 1.0)
    return f * keep + f / case["factor"] * (1 - keep)


def prepare(case, seed):
    r = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    kv, q = _lengths(case)
    cu = np.concatenate([[0], np.cumsum(q)])
    state = dict(case=case, lens=_int(kv), cu=_int(cu), num=_int([len(kv)]), dropped=_int(_dropped(case)))
    if kind == "rotate":
        hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
        tokens = int(q.sum()) + case["pad"]
        qkv = torch.empty((tokens, hq + 2 * hkv, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        at = np.zeros(tokens, np.int64)
        at[:int(q.sum())] = np.concatenate([np.arange(k - n, k) for k, n in zip(kv, q)])
        f = _frequencies(case)
        turns = np.array([round(x / (2 * math.pi) * 2.0**64) % (1 << 64) for x in f.tolist()], np.uint64).view(np.int64)
        weights = [torch.empty(dim, dtype=torch.bfloat16, device="cuda").normal_(1.0, 0.1, generator=g) if case["norm"] else None
                   for _ in range(2)]
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], at=_int(at), frequencies=torch.as_tensor(f, device="cuda"),
                     turns=torch.as_tensor(turns, device="cuda"), q_weight=weights[0], k_weight=weights[1])
        return state
    hkv, page = case["hkv"], case["page"]
    pages = -(-kv // page)
    total = int(pages.sum() * 1.1) + 1
    table = _table(r, pages, total)
    state["table"] = _int(table)
    if kind == "trim":
        free = np.setdiff1d(np.arange(total), table[np.arange(table.shape[1])[None, :] < pages[:, None]])
        stack = np.zeros(total, np.int64)
        stack[:len(free)] = r.permutation(free)
        state.update(free=_int(stack), count=_int([len(free)]))
        return state
    # what earlier steps left: weights as sums of small probabilities, few of them large, and a position for each row
    weights = torch.empty((total, hkv, page), device="cuda").exponential_(generator=g).square_().mul_(0.01)
    positions = torch.zeros((total, hkv, page), dtype=torch.int32, device="cuda")
    state.update(weights=weights, positions=positions)
    if kind == "weigh":
        state["pool"], state["scales"] = _pool(case, total, g)
        state["q"] = torch.empty((int(cu[-1]), case["hq"], case["dim"]), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        return state
    # rows hold tokens in the order that earlier evictions left, each head its own
    slot, inside = _slots(state)
    width = slot.shape[2]
    order = torch.empty((len(kv), hkv, width), device="cuda").uniform_(generator=g)
    order = torch.where(inside, order, 2.0).argsort(-1).argsort(-1).to(torch.int32)
    fresh = torch.arange(width, dtype=torch.int32, device="cuda").expand_as(order)
    gone = state["dropped"][:, None, None] > 0
    held = torch.where(gone, order + state["dropped"][:, None, None], fresh)
    first = (order < case["sinks"]) & gone
    held = torch.where(first, order, held)
    _put(positions, slot, inside, held)
    if kind == "move":
        state["pool"], state["scales"] = _pool(case, total, g)
        state["moves"] = _plain_choose(state)
    return state


# ------------------------------------------------------------------------------------ plain forms
def _slots(s):
    """For each sequence, head and row: the row's place in a ledger, and whether there is one."""
    page, hkv = s["case"]["page"], s["case"]["hkv"]
    row = torch.arange(s["table"].shape[1] * page, device="cuda")
    pages = s["table"].long()[:, row // page]
    head = torch.arange(hkv, device="cuda")[None, :, None]
    inside = (row[None, None, :] < s["lens"].long()[:, None, None]).expand(-1, hkv, -1)
    return (pages[:, None, :] * hkv + head) * page + row % page, inside


def _put(ledger, slot, inside, values):
    """Writes ``values`` to the slots inside the sequences."""
    flat = torch.cat([ledger.flatten(), ledger.new_zeros(1)])
    flat[torch.where(inside, slot, ledger.numel())] = values.to(ledger.dtype)
    ledger.copy_(flat[:-1].view_as(ledger))


def _owners(s, tokens):
    """Each token's sequence, and whether it has one."""
    token = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(s["cu"].long()[1:], token, right=True)
    return seq.clamp(max=s["lens"].numel() - 1), token < s["cu"].long()[-1]


def _plain_rotate(s):
    case = s["case"]
    half = case["rotated"] // 2
    seq, live = _owners(s, s["q"].shape[0])
    at = s["at"].long() + s["dropped"].long()[seq]
    angle = at[:, None, None].double() * s["frequencies"]
    cos, sin = (torch.cos(angle) * case["magnitude"]).float(), (torch.sin(angle) * case["magnitude"]).float()
    got = []
    for x, weight in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        turned, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = turned[..., :half], turned[..., half:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        got.append(torch.where(live[:, None, None], torch.cat([turned, rest], -1), 0.0).to(torch.bfloat16))
    return dict(q=got[0], k=got[1])


def _plain_weigh(s):
    case = s["case"]
    hkv, page = case["hkv"], case["page"]
    tokens, hq, dim = s["q"].shape
    lens, cu = s["lens"].long(), s["cu"].long()
    n, group, most = len(lens), hq // hkv, case["chunk"] if case["chunks"] else 1
    slot, inside = _slots(s)
    rows = slot.shape[2]
    row = torch.arange(rows, device="cuda")
    pages = s["table"].long()[:, row // page]                            # [N, L]
    held = s["pool"].view(torch.uint8) if s["scales"] is not None else s["pool"]
    kv = held.view(-1, hkv, 2, dim)[pages * page + row % page].view(s["pool"].dtype).float()
    if s["scales"] is not None:
        kv = kv * s["scales"][pages][..., None]
    kv = torch.where(inside[:, 0, :, None, None, None], kv, 0.0)
    keys, values = kv[:, :, :, 0].permute(0, 2, 3, 1).contiguous(), kv[:, :, :, 1].transpose(1, 2).contiguous()
    # the sequences' tokens side by side, each in its own row
    step = torch.arange(most, device="cuda")
    token = cu[:-1, None] + step
    mine = token < cu[1:, None]                                          # [N, most]
    q = s["q"][torch.where(mine, token, 0)].float().view(n, most, hkv, group, dim).transpose(1, 2)
    score = torch.matmul(q.reshape(n, hkv, most * group, dim), keys) * dim ** -0.5
    if case["soft_cap"]:
        score = case["soft_cap"] * torch.tanh(score / case["soft_cap"])
    at = lens[:, None] - cu[1:, None] + token
    seen = (mine[:, :, None] & (row <= at[:, :, None]))[:, None, :, None].expand(-1, -1, -1, group, -1).reshape(n, 1, most * group, rows)
    score = torch.where(seen, score, float("-inf"))
    weight = torch.where(seen, torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30)), 0.0)
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    result = torch.matmul(weight, values).view(n, hkv, most, group, dim).transpose(1, 2).reshape(n * most, hq, dim)
    out = torch.zeros((tokens + 1, hq, dim), device="cuda")
    out[torch.where(mine, token, tokens).flatten()] = result
    # the ledger: keys of this step start anew
    new = (row >= (lens - cu[1:] + cu[:-1])[:, None])[:, None]
    old = s["weights"].flatten()[slot]
    old = torch.where(new, 0.0, old * case["decay"])
    _put(s["weights"], slot, inside, old + weight.sum(2))
    known = s["positions"].flatten()[slot]
    _put(s["positions"], slot, inside, torch.where(new, s["dropped"][:, None, None] + row.to(torch.int32), known))
    return dict(out=out[:-1].to(torch.bfloat16), weights=s["weights"], positions=s["positions"])


def _plain_choose(s):
    case = s["case"]
    hkv, page, budget, most = case["hkv"], case["page"], case["budget"], case["max_moves"]
    slot, inside = _slots(s)
    n, _, rows = slot.shape
    end = (s["lens"] + s["dropped"])[:, None, None]
    position = s["positions"].flatten()[slot]
    kept_anyway = (position < case["sinks"]) | (position >= end - case["recent"])
    key = torch.where(kept_anyway, float("inf"), s["weights"].flatten()[slot])
    key = torch.where(inside, key, float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.zeros((n, hkv, rows), dtype=torch.bool, device="cuda").scatter_(2, order, True)
    row = torch.arange(rows, device="cuda")
    cut = (s["lens"] > case["limit"])[:, None, None]
    # the i-th kept row past the budget takes the place of the i-th row before it that goes
    place = s["table"].long()[:, row // page] * page + row % page
    moves = torch.full((n, hkv, most + 1, 2), -1, dtype=torch.int32, device="cuda")
    count = None
    for side, which in ((1, kept & cut & (row >= budget)), (0, ~kept & cut & (row < budget))):
        rank = torch.cumsum(which, -1) - 1
        count = which.sum(-1) if count is None else count
        rank = torch.where(which & (rank < count[..., None]), rank, most).clamp(max=most)
        moves[..., side].scatter_(2, rank, place[:, None].expand(-1, hkv, -1).to(torch.int32))
    return moves[:, :, :most].contiguous()


def _plain_move(s):
    case = s["case"]
    hkv, page, dim = case["hkv"], case["page"], case["dim"]
    to, origin = s["moves"].long().unbind(-1)                            # [N, Hkv, M]
    head = torch.arange(hkv, device="cuda")[None, :, None].expand_as(to)
    live = to >= 0
    held = torch.uint8 if s["scales"] is not None else torch.bfloat16
    pool = s["pool"].view(held).view(-1, hkv, 2 * dim)
    safe_to, safe = torch.where(live, to, 0), torch.where(live, origin, 0)
    rows = pool[safe, head]                                              # [N, Hkv, M, 2 D]
    if s["scales"] is not None:
        values = rows.view(torch.float8_e4m3fn).float().view(*to.shape, 2, dim) * s["scales"][safe // page, head][..., None]
        values = (values / s["scales"][safe_to // page, head][..., None]).clamp(-FP8_MAX, FP8_MAX)
        rows = values.to(torch.float8_e4m3fn).view(held).view(*to.shape, 2 * dim)
    # entries that name no move write a row of their own head, unchanged, to a place past the pool
    spare = torch.cat([pool, pool[:1]])
    spare[torch.where(live, to, pool.shape[0]), head] = rows
    pool.copy_(spare[:-1])
    for ledger in (s["weights"], s["positions"]):
        flat = torch.cat([ledger.flatten(), ledger.new_zeros(1)])
        values = flat[(safe // page * hkv + head) * page + safe % page]
        flat[torch.where(live, (safe_to // page * hkv + head) * page + safe_to % page, ledger.numel())] = values
        ledger.copy_(flat[:-1].view_as(ledger))
    return dict(pool=s["pool"], weights=s["weights"], positions=s["positions"])


def _plain_trim(s):
    case = s["case"]
    page, budget = case["page"], case["budget"]
    lens, table, count = s["lens"].long(), s["table"].long(), s["count"].long()
    cut = lens > case["limit"]
    keep = (budget + page - 1) // page
    back = torch.where(cut, (lens + page - 1) // page - keep, 0)
    ends = torch.cumsum(back, 0)
    place = torch.arange(s["free"].numel(), device="cuda") - count
    owner = torch.searchsorted(ends, place, right=True).clamp(max=len(lens) - 1)
    given = table[owner, (keep + place - (ends - back)[owner]).clamp(0, table.shape[1] - 1)]
    free = torch.where((place >= 0) & (place < ends[-1]), given, s["free"].long())
    whole = lambda x: x.to(torch.int32)  # noqa: E731
    return dict(lens=whole(torch.where(cut, budget, lens)), dropped=whole(s["dropped"] + torch.where(cut, lens - budget, 0)),
                count=whole(count + ends[-1]), free=whole(free))


# ---------------------------------------------------------------------------------------- one pass
def _own(s):
    rotary, eviction, paging = _package()
    case = s["case"]
    kind = case["kind"]
    if kind == "rotate":
        q, k = rotary.rotate_heads(s["q"], s["k"], s["at"], s["turns"], interleaved=case["interleaved"], magnitude=case["magnitude"],
                                   q_weight=s["q_weight"], k_weight=s["k_weight"], dropped=s["dropped"], cu_q_lens=s["cu"],
                                   num_seqs=s["num"])
        return dict(q=q, k=k)
    if kind == "trim":
        lens, dropped, count = paging.trim_pages(s["lens"], s["dropped"], s["table"], s["free"], s["count"], page_size=case["page"],
                                                 budget=case["budget"], limit=case["limit"])
        return dict(lens=lens, dropped=dropped, count=count, free=s["free"])
    ledger = eviction.Ledger(s["weights"], s["positions"])
    if kind == "weigh":
        out = eviction.weighed_attention(s["q"], s["pool"], ledger, s["lens"], s["table"], s["cu"], s["num"], dropped=s["dropped"],
                                         sm_scale=case["dim"] ** -0.5, soft_cap=case["soft_cap"] or None, decay=case["decay"],
                                         kv_scales=s["scales"])
        return dict(out=out, weights=s["weights"], positions=s["positions"])
    if kind == "choose":
        return eviction.choose_moves(ledger, s["lens"], s["table"], s["num"], dropped=s["dropped"], budget=case["budget"],
                                     limit=case["limit"], sinks=case["sinks"], recent=case["recent"], max_moves=case["max_moves"])
    eviction.move_rows(s["pool"], ledger, s["moves"], kv_scales=s["scales"])
    return dict(pool=s["pool"], weights=s["weights"], positions=s["positions"])


def run(state):
    if own:
        return _own(state)
    return {"rotate": _plain_rotate, "weigh": _plain_weigh, "choose": _plain_choose, "move": _plain_move,
            "trim": _plain_trim}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------ in 64 bits
def _exact_rotate(s):
    case = s["case"]
    cu, dropped, f = s["cu"].tolist(), s["dropped"].tolist(), _frequencies(case)
    at = s["at"].cpu().numpy().astype(np.float64)
    for i, d in enumerate(dropped):
        at[cu[i]:cu[i + 1]] += d
    z = torch.as_tensor(np.exp(1j * at[:, None] * f[None, :]) * case["magnitude"], device="cuda")[:, None]
    got = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * w.double()
        r = case["rotated"]
        even, odd = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        turned = torch.complex(y[..., even], y[..., odd]) * z
        y[..., even], y[..., odd] = turned.real, turned.imag
        y[cu[-1]:] = 0
        got.append(y)
    return dict(q=got[0], k=got[1])


def _exact_weigh(s):
    case = s["case"]
    page, hkv = case["page"], case["hkv"]
    lens, cu, dropped = s["lens"].tolist(), s["cu"].tolist(), s["dropped"].tolist()
    tokens, hq, dim = s["q"].shape
    group = hq // hkv
    out = torch.zeros((tokens, hq, dim), dtype=torch.float64, device="cuda")
    weights, positions = s["weights"].double(), s["positions"].clone()
    pool = s["pool"].view(torch.uint8) if s["scales"] is not None else s["pool"]
    for i, n in enumerate(lens):
        first = n - (cu[i + 1] - cu[i])
        ids = s["table"][i, :-(-n // page)].long()
        for h in range(hkv):
            rows = pool[ids][:, :, 2 * h:2 * h + 2].contiguous().view(s["pool"].dtype).double()
            if s["scales"] is not None:
                rows = rows * s["scales"][ids, h].double()[:, None, :, None]
            k, v = rows.permute(2, 0, 1, 3).reshape(2, -1, dim)[:, :n]
            got = weights[ids, h].flatten()
            got[:n] *= case["decay"]
            got[first:n] = 0
            for t0 in range(cu[i], cu[i + 1], 256):
                t1 = min(t0 + 256, cu[i + 1])
                q = s["q"][t0:t1, h * group:(h + 1) * group].double()
                score = (q.reshape(-1, dim) @ k.T.contiguous()).view(t1 - t0, group, n) / math.sqrt(dim)
                if case["soft_cap"]:
                    score = case["soft_cap"] * torch.tanh(score / case["soft_cap"])
                late = torch.arange(n, device="cuda") > first + torch.arange(t0 - cu[i], t1 - cu[i], device="cuda")[:, None, None]
                p = torch.softmax(score.masked_fill(late, float("-inf")), -1)
                out[t0:t1, h * group:(h + 1) * group] = (p.view(-1, n) @ v).view(t1 - t0, group, dim)
                got[:n] += p.sum((0, 1))
            weights[ids, h] = got.view(-1, page)
            there = positions[ids, h].flatten()
            there[first:n] = torch.arange(first + dropped[i], n + dropped[i], device="cuda", dtype=torch.int32)
            positions[ids, h] = there.view(-1, page)
    return dict(out=out, weights=weights, positions=positions)


def _exact_choose(s):
    case = s["case"]
    page, budget = case["page"], case["budget"]
    weights, positions = s["weights"].cpu().numpy(), s["positions"].cpu().numpy()
    table, lens, dropped = (s[k].cpu().numpy().astype(np.int64) for k in ("table", "lens", "dropped"))
    moves = np.full((len(lens), case["hkv"], case["max_moves"], 2), -1, np.int32)
    for i in np.nonzero(lens > case["limit"])[0]:
        n = int(lens[i])
        ids = table[i, :-(-n // page)]
        slots = (ids[:, None] * page + np.arange(page)).reshape(-1)
        for h in range(case["hkv"]):
            w, p = weights[ids, h].reshape(-1)[:n].astype(np.float64), positions[ids, h].reshape(-1)[:n]
            safe = (p < case["sinks"]) | (p >= n + dropped[i] - case["recent"])
            kept = np.zeros(n, bool)
            kept[np.lexsort((np.arange(n), -w, ~safe))[:budget]] = True
            late, holes = np.nonzero(kept[budget:])[0] + budget, np.nonzero(~kept[:budget])[0]
            moves[i, h, :len(late), 0], moves[i, h, :len(late), 1] = slots[holes], slots[late]
    return moves


def _exact_move(s):
    """The pool's values before their rounding; the ledger is carried over as it is."""
    case = s["case"]
    page, hkv, dim = case["page"], case["hkv"], case["dim"]
    pool = s["pool"].double()
    rows = pool.view(-1, hkv, 2, dim)
    weights, positions = s["weights"].double(), s["positions"].clone()
    for h in range(hkv):
        list_of = s["moves"][:, h].reshape(-1, 2).long()
        to, origin = list_of[list_of[:, 0] >= 0].unbind(1)
        x = rows[origin, h]
        if s["scales"] is not None:
            there, here = s["scales"].double()[origin // page, h], s["scales"].double()[to // page, h]
            x = (x * (there / here)[..., None]).clamp(-FP8_MAX, FP8_MAX)
        rows[to, h] = x
        for ledger in (weights, positions):
            ledger[to // page, h, to % page] = ledger[origin // page, h, origin % page]
    return dict(pool=pool, weights=weights, positions=positions)


def _exact_trim(s):
    case = s["case"]
    page, budget = case["page"], case["budget"]
    lens, dropped, table, free = (s[k].cpu().numpy().copy() for k in ("lens", "dropped", "table", "free"))
    count = int(s["count"])
    for i in np.nonzero(lens > case["limit"])[0]:
        back = table[i, -(-budget // page):-(-int(lens[i]) // page)]
        free[count:count + len(back)] = back
        count += len(back)
        dropped[i] += lens[i] - budget
        lens[i] = budget
    return dict(lens=lens, dropped=dropped, count=np.array([count], np.int32), free=free)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "weigh": _exact_weigh, "choose": _exact_choose, "move": _exact_move,
            "trim": _exact_trim}[case["kind"]](s)
