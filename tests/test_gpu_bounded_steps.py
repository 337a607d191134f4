"""A serving loop with a bounded cache: rotation, append, weighed attention, eviction and pages together, against a host
model that keeps each head's keys as a plain list."""

import numpy as np
import pytest
import torch

from oracle import bounded_oracle as orc
from tpu_cake_amd import eviction, paging, rotary, sparse

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, PAGE = 8, 2, 64, 16
BUDGET, RECENT, SINKS, LIMIT = 40, 12, 2, 48


def _i32(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda")


def test_a_serving_loop(cuda):
    rng = np.random.default_rng(0)
    n, pps, total, room = 5, 8, 40, 96
    pool = torch.zeros((total, PAGE, 2 * HKV, DIM), dtype=torch.bfloat16, device="cuda")
    ledger = eviction.make_ledger(pool)
    table, stack = _i32(np.zeros((n, pps))), _i32(rng.permutation(total))
    lens, dropped, count = _i32(np.zeros(n)), _i32(np.zeros(n)), _i32([total])
    turns = rotary.turns_of(rotary.frequencies(DIM))
    whole = [t % (1 << 64) for t in turns.tolist()]
    weight = torch.from_numpy(rng.uniform(0.5, 1.5, DIM).astype(np.float32)).cuda()
    # the model: for each sequence and head {position: (key, value, weight)} as the pool holds them
    model = [[{} for _ in range(HKV)] for _ in range(n)]
    seen = np.zeros(n, np.int64)
    for step in range(30):
        new = rng.integers(1, 3, n) if step else np.array([30, 70, 5, 1, 44]) // 2
        meta = paging.assign_pages(lens, _i32(new), table, stack, count, page_size=PAGE, max_tokens=room)
        tokens = int(meta.cu_q_lens[-1])
        assert tokens == new.sum()
        qkv = torch.from_numpy(rng.standard_normal((room, HQ + 2 * HKV, DIM), np.float32)).to(torch.bfloat16).cuda()
        q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
        raw_q, raw_k = q.double().cpu().numpy(), k.double().cpu().numpy()
        rotary.rotate_heads(q, k, meta.positions, turns, q_weight=weight, k_weight=weight, cu_q_lens=meta.cu_q_lens,
                            num_seqs=meta.num_seqs, dropped=dropped, out=(q, k))
        sparse.append_kv(k, v, pool, meta.slot_mapping)
        out = eviction.weighed_attention(q, pool, ledger, meta.kv_lens, table, meta.cu_q_lens, meta.num_seqs, dropped=dropped,
                                         sm_scale=DIM ** -0.5)
        # positions: those of the whole sequence, whatever the cache has lost
        at = np.concatenate([np.arange(s, s + m) for s, m in zip(seen, new)])
        for got, raw in ((q, raw_q), (k, raw_k)):
            want, size = orc.rotate_heads(raw[:tokens], at, whole, weight=weight.double().cpu().numpy())
            assert (np.abs(got[:tokens].double().cpu().numpy() - want) <= 2.0**-8 * np.abs(want) + 2.0**-19 * size).all()
            assert np.array_equal(got[tokens:].double().cpu().numpy(), raw[tokens:])
        kk, vv, qq = (x[:tokens].double().cpu().numpy() for x in (k, v, q))
        cu = np.concatenate([[0], np.cumsum(new)])
        got = out.double().cpu().numpy()
        for i in range(n):
            for h in range(HKV):
                cache = model[i][h]
                for t in range(cu[i], cu[i + 1]):
                    cache[int(at[t])] = [kk[t, h], vv[t, h], 0.0]
                order = sorted(cache)
                if not order:
                    continue
                keys, values = np.stack([cache[p][0] for p in order]), np.stack([cache[p][1] for p in order])
                for t in range(cu[i], cu[i + 1]):
                    s = qq[t, h * 4:h * 4 + 4] @ keys.T / 8
                    s[:, np.array(order) > at[t]] = -np.inf
                    w = np.exp(s - s.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    want = w @ values
                    # 2^-8 for the rounding, 2^-15 for scores of 64 products and sums of up to 100 keys in 32 bits
                    assert (np.abs(got[t, h * 4:h * 4 + 4] - want) <= 2.0**-8 * np.abs(want) + 2.0**-15).all()
                    for p, x in zip(order, w.sum(0)):
                        cache[p][2] += x
        assert not out[tokens:].any()
        seen += new
        moves = eviction.choose_moves(ledger, meta.kv_lens, table, meta.num_seqs, budget=BUDGET, recent=RECENT, sinks=SINKS,
                                      limit=LIMIT, dropped=dropped)
        eviction.move_rows(pool, ledger, moves)
        lens, dropped, count = paging.trim_pages(meta.kv_lens, dropped, table, stack, meta.free_count, page_size=PAGE, budget=BUDGET,
                                                 limit=LIMIT)
        held, gone, t = lens.cpu().numpy(), dropped.cpu().numpy(), table.cpu().numpy()
        assert np.array_equal(held + gone, seen)
        pages = np.concatenate([t[i, :-(-int(held[i]) // PAGE)] for i in range(n)] + [stack.cpu().numpy()[:count.item()]])
        assert sorted(pages.tolist()) == list(range(total))  # no page is lost, none is held twice
        weights, places = ledger.weights.double().cpu().numpy(), ledger.positions.cpu().numpy()
        rows = pool.view(total, PAGE, HKV, 2, DIM).double().cpu().numpy()
        for i in range(n):
            page, off = t[i, np.arange(held[i]) // PAGE], np.arange(held[i]) % PAGE
            for h in range(HKV):
                cache = model[i][h]
                stay = [int(p) for p in places[page, h, off]]
                assert len(set(stay)) == len(stay) == held[i] and set(stay) <= set(cache)
                if len(cache) > LIMIT:
                    forced = {p for p in cache if p < SINKS or p >= seen[i] - RECENT}
                    assert forced <= set(stay)
                    # the others: none that went weighs more than one that stayed
                    least = min([cache[p][2] for p in stay if p not in forced])
                    assert all(cache[p][2] <= least + 1e-4 for p in cache if p not in set(stay))
                else:
                    assert set(stay) == set(cache)
                for p, kx, vx, w in zip(stay, rows[page, off, h, 0], rows[page, off, h, 1], weights[page, h, off]):
                    assert np.array_equal(kx, cache[p][0]) and np.array_equal(vx, cache[p][1]) and abs(w - cache[p][2]) < 1e-4
                model[i][h] = {p: cache[p] for p in stay}


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_a_captured_step(cuda, kind):
    """A decode step with everything in one graph, replayed, against the same calls made one by one on a second cache."""
    rng = np.random.default_rng(1)
    n, pps, total = 6, 6, 40
    fp8 = kind == "fp8"
    turns = rotary.turns_of(rotary.frequencies(DIM))
    held = rng.integers(20, 48, n)
    start = torch.from_numpy(rng.standard_normal((total, PAGE, 2 * HKV, DIM), np.float32)).cuda().to(torch.float8_e4m3fn if fp8 else torch.bfloat16)
    order = rng.permutation(total)
    pages, rows = -(-held // PAGE), np.zeros((n, pps), np.int64)
    for i, at in enumerate(np.cumsum(pages) - pages):
        rows[i, :pages[i]] = order[at:at + pages[i]]
    used = int(pages.sum())

    class Side:
        def __init__(self):
            self.pool = start.clone()
            self.ledger = eviction.make_ledger(self.pool)
            self.scales = torch.full((total, HKV, 2), 0.5, device="cuda") if fp8 else None
            self.table, self.stack = _i32(rows), _i32(np.concatenate([order[used:][::-1], np.zeros(used)]))
            self.lens, self.dropped, self.count = _i32(held), _i32(np.zeros(n)), _i32([total - used])
            self.qkv = torch.zeros((n, HQ + 2 * HKV, DIM), dtype=torch.bfloat16, device="cuda")
            self.out = torch.zeros((n, HQ, DIM), dtype=torch.bfloat16, device="cuda")

        def step(self):
            meta = paging.assign_pages(self.lens, torch.ones_like(self.lens), self.table, self.stack, self.count, page_size=PAGE, max_tokens=n)
            q, k, v = self.qkv[:, :HQ], self.qkv[:, HQ:HQ + HKV], self.qkv[:, HQ + HKV:]
            rotary.rotate_heads(q, k, meta.positions, turns, cu_q_lens=meta.cu_q_lens, num_seqs=meta.num_seqs, dropped=self.dropped, out=(q, k))
            sparse.append_kv(k, v, self.pool, meta.slot_mapping, **(dict(kv_scales=self.scales) if fp8 else {}))
            eviction.weighed_attention(q, self.pool, self.ledger, meta.kv_lens, self.table, meta.cu_q_lens, meta.num_seqs,
                                       dropped=self.dropped, sm_scale=0.125, kv_scales=self.scales, out=self.out)
            moves = eviction.choose_moves(self.ledger, meta.kv_lens, self.table, meta.num_seqs, budget=BUDGET, recent=RECENT, sinks=SINKS,
                                          limit=LIMIT, dropped=self.dropped, max_moves=16)
            eviction.move_rows(self.pool, self.ledger, moves, kv_scales=self.scales)
            lens, dropped, count = paging.trim_pages(meta.kv_lens, self.dropped, self.table, self.stack, meta.free_count, page_size=PAGE,
                                                     budget=BUDGET, limit=LIMIT)
            self.lens.copy_(lens), self.dropped.copy_(dropped), self.count.copy_(count)

        def state(self):
            return [self.pool.view(torch.uint8), *self.ledger, self.table, self.stack, self.lens, self.dropped, self.count, self.out]

    warm, graphed, eager = Side(), Side(), Side()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        warm.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        graphed.step()
    for turn in range(30):
        x = torch.from_numpy(rng.standard_normal((n, HQ + 2 * HKV, DIM), np.float32)).to(torch.bfloat16).cuda()
        graphed.qkv.copy_(x), eager.qkv.copy_(x)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphed.state(), eager.state())), turn
    assert bool((eager.dropped > 0).all())
    assert eviction.read_error_word(clear=True) == 0 and paging.read_error_word(clear=True) == 0


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_a_pool_past_32_bits(cuda, kind):
    """The last pages of a pool of more than 2^32 values, against the same pages in a small one."""
    rng = np.random.default_rng(2)
    fp8 = kind == "fp8"
    held, new = np.array([700, 333, 60]), np.array([1, 40, 1])
    pages = -(-held // 64)
    small, shift = int(pages.sum()), 140000
    table = np.zeros((3, int(pages.max())), np.int64)
    for i, at in enumerate(np.cumsum(pages) - pages):
        table[i, :pages[i]] = rng.permutation(pages[i]) + at
    values = torch.from_numpy(rng.standard_normal((small, 64, 4, 128), np.float32)).cuda().to(torch.float8_e4m3fn if fp8 else torch.bfloat16)
    q = torch.from_numpy(rng.standard_normal((42, 8, 128), np.float32)).to(torch.bfloat16).cuda()
    got = []
    for first in (0, shift):
        pool = torch.empty((first + small, 64, 4, 128), dtype=values.dtype, device="cuda")
        pool[first:] = values
        scales = torch.full((first + small, 2, 2), 0.25, device="cuda") if fp8 else None
        ledger = eviction.make_ledger(pool)
        at = _i32(table + first)
        out = eviction.weighed_attention(q, pool, ledger, _i32(held), at, _i32([0, 1, 41, 42]), _i32([3]), sm_scale=0.1, kv_scales=scales)
        moves = eviction.choose_moves(ledger, _i32(held), at, _i32([3]), budget=50, recent=10, sinks=2)
        eviction.move_rows(pool, ledger, moves, kv_scales=scales)
        got.append((out, torch.where(moves < 0, moves, moves - first * 64), *(x[first:].clone() for x in (pool.view(torch.uint8), *ledger))))
        assert not first or pool.numel() > 2**32
        del pool
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert eviction.read_error_word(clear=True) == 0
