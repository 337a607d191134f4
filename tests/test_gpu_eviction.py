"""The choice of rows to keep, their moves and the pages back: whole numbers and copies, so equal to the oracles."""

import numpy as np
import pytest
import torch

from oracle import bounded_oracle as orc
from oracle import sparse_oracle
from tests.sparse_cases import i32
from tpu_cake_amd import eviction, paging

pytestmark = pytest.mark.gpu


class Cache:
    def __init__(self, seed, lens, page, hkv, *, ties=False, spare=0, dropped=None):
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.page, self.hkv = np.array(lens), page, hkv
        pages = -(-np.maximum(self.lens, 0) // page)
        self.total = int(pages.sum()) + 3
        self.table = np.zeros((len(lens), int(pages.max(initial=0)) + 2), np.int64)
        order, at = rng.permutation(self.total), 0
        for i, p in enumerate(pages):
            self.table[i, :p] = order[at:at + p]
            at += p
        self.n = len(lens) - spare
        self.dropped = rng.integers(0, 5, len(lens)) * 100 if dropped is None else np.array(dropped)
        shape = (self.total, hkv, page)
        self.weights = (rng.integers(0, 4, shape) / 4 if ties else rng.exponential(1.0, shape)).astype(np.float32)
        self.positions = np.zeros(shape, np.int32)
        for i, n in enumerate(self.lens):
            for h in range(hkv):
                at = np.arange(n) + self.dropped[i]
                if self.dropped[i]:
                    at[:3] = np.arange(3)[:n]
                    rng.shuffle(at)
                self.positions[self.table[i, np.arange(n) // page], h, np.arange(n) % page] = at

    def ledger(self):
        return eviction.Ledger(torch.from_numpy(self.weights).cuda(), torch.from_numpy(self.positions).cuda())

    def choose(self, **kw):
        got = eviction.choose_moves(self.ledger(), i32(self.lens), i32(self.table), i32([self.n]), dropped=i32(self.dropped), **kw)
        want = orc.choose_moves(self.weights, self.positions, self.lens, self.table, self.n, dropped=self.dropped, **kw)
        np.testing.assert_array_equal(got.cpu().numpy(), want)
        return got


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("page,hkv", [(16, 2), (64, 1), (1, 1), (7, 3)])
@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (1, 1, 0), (32, 0, 0), (32, 8, 4), (32, 32, 0), (100, 10, 3), (1000, 500, 4)])
def test_choice(cuda, ties, page, hkv, budget, recent, sinks):
    c = Cache(budget + page, [0, 1, 31, 32, 33, 99, 101, 500, 1001, 2300, 40], page, hkv, ties=ties, spare=1)
    c.choose(budget=budget, recent=recent, sinks=sinks)
    c.choose(budget=budget, recent=recent, sinks=sinks, limit=budget + 68)


def test_long_sequences(cuda):
    c = Cache(1, [70000, 20000, 33000], 16, 1)
    c.choose(budget=4096, recent=64, sinks=4)
    c.choose(budget=19999, recent=64, sinks=4, max_moves=20000)
    c = Cache(2, [50000], 64, 2, ties=True)
    c.choose(budget=3000, recent=64)


@pytest.mark.parametrize("lens,hkv", [([1500] * 20 + [40] * 130, 2), ([9000] + [300] * 140, 2), ([40000] + [500] * 40, 7)])
def test_many_lists(cuda, lens, hkv):
    c = Cache(len(lens), lens, 16, hkv)
    c.choose(budget=200, recent=20, sinks=4, limit=260, max_moves=200)


def test_long_sequences_of_one_weight(cuda):
    """More rows begin with the bound's first digit than LDS holds."""
    c = Cache(7, [40000, 35000], 16, 2)
    c.weights[:] = 0.25
    c.choose(budget=3000, recent=64, sinks=4)
    c.weights.reshape(-1)[::3] = 0.25000003
    c.choose(budget=13500, recent=64, max_moves=13500)


def test_lists_that_are_too_short(cuda):
    c = Cache(3, [300, 120], 16, 2, ties=True)
    eviction.read_error_word(clear=True)
    c.choose(budget=100, recent=10, max_moves=20)  # 120 - 100 suffice for the second, not for the first
    assert eviction.read_error_word(clear=True) == eviction._bounded_lib.ERR_LEN
    c.choose(budget=100, recent=10, max_moves=100)
    assert eviction.read_error_word(clear=True) == 0


def test_weights_that_are_not_numbers(cuda):
    c = Cache(4, [200, 90], 16, 2)
    w = c.weights.reshape(-1)
    for value in (np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5, 1e-45, 3e38):
        w[c.rng.permutation(w.size)[:w.size // 12]] = value
    c.choose(budget=64, recent=5, sinks=2)
    c.weights[:] = np.nan
    c.choose(budget=64, recent=5, sinks=2)
    c.weights[:] = -0.0
    c.weights[::2] = 0.0
    c.choose(budget=64, recent=5, sinks=2)


def test_positions_that_are_all_forced(cuda):
    """A ledger that was never kept (all positions 0): every row is a first one; the lowest stay."""
    c = Cache(5, [200], 16, 1, dropped=[0])
    c.positions[:] = 0
    moves = c.choose(budget=50, recent=5, sinks=3)
    assert bool((moves == -1).all())


def test_bad_pages(cuda):
    c = Cache(6, [200, 100], 16, 2)
    eviction.read_error_word(clear=True)
    table = i32(c.table)
    table[0, 3], table[1, 0] = c.total, -1
    moves = eviction.choose_moves(c.ledger(), i32(c.lens), table, i32([2]), budget=64, recent=8)
    got = moves.cpu().numpy()
    assert ((got >= -1) & (got < c.total * 16)).all() and eviction.read_error_word(clear=True) == eviction._bounded_lib.ERR_PAGE
    # a length past the table
    lens = i32([c.table.shape[1] * 16 + 5, 100])
    moves = eviction.choose_moves(c.ledger(), lens, i32(c.table), i32([2]), budget=64, recent=8)
    assert eviction.read_error_word(clear=True) & eviction._bounded_lib.ERR_LEN


def _pool(c, dim, kind):
    x = c.rng.standard_normal((c.total, c.page, 2 * c.hkv, dim), np.float32)
    if kind == "bf16":
        return torch.from_numpy(x).to(torch.bfloat16), None
    scales = c.rng.uniform(0.005, 0.02, (c.total, c.hkv, 2)).astype(np.float32)
    scales[::3] = scales[0]  # some pages share a scale
    return torch.from_numpy(np.clip(x * 150, -448, 448)).to(torch.float8_e4m3fn), scales


@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (64, "bf16"), (256, "bf16"), (40, "bf16"), (128, "fp8"), (112, "fp8"), (256, "fp8"),
                                      (128, "codes")])
def test_moves(cuda, dim, kind):
    c = Cache(dim, [300, 64, 1000, 5, 129], 16, 3)
    moves = c.choose(budget=128, recent=16, sinks=4)
    pool, scales = _pool(c, dim, "bf16" if kind == "bf16" else "fp8")
    ledger, device = c.ledger(), pool.cuda().view(torch.uint8) if kind == "codes" else pool.cuda()
    use = None if scales is None or kind == "codes" else torch.from_numpy(scales).cuda()
    eviction.move_rows(device, ledger, moves, kv_scales=use)
    raw = pool.view(torch.int16 if kind == "bf16" else torch.uint8).numpy()

    def requantise(rows, h, there, here):
        s = scales[there, h], scales[here, h]
        x = torch.from_numpy(rows.copy()).view(torch.float8_e4m3fn).float().numpy() * s[0][:, None]
        y = torch.from_numpy(np.clip(x / s[1][:, None], np.float32(-448), np.float32(448))).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        return np.where((s[0] == s[1])[:, None], rows, y)

    want = orc.move_rows(raw, c.weights, c.positions, moves.cpu().numpy(), None if use is None else requantise)
    np.testing.assert_array_equal(device.view(torch.int16 if kind == "bf16" else torch.uint8).cpu().numpy(), want[0])
    np.testing.assert_array_equal(ledger.weights.cpu().numpy(), want[1])
    np.testing.assert_array_equal(ledger.positions.cpu().numpy(), want[2])
    again = device.clone()
    eviction.move_rows(device, ledger, moves, kv_scales=use)  # moves read and write apart: once more changes nothing
    assert torch.equal(again.view(torch.uint8), device.view(torch.uint8))


def test_codes_that_are_not_numbers_or_too_large(cuda):
    """NaN stays NaN and what passes the grid saturates."""
    pool = torch.zeros((2, 16, 2, 64), dtype=torch.uint8)
    pool[0, 0, 0, :4] = torch.tensor([0x7F, 0xFF, 0x7E, 0xFE], dtype=torch.uint8)  # NaN, -NaN, 448, -448
    pool[0, 0, 1, :2] = torch.tensor([0x38, 0xB8], dtype=torch.uint8)              # 1, -1
    scales = torch.tensor([[[1.0, 1.0]], [[0.25, 2.0]]]).cuda()
    ledger = eviction.make_ledger(pool)
    ledger = eviction.Ledger(ledger.weights.cuda(), ledger.positions.cuda())
    moves = i32([[[[16, 0], [-1, -1], [5, -1], [-7, 3]]]])
    pool = pool.cuda()
    eviction.move_rows(pool, ledger, moves, kv_scales=scales)
    got = pool[1, 0].view(torch.float8_e4m3fn).float().cpu()
    assert bool(got[0, :2].isnan().all()) and got[0, 2:4].tolist() == [448.0, -448.0] and got[1, :2].tolist() == [0.5, -0.5]
    assert not pool[0, 5].any()


def test_slots_outside_the_pool(cuda):
    c = Cache(8, [64], 16, 2)
    pool, _ = _pool(c, 64, "bf16")
    device, ledger = pool.cuda(), c.ledger()
    eviction.read_error_word(clear=True)
    rows = c.total * 16
    eviction.move_rows(device, ledger, i32([[[[rows, 3], [4, rows]], [[2**31 - 1, 0], [1, 2**31 - 1]]]]))
    assert torch.equal(device.cpu(), pool) and eviction.read_error_word(clear=True) == eviction._bounded_lib.ERR_SLOT
    eviction.move_rows(device, ledger, torch.empty((0, 2, 4, 2), dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("n,page", [(1, 16), (5, 1), (64, 64), (65, 16), (700, 16), (3000, 24)])
def test_trim(cuda, n, page):
    rng = np.random.default_rng(n)
    budget, limit = 5 * page + 1, 6 * page
    pps = 40
    lens, dropped = rng.integers(0, pps * page + 1, n), rng.integers(0, 1000, n)
    table, stack = rng.permutation(n * pps).reshape(n, pps), rng.integers(0, 9, n * pps + 50)
    for capacity in (len(stack), len(stack) // 3):
        free = i32(stack[:capacity])
        got = paging.trim_pages(i32(lens), i32(dropped), i32(table), free, i32([min(17, capacity)]), page_size=page, budget=budget,
                                limit=limit)
        want = orc.trim_pages(lens, dropped, table, stack[:capacity], min(17, capacity), page, budget, limit)
        for g, w in zip((*got[:2], free, got[2]), (*want[:3], [want[3]])):
            np.testing.assert_array_equal(g.cpu().numpy(), w)
    paging.read_error_word(clear=True)


def test_trim_flags_lengths_and_capacity(cuda):
    paging.read_error_word(clear=True)
    table = i32([[1, 2, 3, 4], [5, 6, 7, 8]])
    got = paging.trim_pages(i32([-3, 100]), i32([1, 2]), table, i32([0] * 9), i32([0]), page_size=8, budget=8)
    assert paging.read_error_word(clear=True) == paging._sparse_lib.ERR_LEN
    assert got[0].tolist() == [-3, 8] and got[1].tolist() == [1, 94] and got[2].tolist() == [3]
    stack = i32([9, 0])
    got = paging.trim_pages(i32([0, 32]), i32([0, 0]), table, stack, i32([1]), page_size=8, budget=8)
    assert paging.read_error_word(clear=True) == paging._sparse_lib.ERR_FREE and stack.tolist() == [9, 6] and got[2].tolist() == [2]


def test_release_is_as_before(cuda):
    rng = np.random.default_rng(9)
    lens, finished, table = rng.integers(0, 65, 100), rng.random(100) < 0.4, rng.permutation(800).reshape(100, 8)
    free = i32(np.zeros(900))
    got = paging.release_pages(i32(lens), torch.as_tensor(finished, device="cuda"), i32(table), free, i32([5]), page_size=8)
    want = sparse_oracle.release_pages(lens, finished, table, np.zeros(900), 5, 8)
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(free.cpu().numpy(), want[1]) and got[1].tolist() == [want[2]]


def test_captured(cuda):
    """Choice, moves and trim in one graph, replayed on other weights and lengths."""
    c = Cache(10, [400, 300, 200, 350], 16, 2)
    pool, _ = _pool(c, 64, "bf16")
    lens, dropped, table, num = i32(c.lens), i32(c.dropped), i32(c.table), i32([4])
    free, count = i32(np.zeros(c.total)), i32([0])
    ledger, device = c.ledger(), pool.cuda()

    def step():
        moves = eviction.choose_moves(ledger, lens, table, num, budget=128, recent=16, sinks=2, dropped=dropped)
        eviction.move_rows(device, ledger, moves)
        return (moves, *paging.trim_pages(lens, dropped, table, free, count, page_size=16, budget=128))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for turn in range(4):
        lens.copy_(i32([c.rng.integers(0, n + 1) for n in c.lens]))
        ledger.weights.copy_(torch.from_numpy(c.rng.exponential(1.0, c.weights.shape).astype(np.float32)))
        ledger.positions.copy_(torch.from_numpy(c.positions))
        device.copy_(pool)
        h = [x.cpu().numpy() for x in (ledger.weights, ledger.positions, lens)]
        graph.replay()
        torch.cuda.synchronize()
        moves = orc.choose_moves(h[0], h[1], h[2], c.table, 4, budget=128, recent=16, sinks=2, dropped=c.dropped)
        np.testing.assert_array_equal(out[0].cpu().numpy(), moves, err_msg=f"replay {turn}")
        rows = orc.move_rows(pool.view(torch.int16).numpy(), h[0], h[1], moves)
        np.testing.assert_array_equal(device.view(torch.int16).cpu().numpy(), rows[0])
        np.testing.assert_array_equal(ledger.weights.cpu().numpy(), rows[1])
        want = orc.trim_pages(h[2], c.dropped, c.table, np.zeros(c.total), 0, 16, 128)
        assert out[1].tolist() == want[0].tolist() and out[2].tolist() == want[1].tolist() and out[3].tolist() == [want[3]]
        torch.empty(1000, device="cuda").normal_()
