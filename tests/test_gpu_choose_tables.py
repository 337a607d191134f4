"""choose_moves over page tables that are much wider than their sequences, and over more rows than its scratch is made for:
equal to the oracle."""

import numpy as np
import pytest
import torch

from oracle import bounded_oracle as orc
from tests.sparse_cases import i32
from tests.test_gpu_eviction import Cache
from tpu_cake_amd import eviction

pytestmark = pytest.mark.gpu


def _widen(c, rows):
    """The same pages in a table of room for ``rows``; what is past them is nobody's."""
    wide = np.full((len(c.lens), -(-rows // c.page)), 2**31 - 1, np.int64)
    width = min(c.table.shape[1], wide.shape[1])
    wide[:, :width] = c.table[:, :width]
    c.table = wide


@pytest.mark.parametrize("rows", [32768, 32784, 131072, 1 << 20])
@pytest.mark.parametrize("lens,hkv", [([2100, 2112, 30, 2049, 0, 2300] * 5, 2), ([2100, 32768, 2300, 32769, 40000], 1),
                                      ([33000, 100, 70000, 2300, 36864, 36865], 2)])
def test_tables_wider_than_their_sequences(cuda, rows, lens, hkv):
    c = Cache(len(lens), np.minimum(lens, rows), 16, hkv, spare=1)
    _widen(c, rows)
    eviction.read_error_word(clear=True)
    c.choose(budget=2048, recent=256, sinks=4, limit=2111)
    c.choose(budget=30000, recent=1, max_moves=50000)
    assert eviction.read_error_word(clear=True) == 0


def test_pages_that_are_not_divided_by_four(cuda):
    c = Cache(3, [40000, 33001, 12], 7, 2, ties=True)
    _widen(c, 60000)
    c.choose(budget=2048, recent=256, sinks=4)


@pytest.mark.parametrize("lens", [[40000] * 6, [33000, 40000, 100, 40000, 40000, 2500]])
def test_long_sequences_that_share_pages(cuda, lens):
    """More rows than distinct pages have, so that some sequences' keys find no room: their lists are right all the same."""
    c = Cache(4, lens, 16, 2, ties=True)
    longest = int(np.argmax(lens))
    for i, n in enumerate(lens):
        c.table[i] = c.table[longest]
    order = np.unique(c.table[longest])  # the pool: only what the longest holds
    c.weights, c.positions, c.total = c.weights[order], c.positions[order], len(order)
    c.table = np.searchsorted(order, c.table)
    c.choose(budget=2048, recent=256, sinks=4)


def test_captured_with_long_and_short_sequences(cuda):
    """One graph whose replays find long sequences at other places, or none."""
    c = Cache(5, [40000, 36000, 50000, 3000], 16, 2)
    _widen(c, 131072)
    ledger, lens, table, dropped = c.ledger(), i32(c.lens), i32(c.table), i32(c.dropped)
    num = i32([4])
    kw = dict(budget=2048, recent=64, sinks=4, limit=2100)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eviction.choose_moves(ledger, lens, table, num, dropped=dropped, **kw)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = eviction.choose_moves(ledger, lens, table, num, dropped=dropped, **kw)
        graphs.append((graph, out))
    for turn, (now, count) in enumerate([([40000, 36000, 50000, 3000], 4), ([2100, 2000, 0, 2500], 4), ([100, 36000, 2600, 2200], 4),
                                         ([40000, 32768, 32769, 1], 3), ([40000, 36000, 50000, 3000], 1), ([33000, 36000, 50000, 3000], 4)]):
        lens.copy_(i32(now)), num.copy_(i32([count]))
        c.weights = c.rng.exponential(1.0, c.weights.shape).astype(np.float32)
        ledger.weights.copy_(torch.from_numpy(c.weights))
        graph, out = graphs[turn % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = orc.choose_moves(c.weights, c.positions, now, c.table, count, dropped=c.dropped, **kw)
        np.testing.assert_array_equal(out.cpu().numpy(), want, err_msg=f"replay {turn}")
        torch.empty(1000, device="cuda").normal_()


def test_scratch_follows_the_pool(cuda):
    """What a call takes from the allocator is no more than the keys of the pool's rows need, however wide the table."""
    lens = [2100] * 64
    c = Cache(6, lens, 16, 2)
    _widen(c, 131072)
    ledger, args = c.ledger(), (i32(c.lens), i32(c.table), i32([64]))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    eviction.choose_moves(ledger, *args, budget=2048, recent=256, max_moves=64)
    torch.cuda.synchronize()
    rows = c.total * 16 * 2  # of all heads
    assert torch.cuda.max_memory_allocated() - before < 13 * rows + (1 << 20)
