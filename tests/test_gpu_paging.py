"""Page allocation on the GPU: every whole number equals the oracle's."""

import numpy as np
import pytest
import torch

from oracle import sparse_oracle as orc
from tpu_cake_amd import paging

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda")


def _state(rng, n, pps, page, spare):
    """Requests of random lengths whose pages are distinct, and a stack of the other pages."""
    cached = rng.integers(0, pps * page + 1, n)
    cached[rng.random(n) < 0.3] = 0
    held = -(-cached // page)
    total = int(held.sum()) + spare
    order = rng.permutation(total)
    table = rng.integers(-5, total + 5, (n, pps))  # what lies past a request's pages is anything
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    free = np.full(total, -7)
    free[:spare] = order[at:]
    return cached, table, free, spare


def _assign(cached, new, table, free, count, page, max_tokens):
    want = orc.assign_pages(cached, new, table, free, count, page, max_tokens)
    t = _i32(table)
    inputs = [_i32(cached), _i32(new), t, _i32(free), _i32([count])]
    before = [x.clone() for x in inputs]
    got = paging.assign_pages(*inputs, page_size=page, max_tokens=max_tokens)
    for name, g, w in zip(("kv_lens", "cu_q_lens", "slots", "positions", "table", "count"),
                          (got.kv_lens, got.cu_q_lens, got.slot_mapping, got.positions, t, got.free_count),
                          (*want[:5], [want[5]])):
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
    assert got.num_seqs.tolist() == [len(cached)]
    for i in (0, 1, 3, 4):
        assert torch.equal(inputs[i], before[i])
    return got


@pytest.mark.parametrize("n,pps,page,chunk", [
    (1, 1, 1, 1), (1, 4, 16, 64), (7, 3, 5, 9), (64, 128, 64, 1), (63, 9, 16, 40), (1025, 6, 24, 30), (4096, 8, 16, 3),
    (4097, 4, 1, 4), (9000, 5, 7, 2)])
@pytest.mark.parametrize("limits", ["ample", "pages", "tokens"])
def test_assign_equals_the_oracle(cuda, n, pps, page, chunk, limits):
    rng = np.random.default_rng(n * 100 + page)
    new = rng.integers(0, chunk + 1, n)
    new[rng.random(n) < 0.2] = 0
    if n > 20:
        new[rng.integers(0, n, 4)] = pps * page + 1  # past the table: not valid
    ample = int(new.sum()) + 2
    cached, table, free, count = _state(rng, n, pps, page, ample if limits != "pages" else max(1, n // 3))
    max_tokens = ample + 5 if limits != "tokens" else max(1, ample // 3)
    _assign(cached, new, table, free, count, page, max_tokens)


def test_a_long_prompt_spans_many_workgroups(cuda):
    rng = np.random.default_rng(3)
    page, pps = 16, 1000
    cached, new = np.array([5, 0, 0, 31, 7]), np.array([1, 9001, 0, 4000, 1])
    table = np.zeros((5, pps), np.int64)
    table[:, :2] = np.arange(10).reshape(5, 2)
    free = 10 + rng.permutation(2000)
    _assign(cached, new, table, free, 2000, page, 13100)


def test_invalid_lengths_get_nothing_and_are_flagged(cuda):
    paging.read_error_word(clear=True)
    cached, new = np.array([3, -4, 8, 2**31 - 1, 5]), np.array([1, 1, -2, 7, 2])
    table = np.arange(20).reshape(5, 4)
    got = _assign(cached, new, table, np.arange(20, 30), 10, 8, 16)
    assert got.cu_q_lens.tolist() == [0, 1, 1, 1, 1, 3]
    assert paging.read_error_word(clear=True) == paging._sparse_lib.ERR_LEN
    assert paging.read_error_word() == 0


def test_bad_counts_and_pages_are_flagged_and_never_read(cuda):
    paging.read_error_word(clear=True)
    table = _i32(np.full((2, 4), -9))  # held pages that are no pages
    got = paging.assign_pages(_i32([3, 3]), _i32([1, 1]), table, _i32([1, 2]), _i32([2]), page_size=8, max_tokens=4)
    assert got.slot_mapping.tolist() == [-1, -1, -1, -1] and paging.read_error_word(clear=True) == paging._sparse_lib.ERR_PAGE
    got = paging.assign_pages(_i32([0]), _i32([30]), _i32([[0] * 8]), _i32([5, 6]), _i32([99]), page_size=8, max_tokens=64)
    assert got.cu_q_lens.tolist() == [0, 0] and got.free_count.tolist() == [2]  # two pages, four needed
    assert paging.read_error_word(clear=True) == paging._sparse_lib.ERR_FREE


def test_no_tokens_at_all(cuda):
    got = _assign(np.array([3, 0]), np.array([0, 0]), np.zeros((2, 4), np.int64), np.arange(4), 4, 8, 0)
    assert got.slot_mapping.numel() == 0


@pytest.mark.parametrize("n,pps,page", [(1, 1, 1), (5, 4, 16), (64, 128, 64), (65, 70, 3), (1000, 9, 24), (4100, 3, 1)])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
def test_release_equals_the_oracle(cuda, n, pps, page, share):
    rng = np.random.default_rng(n + pps)
    cached, table, free, count = _state(rng, n, pps, page, 11)
    finished = rng.random(n) < share
    want = orc.release_pages(cached, finished, table, free, count, page)
    stack, lens, cnt = _i32(free), _i32(cached), _i32([count])
    got_lens, got_count = paging.release_pages(lens, torch.as_tensor(finished, device="cuda"), _i32(table), stack, cnt,
                                               page_size=page)
    np.testing.assert_array_equal(got_lens.cpu().numpy(), want[0])
    np.testing.assert_array_equal(stack.cpu().numpy(), want[1])
    assert got_count.item() == want[2]
    np.testing.assert_array_equal(lens.cpu().numpy(), cached)
    assert cnt.item() == count


def test_release_past_the_stack_is_dropped_and_flagged(cuda):
    paging.read_error_word(clear=True)
    stack = _i32([7, 0, 0])
    lens, count = paging.release_pages(_i32([30]), torch.ones(1, dtype=torch.bool, device="cuda"), _i32([[1, 2, 3, 4]]), stack,
                                       _i32([1]), page_size=8)
    assert stack.tolist() == [7, 1, 2] and count.tolist() == [3] and lens.tolist() == [0]
    assert paging.read_error_word(clear=True) == paging._sparse_lib.ERR_FREE


def test_steps_conserve_pages(cuda):
    """Sixty steps of arrivals, growth and ends: no page is lost, none is held twice."""
    rng = np.random.default_rng(8)
    n, pps, page, total = 40, 16, 4, 300
    table, stack = _i32(np.zeros((n, pps))), _i32(rng.permutation(total))
    lens, count = _i32(np.zeros(n)), _i32([total])
    for _ in range(60):
        held = lens.cpu().numpy()
        finished = (held > 0) & (rng.random(n) < 0.1)
        lens, count = paging.release_pages(lens, torch.as_tensor(finished, device="cuda"), table, stack, count, page_size=page)
        new = np.where(lens.cpu().numpy() > 0, 1, rng.integers(0, 20, n))
        step = paging.assign_pages(lens, _i32(new), table, stack, count, page_size=page, max_tokens=128)
        lens, count = step.kv_lens, step.free_count
        held, t = lens.cpu().numpy(), table.cpu().numpy()
        pages = np.concatenate([t[i, :-(-int(held[i]) // page)] for i in range(n)] + [stack.cpu().numpy()[:count.item()]])
        assert sorted(pages.tolist()) == list(range(total))
        slots = step.slot_mapping.cpu().numpy()
        slots = slots[slots >= 0]
        assert len(set(slots.tolist())) == len(slots) == step.cu_q_lens[-1].item()


def test_captured_steps_replay_on_new_lengths(cuda):
    n, pps, page = 6, 8, 4
    lens, new = _i32(np.zeros(n)), _i32(np.ones(n))
    finished = torch.zeros(n, dtype=torch.bool, device="cuda")
    table, stack, count = _i32(np.zeros((n, pps))), _i32(np.arange(60)), _i32([60])

    def step():
        after, left = paging.release_pages(lens, finished, table, stack, count, page_size=page)
        got = paging.assign_pages(after, new, table, stack, left, page_size=page, max_tokens=32)
        lens.copy_(got.kv_lens)
        count.copy_(got.free_count)
        return got

    state = [x.clone() for x in (lens, table, stack, count)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    for x, y in zip((lens, table, stack, count), state):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    rng = np.random.default_rng(1)
    h = [x.cpu().numpy() for x in (lens, table, stack, count)]
    for turn in range(6):
        fin, fresh = (h[0] > 0) & (rng.random(n) < 0.3), rng.integers(0, 5, n)
        finished.copy_(torch.as_tensor(fin))
        new.copy_(_i32(fresh))
        graph.replay()
        torch.cuda.synchronize()
        l2, s2, c2 = orc.release_pages(h[0], fin, h[1], h[2], h[3][0], page)
        want = orc.assign_pages(l2, fresh, h[1], s2, c2, page, 32)
        for g, w in zip((got.kv_lens, got.cu_q_lens, got.slot_mapping, got.positions, table, count, stack),
                        (*want[:5], [want[5]], s2)):
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=f"replay {turn}")
        torch.empty(1000, device="cuda").normal_()  # the program's own work between replays
        h = [x.cpu().numpy() for x in (lens, table, stack, count)]


def test_out_buffers_and_another_stream(cuda):
    cached, new, table, free = [3, 9], [2, 1], [[4, 0, 0], [1, 2, 0]], [8, 9, 10]
    args = [_i32(x) for x in (cached, new, table, free, [3])]
    fresh = paging.assign_pages(*[x.clone() for x in args], page_size=4, max_tokens=5)
    out = paging.StepMetadata(*(torch.full_like(x, 77) for x in fresh))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = paging.assign_pages(*args, page_size=4, max_tokens=5, out=out)
    stream.synchronize()
    assert got is out and all(torch.equal(a, b) for a, b in zip(fresh, out))
