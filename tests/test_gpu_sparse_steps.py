"""The sparse entry points together, as a serving loop runs them: pages are assigned, keys appended,
pages chosen and attended to, and finished requests give their pages back."""

import threading

import numpy as np
import pytest
import torch

from oracle import sparse_oracle as orc
from sparse_cases import i32
from tpu_cake_amd import ops, paging, sparse

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, PAGE, TOP = 8, 2, 128, 16, 6
SCALE = DIM**-0.5


class Loop:
    """Requests in a pool on the GPU, and their keys and values on the host."""

    def __init__(self, seed, requests, pages, columns, kind, max_tokens):
        self.rng, self.n, self.kind, self.max_tokens = np.random.default_rng(seed), requests, kind, max_tokens
        dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
        self.pool = torch.zeros((pages, PAGE, 2 * HKV, DIM), device="cuda").to(dtype)
        self.scales = None
        if kind == "fp8":
            self.scales = torch.from_numpy(self.rng.uniform(0.006, 0.012, (pages, HKV, 2)).astype(np.float32)).cuda()
        self.index = sparse.make_page_index(self.pool)
        self.table, self.free = i32(np.zeros((requests, columns))), i32(self.rng.permutation(pages))
        self.lens, self.count = i32(np.zeros(requests)), i32([pages])
        self.new, self.finished = i32(np.zeros(requests)), torch.zeros(requests, dtype=torch.bool, device="cuda")
        self.qkv = torch.zeros((max_tokens, HQ + 2 * HKV, DIM), dtype=torch.bfloat16, device="cuda")

    def fill(self, new, finished):
        self.new.copy_(i32(new))
        self.finished.copy_(torch.as_tensor(finished))
        self.qkv.copy_(torch.from_numpy(self.rng.standard_normal(self.qkv.shape).astype(np.float32)))

    def step(self):
        lens, count = paging.release_pages(self.lens, self.finished, self.table, self.free, self.count, page_size=PAGE)
        meta = paging.assign_pages(lens, self.new, self.table, self.free, count, page_size=PAGE, max_tokens=self.max_tokens)
        q, k, v = self.qkv[:, :HQ], self.qkv[:, HQ:HQ + HKV], self.qkv[:, HQ + HKV:]
        sparse.append_kv(k, v, self.pool, meta.slot_mapping, kv_scales=self.scales, index=self.index)
        batch = (meta.kv_lens, self.table, meta.cu_q_lens, meta.num_seqs)
        picked = sparse.select_pages(q, self.index, *batch, page_size=PAGE, num_pages=TOP)
        out = sparse.sparse_paged_attention(q, self.pool, picked, *batch, sm_scale=SCALE, kv_scales=self.scales)
        self.lens.copy_(meta.kv_lens)
        self.count.copy_(meta.free_count)
        return meta, picked, out

    def check(self, meta, picked, out, what=""):
        """The step's choice equals the oracle's on the pool's index, the index that of the pool's keys, and
        the output the oracle's within bf16 and the sums' roundings."""
        lens, cu, table = meta.kv_lens.cpu().numpy(), meta.cu_q_lens.cpu().numpy(), self.table.cpu().numpy()
        held = self.pool.double().cpu().numpy().reshape(-1, PAGE, HKV, 2, DIM)
        if self.scales is not None:
            held = held * self.scales.double().cpu().numpy()[:, None, :, :, None]
        bounds, exps = self.index.bounds.cpu().numpy(), self.index.exponents.cpu().numpy()
        for i in range(self.n):
            for p in range(-(-int(lens[i]) // PAGE)):
                rows = held[table[i, p], :min(PAGE, lens[i] - p * PAGE), :, 0].astype(np.float32)
                for h in range(HKV):
                    b, e = orc.page_bounds(rows[:, h])
                    assert e == exps[table[i, p], h] and (b == bounds[table[i, p], h]).all(), (what, i, p, h)
        q = self.qkv[:, :HQ].double().cpu().numpy()
        want = orc.select_pages(q, bounds, exps, lens, table, cu, self.n, PAGE, TOP)
        np.testing.assert_array_equal(picked.cpu().numpy(), want, err_msg=what)
        ref = orc.sparse_attention(q, held[:, :, :, 0], held[:, :, :, 1], want, lens, table, cu, self.n, SCALE)
        # the output's rounding; weights off by twice the scores' error (132 products and sums of |q k| <= 8 * 6)
        tol = 2.0**-8 * np.abs(ref) + 6 * (2 * 132 * 2.0**-24 * DIM * SCALE * 8 + 2.0**-15)
        assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all(), what
        assert (out[int(cu[-1]):] == 0).all() and (picked[int(cu[-1]):] == -1).all()


def _traffic(rng, lens, n):
    finished = (lens > 0) & (rng.random(n) < 0.15)
    alive = np.where(finished, 0, lens)
    new = np.where(alive > 0, np.where(rng.random(n) < 0.2, rng.integers(2, 40, n), 1), rng.choice([0, 3, 60, 130], n))
    return np.where(finished, 0, new), finished


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("pages", [160, 40])  # ample, and so few that requests have to wait
def test_steps(cuda, kind, pages):
    loop = Loop(3, 9, pages, 20, kind, 256)
    for turn in range(10):
        loop.fill(*_traffic(loop.rng, loop.lens.cpu().numpy(), loop.n))
        loop.check(*loop.step(), f"step {turn}")
    assert sparse.read_error_word() == 0


def test_step_metadata_feeds_the_dense_operator(cuda):
    """Requests without tokens among the others, pages of the allocator: lists of every page give what the
    dense operator gives, within both operators' roundings."""
    loop = Loop(4, 6, 200, 16, "bf16", 192)
    for new in ([100, 0, 17, 1, 0, 30], [1, 60, 1, 0, 0, 1], [1, 1, 1, 50, 0, 1]):
        loop.fill(np.array(new), np.zeros(6, bool))
        meta, _, _ = loop.step()
        q = loop.qkv[:, :HQ].contiguous()
        batch = (meta.kv_lens, loop.table, meta.cu_q_lens, meta.num_seqs)
        whole = torch.arange(16, dtype=torch.int32, device="cuda").expand(192, HKV, 16).contiguous()
        got = sparse.sparse_paged_attention(q, loop.pool, whole, *batch, sm_scale=SCALE)
        dense = ops.ragged_paged_attention(q, loop.pool, *batch, sm_scale=SCALE)
        assert (got.float() - dense.float()).abs().max().item() <= 2e-2
        assert ops.read_error_word() == 0


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_captured_steps(cuda, kind):
    """A decode step captured once and replayed over growing lengths, with work of the program between."""
    loop = Loop(5, 7, 120, 16, kind, 7)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        loop.fill(np.ones(7, int), np.zeros(7, bool))
        loop.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        result = loop.step()
    for turn in range(40):
        lens = loop.lens.cpu().numpy()
        finished = (lens > 20) & (loop.rng.random(7) < 0.05)
        loop.fill(np.where(finished, 0, 1), finished)
        graph.replay()
        torch.cuda.synchronize()
        if turn % 8 == 7:
            loop.check(*result, f"replay {turn}")
        torch.randn(4096, device="cuda").sum().item()


def test_two_graphs_replay_side_by_side(cuda):
    """Graphs captured on one stream and replayed on two at once share no scratch: split lists and split rows."""
    rng = np.random.default_rng(0)
    calls = []
    capture = torch.cuda.Stream()
    for seed in range(2):
        pages, n = 20000, 2
        q = torch.randn((n, HQ, DIM), device="cuda").to(torch.bfloat16)
        pool = torch.randn((pages, 1, 2 * HKV, DIM), device="cuda").to(torch.bfloat16)
        index = sparse.PageIndex(torch.randint(-127, 128, (pages, HKV, 2, DIM), dtype=torch.int8, device="cuda"),
                                 torch.randint(-6, -3, (pages, HKV), dtype=torch.int8, device="cuda"))
        batch = (i32([9990, 9000 + seed]), i32(rng.permutation(pages).reshape(2, -1)), i32([0, 1, 2]), i32([2]))

        def step(q=q, pool=pool, index=index, batch=batch):
            picked = sparse.select_pages(q, index, *batch, page_size=1, num_pages=700)
            return picked, sparse.sparse_paged_attention(q, pool, picked, *batch, sm_scale=SCALE)

        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        with torch.cuda.stream(capture):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            got = step()
        calls.append((graph, got, want, torch.cuda.Stream(), step))  # step holds the inputs: a graph does not
    for _ in range(20):
        for graph, _, _, stream, _ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, got, want, _, _ in calls:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            got[1].zero_()


def test_captured_chunks_with_other_lengths(cuda):
    """A chunk's choice and attention, lists split over workgroups: captured once, replayed with other lengths and tokens."""
    n, tokens, width = 3, 40, 64
    rng = np.random.default_rng(3)
    pool = torch.randn((n * width, 64, 2 * HKV, DIM), device="cuda").to(torch.bfloat16)
    index = sparse.PageIndex(torch.randint(-127, 128, (n * width, HKV, 2, DIM), dtype=torch.int8, device="cuda"),
                             torch.randint(-6, -3, (n * width, HKV), dtype=torch.int8, device="cuda"))
    q = torch.empty((tokens, HQ, DIM), dtype=torch.bfloat16, device="cuda")
    lens, table, cu, num = i32([0] * n), i32(rng.permutation(n * width).reshape(n, width)), i32([0] * (n + 1)), i32([n])

    def fill(kv_lens, q_lens):
        lens.copy_(i32(kv_lens))
        cu.copy_(i32(np.concatenate([[0], np.cumsum(q_lens)])))
        q.copy_(torch.from_numpy(rng.standard_normal(q.shape, np.float32)))

    def step():
        picked = sparse.select_pages(q, index, lens, table, cu, num, page_size=64, num_pages=20)
        return picked, sparse.sparse_paged_attention(q, pool, picked, lens, table, cu, num, sm_scale=SCALE)

    fill([4000, 100, 9], [30, 1, 1])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    for kv_lens, q_lens in (([4000, 100, 9], [30, 1, 1]), ([64 * 64, 64, 1], [1, 38, 1]), ([0, 0, 0], [0, 0, 0]), ([700, 3000, 2], [0, 40, 0])):
        fill(kv_lens, q_lens)
        want = [x.clone() for x in step()]
        for _ in range(2):
            got[1].fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            torch.randn(4096, device="cuda").sum().item()


def test_threads_on_streams_of_their_own(cuda):
    """Two threads at once, split forms, each on its stream: the results of one after the other."""
    rng = np.random.default_rng(4)
    jobs = []
    for rows in (2, 30):
        pages = 6000
        q = torch.randn((rows, HQ, DIM), device="cuda").to(torch.bfloat16)
        pool = torch.randn((pages, 4, 2 * HKV, DIM), device="cuda").to(torch.bfloat16)
        index = sparse.PageIndex(torch.randint(-127, 128, (pages, HKV, 2, DIM), dtype=torch.int8, device="cuda"),
                                 torch.randint(-6, -3, (pages, HKV), dtype=torch.int8, device="cuda"))
        cu = [0, 1, rows]
        jobs.append((q, pool, index, (i32([11000, 12000]), i32(rng.permutation(pages).reshape(2, -1)), i32(cu), i32([2]))))

    def step(q, pool, index, batch):
        picked = sparse.select_pages(q, index, *batch, page_size=4, num_pages=300)
        return picked, sparse.sparse_paged_attention(q, pool, picked, *batch, sm_scale=SCALE)

    want = [step(*job) for job in jobs]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(step(*jobs[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x[0], want[i][0]) and torch.equal(x[1], want[i][1])
