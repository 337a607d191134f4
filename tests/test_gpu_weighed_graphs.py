"""weighed_attention with prompt chunks in captured graphs, replayed on other lengths and offsets: equal to the eager call."""

import numpy as np
import pytest
import torch

from tests.sparse_cases import Batch, i32
from tpu_cake_amd import eviction

pytestmark = pytest.mark.gpu

# (tokens, keys) of each of five sequences, and how many of them there are; 90 tokens at most
STEPS = [([60, 1, 25, 1, 3], [900, 3000, 25, 70, 500], 5), ([1, 1, 1, 1, 1], [3000, 3000, 1, 700, 64], 5),
         ([2, 40, 1, 0, 40], [2, 3000, 1, 900, 41], 5), ([90, 0, 0, 0, 0], [2500, 7, 9, 0, 1], 1),
         ([0, 0, 0, 0, 0], [900, 3000, 25, 70, 500], 5), ([1, 88, 0, 1, 0], [3000, 3000, 0, 3000, 0], 4),
         ([30, 30, 30, 0, 0], [3000, 30, 1500, 2, 2], 3), ([90, 5, 5, 5, 5], [2500, 7, 9, 8, 6], 0)]


@pytest.mark.parametrize("dim,kind,hq,hkv", [(128, "bf16", 8, 2), (128, "fp8", 8, 2), (256, "bf16", 4, 1), (64, "bf16", 16, 2)])
def test_captured_with_chunks(cuda, dim, kind, hq, hkv):
    rng = np.random.default_rng(dim)
    b = Batch(dim, [3000] * 5, [18] * 5, 16, hq, hkv, dim)
    pool, scales, *_ = b.pool(kind)
    pool, scales = pool.cuda(), None if scales is None else torch.from_numpy(scales).cuda()
    q, (lens, table, cu, num) = b.q.cuda(), b.meta()
    ledger = eviction.make_ledger(pool)
    dropped = i32([0, 100, 7, 0, 5])

    def call(led):
        return eviction.weighed_attention(q, pool, led, lens, table, cu, num, sm_scale=dim ** -0.5, decay=0.75, dropped=dropped,
                                          kv_scales=scales)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call(ledger)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call(ledger)
        graphs.append((graph, out))
    eviction.read_error_word(clear=True)
    order = list(range(len(STEPS))) + [int(x) for x in rng.permutation(len(STEPS))]
    for turn, step in enumerate(order):
        new, keys, count = STEPS[step]
        lens.copy_(i32(keys)), cu.copy_(i32(np.concatenate([[0], np.cumsum(new)]))), num.copy_(i32([count]))
        q.normal_()
        graph, out = graphs[turn % 2]
        before = eviction.Ledger(ledger.weights.clone(), ledger.positions.clone())
        graph.replay()
        torch.cuda.synchronize()
        want = call(before)
        assert torch.equal(out, want), turn
        assert torch.equal(ledger.weights, before.weights) and torch.equal(ledger.positions, before.positions), turn
        torch.empty(1000, device="cuda").normal_()
    assert eviction.read_error_word(clear=True) == 0
