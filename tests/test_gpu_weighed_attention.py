"""Attention that accounts for the weight of each key, against the formula in 64 bits.

Tolerance: the output is rounded once, half a step of bf16, 2^-8 of the value; scores and sums in 32 bits add what the
oracle bounds from the inputs (a score's dim products and sums, the row's sum of n terms, an exponential's argument).
Weights are 32-bit sums: the same bound of each probability, and a step a term.
"""

import numpy as np
import pytest
import torch

from oracle import bounded_oracle as orc
from tests.sparse_cases import Batch, i32
from tpu_cake_amd import eviction, ops

pytestmark = pytest.mark.gpu


def _state(b, kind="bf16", seed=0):
    rng = np.random.default_rng(seed)
    pool, scales, keys, values = b.pool(kind)
    weights = rng.uniform(0, 0.1, (b.total, b.hkv, b.page_size)).astype(np.float32)
    positions = rng.integers(0, 1000, weights.shape).astype(np.int32)
    return pool, scales, keys, values, weights, positions


def _check(b, state, *, sm_scale=None, q=None, pool=None, **kw):
    pool_, scales, keys, values, weights, positions = state
    pool = pool_.cuda() if pool is None else pool
    sm_scale = b.dim ** -0.5 if sm_scale is None else sm_scale
    ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.from_numpy(positions).cuda())
    lens, table, cu, num = b.meta()
    q = b.q.cuda() if q is None else q
    dropped = kw.pop("dropped", None)
    out = eviction.weighed_attention(q, pool, ledger, lens, table, cu, num, sm_scale=sm_scale,
                                     kv_scales=None if scales is None else torch.from_numpy(scales).cuda(),
                                     dropped=None if dropped is None else i32(dropped), **kw)
    want = orc.weighed_attention(b.q.double().numpy(), keys, values, weights, positions, b.lens, b.table, b.cu, b.n, sm_scale,
                                 dropped=dropped, **kw)
    got = out.double().cpu().numpy()
    bad = ~(np.abs(got - want[0]) <= 2.0**-8 * np.abs(want[0]) + want[3])
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[0][bad][:4])
    got = ledger.weights.double().cpu().numpy()
    bad = ~((np.abs(got - want[1]) <= want[4] + 1e-30) | (np.isnan(got) & np.isnan(want[1])))
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[1][bad][:4], want[4][bad][:4])
    np.testing.assert_array_equal(ledger.positions.cpu().numpy(), want[2])
    return out, ledger


@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (64, "bf16"), (256, "bf16"), (32, "bf16"), (96, "bf16"), (40, "bf16"),
                                      (128, "fp8"), (64, "fp8"), (256, "fp8"), (112, "fp8")])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 5)])
def test_decode(cuda, dim, kind, hq, hkv):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 255, 256, 257, 700, 1500]
    b = Batch(dim, lens, [1] * len(lens), 16, hq, hkv, dim)
    _check(b, _state(b, kind))


@pytest.mark.parametrize("page", [1, 3, 16, 24, 32, 64, 100])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_pages_of_any_size(cuda, page, kind):
    b = Batch(page, [1, page, page + 1, 333, 90, 7], [1, 1, 1, 1, 20, 7], page, 8, 2, 128)
    _check(b, _state(b, kind))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (16, 1), (17, 1), (32, 2), (64, 1), (72, 2), (256, 1)])
def test_groups(cuda, hq, hkv):
    b = Batch(hq, [70, 300, 41], [1, 1, 9], 16, hq, hkv, 64)
    _check(b, _state(b))


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("lens,new", [([40], [40]), ([129], [128]), ([500, 3], [37, 3]), ([1, 200, 64, 900, 5], [1, 200, 1, 33, 2]),
                                      ([2000, 10], [130, 1]), ([65, 65, 65, 65], [2, 3, 4, 65])])
def test_chunks(cuda, kind, lens, new):
    b = Batch(len(lens) + lens[0], lens, new, 16, 8, 2, 128, spare=2, pad=5)
    _check(b, _state(b, kind))


@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0])
def test_decay_dropped_and_stale_entries(cuda, decay):
    """New keys' entries and, with decay 0, all entries start anew whatever is there."""
    b = Batch(3, [50, 100, 9], [1, 4, 9], 16, 4, 2, 64, spare=1)
    pool, scales, keys, values, weights, positions = _state(b)
    for i, (n, new) in enumerate(((50, 1), (100, 4), (9, 9))):
        for r in range(0 if decay == 0.0 else n - new, n):
            weights[b.table[i, r // 16], :, r % 16] = np.nan
    _check(b, (pool, scales, keys, values, weights, positions), decay=decay, dropped=np.array([1000, 0, 5, 9]))


def test_sequences_without_tokens_stay_as_they_are(cuda):
    b = Batch(4, [50, 100, 9, 30], [0, 2, 0, 1], 16, 4, 2, 64)
    _check(b, _state(b))


def test_empty_sequences(cuda):
    """No key: zero rows; and a length shorter than its tokens: the first of them see none."""
    b = Batch(5, [8, 30], [1, 6], 16, 4, 2, 64)
    b.lens = np.array([0, 3])
    pool, scales, keys, values, weights, positions = _state(b)
    ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.from_numpy(positions).cuda())
    out = eviction.weighed_attention(b.q.cuda(), pool.cuda(), ledger, *b.meta(), sm_scale=0.125)
    assert not out[0].any() and not out[1:4].any() and bool(out[4:].any())
    got = ledger.weights[int(b.table[1, 0]), :, :3].double().cpu().numpy()
    np.testing.assert_allclose(got.sum(), 3 * 4, rtol=1e-5)  # three tokens' probabilities for each of four heads
    np.testing.assert_array_equal(ledger.positions[int(b.table[1, 0]), :, :3].cpu().numpy(), [[0, 1, 2]] * 2)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_keys_that_are_not_seen_may_hold_anything(cuda, kind):
    """Rows past a sequence's end, pages of nobody, and a chunk's later tokens hold infinities and NaN."""
    b = Batch(6, [20, 100, 50], [1, 3, 40], 16, 8, 2, 128)
    pool, scales, keys, values, weights, positions = _state(b, kind)
    poison = pool.clone()
    seen = np.zeros((b.total, 16), bool)
    for i, n in enumerate(b.lens):
        for r in range(n):
            seen[b.table[i, r // 16], r % 16] = True
    bad = torch.full((b.dim,), float("nan")).to(poison.dtype)
    for page, off in np.argwhere(~seen):
        poison[page, off] = bad
    # the last token of the last chunk: its values are infinite, and only it sees them
    page, off = int(b.table[2, 49 // 16]), 49 % 16
    if kind == "bf16":
        poison[page, off, 1::2] = float("inf")
    lens, table, cu, num = b.meta()
    ledgers = [eviction.Ledger(torch.from_numpy(weights).cuda(), torch.from_numpy(positions).cuda()) for _ in range(2)]
    sc = None if scales is None else torch.from_numpy(scales).cuda()
    got = eviction.weighed_attention(b.q.cuda(), poison.cuda(), ledgers[0], lens, table, cu, num, kv_scales=sc)
    want = eviction.weighed_attention(b.q.cuda(), pool.cuda(), ledgers[1], lens, table, cu, num, kv_scales=sc)
    last = b.tokens - 1
    assert torch.equal(got[:last], want[:last])
    assert torch.equal(ledgers[0].weights, ledgers[1].weights) and torch.equal(ledgers[0].positions, ledgers[1].positions)


def test_scores_of_minus_infinity(cuda):
    """Keys whose score is -infinity weigh nothing; a row of them only is zero."""
    b = Batch(7, [40, 6], [1, 1], 16, 2, 1, 64)
    pool, scales, keys, values, weights, positions = _state(b)
    b.q = b.q.abs() + 0.5
    pool = pool.clone()
    for i, rows in ((0, range(5, 30)), (1, range(6))):
        for r in rows:
            pool[int(b.table[i, r // 16]), r % 16, 0] = float("-inf")
    keys = pool.view(b.total, 16, 1, 2, 64)[..., 0, :].double().numpy()
    with np.errstate(invalid="ignore"):
        ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.from_numpy(positions).cuda())
        out = eviction.weighed_attention(b.q.cuda(), pool.cuda(), ledger, *b.meta(), sm_scale=0.1, decay=0.0)
    assert not out[1].any() and bool(out[0].isfinite().all())
    w = ledger.weights.cpu().numpy()
    assert all(w[b.table[0, r // 16], 0, r % 16] == 0 for r in range(5, 30))
    assert abs(sum(w[b.table[0, r // 16], 0, r % 16] for r in range(40)) - 2) < 1e-5
    assert not w[b.table[1, 0], 0, :6].any()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_soft_cap_and_large_scores(cuda, kind):
    b = Batch(8, [300, 70], [1, 30], 16, 8, 2, 128)
    _check(b, _state(b, kind), soft_cap=5.0, sm_scale=0.7)
    _check(b, _state(b, kind), sm_scale=2.0)


def test_scalar_scales(cuda):
    b = Batch(9, [120, 40], [1, 12], 16, 8, 2, 64)
    pool, scales, keys, values, weights, positions = _state(b, "fp8")
    codes = pool.float().double().numpy().reshape(b.total, 16, 2, 2, 64)
    ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.from_numpy(positions).cuda())
    out = eviction.weighed_attention(b.q.cuda(), pool.view(torch.uint8).cuda(), ledger, *b.meta(), sm_scale=0.125, k_scale=0.01,
                                     v_scale=0.5)
    ks, vs = float(np.float32(0.01)), 0.5
    want = orc.weighed_attention(b.q.double().numpy(), codes[..., 0, :] * ks, codes[..., 1, :] * vs, weights, positions, b.lens, b.table,
                                 b.cu, b.n, 0.125)
    assert (np.abs(out.double().cpu().numpy() - want[0]) <= 2.0**-8 * np.abs(want[0]) + want[3]).all()
    assert (np.abs(ledger.weights.double().cpu().numpy() - want[1]) <= want[4]).all()


def test_long_rows_over_many_workgroups(cuda):
    """A few long sequences beside many short ones: rows whole, in parts and several of them in a workgroup."""
    rng = np.random.default_rng(10)
    lens = [30000, 9000] + rng.integers(1, 600, 60).tolist()
    b = Batch(10, lens, [1] * len(lens), 64, 8, 2, 128)
    _check(b, _state(b))
    b = Batch(11, [20001], [1], 16, 16, 2, 64)
    _check(b, _state(b, "fp8"))


def test_many_sequences(cuda):
    rng = np.random.default_rng(12)
    lens = rng.integers(1, 40, 700)
    b = Batch(12, lens.tolist(), [1] * 700, 16, 4, 1, 64, spare=100)
    _check(b, _state(b))
    new = np.minimum(rng.integers(0, 4, 700), lens)
    b = Batch(13, lens.tolist(), new.tolist(), 16, 4, 1, 64)
    _check(b, _state(b))


def test_chunks_of_many_sequences(cuda):
    """More sequences than one wave counts, some of one token."""
    rng = np.random.default_rng(22)
    lens = rng.integers(1, 60, 300)
    new = np.minimum(rng.integers(1, 9, 300), lens)
    b = Batch(22, lens.tolist(), new.tolist(), 16, 4, 2, 64, spare=3)
    _check(b, _state(b, "fp8"))


@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (256, "bf16"), (40, "bf16"), (128, "fp8"), (256, "fp8"), (112, "fp8")])
def test_chunks_of_many_lengths(cuda, dim, kind):
    """Enough rows of the table, or enough keys, that every wave has keys of its own."""
    rng = np.random.default_rng(25)
    lens = rng.integers(1, 400, 140)
    new = np.minimum(rng.integers(1, 20, 140), lens)
    b = Batch(25, lens.tolist(), new.tolist(), 16, 4, 2, dim)
    _check(b, _state(b, kind))
    b = Batch(26, [40000, 300], [3, 70], 64, 4, 2, dim)
    _check(b, _state(b, kind))


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_chunks_in_a_batch_of_few_tokens(cuda, kind):
    """As many sequences as tokens could be there, but some have more than one."""
    b = Batch(23, [300, 45, 200, 40], [5, 1, 70, 40], 16, 8, 2, 128, spare=150)
    _check(b, _state(b, kind))


@pytest.mark.parametrize("hq,hkv", [(320, 160), (130, 65), (512, 2)])
def test_many_heads(cuda, hq, hkv):
    b = Batch(hq, [70, 300, 5, 16], [1, 1, 1, 1], 16, hq, hkv, 32)
    _check(b, _state(b))


def test_pages_held_twice(cuda):
    """Sequences that share pages, which the ledger does not allow: the outputs are right, and so are the weights of one
    that shares none, behind more keys than the pool has."""
    b = Batch(24, [400, 400, 400, 400, 300], [1] * 5, 16, 8, 2, 64)
    b.table[1:4] = b.table[0]
    state = pool, _, keys, values, weights, positions = _state(b)
    ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.from_numpy(positions).cuda())
    out = eviction.weighed_attention(b.q.cuda(), pool.cuda(), ledger, *b.meta(), sm_scale=0.125)
    want = orc.weighed_attention(b.q.double().numpy(), keys, values, weights, positions, b.lens, b.table, b.cu, b.n, 0.125)
    assert (np.abs(out.double().cpu().numpy() - want[0]) <= 2.0**-8 * np.abs(want[0]) + want[3]).all()
    rows = b.table[4, :300 // 16]
    assert (np.abs(ledger.weights.double().cpu().numpy() - want[1])[rows] <= want[4][rows]).all()


def test_strided_queries(cuda):
    b = Batch(14, [90, 33], [1, 33], 16, 8, 2, 64)
    wide = torch.zeros((b.tokens, 12, 80), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:10, 8:72] = b.q.cuda()
    _check(b, _state(b), q=wide[:, 2:10, 8:72])
    heads = b.q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    _check(b, _state(b), q=heads)


def test_as_the_dense_operator(cuda):
    """The outputs of the framework's own attention, which rounds probabilities to bf16: within two of its steps."""
    b = Batch(15, [700, 300, 64], [1, 100, 1], 16, 8, 2, 128)
    state = _state(b)
    out, _ = _check(b, state)
    dense = ops.ragged_paged_attention(b.q.cuda(), state[0].cuda(), *b.meta(), sm_scale=b.dim ** -0.5)
    assert (out.float() - dense.float()).abs().max() <= 2e-2


def test_bad_pages_and_lengths(cuda):
    """Pages outside the pool count for nothing, lengths past the table end with it; both are flagged."""
    b = Batch(16, [64, 40, 90], [1, 1, 20], 16, 4, 2, 64)
    state = _state(b)
    eviction.read_error_word(clear=True)
    lens, table, cu, num = b.meta()
    broken = table.clone()
    broken[0, 1], broken[1, 0], broken[2, 4] = b.total, -3, 2**31 - 1
    ledger = eviction.Ledger(torch.from_numpy(state[4]).cuda(), torch.from_numpy(state[5]).cuda())
    out = eviction.weighed_attention(b.q.cuda(), state[0].cuda(), ledger, lens, broken, cu, num, sm_scale=0.125)
    assert bool(out.isfinite().all()) and eviction.read_error_word(clear=True) == eviction._bounded_lib.ERR_PAGE
    # the table's 64 keys of sequence 0, as if the length said so
    narrow = table[:, :4].contiguous()
    long = lens.clone()
    long[0] = 1000
    ledgers = [eviction.Ledger(torch.from_numpy(state[4]).cuda(), torch.from_numpy(state[5]).cuda()) for _ in range(2)]
    one = torch.tensor([1], dtype=torch.int32, device="cuda")
    got = eviction.weighed_attention(b.q.cuda(), state[0].cuda(), ledgers[0], long, narrow, cu, one, sm_scale=0.125)
    assert eviction.read_error_word(clear=True) == eviction._bounded_lib.ERR_LEN
    want = eviction.weighed_attention(b.q.cuda(), state[0].cuda(), ledgers[1], lens, narrow, cu, one, sm_scale=0.125)
    assert torch.equal(got[:1], want[:1]) and torch.equal(ledgers[0].weights, ledgers[1].weights)
    assert eviction.read_error_word(clear=True) == 0


def test_the_same_again(cuda):
    """Two runs on the same inputs agree to the bit."""
    b = Batch(17, [5000, 300, 900], [1, 50, 1], 16, 8, 2, 128)
    state = _state(b)
    first, second = _check(b, state), _check(b, state)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1].weights, second[1].weights)


def test_captured_with_other_lengths(cuda):
    rng = np.random.default_rng(18)
    b = Batch(18, [600, 600, 600, 600], [1, 1, 1, 1], 16, 8, 2, 64)
    state = _state(b)
    pool, q = state[0].cuda(), b.q.cuda()
    lens, table, cu, num = b.meta()
    ledger = eviction.Ledger(torch.from_numpy(state[4]).cuda(), torch.from_numpy(state[5]).cuda())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eviction.weighed_attention(q, pool, ledger, lens, table, cu, num, sm_scale=0.125)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = eviction.weighed_attention(q, pool, ledger, lens, table, cu, num, sm_scale=0.125)
        graphs.append((graph, out))
    for turn in range(6):
        lens.copy_(i32(rng.integers(1, 601, 4)))
        q.normal_()
        graph, out = graphs[turn % 2]
        before = eviction.Ledger(ledger.weights.clone(), ledger.positions.clone())
        graph.replay()
        torch.cuda.synchronize()
        want = eviction.weighed_attention(q, pool, before, lens, table, cu, num, sm_scale=0.125)
        assert torch.equal(out, want) and torch.equal(ledger.weights, before.weights), turn
        assert torch.equal(ledger.positions, before.positions)
        torch.empty(1000, device="cuda").normal_()


def test_two_streams_at_once(cuda):
    """Two pools on two streams, calls that may overlap."""
    bs = [Batch(19 + i, [3000, 50, 800], [1, 20, 1], 16, 8, 2, 128) for i in range(2)]
    states = [_state(b) for b in bs]
    want = [_check(b, s) for b, s in zip(bs, states)]
    args = [(b.q.cuda(), s[0].cuda(), *b.meta()) for b, s in zip(bs, states)]
    ledgers = [eviction.Ledger(torch.from_numpy(s[4]).cuda(), torch.from_numpy(s[5]).cuda()) for s in states]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [None, None]
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            q, pool, *meta = args[i]
            got[i] = eviction.weighed_attention(q, pool, ledgers[i], *meta, sm_scale=128 ** -0.5)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert torch.equal(got[i], want[i][0]) and torch.equal(ledgers[i].weights, want[i][1].weights)


def test_no_tokens(cuda):
    b = Batch(21, [5], [1], 16, 4, 2, 64)
    state = _state(b)
    ledger = eviction.Ledger(torch.from_numpy(state[4]).cuda(), torch.from_numpy(state[5]).cuda())
    lens, table, cu, num = b.meta()
    out = eviction.weighed_attention(b.q[:0].cuda(), state[0].cuda(), ledger, lens, table, torch.zeros_like(cu), num)
    assert out.shape[0] == 0 and np.array_equal(ledger.weights.cpu().numpy(), state[4])
