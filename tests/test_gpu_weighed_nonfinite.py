"""weighed_attention with queries that are not numbers: what they must not reach, against the formula in 64 bits.

Tolerances as in test_gpu_weighed_attention: the output's rounding (bf16, 2^-8 of the value) and what the oracle bounds for
scores and sums in 32 bits.
"""

import numpy as np
import pytest
import torch

from oracle import bounded_oracle as orc
from tests.sparse_cases import Batch
from tpu_cake_amd import eviction

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (128, "fp8"), (256, "bf16"), (64, "bf16"), (96, "bf16"), (112, "fp8")])
@pytest.mark.parametrize("lens,new,spare", [
    ([300, 40], [200, 1], 0),        # few keys: a workgroup's waves share them
    ([40000, 300], [300, 70], 0),    # many: a wave has keys of its own
    ([300] + [9] * 139, [200] + [2] * 139, 0),  # many rows of the table: likewise
    ([300, 40], [200, 1], 250)])     # fewer tokens than rows of the table: no tiles
def test_a_query_that_is_not_a_number(cuda, dim, kind, lens, new, spare):
    """One head of one token of a chunk is NaN: the keys that the token sees weigh NaN for the head's kv head, later ones do not."""
    b = Batch(dim, lens, new, 64, 4, 2, dim, spare=spare)
    token, head = 3 * new[0] // 8, 1  # of the first sequence; kv head 0's second head
    at = lens[0] - new[0] + token     # its position
    pool, scales, keys, values = b.pool(kind)
    weights = np.random.default_rng(dim).uniform(0, 0.1, (b.total, 2, 64)).astype(np.float32)
    positions = np.zeros(weights.shape, np.int32)
    q = b.q.clone()
    q[token, head] = float("nan")
    b.q[token, head] = 0  # the oracle's: what the token adds is not looked at
    ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.from_numpy(positions).cuda())
    out = eviction.weighed_attention(q.cuda(), pool.cuda(), ledger, *b.meta(), sm_scale=dim ** -0.5,
                                     kv_scales=None if scales is None else torch.from_numpy(scales).cuda())
    want = orc.weighed_attention(b.q.double().numpy(), keys, values, weights, positions, b.lens, b.table, b.cu, b.n, dim ** -0.5)
    got = out.double().cpu().numpy()
    rest = np.ones(got.shape[:2], bool)
    rest[token, head] = False
    assert np.isnan(got[token, head]).all()
    assert (np.abs(got - want[0]) <= 2.0**-8 * np.abs(want[0]) + want[3])[rest].all()
    got = ledger.weights.double().cpu().numpy()
    seen = np.zeros(got.shape, bool)
    row = np.arange(at + 1)
    seen[b.table[0, row // 64], 0, row % 64] = True
    assert np.isnan(got[seen]).all()
    bad = ~(np.abs(got - want[1]) <= want[4] + 1e-30) & ~seen
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], got[bad][:4], want[1][bad][:4])
    np.testing.assert_array_equal(ledger.positions.cpu().numpy(), want[2])


def _late_value(b, pool, kind, seq, row, head):
    """A value of one key that is not a number (fp8: the code) or infinite."""
    pool = pool.clone()
    page, off = int(b.table[seq, row // b.page_size]), row % b.page_size
    if kind == "bf16":
        pool[page, off, 2 * head + 1, 3::7] = float("inf")
    else:
        pool.view(torch.uint8)[page, off, 2 * head + 1, 3::7] = 0x7F
    return pool


@pytest.mark.parametrize("dim,kind", [(128, "bf16"), (128, "fp8"), (256, "bf16"), (64, "bf16"), (96, "bf16"), (112, "fp8")])
@pytest.mark.parametrize("lens,new", [([20000], [40]), ([700, 90], [300, 1])])
def test_a_late_value_in_a_tile_of_many_shares(cuda, dim, kind, lens, new):
    """A value that only a chunk's later tokens see is not finite: the earlier ones of its tile are right, though the tile's
    keys are spread over many workgroups."""
    b = Batch(dim, lens, new, 16, 8, 2, dim)
    pool, scales, keys, values = b.pool(kind)
    token = 20  # of the first tile, 32 tokens
    row, head = lens[0] - new[0] + token, 1
    poison = _late_value(b, pool, kind, 0, row, head)
    weights = np.zeros((b.total, 2, 16), np.float32)
    ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.zeros(weights.shape, dtype=torch.int32, device="cuda"))
    out = eviction.weighed_attention(b.q.cuda(), poison.cuda(), ledger, *b.meta(), sm_scale=dim ** -0.5,
                                     kv_scales=None if scales is None else torch.from_numpy(scales).cuda())
    want = orc.weighed_attention(b.q.double().numpy(), keys, values, weights, weights.astype(np.int32), b.lens, b.table, b.cu, b.n,
                                 dim ** -0.5)
    got = out.double().cpu().numpy()
    seen = np.zeros(got.shape, bool)
    seen[token:new[0], 4:, 3::7] = True
    assert not np.isfinite(got[seen]).any()
    bad = ~(np.abs(got - want[0]) <= 2.0**-8 * np.abs(want[0]) + want[3]) & ~seen
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4])
    got = ledger.weights.double().cpu().numpy()
    assert (np.abs(got - want[1]) <= want[4] + 1e-30).all()


def test_a_scale_that_is_not_finite(cuda):
    """The page of a chunk's last tokens has an infinite scale of values: tokens before it do not see it."""
    b = Batch(9, [328], [200], 16, 4, 1, 64)
    pool, scales, keys, values = b.pool("fp8")
    scales[b.table[0, 20], :, 1] = np.inf  # rows 320 .. 327
    weights = np.zeros((b.total, 1, 16), np.float32)
    ledger = eviction.Ledger(torch.from_numpy(weights).cuda(), torch.zeros(weights.shape, dtype=torch.int32, device="cuda"))
    out = eviction.weighed_attention(b.q.cuda(), pool.cuda(), ledger, *b.meta(), sm_scale=0.125, kv_scales=torch.from_numpy(scales).cuda())
    want = orc.weighed_attention(b.q.double().numpy(), keys, values, weights, weights.astype(np.int32), b.lens, b.table, b.cu, b.n, 0.125)
    got = out.double().cpu().numpy()
    assert not np.isfinite(got[192:]).all(-1).any()
    assert (np.abs(got - want[0]) <= 2.0**-8 * np.abs(want[0]) + want[3])[:192].all()


@pytest.mark.parametrize("what", ["an old value", "a query"])
@pytest.mark.parametrize("hq,kind", [(2, "bf16"), (2, "fp8"), (16, "bf16")])
def test_what_is_not_finite_for_all_costs_nothing(cuda, hq, kind, what):
    """A value that every token of the chunk sees, or a token's own query, is not finite: nothing could be done again to mend
    it.  Done again token by token the call took 5 (16 query heads over 2 kv heads) to 25 times (2) as long."""
    b = Batch(hq, [3000], [1500], 16, hq, 2, 128)
    pool, scales, *_ = b.pool(kind)
    q, pool, clean = b.q.cuda(), pool.cuda(), (b.q.cuda(), pool.cuda())
    if what == "a query":
        q = q.clone()
        q[::100] = float("nan")
    else:
        pool = _late_value(b, pool, kind, 0, 700, 0)
    ledger, meta = eviction.make_ledger(pool), b.meta()
    scales = None if scales is None else torch.from_numpy(scales).cuda()
    times = []
    for x, y in (clean, (q, pool)):
        rounds = []
        for _ in range(7):
            a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            eviction.weighed_attention(x, y, ledger, *meta, sm_scale=128 ** -0.5, kv_scales=scales)
            z.record()
            z.synchronize()
            rounds.append(a.elapsed_time(z))
        times.append(sorted(rounds)[3])
    assert times[1] < 2 * times[0], times
