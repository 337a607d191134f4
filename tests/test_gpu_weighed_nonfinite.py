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
