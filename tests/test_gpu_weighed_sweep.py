"""weighed_attention over drawn batches: types, groups, pages, chunks beside single tokens, rows of the table and of the batch that
nobody has, caches shorter than their step.  Tolerances as in test_gpu_weighed_attention."""

import numpy as np
import pytest

from tests.sparse_cases import Batch
from tests.test_gpu_weighed_attention import _check, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(24))
def test_drawn_batches(cuda, seed):
    rng = np.random.default_rng(1000 + seed)
    kind = ["bf16", "fp8"][seed % 2]
    dim = int(rng.choice([64, 80, 112, 128, 256] if kind == "fp8" else [32, 40, 64, 88, 96, 128, 256]))
    hkv = int(rng.choice([1, 2, 3, 5, 8]))
    hq = hkv * int(rng.choice([1, 2, 3, 4, 7, 16, 17]))
    n = int(rng.choice([1, 2, 5, 40]))
    lens = np.maximum(1, np.exp(rng.uniform(0, np.log(1500 if n < 40 else 200), n))).astype(int)
    new = np.minimum(lens, np.exp(rng.uniform(0, np.log(300 if n < 40 else 30), n)).astype(int))
    new[rng.random(n) < 0.3] = 1
    new[rng.random(n) < 0.1] = 0
    b = Batch(seed, lens.tolist(), new.tolist(), int(rng.choice([1, 5, 16, 24, 64])), hq, hkv, dim, spare=int(rng.choice([0, 1, 60])),
              pad=int(rng.choice([0, 3, 100])))
    dropped = rng.integers(0, 1000, len(b.lens))
    _check(b, _state(b, kind, seed), decay=float(rng.choice([0.0, 0.5, 1.0])), dropped=dropped,
           soft_cap=float(rng.choice([0.0, 0.0, 20.0])) or None)


@pytest.mark.parametrize("tokens,keys", [([300, 1], [100, 40]), ([129], [1]), ([700], [650]), ([64, 200, 3], [0, 150, 2])])
def test_caches_shorter_than_their_step(cuda, tokens, keys):
    """The first tokens of such a sequence see no key, and all of its keys are new."""
    b = Batch(len(tokens), np.maximum(tokens, keys).tolist(), tokens, 16, 8, 2, 64)  # pages of their own for all rows
    b.lens = np.array(keys)
    _check(b, _state(b))
