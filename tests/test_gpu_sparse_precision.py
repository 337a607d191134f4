"""sparse_paged_attention where values cancel: what is left of a row is far smaller than its weights.

Keys 0 to count - 1 of a sequence score 0 and the next one -x_h for head h; the first ones' values in dimension h are
the pieces of -exp(-x_h) and the last one's is 1.  So the oracle's output there is what the pieces leave of the
weight, and weights held in 16 bits would lose most of it.

The tolerance is half a step of the output and, relative to values of at most `top`, what fp32 rounds: a weight of at most 1
by 3 * 2^-24 (its score's product, |s| < 1.02, and the constant log2 e together 2^-24 of the weight, exp2 an ulp of 2^-24, weight *
scale 2^-24), and three products of each of count + 1 weights, each added with a rounding of at most 2^-24 of top, as no
partial sum passes it; all that over the sum of weights, which is at least count.
"""

import numpy as np
import pytest
import torch

from oracle import sparse_oracle as orc
from sparse_cases import i32
from tpu_cake_amd import sparse

pytestmark = pytest.mark.gpu

HEADS, DIM, PAGE = 16, 64, 16


def _pieces(x, count, dtype, step):
    """x as `count` values of a type, each the nearest to what the earlier ones leave; `step`: of a code."""
    got = []
    for _ in range(count):
        got.append(float(torch.tensor(x / step, dtype=torch.float64).to(torch.float32).to(dtype).to(torch.float64)) * step)
        x -= got[-1]
    return got


@pytest.mark.parametrize("kind,scale", [("bf16", 1.0), ("fp8", 1.0), ("fp8", 0.0123)])
@pytest.mark.parametrize("tokens,lists", [(1, 1), (1, 40), (5, 1), (5, 40)])  # rows and tiles, whole and split
def test_values_that_cancel(cuda, kind, scale, tokens, lists):
    rng = np.random.default_rng(tokens + lists)
    x = rng.uniform(0.1, 0.7, HEADS)
    q = torch.zeros((tokens, HEADS, DIM), dtype=torch.bfloat16)
    q[:, :, 0] = torch.from_numpy(x.astype(np.float32)).to(torch.bfloat16)
    x = q[0, :, 0].double().numpy()
    count, top = (2, 1.0) if kind == "bf16" else (5, 256.0)
    keys, values = np.zeros((lists, PAGE, 1, DIM)), np.zeros((lists, PAGE, 1, DIM))
    values[0, count, 0, :HEADS], keys[0, count, 0, 0] = top, -1.0
    for h in range(HEADS):
        dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
        values[0, :count, 0, h] = [-p for p in _pieces(np.exp(-x[h]) * top, count, dtype, 1.0)]
    keys[0, count + 1:, 0, 0] = -384.0  # weights of e^-38 and less
    keys[1:, :, 0, 0] = -384.0
    pool = torch.from_numpy(np.stack([keys, values], 3)).float().to(torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn)
    held = pool.double().numpy()
    np.testing.assert_array_equal(held[:, :, :, 0], keys)
    np.testing.assert_array_equal(held[:, :, :, 1], values)
    kw = {}
    if kind == "fp8":
        page_scales = np.ones((lists, 1, 2), np.float32)
        page_scales[:, :, 1] = scale
        values = values * page_scales[:, None, :, 1:].astype(np.float64)
        kw["kv_scales"] = torch.from_numpy(page_scales).cuda()
    picked = np.tile(np.arange(lists), (tokens, 1, 1))
    lens, table, cu = np.array([lists * PAGE]), np.arange(lists)[None], np.array([0, tokens])
    got = sparse.sparse_paged_attention(q.cuda(), pool.view(lists, PAGE, 2, DIM).cuda(), i32(picked), i32(lens), i32(table), i32(cu),
                                        i32([1]), sm_scale=1.0, **kw).double().cpu().numpy()
    want = orc.sparse_attention(q.double().numpy(), keys, values, picked, lens, table, cu, 1, 1.0)
    tol = 2.0**-8 * np.abs(want) + (3 + 3 * (count + 1)) / count * 2.0**-24 * np.abs(values).max()
    left = np.abs(want[:, np.arange(HEADS), np.arange(HEADS)])
    assert (left < 2.0**-15 * np.abs(values).max()).all()  # of weights of 1: they cancel
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, f"{worst} times the tolerance"
