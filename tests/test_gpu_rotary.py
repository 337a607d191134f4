"""Norms and rotation of queries and keys against the formula in 64 bits.

Tolerance: the result is rounded once, half a step of bf16, 2^-8 of the value.  Before that, in 32 bits, of the sum of
the magnitudes a result is made of (|a| + |b|): the norm's sum (21 additions at most, halved by the root), its
quotient, root and products (5), sine and cosine (2 steps each of 2^-24, and 2^-29), their products and sum (3), the
magnitude (1): below 24 * 2^-24 < 2^-19.
"""

import numpy as np
import pytest
import torch

from oracle import bounded_oracle as orc
from tpu_cake_amd import rotary

pytestmark = pytest.mark.gpu


def _turns(rotated, rng):
    whole = [int(x) for x in rng.integers(0, 1 << 63, rotated // 2)]
    whole[:3] = [1 << 63, 1, (1 << 64) - 5][:len(whole)]  # half a turn, next to none, a step back
    return whole, torch.tensor([w - (1 << 64) if w >> 63 else w for w in whole], dtype=torch.int64, device="cuda")


def _close(got, want, size, live=None):
    got = got.double().cpu().numpy()
    bad = np.abs(got - want) > 2.0**-8 * np.abs(want) + 2.0**-19 * size
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


def _both(q, k, at, whole, turns, weights, **kw):
    got = rotary.rotate_heads(q, k, torch.as_tensor(at, dtype=torch.int32, device="cuda"), turns, q_weight=weights[0],
                              k_weight=weights[1], **{x: kw[x] for x in kw if x not in ("add",)})
    for y, x, w in ((got[0], q, weights[0]), (got[1], k, weights[1])):
        want, size = orc.rotate_heads(x.double().cpu().numpy(), np.asarray(at) + kw.get("add", 0), whole,
                                      interleaved=kw.get("interleaved", False), magnitude=kw.get("magnitude", 1.0),
                                      weight=None if w is None else w.double().cpu().numpy(), eps=kw.get("eps", 1e-6))
        _close(y, want, size)
    return got


@pytest.mark.parametrize("tokens,hq,hkv,dim,rotated,interleaved,norm", [
    (1, 1, 1, 128, 128, False, True), (1, 32, 8, 128, 128, False, False), (7, 8, 2, 64, 64, False, True),
    (5, 6, 2, 96, 96, False, True), (5, 6, 2, 96, 24, False, True), (3, 4, 4, 40, 40, False, True), (3, 4, 4, 40, 8, True, True),
    (3, 5, 1, 256, 256, False, True), (3, 5, 1, 256, 64, True, True), (9, 16, 2, 128, 64, False, True),
    (9, 16, 2, 128, 50, True, True), (4, 3, 1, 32, 32, True, False), (4, 3, 3, 32, 0, False, True), (4, 3, 3, 120, 120, False, True),
    (6, 7, 7, 72, 56, False, True), (2500, 9, 2, 128, 128, False, True), (11, 71, 1, 64, 32, True, True)])
def test_shapes(cuda, tokens, hq, hkv, dim, rotated, interleaved, norm):
    rng = np.random.default_rng(tokens * 1000 + dim + rotated)
    whole, turns = _turns(rotated, rng)
    g = torch.Generator(device="cuda").manual_seed(dim)
    q = torch.empty((tokens, hq, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    k = torch.empty((tokens, hkv, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    weights = [torch.empty(dim, dtype=torch.bfloat16, device="cuda").normal_(1.0, 0.2, generator=g) if norm else None for _ in "qk"]
    at = rng.integers(0, 1 << 31, tokens)
    _both(q, k, at, whole, turns, weights, interleaved=interleaved, magnitude=1.25)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_for_each_head_and_for_one_of_the_two(cuda, dtype):
    rng = np.random.default_rng(3)
    whole, turns = _turns(64, rng)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.empty((5, 12, 64), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    k = torch.empty((5, 3, 64), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    per_head = torch.empty((12, 64), dtype=dtype, device="cuda").normal_(generator=g)
    one = torch.empty(64, dtype=dtype, device="cuda").normal_(generator=g)
    at = rng.integers(0, 1 << 20, 5)
    _both(q, k, at, whole, turns, [per_head, one], eps=0.5)
    _both(q, k, at, whole, turns, [None, one])
    _both(q, k, at, whole, turns, [per_head, None])


def test_rows_of_zeros_and_of_infinities(cuda):
    """A row of zeros stays zeros; what is not rotated passes infinities and NaN on as they are."""
    whole, turns = _turns(32, np.random.default_rng(4))
    for interleaved in (False, True):
        q = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
        k = torch.ones((2, 1, 64), dtype=torch.bfloat16, device="cuda")
        k[:, :, 40], k[:, :, 41] = float("inf"), float("nan")
        out = rotary.rotate_heads(q, k, torch.tensor([5, 70], dtype=torch.int32, device="cuda"), turns, interleaved=interleaved,
                                  q_weight=torch.ones(64, dtype=torch.bfloat16, device="cuda"))
        assert torch.equal(out[0], q)
        assert torch.equal(out[1][:, :, 32:41], k[:, :, 32:41]) and torch.equal(out[1][:, :, 42:], k[:, :, 42:])
        assert bool(out[1][:, :, 41].isnan().all()) and bool(out[1][:, :, :32].isfinite().all())


@pytest.mark.parametrize("sequences", [3, 200])
def test_slices_padding_and_dropped(cuda, sequences):
    """Slices of one projection's output, a batch with padding, positions past what the cache holds."""
    rng = np.random.default_rng(5)
    hq, hkv, dim = 8, 2, 128
    lens = rng.integers(0, 4, sequences)
    lens[0] = 5
    cu = np.concatenate([[0], np.cumsum(lens), [cu_end := int(lens.sum()) + 7] * 3])  # rows past num_seqs hold anything
    tokens = int(lens.sum()) + 11
    whole, turns = _turns(dim, rng)
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.empty((tokens, hq + 2 * hkv, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
    dropped = rng.integers(0, 1 << 30, sequences + 3)
    at = rng.integers(0, 1 << 30, tokens)
    seq = np.repeat(np.arange(sequences), lens)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    w = torch.empty(dim, dtype=torch.float32, device="cuda").normal_(generator=g)
    kw = dict(q_weight=w, k_weight=w, cu_q_lens=i32(cu), num_seqs=i32([sequences]), dropped=i32(dropped))
    got = rotary.rotate_heads(q, k, i32(at), turns, **kw)
    live = len(seq)
    for y, x in zip(got, (q, k)):
        want, size = orc.rotate_heads(x.double().cpu().numpy()[:live], at[:live] + dropped[seq], whole, weight=w.double().cpu().numpy())
        _close(y[:live], want, size)
        assert not y[live:].any()
    # in place: the same values, and rows past the last, values and v heads as they were
    held = qkv.clone()
    same = rotary.rotate_heads(q, k, i32(at), turns, out=(q, k), **kw)
    assert same[0].data_ptr() == q.data_ptr()
    assert torch.equal(q[:live], got[0][:live]) and torch.equal(k[:live], got[1][:live])
    assert torch.equal(qkv[live:], held[live:]) and torch.equal(qkv[:, hq + hkv:], held[:, hq + hkv:])


def test_heads_before_tokens(cuda):
    """Tensors of [heads, tokens, dim], transposed; an output of its own layout."""
    rng = np.random.default_rng(6)
    whole, turns = _turns(64, rng)
    q = torch.from_numpy(rng.standard_normal((4, 9, 64), np.float32)).to(torch.bfloat16).cuda().transpose(0, 1)
    k = torch.from_numpy(rng.standard_normal((2, 9, 64), np.float32)).to(torch.bfloat16).cuda().transpose(0, 1)
    at = rng.integers(0, 1000, 9)
    got = _both(q, k, at, whole, turns, [None, None])
    out = torch.full((4, 9, 72), 7.0, dtype=torch.bfloat16, device="cuda")[:, :, :64].transpose(0, 1), torch.empty_like(got[1])
    _both(q, k, at, whole, turns, [None, None], out=out)
    assert torch.equal(out[0], got[0]) and torch.equal(out[1], got[1])


def test_no_tokens(cuda):
    q = torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    k, at = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    out = rotary.rotate_heads(q, k, at, _turns(64, np.random.default_rng(0))[1])
    assert out[0].shape == q.shape and out[1].shape == k.shape


def test_angles_of_far_positions(cuda):
    """A pair (1, 0) becomes the cosine and sine of the angle: within half a step of them at every position."""
    f = rotary.frequencies(128, 1e6, factor=4.0, trained=8192)
    turns = rotary.turns_of(f)
    at = np.concatenate([np.arange(64), np.random.default_rng(1).integers(0, (1 << 31) - 1, 400), [2**31 - 1]])
    q = torch.zeros((len(at), 1, 128), dtype=torch.bfloat16, device="cuda")
    q[:, :, :64] = 1.0
    got, _ = rotary.rotate_heads(q, q.clone(), torch.as_tensor(at, dtype=torch.int32, device="cuda"), turns)
    whole = [t % (1 << 64) for t in turns.tolist()]
    angle = 2 * np.pi * np.array([[(int(p) * w) % (1 << 64) for w in whole] for p in at], np.float64) / 2.0**64
    for part, want in ((got[:, 0, :64], np.cos(angle)), (got[:, 0, 64:], np.sin(angle))):
        assert (np.abs(part.double().cpu().numpy() - want) <= 2.0**-8 * np.abs(want) + 2.0**-21).all()


def test_captured_and_on_another_stream(cuda):
    rng = np.random.default_rng(8)
    whole, turns = _turns(128, rng)
    q = torch.empty((33, 8, 128), dtype=torch.bfloat16, device="cuda").normal_()
    k = torch.empty((33, 2, 128), dtype=torch.bfloat16, device="cuda").normal_()
    at = torch.zeros(33, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        rotary.rotate_heads(q, k, at, turns)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = rotary.rotate_heads(q, k, at, turns)
    for turn in range(4):
        at.copy_(torch.as_tensor(rng.integers(0, 1 << 30, 33), dtype=torch.int32))
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = rotary.rotate_heads(q, k, at, turns)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), turn
        torch.empty(1000, device="cuda").normal_()
