"""append_kv: rows, fp8 codes and the page index equal the oracle's, bit for bit."""

import numpy as np
import pytest
import torch

from oracle import sparse_oracle as orc
from sparse_cases import i32
from tpu_cake_amd import paging, sparse

pytestmark = pytest.mark.gpu


def _codes(x, scale):
    """e4m3 codes (as values) of float32 x / scale, the division rounded to float32."""
    return orc.e4m3(np.clip((x.astype(np.float32) / scale.astype(np.float32)).astype(np.float64), -448, 448))


class Stream:
    """Sequences that grow by chunks, their pool on the GPU beside what it should hold."""

    def __init__(self, seed, lens, page, hkv, dim, kind, scalar=False):
        self.rng = np.random.default_rng(seed)
        self.page, self.hkv, self.dim, self.kind = page, hkv, dim, kind
        pages = -(-np.array(lens) // page)
        self.total = int(pages.sum()) + 2
        order = self.rng.permutation(self.total)
        self.table = [order[int(pages[:i].sum()):int(pages[:i + 1].sum())] for i in range(len(lens))]
        self.at, self.lens = np.zeros(len(lens), int), lens
        shape = (self.total, page, 2 * hkv, dim)
        self.want = self.rng.standard_normal(shape).astype(np.float32)
        self.scales = None
        if kind == "fp8":
            self.pool = torch.from_numpy(self.want).to(torch.float8_e4m3fn).cuda()
            if not scalar:
                self.scales = self.rng.uniform(0.002, 0.02, (self.total, hkv, 2)).astype(np.float32)
        else:
            self.pool = torch.from_numpy(self.want).to(torch.bfloat16).cuda()
        self.want = self.pool.double().cpu().numpy()
        self.scalar = (0.0125, 0.02) if scalar else None
        self.index = sparse.make_page_index(self.pool)
        self.index.bounds.fill_(99)  # what other pages' indices hold is anything
        self.index.exponents.fill_(3)

    def scale(self, page, part):
        if self.kind == "bf16":
            return np.ones(self.hkv, np.float32)
        return self.scales[page, :, part] if self.scales is not None else np.full(self.hkv, self.scalar[part], np.float32)

    def grow(self, chunks, pad=0, strided=True, magnitude=1.0):
        chunks = np.minimum(chunks, np.array(self.lens) - self.at)
        slots = [int(self.table[i][p // self.page]) * self.page + p % self.page
                 for i, c in enumerate(chunks) for p in range(self.at[i], self.at[i] + c)]
        self.at += chunks
        tokens = len(slots) + pad
        x = self.rng.standard_normal((tokens, 3 * self.hkv, self.dim)).astype(np.float32) * magnitude
        x = torch.from_numpy(x).to(torch.bfloat16)
        k, v = x[:, self.hkv:2 * self.hkv], x[:, 2 * self.hkv:]
        for t, s in enumerate(slots):
            for part, y in enumerate((k, v)):
                y = y[t].float().numpy()
                if self.kind == "fp8":
                    y = _codes(y, self.scale(s // self.page, part)[:, None])
                self.want[s // self.page, s % self.page, part::2] = y
        x = x.cuda()
        k, v = x[:, self.hkv:2 * self.hkv], x[:, 2 * self.hkv:]
        if not strided:
            k, v = k.contiguous(), v.contiguous()
        slots = i32(slots + [-1] * pad)
        sparse.preflight_append(slots, self.pool)
        kw = dict(kv_scales=torch.from_numpy(self.scales).cuda()) if self.scales is not None else {}
        if self.scalar:
            kw = dict(k_scale=self.scalar[0], v_scale=self.scalar[1])
        sparse.append_kv(k, v, self.pool, slots, index=self.index, **kw)

    def check(self):
        np.testing.assert_array_equal(self.pool.double().cpu().numpy(), self.want)
        bounds, exps = np.full((self.total, self.hkv, 2, self.dim), 99), np.full((self.total, self.hkv), 3)
        for i, n in enumerate(self.at):
            for p in range(-(-int(n) // self.page)):
                page, rows = self.table[i][p], min(self.page, int(n) - p * self.page)
                keys = self.want[page, :rows, ::2].astype(np.float32) * self.scale(page, 0)[:, None]
                for h in range(self.hkv):
                    bounds[page, h], exps[page, h] = orc.page_bounds(keys[:, h])
        np.testing.assert_array_equal(self.index.exponents.cpu().numpy(), exps)
        np.testing.assert_array_equal(self.index.bounds.cpu().numpy(), bounds)


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("bf16", 64), ("bf16", 256), ("bf16", 32), ("bf16", 40), ("bf16", 96),
                                      ("bf16", 120), ("fp8", 128), ("fp8", 64), ("fp8", 256), ("fp8", 112)])
@pytest.mark.parametrize("page,hkv", [(16, 8), (1, 2), (7, 1), (64, 3), (200, 12)])
def test_grown_by_chunks_equals_from_scratch(cuda, kind, dim, page, hkv):
    s = Stream(dim + page, [40, 1, 0, 333, 97], page, hkv, dim, kind)
    s.grow(np.array([5, 1, 0, 17, 64]), pad=3)
    s.check()
    s.grow(np.array([1, 1, 1, 1, 1]), magnitude=40.0)  # the grids of open pages coarsen
    s.grow(np.array([1, 1, 1, 200, 0]), strided=False)
    s.check()
    s.grow(np.array([100, 100, 100, 100, 100]), pad=1, magnitude=0.01)
    s.check()


def test_scalar_scales_and_uint8_pools(cuda):
    s = Stream(5, [70, 9], 16, 4, 128, "fp8", scalar=True)
    s.grow(np.array([33, 9]))
    s.grow(np.array([37, 0]))
    s.check()
    pool = s.pool.clone().view(torch.uint8)
    k = torch.randn(2, 4, 128, device="cuda", dtype=torch.bfloat16)
    sparse.append_kv(k, k, pool, i32([0, 17]), k_scale=0.5, v_scale=0.25)
    sparse.append_kv(k, k, s.pool, i32([0, 17]), k_scale=0.5, v_scale=0.25)
    assert torch.equal(pool, s.pool.view(torch.uint8))


def test_every_rounding_of_fp8(cuda):
    """All bf16 values at scale 1: codes to nearest even, saturated, NaN kept."""
    bits = np.arange(1 << 16).astype(np.uint16)
    x = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).reshape(512, 1, 128)
    pool = torch.zeros((512, 1, 2, 128), dtype=torch.float8_e4m3fn, device="cuda")
    sparse.append_kv(x.cuda(), x.cuda(), pool, i32(np.arange(512)))
    got = pool[:, 0].double().cpu().numpy()
    want = x.double().numpy()
    nan = np.isnan(want)
    want = orc.e4m3(np.clip(np.where(nan, 0, want), -448, 448))
    for part in range(2):
        np.testing.assert_array_equal(np.isnan(got[:, part:part + 1]), nan)
        np.testing.assert_array_equal(got[:, part:part + 1][~nan], want[~nan])


def test_extreme_keys_in_the_index(cuda):
    """Zeros, subnormals, the largest values, infinities and NaN: the oracle's bounds."""
    values = [0.0, -0.0, 1e-40, -1e-40, 3e38, -3e38, np.inf, -np.inf, np.nan, 127.0, 127.5, -128.0, 1.0]
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.choice(values, (60, 2, 64)).astype(np.float32)).to(torch.bfloat16)
    x[:8] = torch.from_numpy(rng.choice([0.0, 1e-40, -1e-40], (8, 2, 64)).astype(np.float32)).to(torch.bfloat16)
    x[8:16] = 0
    x[16:24] = 127.0
    x[24:32, :, 3:] = 1e-3  # the first dimensions' magnitudes make the others vanish on the grid
    pool = torch.zeros((8, 8, 4, 64), dtype=torch.bfloat16, device="cuda")
    index = sparse.make_page_index(pool)
    sparse.append_kv(x.cuda(), x.cuda(), pool, i32(np.arange(60)), index=index)
    for p in range(8):
        keys = x[8 * p:min(60, 8 * p + 8)].double().numpy()
        for h in range(2):
            bounds, e = orc.page_bounds(keys[:, h])
            assert index.exponents[p, h].item() == e, (p, h)
            np.testing.assert_array_equal(index.bounds[p, h].cpu().numpy(), bounds, err_msg=f"{p} {h}")


def test_extreme_scales_in_the_index(cuda):
    """Page scales of 0, NaN and infinity: keys that the pool holds as NaN times them count as 0."""
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.choice([0.0, 1.0, -2.5, 3e38, -np.inf, np.nan], (40, 1, 64)).astype(np.float32)).to(torch.bfloat16)
    scales = np.array([0.0, np.nan, np.inf, 1e-30, 1e30], np.float32)
    pool = torch.zeros((5, 8, 2, 64), dtype=torch.float8_e4m3fn, device="cuda")
    index = sparse.make_page_index(pool)
    both = torch.from_numpy(np.repeat(scales[:, None, None], 2, axis=2)).contiguous().cuda()
    sparse.append_kv(x.cuda(), x.cuda(), pool, i32(np.arange(40)), kv_scales=both, index=index)
    with np.errstate(all="ignore"):
        keys = pool[:, :, 0].double().cpu().numpy().astype(np.float32) * scales[:, None, None]
    for p in range(5):
        bounds, e = orc.page_bounds(keys[p])
        assert index.exponents[p, 0].item() == e, p
        np.testing.assert_array_equal(index.bounds[p, 0].cpu().numpy(), bounds, err_msg=str(p))


def test_slots_outside_the_pool_are_skipped_and_flagged(cuda):
    sparse.read_error_word(clear=True)
    pool = torch.zeros((2, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    index = sparse.make_page_index(pool)
    x = torch.ones((5, 1, 64), dtype=torch.bfloat16, device="cuda")
    sparse.append_kv(x, x, pool, i32([8, -2, -1, 2**31 - 1, 3]), index=index)
    assert sparse.read_error_word(clear=True) == sparse._sparse_lib.ERR_SLOT
    want = torch.zeros_like(pool)
    want[0, 3] = 1
    assert torch.equal(pool, want)


@pytest.mark.parametrize("tokens", [6, 64])  # one workgroup's teams, and several workgroups'
def test_slots_outside_an_fp8_pool_read_no_scales(cuda, tokens):
    """Far slots beside pages that begin: per-page scales and bounds of the pool's pages only."""
    rng = np.random.default_rng(tokens)
    pages = tokens // 2
    pool = torch.zeros((pages, 4, 4, 128), dtype=torch.float8_e4m3fn, device="cuda")
    index = sparse.make_page_index(pool)
    scales = rng.uniform(0.002, 0.02, (pages, 2, 2)).astype(np.float32)
    x = torch.from_numpy(rng.standard_normal((tokens, 2, 128)).astype(np.float32)).to(torch.bfloat16)
    slots = np.full(tokens, 2**31 - 1, np.int64)
    slots[::2] = 4 * np.arange(pages)
    slots[1] = -7
    sparse.read_error_word(clear=True)
    sparse.append_kv(x.cuda(), x.cuda(), pool, i32(slots), kv_scales=torch.from_numpy(scales).cuda(), index=index)
    assert sparse.read_error_word(clear=True) == sparse._sparse_lib.ERR_SLOT
    codes = _codes(x[::2].float().numpy(), scales[:, :, :1])
    got = pool.double().cpu().numpy()
    np.testing.assert_array_equal(got[:, 0, ::2], codes)
    assert (got[:, 1:] == 0).all()
    for p in range(pages):
        for h in range(2):
            bounds, e = orc.page_bounds((codes[p, h].astype(np.float32) * scales[p, h, 0])[None])
            assert index.exponents[p, h].item() == e
            np.testing.assert_array_equal(index.bounds[p, h].cpu().numpy(), bounds)


def test_rows_past_a_page_that_grows_are_left_alone(cuda):
    pool = torch.full((3, 8, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    x = torch.randn((3, 1, 128), device="cuda").to(torch.bfloat16)
    sparse.append_kv(x, x, pool, i32([10, 11, 12]))
    left = pool.view(24, 2, 128)
    assert torch.equal(left[10:13, 0], x[:, 0]) and torch.equal(left[10:13, 1], x[:, 0])
    assert (left[:10] == 7).all() and (left[13:] == 7).all()


def test_no_tokens(cuda):
    pool = torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    x = torch.zeros((0, 1, 64), dtype=torch.bfloat16, device="cuda")
    sparse.append_kv(x, x, pool, i32([]))


def test_slots_past_32_bit_byte_offsets(cuda):
    """A pool of over 4 GiB: rows at its end."""
    pages, page = 4200, 256  # 4200 * 256 rows of 4 KiB
    pool = torch.empty((pages, page, 16, 128), dtype=torch.bfloat16, device="cuda")
    pool[-1].zero_()
    x = torch.randn((3, 8, 128), device="cuda").to(torch.bfloat16)
    last = pages * page
    index = sparse.make_page_index(pool)
    sparse.append_kv(x, -x, pool, i32([last - 256, last - 255, last - 254]), index=index)
    assert torch.equal(pool[-1, :3, ::2], x) and torch.equal(pool[-1, :3, 1::2], -x)
    assert (pool[-1, 3:] == 0).all()
    bounds, e = orc.page_bounds(x[:, 5].double().cpu().numpy())
    assert index.exponents[-1, 5].item() == e
    np.testing.assert_array_equal(index.bounds[-1, 5].cpu().numpy(), bounds)
