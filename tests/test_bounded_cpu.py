"""Refusals of rotation, weighed attention, eviction and trimming before any launch, and their binding: no GPU needed."""

import ctypes
import math
import pathlib
import re
import subprocess

import pytest
import torch

from tpu_cake_amd import _bounded_lib, _sparse_lib, eviction, paging, rotary, sparse

ROOT = pathlib.Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "rpa_bounded.h").read_text()
FAKE = [ctypes.c_void_p((i + 1) << 44) for i in range(16)]  # far apart, never dereferenced: every call here is refused
MOST = 2**31 - 2**16 - 1


@pytest.fixture(scope="module")
def lib():
    if not _bounded_lib.library_path().exists():
        from tpu_cake_amd import build
        build.build()
    return _bounded_lib.load()


def _functions():
    text = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    return dict(re.findall(r"\b(rpa_[a-z_]+)\s*\(([^)]*)\)\s*;", text))


def test_header_binding_and_library_agree(lib):
    assert sorted(_functions()) == sorted(_bounded_lib.EXPORTED_SYMBOLS)
    for name, params in _functions().items():
        count = 0 if params.strip() == "void" else params.count(",") + 1
        assert len(getattr(lib, name).argtypes) == count, name
    assert lib.rpa_bounded_abi_version() == _bounded_lib.ABI_VERSION


def test_structs_match_c(tmp_path):
    structs = {"rpa_rotate_shape_t": _bounded_lib.RpaRotateShape, "rpa_weigh_shape_t": _bounded_lib.RpaWeighShape,
               "rpa_weigh_options_t": _bounded_lib.RpaWeighOptions, "rpa_choose_shape_t": _bounded_lib.RpaChooseShape,
               "rpa_move_shape_t": _bounded_lib.RpaMoveShape}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "rpa_bounded.h"\nint main(void){' + "\n".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == want


# ---- rotation ----
def _rotate(**kw):
    return _bounded_lib.RpaRotateShape(**{**dict(
        num_tokens=4, num_q_heads=8, num_kv_heads=2, head_dim=128, rotated=128, interleaved=0, max_num_seqs=4, weight_bytes=2,
        q_token_stride=1024, q_head_stride=128, k_token_stride=256, k_head_stride=128, q_out_token_stride=1024,
        q_out_head_stride=128, k_out_token_stride=256, k_out_head_stride=128, q_weight_stride=0, k_weight_stride=0), **kw})


def _call_rotate(lib, shape, ptrs=None):
    return lib.rpa_rotate_heads(None if shape is None else ctypes.byref(shape), 1e-6, 1.0, *(FAKE[:11] if ptrs is None else ptrs), None)


@pytest.mark.parametrize("bad,code,message", [
    (dict(num_tokens=-1), -1, b"num_tokens"), (dict(num_tokens=1 << 30), -1, b"2^30"), (dict(num_q_heads=0), -1, b"non-positive"),
    (dict(num_kv_heads=0), -1, b"non-positive"), (dict(num_kv_heads=65536), -2, b"65535"), (dict(head_dim=192), -2, b"head_dim 192"),
    (dict(head_dim=36), -2, b"head_dim 36"), (dict(rotated=130), -1, b"rotated=130"), (dict(rotated=-2), -1, b"rotated"),
    (dict(rotated=12), -1, b"multiple of 8"), (dict(rotated=7, interleaved=1), -1, b"multiple of 2"), (dict(interleaved=2), -1, b"interleaved"),
    (dict(weight_bytes=3), -1, b"weight_bytes"), (dict(max_num_seqs=0), -1, b"max_num_seqs"), (dict(max_num_seqs=MOST + 1), -1, b"max_num_seqs"),
    (dict(q_token_stride=1023), -1, b"q must"), (dict(k_head_stride=4), -1, b"k must"), (dict(q_out_head_stride=12), -1, b"q_out must"),
    (dict(q_token_stride=-1024), -1, b"negative stride"), (dict(q_weight_stride=-8), -1, b"negative stride"),
    (dict(q_out_head_stride=64), -1, b"overlap"), (dict(q_out_token_stride=512), -1, b"overlap"), (dict(k_out_token_stride=0), -1, b"overlap"),
    (dict(num_tokens=(1 << 30) - 1), -2, b"one launch")])
def test_rotate_refuses(lib, bad, code, message):
    assert _call_rotate(lib, _rotate(**bad)) == code and message in lib.rpa_bounded_last_error()


def test_rotate_refuses_pointers_and_overlaps(lib):
    shape = _rotate()
    for hole in (0, 1, 2, 3, 9, 10):
        assert _call_rotate(lib, shape, [None if i == hole else p for i, p in enumerate(FAKE[:11])]) == -1
        assert b"NULL" in lib.rpa_bounded_last_error()
    assert _call_rotate(lib, shape, [*FAKE[:6], None, None, *FAKE[8:11]]) == -1 and b"dropped needs" in lib.rpa_bounded_last_error()
    assert _call_rotate(lib, shape, [*FAKE[:6], None, *FAKE[7:11]]) == -1 and b"NULL" in lib.rpa_bounded_last_error()
    assert _call_rotate(lib, None) == -1
    at = lambda p, n: ctypes.c_void_p(p.value + n)  # noqa: E731
    for outs in ((at(FAKE[0], 16), FAKE[10]), (FAKE[9], at(FAKE[1], 512)), (FAKE[2], FAKE[10]), (FAKE[9], at(FAKE[9], 1024)),
                 (FAKE[9], FAKE[5])):
        assert _call_rotate(lib, shape, [*FAKE[:9], *outs]) == -1 and b"overlap" in lib.rpa_bounded_last_error()
    # one in place and the other not
    assert _call_rotate(lib, shape, [*FAKE[:9], FAKE[0], FAKE[10]]) == -1 and b"in place" in lib.rpa_bounded_last_error()
    # in place, and both the same
    assert _call_rotate(lib, _rotate(num_q_heads=2, q_token_stride=256, q_out_token_stride=256), [FAKE[0], FAKE[0], *FAKE[2:9], FAKE[0], FAKE[0]]) == -1
    assert b"overlap" in lib.rpa_bounded_last_error()
    assert _call_rotate(lib, _rotate(num_tokens=0), [None] * 11) == 0


def test_frequencies():
    f = rotary.frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(rotary.frequencies(8, factor=4.0), f / 4)
    g = rotary.frequencies(64, 10000.0, factor=8.0, trained=4096, slow=1.0, fast=32.0)
    f = rotary.frequencies(64, 10000.0)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.equal(g[turns <= 1], f[turns <= 1] / 8)
    between = (turns > 1) & (turns < 32)
    assert bool(((g > f / 8) & (g < f))[between].all()) and bool(between.any())
    assert rotary.frequencies(0).numel() == 0
    for bad in (dict(rotated=7), dict(rotated=-2), dict(rotated=8, base=0.0), dict(rotated=8, factor=-1.0),
                dict(rotated=8, trained=0), dict(rotated=8, trained=10, slow=2.0, fast=2.0)):
        with pytest.raises(ValueError):
            rotary.frequencies(**bad)


def test_turns_of():
    got = rotary.turns_of([2 * math.pi / 4, -2 * math.pi / 4, 0.0, 2 * math.pi * 0.75], device="cpu")
    assert got.tolist() == [1 << 62, -(1 << 62), 0, -(1 << 62)]  # quarter turns; three quarters are one back
    f = rotary.frequencies(64, 10000.0)
    whole = torch.tensor([float(t % (1 << 64)) for t in rotary.turns_of(f, device="cpu").tolist()], dtype=torch.float64)
    assert torch.allclose(whole / 2.0**64 * 2 * math.pi, f, rtol=1e-15)
    with pytest.raises(ValueError, match="finite"):
        rotary.turns_of([float("nan")], device="cpu")


# ---- weighed attention ----
OPTIONS = _bounded_lib.RpaWeighOptions(1.0, 0.0, 1.0, 1.0, 1.0)


def _weigh(**kw):
    return _bounded_lib.RpaWeighShape(**{**dict(num_tokens=4, num_q_heads=8, num_kv_heads=2, head_dim=128, total_pages=64, page_size=16,
                                                max_num_seqs=4, pages_per_seq=8, kv_dtype=0, reserved=0, q_token_stride=1024,
                                                q_head_stride=128), **kw})


def _call_weigh(lib, shape, ptrs=None, options=OPTIONS, need=1 << 39):
    ptrs = [*FAKE[:2], None, *FAKE[3:12]] if ptrs is None else ptrs
    return lib.rpa_weighed_attention(ctypes.byref(shape), None if options is None else ctypes.byref(options), *ptrs, need, None)


@pytest.mark.parametrize("bad,code,message", [
    (dict(num_q_heads=7), -1, b"divisible"), (dict(num_q_heads=0), -1, b"non-positive"), (dict(max_num_seqs=0), -1, b"non-positive"),
    (dict(pages_per_seq=1 << 28), -1, b"int32"), (dict(num_tokens=-3), -1, b"num_tokens"), (dict(kv_dtype=3), -1, b"kv_dtype"),
    (dict(head_dim=160), -2, b"head_dim 160"), (dict(head_dim=48, kv_dtype=1), -2, b"head_dim 48"), (dict(q_token_stride=1020), -1, b"q must"),
    (dict(num_q_heads=1024), -2, b"256 query heads"), (dict(num_tokens=1 << 29), -1, b"num_tokens * num_q_heads"),
    (dict(pages_per_seq=MOST + 1, page_size=1), -2, b"2^31 - 2^16 - 1"), (dict(total_pages=0), -1, b"non-positive")])
def test_weigh_refuses_shapes(lib, bad, code, message):
    assert _call_weigh(lib, _weigh(**bad)) == code and message in lib.rpa_bounded_last_error()
    if "q_token_stride" not in bad:
        assert lib.rpa_weigh_workspace_size(ctypes.byref(_weigh(**bad))) == 0


def test_weigh_refuses(lib):
    need = lib.rpa_weigh_workspace_size(ctypes.byref(_weigh()))
    assert need > 0
    good = [*FAKE[:2], None, *FAKE[3:12]]
    for hole in (0, 1, 3, 4, 5, 6, 8, 9, 10):
        assert _call_weigh(lib, _weigh(), [None if i == hole else p for i, p in enumerate(good)]) == -1
        assert b"NULL" in lib.rpa_bounded_last_error()
    assert _call_weigh(lib, _weigh(), need=need - 1) == -3
    assert _call_weigh(lib, _weigh(), [*good[:11], None], need=need) == -3
    assert _call_weigh(lib, _weigh(), options=None) == -1 and b"options" in lib.rpa_bounded_last_error()
    for decay in (-0.1, float("nan"), float("inf")):
        assert _call_weigh(lib, _weigh(), options=_bounded_lib.RpaWeighOptions(1.0, 0.0, 1.0, 1.0, decay)) == -1
        assert b"decay" in lib.rpa_bounded_last_error()
    assert _call_weigh(lib, _weigh(), FAKE[:12]) == -1 and b"fp8" in lib.rpa_bounded_last_error()
    for a, b in ((10, 0), (8, 1), (9, 8), (10, 9), (8, 4), (10, 11)):  # out, weights, positions: apart from inputs and each other
        same = list(good)
        same[a] = good[b]
        assert _call_weigh(lib, _weigh(), same) == -1 and b"overlap" in lib.rpa_bounded_last_error(), (a, b)
    odd = [good[0], ctypes.c_void_p(good[1].value + 8), *good[2:]]
    assert _call_weigh(lib, _weigh(), odd) == -1 and b"aligned" in lib.rpa_bounded_last_error()
    assert _call_weigh(lib, _weigh(num_tokens=0), [None] * 12, need=0) == 0


def test_weigh_workspaces_stay_in_bounds(lib):
    """The scores' room is what the pool or the sequences can hold, whichever is less."""
    size = lambda **kw: lib.rpa_weigh_workspace_size(ctypes.byref(_weigh(**kw)))  # noqa: E731
    wide, pool = size(pages_per_seq=1 << 20), size(pages_per_seq=1 << 20, total_pages=1 << 10)
    assert size() <= wide < pool
    assert wide < 64 * 16 * 8 * 4 + (1 << 26)  # scores of all the pool's rows, and parts
    assert size(num_tokens=2000) > size(num_tokens=8)


# ---- eviction ----
def _choose(**kw):
    return _bounded_lib.RpaChooseShape(**{**dict(max_num_seqs=4, pages_per_seq=8, num_kv_heads=2, total_pages=64, page_size=16, budget=64,
                                                 limit=80, sinks=4, recent=16, max_moves=64), **kw})


@pytest.mark.parametrize("bad,code,message", [
    (dict(max_num_seqs=0), -1, b"non-positive"), (dict(pages_per_seq=0), -1, b"non-positive"), (dict(max_moves=0), -1, b"non-positive"),
    (dict(num_kv_heads=65536), -2, b"65535"), (dict(total_pages=0), -1, b"non-positive"), (dict(budget=0), -1, b"budget"),
    (dict(limit=63), -1, b"limit"), (dict(sinks=-1), -1, b"sinks"), (dict(recent=-1), -1, b"recent"), (dict(sinks=60), -1, b"budget together"),
    (dict(sinks=2**31 - 1, recent=2**31 - 1), -1, b"budget together"), (dict(max_moves=1 << 30), -1, b"2^30"),
    (dict(pages_per_seq=1 << 28), -1, b"2^31"), (dict(max_num_seqs=1 << 28), -2, b"one launch")])
def test_choose_refuses(lib, bad, code, message):
    assert lib.rpa_choose_moves(ctypes.byref(_choose(**bad)), *FAKE[:8], 1 << 39, None) == code
    assert message in lib.rpa_bounded_last_error()
    assert lib.rpa_choose_workspace_size(ctypes.byref(_choose(**bad))) == 0


def test_choose_refuses_pointers(lib):
    for hole in (0, 1, 2, 3, 4, 6):
        assert lib.rpa_choose_moves(ctypes.byref(_choose()), *[None if i == hole else p for i, p in enumerate(FAKE[:8])], 0, None) == -1
        assert b"NULL" in lib.rpa_bounded_last_error()
    for other in (0, 1, 2, 3, 4, 5):
        assert lib.rpa_choose_moves(ctypes.byref(_choose()), *FAKE[:6], FAKE[other], FAKE[7], 0, None) == -1
        assert b"overlap" in lib.rpa_bounded_last_error()
    long = _choose(pages_per_seq=1 << 14)
    need = lib.rpa_choose_workspace_size(ctypes.byref(long))
    assert need > 0 and lib.rpa_choose_workspace_size(ctypes.byref(_choose())) == 0
    assert lib.rpa_choose_moves(ctypes.byref(long), *FAKE[:8], need - 1, None) == -3
    assert lib.rpa_choose_moves(ctypes.byref(long), *FAKE[:7], None, need, None) == -3
    assert lib.rpa_choose_moves(None, *FAKE[:8], 0, None) == -1


def _move(**kw):
    return _bounded_lib.RpaMoveShape(**{**dict(num_lists=4, max_moves=16, num_kv_heads=2, head_dim=128, total_pages=64, page_size=16,
                                               kv_dtype=0), **kw})


@pytest.mark.parametrize("bad,code,message", [
    (dict(num_lists=-1), -1, b"non-positive"), (dict(max_moves=0), -1, b"non-positive"), (dict(head_dim=24), -2, b"head_dim 24"),
    (dict(kv_dtype=2), -1, b"kv_dtype"), (dict(page_size=0), -1, b"non-positive"), (dict(num_lists=1 << 30), -2, b"one launch"),
    (dict(num_lists=2**31 - 1, max_moves=2**31 - 1, num_kv_heads=65535), -2, b"one launch")])
def test_move_refuses(lib, bad, code, message):
    assert lib.rpa_move_rows(ctypes.byref(_move(**bad)), FAKE[0], None, *FAKE[2:5], None) == code
    assert message in lib.rpa_bounded_last_error()


def test_move_refuses_pointers(lib):
    ok = ctypes.byref(_move())
    good = [FAKE[0], None, *FAKE[2:5]]
    for hole in (0, 2, 3, 4):
        assert lib.rpa_move_rows(ok, *[None if i == hole else p for i, p in enumerate(good)], None) == -1
        assert b"NULL" in lib.rpa_bounded_last_error()
    assert lib.rpa_move_rows(ok, *FAKE[:5], None) == -1 and b"fp8" in lib.rpa_bounded_last_error()
    for a, b in ((2, 0), (3, 2), (4, 3), (4, 0)):
        same = list(good)
        same[a] = good[b]
        assert lib.rpa_move_rows(ok, *same, None) == -1 and b"overlap" in lib.rpa_bounded_last_error()
    assert lib.rpa_move_rows(ok, FAKE[0], None, ctypes.c_void_p(FAKE[2].value + 4), *FAKE[3:5], None) == -1
    assert b"aligned" in lib.rpa_bounded_last_error()
    assert lib.rpa_move_rows(ctypes.byref(_move(num_lists=0)), *[None] * 5, None) == 0


# ---- trim ----
def test_trim_refuses():
    lib = _sparse_lib.load()
    shape = _sparse_lib.RpaPagingShape(4, 8, 16, 9, 0)
    call = lambda budget, limit, ptrs: lib.rpa_trim_pages(ctypes.byref(shape), budget, limit, *ptrs, None)  # noqa: E731
    for budget, limit in ((0, 5), (-1, 5), (8, 7)):
        assert call(budget, limit, FAKE[:8]) == -1 and b"budget" in lib.rpa_sparse_last_error()
    for hole in range(8):
        assert call(5, 5, [None if i == hole else p for i, p in enumerate(FAKE[:8])]) == -1 and b"NULL" in lib.rpa_sparse_last_error()
    for a, b in ((5, 0), (6, 1), (7, 4), (6, 5), (7, 6), (5, 3)):
        same = list(FAKE[:8])
        same[a] = FAKE[b]
        assert call(5, 5, same) == -1 and b"overlap" in lib.rpa_sparse_last_error()
    assert lib.rpa_trim_pages(None, 5, 5, *FAKE[:8], None) == -1


# ---- Python checks, with the device check out of the way ----
@pytest.fixture
def anywhere(monkeypatch):
    real = sparse._tensor
    for module in (sparse, rotary, eviction, paging):
        if hasattr(module, "_require_cuda"):
            monkeypatch.setattr(module, "_require_cuda", lambda name, t: None)
        if hasattr(module, "_tensor"):
            monkeypatch.setattr(module, "_tensor", lambda *a, **kw: real(*a))


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_cpu_tensors_are_refused():
    pool = _bf(4, 16, 4, 128)
    ledger = eviction.make_ledger(pool)
    assert ledger.weights.shape == ledger.positions.shape == (4, 2, 16)
    meta = (_i(2), _i(2, 8), _i(3), _i(1))
    for call in (lambda: rotary.rotate_heads(_bf(3, 4, 128), _bf(3, 2, 128), _i(3), torch.zeros(64, dtype=torch.int64)),
                 lambda: eviction.weighed_attention(_bf(3, 4, 128), pool, ledger, *meta),
                 lambda: eviction.choose_moves(ledger, _i(2), _i(2, 8), _i(1), budget=8, recent=1),
                 lambda: eviction.move_rows(pool, ledger, _i(2, 2, 4, 2)),
                 lambda: paging.trim_pages(_i(2), _i(2), _i(2, 8), _i(9), _i(1), page_size=16, budget=8)):
        with pytest.raises(ValueError, match="GPU device"):
            call()


@pytest.mark.parametrize("change,message", [
    (dict(q=_bf(3, 4)), "q must be"), (dict(k=_bf(2, 2, 128)), "k has shape"), (dict(k=_bf(3, 2, 64)), "k has shape"),
    (dict(q=torch.zeros(3, 4, 128)), "q dtype"), (dict(at=_i(4)), "positions has shape"), (dict(at=torch.zeros(3, dtype=torch.int64)), "positions dtype"),
    (dict(turns=torch.zeros(64)), "turns dtype"), (dict(turns=torch.zeros(65, dtype=torch.int64)), "65 turns"),
    (dict(turns=torch.zeros(6, dtype=torch.int64)), "6 turns"), (dict(q_weight=_bf(64)), "q_weight has shape"),
    (dict(k_weight=_bf(4, 128)), "k_weight has shape"), (dict(q_weight=torch.ones(128, dtype=torch.float16)), "q_weight dtype"),
    (dict(q_weight=_bf(128), k_weight=torch.ones(128)), "must be the same"), (dict(cu_q_lens=_i(3)), "come together"),
    (dict(dropped=_i(2)), "dropped needs"), (dict(cu_q_lens=_i(1), num_seqs=_i(1)), "two entries"),
    (dict(cu_q_lens=_i(3), num_seqs=_i(1), dropped=_i(3)), "dropped has shape"), (dict(magnitude=1), "floats"), (dict(interleaved=1), "bool"),
    (dict(out=(_bf(3, 4, 128), _bf(3, 3, 128))), "out k has shape")])
def test_rotate_python_refuses(anywhere, change, message):
    args = dict(q=_bf(3, 4, 128), k=_bf(3, 2, 128), at=_i(3), turns=torch.zeros(64, dtype=torch.int64))
    args.update({k: v for k, v in change.items() if k in args})
    kw = {k: v for k, v in change.items() if k not in args}
    with pytest.raises(ValueError, match=message):
        rotary.rotate_heads(args["q"], args["k"], args["at"], args["turns"], **kw)


@pytest.mark.parametrize("change,message", [
    (dict(soft_cap=0.0), "soft_cap"), (dict(soft_cap=torch.ones(())), "must be a float"), (dict(sm_scale=torch.ones(())), "must be a float"),
    (dict(sm_scale=None), "must be a float"), (dict(q=_bf(3, 3, 128)), "divisible"), (dict(q=_bf(3, 4, 64)), "q has shape"),
    (dict(decay=-1.0), "decay"), (dict(decay=float("nan")), "decay"), (dict(decay=float("inf")), "decay"), (dict(dropped=_i(3)), "dropped has shape"),
    (dict(ledger=eviction.Ledger(torch.zeros(4, 2, 8), _i(4, 2, 16))), "ledger.weights has shape"),
    (dict(ledger=eviction.Ledger(torch.zeros(4, 2, 16), _i(4, 2, 8))), "ledger.positions has shape"),
    (dict(ledger=eviction.Ledger(_i(4, 2, 16), _i(4, 2, 16))), "ledger.weights dtype"), (dict(v_scale=2), "float or None"),
    (dict(kv_scales=torch.ones(4, 2, 2)), "requires fp8"), (dict(lens=_i(3)), "kv_lens has shape"), (dict(pool=torch.zeros(4, 16, 4, 128)), "not bf16")])
def test_weigh_python_refuses(anywhere, change, message):
    args = dict(q=_bf(3, 4, 128), pool=_bf(4, 16, 4, 128), ledger=eviction.Ledger(torch.zeros(4, 2, 16), _i(4, 2, 16)), lens=_i(2))
    args.update({k: v for k, v in change.items() if k in args})
    kw = {k: v for k, v in change.items() if k not in args}
    with pytest.raises(ValueError, match=message):
        eviction.weighed_attention(args["q"], args["pool"], args["ledger"], args["lens"], _i(2, 8), _i(3), _i(1), **kw)


@pytest.mark.parametrize("change,message", [
    (dict(budget=0), "budget"), (dict(budget=2.0), "budget"), (dict(limit=7), "limit"), (dict(max_moves=0), "max_moves"), (dict(sinks=-1), "sinks"),
    (dict(recent=-1), "recent"), (dict(recent=6, sinks=3), "exceed budget"), (dict(dropped=_i(3)), "dropped has shape"),
    (dict(ledger=(torch.zeros(4, 2, 16), _i(4, 2, 15))), "ledger.positions has shape")])
def test_choose_python_refuses(anywhere, change, message):
    kw = dict(budget=8, recent=1)
    ledger = change.get("ledger", eviction.Ledger(torch.zeros(4, 2, 16), _i(4, 2, 16)))
    kw.update({k: v for k, v in change.items() if k != "ledger"})
    with pytest.raises(ValueError, match=message):
        eviction.choose_moves(ledger, _i(2), _i(2, 8), _i(1), **kw)
    with pytest.raises(TypeError, match="Ledger"):
        eviction._ledger(3, (None, None, None), None)


@pytest.mark.parametrize("moves,scales,message", [
    (_i(2, 3, 4, 2), None, "moves has shape"), (_i(2, 2, 4), None, "moves has shape"), (_i(2, 2, 0, 2), None, "room"),
    (torch.zeros(2, 2, 4, 2), None, "moves dtype"), (_i(2, 2, 4, 2), torch.ones(4, 2, 2), "requires fp8")])
def test_move_python_refuses(anywhere, moves, scales, message):
    with pytest.raises(ValueError, match=message):
        eviction.move_rows(_bf(4, 16, 4, 128), eviction.Ledger(torch.zeros(4, 2, 16), _i(4, 2, 16)), moves, kv_scales=scales)


@pytest.mark.parametrize("change,message", [
    (dict(budget=0), "budget"), (dict(limit=7), "limit"), (dict(budget=1.5), "budget"), (dict(dropped=_i(3)), "dropped has shape"),
    (dict(page_size=0), "page_size")])
def test_trim_python_refuses(anywhere, monkeypatch, change, message):
    kw = dict(page_size=16, budget=8)
    kw.update({k: v for k, v in change.items() if k != "dropped"})
    with pytest.raises(ValueError, match=message):
        paging.trim_pages(_i(2), change.get("dropped", _i(2)), _i(2, 8), _i(9), _i(1), **kw)


def test_preflight_pages():
    table = torch.tensor([[3, 1, 9], [2, 3, 0]], dtype=torch.int32)
    eviction.preflight_pages(torch.tensor([20, 16]), table, 16)  # 3, 1 and 2
    with pytest.raises(ValueError, match="twice"):
        eviction.preflight_pages(torch.tensor([20, 17]), table, 16)
    eviction.preflight_pages(torch.tensor([0, -4]), table, 16)
