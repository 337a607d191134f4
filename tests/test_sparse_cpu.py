"""Refusals of the sparse entry points before any launch, and their binding: no GPU needed."""

import ctypes
import pathlib
import re
import subprocess

import pytest
import torch

from tpu_cake_amd import _sparse_lib, sparse

ROOT = pathlib.Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "rpa_sparse.h").read_text()


@pytest.fixture(scope="module")
def lib():
    if not _sparse_lib.library_path().exists():
        from tpu_cake_amd import build
        build.build()
    return _sparse_lib.load()


def _functions():
    text = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    return dict(re.findall(r"\b(rpa_[a-z_]+)\s*\(([^)]*)\)\s*;", text))


def test_header_binding_and_library_agree(lib):
    assert sorted(_functions()) == sorted(_sparse_lib.EXPORTED_SYMBOLS)
    for name, params in _functions().items():
        count = 0 if params.strip() == "void" else params.count(",") + 1
        assert len(getattr(lib, name).argtypes) == count, name
    for name, value in re.findall(r"RPA_SPARSE_(ERR_\w+) = (\d+)", HEADER):
        assert getattr(_sparse_lib, name) == int(value)
    assert lib.rpa_sparse_abi_version() == _sparse_lib.ABI_VERSION


def test_structs_match_c(tmp_path):
    structs = {"rpa_paging_shape_t": _sparse_lib.RpaPagingShape, "rpa_append_shape_t": _sparse_lib.RpaAppendShape,
               "rpa_sparse_shape_t": _sparse_lib.RpaSparseShape, "rpa_sparse_options_t": _sparse_lib.RpaSparseOptions}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "rpa_sparse.h"\nint main(void){' + "\n".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == want


FAKE = [ctypes.c_void_p(4096 * (i + 1)) for i in range(16)]  # never dereferenced: every call here is refused


def _append(**kw):
    return _sparse_lib.RpaAppendShape(**{**dict(num_tokens=4, num_kv_heads=2, head_dim=128, total_pages=8, page_size=16, kv_dtype=0,
                                                k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128), **kw})


@pytest.mark.parametrize("bad,code,message", [
    (dict(num_tokens=-1), -1, b"num_tokens"), (dict(num_kv_heads=0), -1, b"non-positive"), (dict(kv_dtype=7), -1, b"kv_dtype"),
    (dict(total_pages=0), -1, b"non-positive"), (dict(page_size=1 << 20, total_pages=1 << 12), -1, b"int32"),
    (dict(k_token_stride=257), -1, b"keys must"), (dict(v_head_stride=4), -1, b"values must"),
    (dict(head_dim=24), -2, b"head_dim 24"), (dict(head_dim=36), -2, b"head_dim 36"), (dict(head_dim=192), -2, b"head_dim 192"),
    (dict(head_dim=48, kv_dtype=1), -2, b"head_dim 48"), (dict(head_dim=72, kv_dtype=1), -2, b"head_dim 72")])
def test_append_refuses(lib, bad, code, message):
    assert lib.rpa_append_kv(ctypes.byref(_append(**bad)), *FAKE[:5], 1.0, 1.0, *FAKE[5:7], None) == code
    assert message in lib.rpa_sparse_last_error()


def test_append_refuses_pointers(lib):
    ok = ctypes.byref(_append())
    for hole in (0, 1, 2, 3):
        ptrs = [None if i == hole else p for i, p in enumerate(FAKE[:5])]
        assert lib.rpa_append_kv(ok, *ptrs, 1.0, 1.0, *FAKE[5:7], None) == -1 and b"NULL" in lib.rpa_sparse_last_error()
    assert lib.rpa_append_kv(ok, *FAKE[:5], 1.0, 1.0, FAKE[5], None, None) == -1  # bounds without exponents
    odd = [ctypes.c_void_p(4104), *FAKE[1:5]]
    assert lib.rpa_append_kv(ok, *odd, 1.0, 1.0, *FAKE[5:7], None) == -1 and b"aligned" in lib.rpa_sparse_last_error()
    assert lib.rpa_append_kv(None, *FAKE[:5], 1.0, 1.0, *FAKE[5:7], None) == -1


@pytest.mark.parametrize("bad", [0.0, -0.5, float("inf"), float("nan")])
def test_append_refuses_scales(lib, monkeypatch, anywhere, bad):
    ok = ctypes.byref(_append(kv_dtype=1))
    for scales in ((bad, 1.0), (1.0, bad)):
        assert lib.rpa_append_kv(ok, *FAKE[:4], None, *scales, *FAKE[5:7], None) == -1
        assert b"positive and finite" in lib.rpa_sparse_last_error()
    real = sparse._tensor
    monkeypatch.setattr(sparse, "_tensor", lambda *a, **kw: real(*a))
    pool = torch.zeros((4, 16, 4, 128), dtype=torch.uint8)
    for scales in (dict(k_scale=bad), dict(v_scale=bad)):
        with pytest.raises(ValueError, match="positive and finite"):
            sparse.append_kv(_bf(3, 2, 128), _bf(3, 2, 128), pool, _i(3), **scales)


def test_counts_that_pass_32_bits_are_refused(lib):
    many = ctypes.byref(_append(num_tokens=1 << 30))
    assert lib.rpa_append_kv(many, *FAKE[:5], 1.0, 1.0, *FAKE[5:7], None) == -1 and b"2^30" in lib.rpa_sparse_last_error()
    wide = ctypes.byref(_sparse(max_num_seqs=1 << 27))
    assert lib.rpa_select_pages(wide, 1, 1, *FAKE[:9], 1 << 40, None) == -1 and b"max_num_seqs" in lib.rpa_sparse_last_error()
    assert lib.rpa_sparse_workspace_size(wide) == 0
    heads = ctypes.byref(_append(num_kv_heads=65536))
    assert lib.rpa_append_kv(heads, *FAKE[:5], 1.0, 1.0, *FAKE[5:7], None) == -2 and b"65535 kv heads" in lib.rpa_sparse_last_error()
    heads = ctypes.byref(_sparse(num_kv_heads=65536, num_q_heads=65536, num_tokens=1))
    assert lib.rpa_select_pages(heads, 1, 1, *FAKE[:9], 1 << 40, None) == -2 and b"65535 kv heads" in lib.rpa_sparse_last_error()


def _sparse(**kw):
    return _sparse_lib.RpaSparseShape(**{**dict(num_tokens=4, num_q_heads=8, num_kv_heads=2, head_dim=128, total_pages=64, page_size=16,
                                                max_num_seqs=4, pages_per_seq=8, kv_dtype=0, num_pages=6, q_token_stride=1024,
                                                q_head_stride=128), **kw})


SHAPES = [
    (dict(num_q_heads=7), -1, b"divisible"), (dict(num_q_heads=0), -1, b"non-positive"), (dict(num_pages=0), -1, b"non-positive"),
    (dict(max_num_seqs=0), -1, b"non-positive"), (dict(pages_per_seq=1 << 28), -1, b"int32"), (dict(num_tokens=-3), -1, b"num_tokens"),
    (dict(kv_dtype=3), -1, b"kv_dtype"), (dict(head_dim=160), -2, b"head_dim 160"), (dict(q_token_stride=1020), -1, b"q must"),
    (dict(num_q_heads=1024), -2, b"256 query heads"), (dict(num_tokens=1 << 30, num_kv_heads=4), -1, b"overflows")]


@pytest.mark.parametrize("bad,code,message", SHAPES)
def test_select_and_attention_refuse_shapes(lib, bad, code, message):
    shape = ctypes.byref(_sparse(**bad))
    options = _sparse_lib.RpaSparseOptions(1.0, 0.0, 1.0, 1.0)
    assert lib.rpa_select_pages(shape, 1, 1, *FAKE[:9], 1 << 40, None) == code and message in lib.rpa_sparse_last_error()
    assert lib.rpa_sparse_paged_attention(shape, ctypes.byref(options), *FAKE[:2], None, *FAKE[3:10], 1 << 40, None) == code
    assert message in lib.rpa_sparse_last_error()
    if "q_token_stride" not in bad:
        assert lib.rpa_select_workspace_size(shape) == lib.rpa_sparse_workspace_size(shape) == 0


def test_select_refuses_counts_and_workspaces(lib):
    for sink, recent in ((-1, 1), (1, -1), (4, 3), (2**31 - 1, 2**31 - 1)):
        assert lib.rpa_select_pages(ctypes.byref(_sparse()), sink, recent, *FAKE[:9], 0, None) == -1
        assert b"sink_pages" in lib.rpa_sparse_last_error()
    long = _sparse(pages_per_seq=100000)
    need = lib.rpa_select_workspace_size(ctypes.byref(long))
    assert need > 0
    assert lib.rpa_select_pages(ctypes.byref(long), 1, 1, *FAKE[:9], need - 1, None) == -3
    assert lib.rpa_select_pages(ctypes.byref(long), 1, 1, *FAKE[:8], None, need, None) == -3


def test_attention_refuses(lib):
    options = _sparse_lib.RpaSparseOptions(1.0, 0.0, 1.0, 1.0)
    shape = _sparse(num_pages=64)
    need = lib.rpa_sparse_workspace_size(ctypes.byref(shape))
    assert need > 0
    call = lambda s, o, ptrs, n: lib.rpa_sparse_paged_attention(ctypes.byref(s), o, *ptrs, n, None)  # noqa: E731
    no_scales = [FAKE[0], FAKE[1], None, *FAKE[3:10]]
    assert call(shape, ctypes.byref(options), no_scales, need - 1) == -3
    assert call(shape, None, no_scales, need) == -1 and b"options" in lib.rpa_sparse_last_error()
    assert call(shape, ctypes.byref(options), FAKE[:10], need) == -1 and b"fp8" in lib.rpa_sparse_last_error()
    same = [*no_scales[:8], FAKE[0], FAKE[9]]
    assert call(shape, ctypes.byref(options), same, need) == -1 and b"out" in lib.rpa_sparse_last_error()
    huge = _sparse(num_pages=1 << 20, page_size=2048)
    assert lib.rpa_sparse_workspace_size(ctypes.byref(huge)) == 0 and b"2^24" in lib.rpa_sparse_last_error()


def test_no_tokens_is_no_error(lib):
    options = _sparse_lib.RpaSparseOptions(1.0, 0.0, 1.0, 1.0)
    empty = ctypes.byref(_sparse(num_tokens=0))
    assert lib.rpa_select_pages(empty, 1, 1, *[None] * 9, 0, None) == 0
    assert lib.rpa_sparse_paged_attention(empty, ctypes.byref(options), *[None] * 10, 0, None) == 0
    assert lib.rpa_append_kv(ctypes.byref(_append(num_tokens=0)), *[None] * 5, 1.0, 1.0, None, None, None) == 0


# ---- Python checks, with the device check out of the way ----
@pytest.fixture
def anywhere(monkeypatch):
    monkeypatch.setattr(sparse, "_require_cuda", lambda name, t: None)


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_cpu_tensors_are_refused():
    pool = _bf(4, 16, 4, 128)
    with pytest.raises(ValueError, match="GPU device"):
        sparse.append_kv(_bf(3, 2, 128), _bf(3, 2, 128), pool, _i(3))
    index = sparse.make_page_index(pool)
    assert index.bounds.shape == (4, 2, 2, 128) and index.exponents.shape == (4, 2)
    meta = (_i(2), _i(2, 8), _i(3), _i(1))
    with pytest.raises(ValueError, match="GPU device"):
        sparse.select_pages(_bf(3, 4, 128), index, *meta, page_size=16, num_pages=4)
    with pytest.raises(ValueError, match="GPU device"):
        sparse.sparse_paged_attention(_bf(3, 4, 128), pool, _i(3, 2, 4), *meta)


@pytest.mark.parametrize("change,message", [
    (dict(k=_bf(3, 4, 128)), "k has shape"), (dict(v=_bf(2, 2, 128)), "v has shape"), (dict(k=torch.zeros(3, 2, 128)), "k dtype"),
    (dict(slots=_i(4)), "slot_mapping has shape"), (dict(slots=torch.zeros(3, dtype=torch.int64)), "slot_mapping dtype"),
    (dict(pool=_bf(4, 16, 3, 128)), "2 \\* kv heads"), (dict(pool=torch.zeros(4, 16, 4, 128)), "not bf16 or fp8"),
    (dict(kv_scales=torch.zeros(4, 2, 2)), "requires fp8"), (dict(k_scale=0.5), "require fp8"), (dict(k_scale=1), "float or None"),
    (dict(index=(torch.zeros(4, 2, 2, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.int8))), "bounds has shape"),
    (dict(index=(torch.zeros(4, 2, 2, 128, dtype=torch.int8), torch.zeros(4, 2))), "exponents dtype"), (dict(index=3), "PageIndex")])
def test_append_python_refuses(monkeypatch, anywhere, change, message):
    real = sparse._tensor
    monkeypatch.setattr(sparse, "_tensor", lambda *a, **kw: real(*a))  # the rows' device check aside
    args = dict(k=_bf(3, 2, 128), v=_bf(3, 2, 128), pool=_bf(4, 16, 4, 128), slots=_i(3), kv_scales=None, k_scale=None, v_scale=None,
                index=None)
    args.update(change)
    with pytest.raises((ValueError, TypeError), match=message):
        if change.get("index") == 3:
            sparse._index(3, 4, 2, 128, None)
        sparse.append_kv(args["k"], args["v"], args["pool"], args["slots"], kv_scales=args["kv_scales"], k_scale=args["k_scale"],
                         v_scale=args["v_scale"], index=args["index"])


@pytest.mark.parametrize("change,message", [
    (dict(page_size=0), "page_size"), (dict(num_pages=0), "num_pages"), (dict(sink_pages=-1), "sink_pages"),
    (dict(sink_pages=3, recent_pages=2), "exceed num_pages"), (dict(num_pages=2.0), "num_pages"), (dict(q=_bf(3, 5, 128)), "divisible"),
    (dict(q=_bf(3, 4, 64)), "q has shape"), (dict(lens=_i(3)), "kv_lens has shape"), (dict(cu=_i(2)), "cu_q_lens has shape"),
    (dict(num=_i(2)), "num_seqs has shape"), (dict(table=torch.zeros(2, 8)), "page_indices dtype")])
def test_select_python_refuses(monkeypatch, anywhere, change, message):
    real = sparse._tensor
    monkeypatch.setattr(sparse, "_tensor", lambda *a, **kw: real(*a))
    t = dict(q=_bf(3, 4, 128), lens=_i(2), table=_i(2, 8), cu=_i(3), num=_i(1))
    t.update({k: v for k, v in change.items() if k in t})
    kw = dict(page_size=16, num_pages=4)
    kw.update({k: v for k, v in change.items() if k not in t})
    index = sparse.make_page_index(_bf(4, 16, 4, 128))
    with pytest.raises(ValueError, match=message):
        sparse.select_pages(t["q"], index, t["lens"], t["table"], t["cu"], t["num"], **kw)


@pytest.mark.parametrize("change,message", [
    (dict(soft_cap=0.0), "soft_cap"), (dict(picked=_i(3, 1, 4)), "selected_pages has shape"), (dict(picked=_i(3, 2, 0)), "room"),
    (dict(q=_bf(3, 3, 128)), "divisible"), (dict(v_scale=2), "float or None"), (dict(kv_scales=torch.ones(4, 2, 2)), "requires fp8"),
    (dict(pool=torch.zeros(4, 16, 4, 128, dtype=torch.uint8), kv_scales=torch.ones(4, 2, 2), k_scale=1.0), "not both"),
    (dict(pool=torch.zeros(4, 16, 4, 128, dtype=torch.uint8), kv_scales=torch.ones(4, 1, 2)), "kv_scales has shape")])
def test_attention_python_refuses(monkeypatch, anywhere, change, message):
    real = sparse._tensor
    monkeypatch.setattr(sparse, "_tensor", lambda *a, **kw: real(*a))
    t = dict(q=_bf(3, 4, 128), pool=_bf(4, 16, 4, 128), picked=_i(3, 2, 4))
    t.update({k: v for k, v in change.items() if k in t})
    kw = {k: v for k, v in change.items() if k not in t}
    with pytest.raises(ValueError, match=message):
        sparse.sparse_paged_attention(t["q"], t["pool"], t["picked"], _i(2), _i(2, 8), _i(3), _i(1), **kw)


def test_rows_of_odd_strides_are_refused(monkeypatch):
    class Cuda(torch.Tensor):  # a CPU tensor that says it is on the GPU
        device = torch.device("cuda", 0)

    def on(t):
        return t.as_subclass(Cuda)

    wide = _bf(4, 8, 136)
    sparse._tensor("q", on(wide[:, 1:5, :128]), torch.bfloat16, (None, 4, 128), None, rows=True)
    for bad in (_bf(4, 8, 132)[:, :, :128], _bf(4, 128, 8).transpose(1, 2), _bf(4, 8, 256)[:, :, ::2]):
        with pytest.raises(ValueError, match="contiguous rows"):
            sparse._tensor("q", on(bad), torch.bfloat16, (None, 8, 128), None, rows=True)


@pytest.mark.parametrize("slots,message", [
    ([0, 1, 2, -1, 17], None), ([3, 4, 5, 15, 16, 17], None), ([-1], None), ([], None), ([5, 9, 12], "consecutive"),
    ([5, -1, 6], "consecutive"), ([6, 5], "consecutive"), ([4, 4], "twice"), ([-2], "outside"), ([32], "outside"), ([16, 15], None),
    ([15, 16], None)])
def test_preflight_append(slots, message):
    pool, slots = _bf(4, 8, 2, 64), torch.tensor(slots, dtype=torch.int32)
    if message is None:
        sparse.preflight_append(slots, pool)
    else:
        with pytest.raises(ValueError, match=message):
            sparse.preflight_append(slots, pool)
