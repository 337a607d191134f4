"""Tensors of one call on different GPUs are refused, each by its name: no GPU needed."""

import pytest
import torch

from tpu_cake_amd import sparse


class First(torch.Tensor):  # CPU tensors that say they are on a GPU
    device = torch.device("cuda", 0)


class Second(torch.Tensor):
    device = torch.device("cuda", 1)


def _tensors():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    b = lambda *s: torch.zeros(s, dtype=torch.int8)  # noqa: E731
    return dict(q=torch.zeros((3, 4, 128), dtype=torch.bfloat16), bounds=b(4, 2, 2, 128), exponents=b(4, 2), kv_lens=i(2),
                page_indices=i(2, 8), cu_q_lens=i(3), num_seqs=i(1), pool=torch.zeros((4, 16, 4, 128), dtype=torch.bfloat16),
                lists=i(3, 2, 4), k=torch.zeros((3, 2, 128), dtype=torch.bfloat16), v=torch.zeros((3, 2, 128), dtype=torch.bfloat16),
                slots=i(3))


META = ["kv_lens", "page_indices", "cu_q_lens", "num_seqs"]


def _call(entry, t):
    index = sparse.PageIndex(t["bounds"], t["exponents"])
    if entry == "select":
        sparse.select_pages(t["q"], index, *[t[x] for x in META], page_size=16, num_pages=4)
    elif entry == "attend":
        sparse.sparse_paged_attention(t["q"], t["pool"], t["lists"], *[t[x] for x in META])
    else:
        sparse.append_kv(t["k"], t["v"], t["pool"], t["slots"], index=index)


@pytest.mark.parametrize("entry,names", [("select", ["q", "bounds", "exponents", *META]), ("attend", ["q", "pool", "lists", *META]),
                                         ("append", ["k", "v", "pool", "slots", "bounds", "exponents"])])
def test_each_tensor(monkeypatch, entry, names):
    monkeypatch.setattr(sparse, "_require_cuda", lambda name, t: None)
    for name in names:
        t = {x: y.as_subclass(Second if x == name else First) for x, y in _tensors().items()}
        with pytest.raises(ValueError, match="cuda:[01], expected cuda:[01]"):
            _call(entry, t)
