"""Paged cache calls without a GPU: arguments that must not reach a kernel as they are."""
import pytest
import torch

from cast_b200 import paged, tree_attn

from .test_paged_cpu import L, _decode, _tree  # noqa: F401  (L: fixture)


def _aligned_bytes(n):
    base = torch.zeros(n + 256, dtype=torch.uint8)
    return base[-base.data_ptr() % 256:][:n]


@pytest.mark.parametrize("which", ["paged", "ragged and store"])
def test_workspace_with_gaps_or_repeats_is_not_used(monkeypatch, which):
    # its address is good for fewer bytes than it counts: a kernel would write past it
    whole = _aligned_bytes(4096)
    short, strided = whole[:1].expand(4096), whole[::2]
    assert short.nbytes == 4096 and short.data_ptr() % 256 == 0 and strided.nbytes == 2048
    monkeypatch.setattr(torch, "empty", lambda *a, **k: "new")
    ask = (lambda w, n: paged._workspace(w, n, -1)) if which == "paged" else (lambda w, n: tree_attn._workspace(w, n, torch.device("cpu")))
    assert ask(whole, 4096) is whole and ask(whole, 4097) == "new" and ask(None, 1) == "new"
    assert ask(short, 4096) == "new" and ask(strided, 2048) == "new"
    elsewhere = (lambda n: paged._workspace(whole, n, 0)) if which == "paged" else (
        lambda n: tree_attn._workspace(whole, n, torch.device("cuda", 0)))
    assert elsewhere(4096) == "new"                  # another device's memory


def test_lengths_near_the_end_of_32_bits(L):  # noqa: F811
    # the kernels look up to 4224 keys past a tile: nothing above 2^31 - 8193 keys
    most = (1 << 31) - 1 - 8192
    assert _tree(L, max_prefix=most, max_pack=4) == -2 and _tree(L, max_prefix=most + 1, max_pack=0) == -2
    assert _tree(L, max_prefix=most - 4, max_pack=4, vp=None) == -1               # passes the sizes, fails the next check
    assert _tree(L, ps=most + 1) == -2 and _decode(L, ps=most + 1) == -2
    size = L.cast_tree_attn_paged_workspace_size
    assert size(1, 1, 17, 32, 8, 128, 17, most) == 0 and size(1, 1, 17, 32, 8, 128, 17, (1 << 31) - 1) == 0
    assert size(1, 1, 17, 32, 8, 128, -1, 10) == 0 and size(1, 1, 17, 32, 8, 128, 17, -1) == 0
    assert 0 < size(0, 1, 17, 32, 8, 128, 17, 100000) < size(0, 1, 34, 32, 8, 128, 17, 100000)
