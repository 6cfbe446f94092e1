"""Paged cache calls without a GPU: arguments that must not reach a kernel as they are."""
import os
import subprocess
import sysconfig
from pathlib import Path

import pytest
import torch

import cast_b200
from cast_b200 import _lib, paged, tree_attn

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


# ------------------------------------------------------------------------------------- building the binding
def test_binding_is_named_for_its_python_and_torch():
    name = _lib.build_binding().name
    assert torch.__version__ in name and sysconfig.get_config_var("SOABI") in name


@pytest.mark.parametrize("build", ["build", "build_binding"])
def test_builds_at_once_do_not_share_a_temporary_file(monkeypatch, tmp_path, build):
    # whatever a process writes before the last rename is its own; nothing is left when the compiler fails
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "lib.so")
    monkeypatch.setattr(_lib, "PKG", tmp_path)
    seen = []

    def run(cmd, **_):
        out = Path(cmd[cmd.index("-o") + 1])
        seen.append(out.name)
        out.write_bytes(b"x")
        return subprocess.CompletedProcess(cmd, len(seen) - 1, "", "no luck")

    monkeypatch.setattr(subprocess, "run", run)
    made = getattr(_lib, build)(force=True)
    assert made.read_bytes() == b"x" and os.listdir(tmp_path) == [made.name]
    with pytest.raises(RuntimeError, match="no luck"):
        getattr(_lib, build)(force=True)
    assert os.listdir(tmp_path) == [made.name] and all(str(os.getpid()) in n for n in seen)


def test_calls_go_through_ctypes_where_the_binding_cannot_be_built(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "PKG", tmp_path)
    monkeypatch.setattr(_lib, "_BINDING", None)
    monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    pages, row = torch.zeros(4, 2, 16, 64), torch.zeros(1, 2, 64)
    ints = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.warns(UserWarning, match="ctypes"):
        assert cast_b200.append_paged([], [], ints, ints[0, :1], [], []) is None
    for call in (lambda: cast_b200.append_paged(pages, pages, ints, ints[0, :1], row, row),
                 lambda: cast_b200.decode_attention_paged(row, pages, pages, ints, ints[0, :1]),
                 lambda: cast_b200.varlen_tree_attention_paged(row, pages, pages, ints, row, row, [0, 1], [0], [1], parent=[-1])):
        with pytest.raises(RuntimeError, match="CUDA"):       # paged.py's own check, not the compiler's failure
            call()
