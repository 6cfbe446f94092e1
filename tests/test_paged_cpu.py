"""Paged cache entry points without a GPU: argument errors come back before any CUDA call."""
import ctypes

import pytest
import torch

import cast_b200
from cast_b200 import _lib

P = 1 << 12


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _i64(*x):
    return (ctypes.c_int64 * len(x))(*x)


def _append(L, **o):
    ptrs = (ctypes.c_void_p * 2)(P, P)
    a = dict(n=1, pages=ptrs, new=ptrs, dtype=1, H=8, D=128, num_pages=4, ps=16, pst=_i64(*[16384, 2048, 128] * 2),
             total=3, nst=_i64(1024, 128, 1024, 128), table=P, ts=2, mp=2, sl=P, B=3, cu=None, keep=None, ks=0, acc=None,
             pos=None, inv=None, nf=0, il=0, sc=1.0, q=None, qo=None, Hq=0, qs=None, stream=None)
    a.update(o)
    return L.cast_paged_append(*a.values())


def test_append_argument_checks(L):
    assert _append(L, dtype=3) == -3
    assert _append(L, H=0) == -2 and _append(L, num_pages=0) == -2 and _append(L, ps=0) == -2
    assert _append(L, total=-1) == -2 and _append(L, mp=0) == -2 and _append(L, ts=-1) == -2
    assert _append(L, total=1 << 31) == -2
    assert _append(L, nf=65, inv=P) == -2                       # more pairs than half a head
    assert _append(L, D=512) == -4
    assert _append(L, table=None) == -1 and _append(L, sl=None) == -1 and _append(L, nf=64) == -1
    assert _append(L, q=P) == -1                                # q without q_out
    assert _append(L, q=P, qo=P, Hq=32, qs=_i64(1, 1, 1, 1)) == -2    # q without rotation
    assert _append(L, keep=P) == -1 and _append(L, keep=P, acc=P) == -1   # keep needs accepted and cu_q
    assert _append(L, q=P, qo=P, Hq=32, nf=64, inv=P, keep=P, acc=P, cu=P, ks=1, qs=_i64(1, 1, 1, 1)) == -2
    two = (ctypes.c_void_p * 2)(P, None)
    assert _append(L, new=two) == -1
    for nothing in (dict(n=0), dict(B=0), dict(total=0), dict(keep=P, acc=P, cu=P, ks=0)):
        assert _append(L, **nothing) == 0


def _decode(L, **o):
    a = dict(q=P, k=P, v=P, out=P, lse=None, dtype=1, st=_i64(4096, 128, 16384, 2048, 128, 4096, 128), table=P, ts=2,
             mp=2, sl=P, B=2, Hq=32, Hkv=8, D=128, np=4, ps=16, scale=0.0, cap=0.0, win=0, slopes=None, ws=None, n=0,
             stream=None)
    a.update(o)
    return L.cast_paged_decode_attn(*a.values())


def test_decode_argument_checks(L):
    assert _decode(L, dtype=3) == -3
    assert _decode(L, Hq=30) == -2 and _decode(L, np=0) == -2 and _decode(L, ps=0) == -2 and _decode(L, win=-1) == -2
    assert all(_decode(L, cap=x) == -2 for x in (-1.0, 1e-7, 1e31, float("inf"), float("nan")))
    assert _decode(L, D=96) == -4
    assert _decode(L, q=None) == -1 and _decode(L, table=None) == -1 and _decode(L, sl=None) == -1
    assert _decode(L, q=P + 8) == -7 and _decode(L, k=P + 8) == -7
    assert _decode(L, st=_i64(4096, 130, 16384, 2048, 128, 4096, 128)) == -7
    assert _decode(L, st=_i64(4096, 128, 16384, 2048, 132, 4096, 128)) == -7     # page rows off 16 bytes
    assert _decode(L, dtype=0, st=_i64(4096, 128, 16384, 2048, 130, 4096, 128)) == -7
    assert _decode(L, B=0) == 0
    assert _decode(L) in (-6, -10)                              # no workspace (or no device here)


def test_decode_workspace_size(L):
    f = L.cast_paged_decode_workspace_size
    small, large = f(1, 1, 32, 8, 128), f(1, 4096, 32, 8, 128)
    assert 0 < small == large                                   # neither the lengths nor their number play a part
    assert f(1, 1, 30, 8, 128) == 0 and f(1, 1, 32, 8, 96) == 0 and f(3, 1, 32, 8, 128) == 0 and f(1, 0, 32, 8, 128) == 0
    assert cast_b200.decode_workspace_size(torch.bfloat16, 1, 32, 8, 128) == small


def _tree(L, **o):
    a = dict(q=P, k=P, v=P, kp=P, vp=P, out=P, dtype=1,
             st=_i64(4096, 128, 16384, 2048, 128, 1024, 128, 1024, 128, 4096, 128), table=P, ts=2, mp=2, cu=P, pre=P,
             pack=P, anc=None, wpr=0, par=P, B=1, tq=4, np=4, ps=16, Hq=32, Hkv=8, D=128, scale=0.0, max_pack=4,
             max_prefix=32, ws=None, n=0, stream=None)
    a.update(o)
    return L.cast_tree_attn_paged_fwd(*a.values())


def test_tree_argument_checks(L):
    assert _tree(L, dtype=3) == -3
    assert _tree(L, Hq=30) == -2 and _tree(L, np=0) == -2 and _tree(L, ps=0) == -2
    assert _tree(L, max_prefix=(1 << 31) - 1, max_pack=1024) == -2
    assert _tree(L, D=96) == -4 and _tree(L, max_pack=4096) == -5
    assert _tree(L, kp=None) == -1 and _tree(L, table=None) == -1 and _tree(L, cu=None) == -1
    assert _tree(L, par=None) == -11 and _tree(L, anc=P, wpr=1) == -11 and _tree(L, par=None, anc=P) == -5
    assert _tree(L, vp=P + 8) == -7
    assert _tree(L, st=_i64(4096, 128, 16384, 2048, 132, 1024, 128, 1024, 128, 4096, 128)) == -7
    assert _tree(L, B=0) == 0 and _tree(L, max_pack=0) == 0


def test_python_refusals():
    pages = torch.zeros(4, 2, 16, 64)
    table, length = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    row = torch.zeros(1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        cast_b200.append_paged(pages, pages, table, length, row, row)
    with pytest.raises(RuntimeError, match="CUDA"):
        cast_b200.decode_attention_paged(torch.zeros(1, 4, 64), pages, pages, table, length)
    with pytest.raises(RuntimeError, match="CUDA"):
        cast_b200.varlen_tree_attention_paged(torch.zeros(1, 4, 64), pages, pages, table, row, row, [0, 1], length,
                                              length, parent=length)
    with pytest.raises(ValueError, match="per layer"):
        cast_b200.append_paged([pages], [pages], table, length, [row, row], [row])
    assert cast_b200.append_paged([], [], table, length, [], []) is None


def test_binding_leaves_what_it_does_not_take():
    # no CUDA tensor, too few arguments, no tensor at all: paged.py goes on (and refuses above)
    b = _lib.binding()
    pages, row, ints = torch.zeros(4, 2, 16, 64), torch.zeros(1, 2, 64), torch.zeros(1, 2, dtype=torch.int32)
    args = (pages, pages, ints, ints[0], row, row, None, None, None, None, None, False, 1.0, None, None)
    assert b.append(*args) is NotImplemented
    assert b.append(*args[:5]) is NotImplemented and b.decode() is NotImplemented and b.tree(None) is NotImplemented
    assert b.append([], [], ints, ints, [], [], *args[6:]) is NotImplemented
    assert b.decode(*[3] * 12) is NotImplemented and b.tree(*[None] * 16) is NotImplemented
    with pytest.raises(TypeError):
        b.bind(1)
    with pytest.raises(TypeError):
        b.bind(*["x"] * 5)
