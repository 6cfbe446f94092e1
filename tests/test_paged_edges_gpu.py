"""Paged cache operators where a value that is no part of a result, or a number at the edge of its type, could reach it.

The helpers and their bounds are those of test_paged_gpu.py.
"""
import math

import numpy as np
import pytest
import torch

import cast_b200
from cast_b200 import _lib

from .test_paged_gpu import TYPES, U32, Cache, _attend, _check_attention, _tree_inputs

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------- rows of other requests
# one pack tile holds up to 128 rows from the pack's first: rows of the next packs, and rows behind the last one
SPLIT = ([3000, 2000, 2500], [17, 20, 40])          # few units: the launch cuts the keys into chunks
WHOLE = ([0, 128, 300, 64], [9, 1, 130, 64])        # one and two query tiles, one and two pack tiles
MANY = ([40] * 24, [3] * 24)                        # 192 units of one chunk each


def _poisoned(x, value, rows):
    y = x.clone()
    y[rows] = value
    return y


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("S,P", [SPLIT, WHOLE, MANY], ids=["split", "whole", "many"])
@pytest.mark.parametrize("ps,Hq,Hkv,D", [(16, 8, 2, 128), (1, 8, 2, 128), (24, 12, 4, 64), (3, 6, 2, 64)])
def test_tree_keeps_other_packs_out(cuda, dtype, S, P, ps, Hq, Hkv, D):
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 51, S, P, Hq, Hkv, D, ps, dt)
    pad = torch.zeros(67, Hkv, D, dtype=dt, device=cuda)
    kp, vp = torch.cat((kp, pad)), torch.cat((vp, pad))            # 67 rows behind the last pack
    q = torch.cat((q, torch.zeros(67, Hq, D, dtype=dt, device=cuda)))
    total = int(cu[-1])
    par = np.concatenate(parents + [[-1] * 67]).astype(np.int32)

    def run(k, v):
        out = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, k, v, cu, c.len, P, parent=par,
                                                    out=torch.zeros_like(q))
        assert _lib.device_error() == 0
        return out

    good = run(kp, vp)
    assert torch.isfinite(good).all()
    behind = slice(total, total + 67)
    one = slice(int(cu[1]), int(cu[2]))                            # request 1's own rows
    rest = torch.ones(total, dtype=torch.bool, device=cuda)
    rest[one] = False
    for kv, vv in ((math.nan, math.inf), (math.inf, math.nan), (1.0, -math.inf)):
        got = run(_poisoned(kp, kv, behind), _poisoned(vp, vv, behind))
        assert torch.equal(got[:total], good[:total])
        got = run(_poisoned(_poisoned(kp, kv, behind), kv, one), _poisoned(_poisoned(vp, vv, behind), vv, one))
        assert torch.equal(got[:total][rest], good[:total][rest])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("S,P", [SPLIT, WHOLE, MANY], ids=["split", "whole", "many"])
def test_store_form_keeps_other_packs_out(cuda, dtype, S, P):
    dt = TYPES[dtype]
    g = torch.Generator(device=cuda).manual_seed(52)
    rnd = lambda *s: torch.empty(s, dtype=dt, device=cuda).normal_(generator=g)
    B, Hq, Hkv, D, total = len(S), 8, 2, 128, sum(P)
    ks, vs, q = rnd(B, Hkv, max(S) + 5, D), rnd(B, Hkv, max(S) + 5, D), rnd(total + 67, Hq, D)
    kp, vp = rnd(total + 67, Hkv, D), rnd(total + 67, Hkv, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    cu = np.concatenate([[0], np.cumsum(P)]).tolist()
    par = i32(sum([[-1] + list(range(p - 1)) for p in P], []) + [-1] * 67)

    def run(k, v):
        out = cast_b200.varlen_tree_attention_store(q, ks, vs, k, v, i32(cu), i32(S), i32(P), parent=par,
                                                    out=torch.zeros_like(q))
        assert _lib.device_error() == 0
        return out

    good = run(kp, vp)
    behind, one = slice(total, total + 67), slice(cu[1], cu[2])
    rest = torch.ones(total, dtype=torch.bool, device=cuda)
    rest[one] = False
    got = run(_poisoned(_poisoned(kp, math.nan, behind), math.nan, one), _poisoned(_poisoned(vp, math.inf, behind), math.nan, one))
    assert torch.equal(got[:total][rest], good[:total][rest])


# ------------------------------------------------------------------------------------- workspaces
def test_workspaces_with_gaps_or_repeats(cuda):
    """A workspace view that is not one piece is left alone: a new one is taken, the bytes between its own stay."""
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 57, [3000, 2000], [17, 20], 8, 2, 128, 16, torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    par, P = i32(sum(parents, [])), i32([17, 20])
    ks, vs = (torch.stack([torch.nn.functional.pad(c.rows(pg, b, 0, n), (0, 0, 0, 0, 0, 3000 - n)).transpose(0, 1).contiguous()
                           for b, n in enumerate(c.lens)]) for pg in (c.k[0], c.v[0]))
    k, v = (torch.cat([t for b, n in enumerate(c.lens) for t in (c.rows(pg, b, 0, n), pk[cu[b]:cu[b + 1]])])
            for pg, pk in ((c.k[0], kp), (c.v[0], vp)))
    cu = i32(cu.tolist())
    calls = [
        lambda w: cast_b200.decode_attention_paged(q[:2], c.k[0], c.v[0], c.table, c.len, workspace=w),
        lambda w: cast_b200.decode_attention_paged(q[:2], c.k[0], c.v[0], c.table, c.len.long(), workspace=w),
        lambda w: cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P, parent=par,
                                                        max_pack=20, max_prefix=3000, workspace=w),
        lambda w: cast_b200.varlen_tree_attention_store(q, ks, vs, kp, vp, cu, c.len, P, parent=par, workspace=w),
        lambda w: cast_b200.varlen_tree_attention(q, k, v, cu, i32([0, 3017, 5037]), c.len, P, parent=par, workspace=w),
    ]
    big = torch.full((64 << 20,), 7, dtype=torch.uint8, device=cuda)
    for call in calls:
        want = call(None)
        for view in (big[:1].expand(32 << 20), big[::2]):
            assert torch.equal(call(view), want)
        assert (big == 7).all() and _lib.device_error() == 0
        assert torch.equal(call(big), want) and not (big == 7).all()      # one piece: used
        big.fill_(7)


# ------------------------------------------------------------------------------------- rows of no sequence
@pytest.mark.parametrize("dtype", list(TYPES))
def test_tree_rows_of_no_sequence_then_another_call(cuda, dtype):
    """Offsets that give every row to an empty second pack: split launches write nothing, and the calls behind them in the
    stream (which overwrite the cache and reuse the workspace) are not disturbed."""
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 58, [6000, 6000], [17, 20], 8, 2, 128, 16, dt)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    par, cu, P = i32(sum(parents, [])), i32(cu.tolist()), i32([17, 20])
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=cuda)
    tree = lambda cu, P, out: cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P, parent=par,
                                                                    max_pack=20, max_prefix=6000, out=out, workspace=ws)
    keep_k, keep_v = c.k[0].clone(), c.v[0].clone()
    good = tree(cu, P, torch.empty_like(q))
    nowhere, empty = i32([0, 0, 0]), i32([17, 0])
    for _ in range(20):
        left = torch.full_like(q, 7.0)
        tree(nowhere, empty, left)
        c.k[0].fill_(3.0)
        c.v[0].fill_(3.0)
        c.k[0].copy_(keep_k)
        c.v[0].copy_(keep_v)
        assert torch.equal(tree(cu, P, torch.empty_like(q)), good) and (left == 7.0).all()
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------------- visible NaN
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 12, 4), (128, 5, 1)])
def test_decode_shows_every_visible_nan(cuda, dtype, D, Hq, Hkv):
    """NaN in a query head, in the only key, in a whole first step, in every key, in the last key, in a value: rows of that
    head group (that dim) are NaN and their log-sum-exp too (not for a value), all others keep their bits."""
    G = Hq // Hkv
    lens = [700, 1, 700, 40, 5000, 300]
    c = Cache(53, lens, Hkv, D, 16, TYPES[dtype], cuda)
    g = torch.Generator(device=cuda).manual_seed(54)
    q = torch.empty((len(lens), Hq, D), device=cuda).normal_(generator=g).to(TYPES[dtype])

    def run(q):
        lse = torch.zeros(len(lens), Hq, device=cuda)
        out = cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len, lse=lse)
        assert _lib.device_error() == 0
        return out, lse

    good, good_lse = run(q)
    assert torch.isfinite(good).all() and torch.isfinite(good_lse).all()
    bad = torch.zeros(len(lens), Hq, dtype=torch.bool, device=cuda)
    q2 = q.clone()
    q2[0, Hq - 1, 3] = math.nan
    bad[0, Hq - 1] = True

    def spoil(pages, b, h, n, d):
        pages[int(c.table[b, n // 16]), h, n % 16, d] = math.nan

    last = Hkv - 1
    for b, keys in ((1, [0]), (2, range(32)), (3, range(40)), (4, [4999])):
        for n in keys:
            spoil(c.k[0], b, last, n, 7)
        bad[b, last * G:] = True
    spoil(c.v[0], 5, 0, 17, 11)
    out, lse = run(q2)
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert out[5, :G, 11].isnan().all()
    keep = ~bad[..., None].expand_as(out).clone()
    keep[5, :G, 11] = False
    assert torch.equal(out[keep], good[keep]) and torch.equal(lse[~bad], good_lse[~bad])


# ------------------------------------------------------------------------------------- caps
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cap", [1e-3, 1.0, 50.0, 1e3, 1e4, 1e6, 1e8, 1e30])
def test_decode_cap_of_any_size(cuda, dtype, cap):
    """cap tanh(s / cap) is s itself where the cap is large. Its error goes by the score, not by the cap: 2^-19 of the capped
    score (below a quarter of the cap a polynomial off by some 2^-22; above it an exponential and a reciprocal of 2^-22 and
    2^-23, together under 2.5 x 2^-23 of the cap, of which the score has tanh(1/4) or more)."""
    lens, Hq, Hkv, D = [1, 40, 700, 3000], 8, 2, 128
    dt = TYPES[dtype]
    c = Cache(55, lens, Hkv, D, 16, dt, cuda)
    g = torch.Generator(device=cuda).manual_seed(56)
    q = (torch.empty((len(lens), Hq, D), device=cuda).normal_(generator=g) * 3).to(dt)
    lse = torch.zeros(len(lens), Hq, device=cuda)
    got = cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len, softcap=cap, lse=lse)
    assert _lib.device_error() == 0
    for b, n in enumerate(lens):
        k, v = c.rows(c.k[0], b, 0, n), c.rows(c.v[0], b, 0, n)
        _, _, e, _ = _attend(q[b:b + 1], k, v, 1 / math.sqrt(D), 0, None, None)      # the dot products' error
        kk = k.double().repeat_interleave(Hq // Hkv, 1)
        s = torch.einsum("hd,nhd->hn", q[b].double(), kk) / math.sqrt(D)
        s = cap * torch.tanh(s / cap)
        e = e + 2.0 ** -19 * s.abs().amax(-1)
        p = torch.softmax(s, -1)
        vv = v.double().repeat_interleave(Hq // Hkv, 1)
        want, pv = torch.einsum("hn,nhd->hd", p, vv)[None], torch.einsum("hn,nhd->hd", p, vv.abs())[None]
        _check_attention(got[b:b + 1], want, e, pv, n, dt, 0.0 if dtype == "fp32" else 2.0 ** -15)
        want_l = torch.logsumexp(s, -1)
        assert ((lse[b].double() - want_l).abs() <= 2 * e[0] + 2.0 ** -20 + n * U32 + 4 * U32 * want_l.abs()).all()


# ------------------------------------------------------------------------------------- small probabilities
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,Hq,Hkv,n", [(64, 16, 8, 16000), (128, 8, 4, 16000), (64, 32, 2, 40000)])
def test_decode_long_tail_of_small_probabilities(cuda, dtype, D, Hq, Hkv, n):
    """Every 500th key has the score 0 and a value of 0, the others one score near -15.76 (p = 2.4 x 2^-24 of the largest)
    and a value of 1000: the output is all tail. The two 16-bit terms of 2^14 p are off by half a step of the smaller one,
    2^-25 at least in half precision, which is 2^-25 / (2.4 x 2^-10) < 2^-16 of p; by 2^-17 of p in bfloat16."""
    dt = TYPES[dtype]
    B, ps = 16, 64
    pages = -(-n // ps)
    at = torch.arange(pages * ps, device=cuda).view(pages, 1, ps, 1)
    top = (at % 500 == 7).expand(pages, Hkv, ps, D)
    level = torch.tensor(-15.76 / math.sqrt(D), dtype=dt, device=cuda)
    k = torch.where(top, torch.zeros_like(level), level).contiguous()
    v = torch.where(top, torch.zeros_like(level), torch.full_like(level, 1000.0)).contiguous()
    q = torch.ones(B, Hq, D, dtype=dt, device=cuda)
    table = torch.arange(pages, dtype=torch.int32, device=cuda).repeat(B, 1)      # all sequences share the pages
    got = cast_b200.decode_attention_paged(q, k, v, table, torch.full((B,), n, dtype=torch.int32, device=cuda))
    assert _lib.device_error() == 0
    s = level.double() * math.sqrt(D)
    tops = len(range(7, n, 500))
    tail = (n - tops) * torch.exp(s)
    want = (1000.0 * tail / (tops + tail)).expand(B, Hq, D)
    e = (D + 2) * 2 * U32 * s.abs().expand(B, Hq)
    _check_attention(got, want, e, want, n, dt, 2.0 ** -16)


# ------------------------------------------------------------------------------------- numbers above 32 bits
@pytest.mark.parametrize("convert", [False, True], ids=["binding", "python"])
def test_windows_and_page_counts_above_32_bits(cuda, convert):
    """The C ABI takes ints: a window of 2^32 + 5 is no window of 5, and 2^32 + 1 pages are not one."""
    c = Cache(59, [90, 700], 2, 64, 16, torch.bfloat16, cuda)
    lens, table = (c.len.long(), c.table.long()) if convert else (c.len, c.table)
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=cuda)
    want = cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len)
    for window in ((1 << 31) - 1, 1 << 31, (1 << 32) + 5, 1 << 70):
        assert torch.equal(cast_b200.decode_attention_paged(q, c.k[0], c.v[0], table, lens, window=window), want)
    base = torch.zeros(2, 1, 1, 4, 8, device=cuda)
    k, v = (x.expand((1 << 32) + 1, 1, 4, 8) for x in base)          # every page is the one behind the view
    new = torch.ones(1, 1, 8, device=cuda)
    five, zero = torch.full((1, 1), 5, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    cast_b200.append_paged(k, v, five.long() if convert else five, zero, new, new)
    assert (base[:, :, :, 0] == 1).all() and (base[:, :, :, 1:] == 0).all() and _lib.device_error() == 0
    with pytest.raises((ValueError, _lib.CastError)):
        cast_b200.append_paged(base[0, :, :, :1].expand(1, 1, 1 << 32, 8), base[1, :, :, :1].expand(1, 1, 1 << 32, 8), five, zero, new, new)
    one = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    pk = torch.ones(2, 2, 64, dtype=torch.bfloat16, device=cuda)
    for bad in (dict(max_pack=1 << 32, max_prefix=700), dict(max_pack=1, max_prefix=(1 << 32) + 700)):
        with pytest.raises((ValueError, _lib.CastError)):
            cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], table, pk, pk, one, c.len, [1, 1], parent=[-1, -1], **bad)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("convert", [False, True], ids=["binding", "python"])
def test_scales_that_are_not_positive(cuda, convert):
    # the C ABI's "0 or less: the default" is no answer to a caller who asks for 0, a negative scale or NaN
    c = Cache(60, [90, 700], 2, 64, 16, torch.bfloat16, cuda)
    q, pk = (torch.ones(2, h, 64, dtype=torch.bfloat16, device=cuda) for h in (4, 2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    lens = c.len.long() if convert else c.len
    for scale in (0.0, 0, -0.125, math.nan, math.inf, 1e-60):
        with pytest.raises(ValueError):
            cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, lens, scale)
        with pytest.raises(ValueError):
            cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, pk, pk, i32([0, 1, 2]), lens, i32([1, 1]), None, scale,
                                                  parent=i32([-1, -1]), max_pack=1, max_prefix=700)
    a, b = (cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, lens, s) for s in (None, 0.125))
    assert torch.equal(a, b) and _lib.device_error() == 0


@pytest.mark.parametrize("convert", [False, True], ids=["binding", "python"])
def test_append_refuses_queries_written_over_one_another(cuda, convert):
    c = Cache(61, [9, 20, 0], 2, 64, 16, torch.bfloat16, cuda, room=1, poison=False)
    q, k = torch.ones(3, 4, 64, dtype=torch.bfloat16, device=cuda), torch.ones(3, 2, 64, dtype=torch.bfloat16, device=cuda)
    lens, freq = c.len.long() if convert else c.len, torch.ones(32, device=cuda)
    before = c.k[0].clone()
    for q_out in (q[:1].clone().expand(3, 4, 64), q[:, :1].clone().expand(3, 4, 64)):
        with pytest.raises(ValueError, match="q_out"):
            cast_b200.append_paged(c.k[0], c.v[0], c.table, lens, k, k, inv_freq=freq, q=q, q_out=q_out)
    assert torch.equal(c.k[0], before)
    # one source row for every query is fine, and so is a single head or row of any stride
    same = cast_b200.append_paged(c.k[0], c.v[0], c.table, lens, k, k, inv_freq=freq, q=q[:1].expand(3, 4, 64), q_out=torch.empty_like(q))
    assert torch.equal(same, cast_b200.append_paged(c.k[0], c.v[0], c.table, lens, k, k, inv_freq=freq, q=q, q_out=torch.empty_like(q)))
    row = torch.empty(3, 64, dtype=q.dtype, device=cuda)[:, None].expand(3, 1, 64)
    assert cast_b200.append_paged(c.k[0], c.v[0], c.table, lens, k, k, inv_freq=freq, q=q[:, :1], q_out=row) is row
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------------- without the binding
def test_whole_calls_without_the_binding(cuda, monkeypatch):
    c = Cache(62, [90, 0, 33], 2, 128, 16, torch.bfloat16, cuda, room=8, poison=False, layers=2)
    g = torch.Generator(device=cuda).manual_seed(63)
    rnd = lambda *s: torch.empty(s, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    q, k, v = rnd(3, 8, 128), rnd(3, 2, 128), rnd(3, 2, 128)
    first = [t.clone() for t in c.k + c.v]

    def everything():
        for t, f in zip(c.k + c.v, first):
            t.copy_(f)
        lse = torch.zeros(3, 8, device=cuda)
        outs = [cast_b200.append_paged(c.k[0], c.v[0], c.table, c.len, k, v, inv_freq=torch.ones(64, device=cuda), q=q),
                cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len + 1, 0.2, softcap=30.0, window=50,
                                                 alibi_slopes=torch.ones(8, device=cuda), lse=lse), lse,
                cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, k, v, i32([0, 2, 3, 3]), c.len, i32([2, 1, 0]),
                                                      parent=i32([-1, 0, -1]), max_pack=2, max_prefix=90)]
        cast_b200.append_paged(c.k, c.v, c.table, c.len, [k, k], [v, v], i32([0, 2, 3, 3]), keep=i32([[0, 1], [0, -1], [-1, -1]]),
                               accepted=i32([2, 1, 0]))
        return outs + [t.clone() for t in c.k + c.v]

    want = everything()
    monkeypatch.setattr(_lib, "_BINDING", _lib._NoBinding())
    assert all(torch.equal(a, b) for a, b in zip(everything(), want)) and _lib.device_error() == 0


# ------------------------------------------------------------------------------------- refusals, both ways
def _base_calls(dev):
    """Arguments of one good call of each operator, by name, in the binding's order, and the public function."""
    c = Cache(64, [9, 40], 2, 64, 16, torch.bfloat16, dev, room=2, poison=False)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    one = lambda *s: torch.ones(s, dtype=torch.bfloat16, device=dev)
    append = dict(k_pages=c.k[0], v_pages=c.v[0], page_table=c.table, seq_len=c.len, k=one(2, 2, 64), v=one(2, 2, 64), cu_q=None,
                  keep=None, accepted=None, inv_freq=torch.ones(32, device=dev), positions=None, interleaved=False, rope_scale=1.0,
                  q=one(2, 4, 64), q_out=None)
    decode = dict(q=one(2, 4, 64), k_pages=c.k[0], v_pages=c.v[0], page_table=c.table, seq_len=c.len, sm_scale=None, softcap=0.0,
                  window=0, alibi_slopes=None, out=None, lse=None, workspace=None)
    tree = dict(q=one(3, 4, 64), k_pages=c.k[0], v_pages=c.v[0], page_table=c.table, k_pack=one(3, 2, 64), v_pack=one(3, 2, 64),
                cu_q=i32(0, 2, 3), prefix_len=c.len, pack_len=i32(2, 1), ancestor_mask=None, sm_scale=None, parent=i32(-1, 0, -1),
                max_pack=2, max_prefix=40, out=None, workspace=None)
    return {"append": (append, cast_b200.append_paged), "decode": (decode, cast_b200.decode_attention_paged),
            "tree": (tree, cast_b200.varlen_tree_attention_paged)}


def _bad(op, dev):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=dev)
    f = lambda *s: torch.zeros(s, device=dev)
    pages = [dict(k_pages=z(4, 2, 16, 64)), dict(v_pages=z(1, 2, 16, 64)), dict(k_pages=f(4, 2, 16, 64), v_pages=f(4, 2, 16, 64)),
             dict(k_pages=z(4, 2, 16), v_pages=z(4, 2, 16)), dict(k_pages=z(4, 2, 16, 128)[..., ::2], v_pages=z(4, 2, 16, 128)[..., ::2]),
             dict(page_table=i32(1, 2)), dict(page_table=None)]
    if op == "append":
        return pages + [
            dict(seq_len=i32(1, 2, 3)), dict(k=z(2, 3, 64)), dict(v=z(3, 2, 64)), dict(k=z(2, 2, 32)), dict(k=f(2, 2, 64)), dict(k=z(2, 2, 128)[..., ::2]),
            dict(cu_q=i32(0, 2)), dict(keep=i32(0, 0).view(2, 1)), dict(accepted=i32(1, 1)), dict(keep=i32(0, 0).view(2, 1), accepted=i32(1, 1)),
            dict(keep=i32(0, 0), accepted=i32(1, 1), cu_q=i32(0, 1, 2), q=None), dict(keep=i32(0, 0).view(2, 1), accepted=i32(1, 1), cu_q=i32(0, 1, 2)),
            dict(inv_freq=f(33)), dict(inv_freq=None), dict(positions=i32(1)), dict(q=z(3, 4, 64)), dict(q=z(2, 4, 32)), dict(q=f(2, 4, 64)),
            dict(q_out=z(2, 3, 64)), dict(q=None, q_out=z(2, 4, 64)), dict(q_out=f(2, 4, 64)), dict(q_out=z(2, 4, 128)[..., ::2]),
            dict(q_out=z(1, 4, 64).expand(2, 4, 64)), dict(q_out=z(2, 1, 64).expand(2, 4, 64)), dict(page_table=i32(0, 1).view(2, 1)[:, :0])]
    scale = [dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(sm_scale=math.nan)]
    if op == "decode":
        return pages + scale + [
            dict(q=z(3, 4, 64)), dict(q=z(2, 3, 64)), dict(q=f(2, 4, 64)), dict(q=z(2, 4, 32)), dict(q=z(2, 256)), dict(seq_len=i32(1)),
            dict(softcap=-1.0), dict(softcap=1e31), dict(softcap=math.nan), dict(window=-1), dict(alibi_slopes=f(3)), dict(alibi_slopes=f(2, 2)),
            dict(out=z(2, 3, 64)), dict(out=f(2, 4, 64)), dict(out=z(2, 4, 66)[..., 1:65]), dict(out=z(1, 4, 64).expand(2, 4, 64)),
            dict(lse=f(8)), dict(lse=f(4, 2)), dict(lse=z(2, 4)), dict(lse=f(2, 8)[:, ::2]),
            dict(k_pages=z(4, 2, 16, 96), v_pages=z(4, 2, 16, 96), q=z(2, 4, 96)),
            dict(k_pages=z(4, 2, 16, 68)[..., :64], v_pages=z(4, 2, 16, 68)[..., :64])]
    return pages + scale + [
        dict(q=z(3, 3, 64)), dict(q=f(3, 4, 64)), dict(q=z(4, 4, 64)), dict(k_pack=z(2, 2, 64)), dict(v_pack=z(3, 1, 64)), dict(k_pack=f(3, 2, 64)),
        dict(cu_q=i32(0, 3)), dict(prefix_len=i32(1)), dict(pack_len=i32(1, 1, 1)), dict(parent=None), dict(parent=i32(-1, 0)),
        dict(ancestor_mask=torch.ones(3, dtype=torch.int64, device=dev)), dict(parent=None, ancestor_mask=torch.ones(4, dtype=torch.int64, device=dev)),
        dict(max_pack=-1), dict(max_prefix=-1), dict(max_pack=2000), dict(max_pack=1 << 32), dict(max_prefix=(1 << 31) - 1),
        dict(out=z(3, 3, 64)), dict(out=f(3, 4, 64)), dict(out=z(1, 4, 64).expand(3, 4, 64)), dict(out=z(3, 4, 66)[..., 1:65])]


@pytest.mark.parametrize("op", ["append", "decode", "tree"])
def test_binding_and_paged_py_refuse_alike(cuda, op, monkeypatch):
    """What paged.py refuses, the binding leaves to it: each bad call raises the same error with and without the binding,
    which takes none of them, and nothing is written."""
    good, call = _base_calls(cuda)[op]
    bind = getattr(_lib.binding(), op)
    assert bind(*good.values()) is not NotImplemented
    watch = (good["k_pages"].clone(), good["v_pages"].clone())
    for i, bad in enumerate(_bad(op, cuda)):
        kw = dict(good, **bad)
        assert bind(*kw.values()) is NotImplemented, (i, list(bad))
        errors = []
        for without in (False, True):
            with monkeypatch.context() as m:
                if without:
                    m.setattr(_lib, "_BINDING", _lib._NoBinding())
                with pytest.raises((ValueError, AssertionError, _lib.CastError)) as e:
                    call(**kw)
                errors.append((type(e.value), str(e.value)))
        assert errors[0] == errors[1], (i, list(bad))
    assert torch.equal(good["k_pages"], watch[0]) and torch.equal(good["v_pages"], watch[1]) and _lib.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,Hq,Hkv,ps,B,n", [(128, 8, 2, 64, 40, 3000), (128, 32, 8, 16, 2, 16000), (64, 6, 2, 1, 3, 5000), (64, 4, 1, 24, 2, 900)])
def test_tree_long_tail_of_small_probabilities(cuda, dtype, D, Hq, Hkv, ps, B, n):
    """As for decode, over the prefix of one-token packs whose own key has the score -15.76 as well. Probabilities are one
    16-bit term: off by half(type) of p, in half precision by half a step of its smallest, 2^-25, on 2^7 p = 2.4 x 2^-17."""
    dt = TYPES[dtype]
    pages = -(-n // ps)
    at = torch.arange(pages * ps, device=cuda).view(pages, 1, ps, 1)
    top = (at % 500 == 7).expand(pages, Hkv, ps, D)
    level = torch.tensor(-15.76 / math.sqrt(D), dtype=dt, device=cuda)
    k = torch.where(top, torch.zeros_like(level), level).contiguous()
    v = torch.where(top, torch.zeros_like(level), torch.full_like(level, 1000.0)).contiguous()
    q = torch.ones(B, Hq, D, dtype=dt, device=cuda)
    table = torch.arange(pages, dtype=torch.int32, device=cuda).repeat(B, 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    kp, vp = level.expand(B, Hkv, D).contiguous(), torch.full((B, Hkv, D), 1000.0, dtype=dt, device=cuda)
    got = cast_b200.varlen_tree_attention_paged(q, k, v, table, kp, vp, i32(list(range(B + 1))), i32([n] * B), i32([1] * B),
                                                parent=i32([-1] * B), max_pack=1, max_prefix=n)
    assert _lib.device_error() == 0
    s = level.double() * math.sqrt(D)
    tops = len(range(7, n, 500))
    tail = (n + 1 - tops) * torch.exp(s)
    want = (1000.0 * tail / (tops + tail)).expand(B, Hq, D)
    e = (D + 2) * 2 * U32 * s.abs().expand(B, Hq)
    _check_attention(got, want, e, want, 0, dt, 2.0 ** -8 if dtype == "bf16" else 2.0 ** -25 / (2.4 * 2.0 ** -17))


# ------------------------------------------------------------------------------------- graphs and streams
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_tree_and_accept_captured_and_on_two_streams(cuda, dtype):
    """A verify pass and the append of its accepted rows, captured once with the table's capacity as the bound, replayed with
    other lengths, packs, accepted rows and contents beside eager calls on another stream, each with its own workspace."""
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 65, [900, 33, 1500], [17, 1, 20], 8, 2, 128, 16, dt)
    for t in c.k + c.v:
        t.nan_to_num_(0.5, 0.5, 0.5)
    room = int(torch.where(c.table >= 0, c.table < c.num, False).sum(1).min()) * 16       # keys every sequence has pages for
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    par, cu, P = i32(sum(parents, [])), i32(cu.tolist()), i32([17, 1, 20])
    length, keep, acc = i32([20, 33, 5]), i32([[0, 3, 8], [0, -1, -1], [0, 5, -1]]), i32([3, 1, 2])
    cap = c.table.shape[1] * 16
    ws = [torch.full((64 << 20,), 255, dtype=torch.uint8, device=cuda) for _ in range(2)]
    outs = [torch.zeros_like(q) for _ in range(2)]
    pages = [(c.k[0], c.v[0]), (c.k[0].clone(), c.v[0].clone())]

    def step(i):
        k, v = pages[i]
        cast_b200.varlen_tree_attention_paged(q, k, v, c.table, kp, vp, cu, length, P, parent=par, max_pack=20, max_prefix=cap,
                                              out=outs[i], workspace=ws[i])
        cast_b200.append_paged(k, v, c.table, length, kp, vp, cu, keep=keep, accepted=acc)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0)
    g = torch.Generator(device=cuda).manual_seed(66)
    for lens, took in (([20, 33, 5], [3, 1, 2]), ([0, 1, 40], [0, 1, 1]), ([room - 3, 17, 16], [3, 0, 2])):
        length.copy_(i32(lens))
        acc.copy_(i32(took))
        q.normal_(generator=g)
        pages[0][0].normal_(generator=g)
        pages[1][0].copy_(pages[0][0])
        pages[1][1].copy_(pages[0][1])
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            step(1)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()
        assert torch.equal(pages[0][0], pages[1][0]) and torch.equal(pages[0][1], pages[1][1])
    assert _lib.device_error() == 0
