"""Paged cache operators against the formulas in 64 bits.

Bounds, with u = finfo(type).eps / 2 (half a step) and u32 = 2^-24:

* append: the sine and cosine of the reduced angle are within 2 steps of 32 bits (rounding the remainder, the
  function), each product, sum and the scale round once: 5 u32 (|x_a| + |x_b|), then u of the result.
* attention: a dot product of D terms is off by at most (D + 2) 2 u32 sum |q d| |k d| scale =: e (twice u32 for sums
  that drop instead of rounding), a probability by 2 e + 2^-21 (exponential, scale) relative, numerator and
  denominator alike; n added terms by n u32. So |out| is off by (4 e + 2^-20 + 2 n u32 [+ what p is rounded by]) sum p
  |v|, then u of the result. A capped or biased score adds 4 u32 of its largest value to e.
"""
import math

import numpy as np
import pytest
import torch

import cast_b200
from cast_b200 import _lib

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


class Cache:
    """Random pages, page by page in a random order, with poison wherever no key of a sequence is."""

    def __init__(self, seed, lens, Hkv, D, ps, dtype, dev, order="hnd", room=0, poison=True, layers=1):
        g = torch.Generator(device=dev).manual_seed(seed)
        need = [-(-(n + room) // ps) for n in lens]
        width = max(1, max(need, default=1)) + 1
        self.num = sum(need) + 3
        perm = torch.randperm(self.num, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lens), width), 0x7fffffff, dtype=torch.int32, device=dev)   # never to be read
        self.lens, self.ps, self.Hkv, self.D = list(lens), ps, Hkv, D
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            at += n
        self.k, self.v = [], []
        for which in (self.k, self.v):
            for _ in range(layers):
                shape = (self.num, Hkv, ps, D) if order == "hnd" else (self.num, ps, Hkv, D)
                t = torch.empty(shape, dtype=dtype, device=dev).normal_(generator=g)
                which.append(t if order == "hnd" else t.transpose(1, 2))
        self.len = torch.tensor(lens, dtype=torch.int32, device=dev)
        if poison:
            free = torch.ones((self.num, ps), dtype=torch.bool)
            for b, n in enumerate(lens):
                for j in range(need[b]):
                    free[int(self.table[b, j]), :max(0, min(ps, n - j * ps))] = False
            free = free.to(dev)[:, None, :, None]
            for t in self.k:
                t.masked_fill_(free, math.nan)
            for t in self.v:
                t.masked_fill_(free, math.inf)

    def rows(self, pages, b, lo, hi):
        n = torch.arange(lo, hi, device=pages.device)
        return pages[self.table[b].long()[n // self.ps], :, n % self.ps]     # [keys, H, D]


# ------------------------------------------------------------------------------------------------ append
def _turn(x, pos, freq, interleaved, scale):
    """x [rows, H, D] in 64 bits turned by pos * freq; and the sum of magnitudes the bound goes by."""
    h = freq.numel()
    ang = pos.double()[:, None] * freq.double()
    c, s = (ang.cos() * scale)[:, None], (ang.sin() * scale)[:, None]
    y, mag = x.clone(), torch.zeros_like(x)
    ia = torch.arange(h, device=x.device) * (2 if interleaved else 1)
    ib = ia + 1 if interleaved else ia + h
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * scale
    return y, mag


def _check_turned(got, x, pos, freq, interleaved, scale):
    if freq is None:
        assert torch.equal(got, x)
        return
    want, mag = _turn(x.double(), pos, freq, interleaved, scale)
    bound = 5 * U32 * mag + _half(got.dtype) * (want.abs() + 5 * U32 * mag) + 2.0 ** -25 * (got.dtype == torch.float16)
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max().item()
    h2 = 2 * freq.numel()
    assert torch.equal(got[..., h2:], x[..., h2:])


def _freq(rot, dev):
    return (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().to(dev) if rot else None


def _run_append(dev, seed, lens, new, Hq, Hkv, D, ps, dtype, rot, interleaved=False, order="hnd", mode="rows", shift=0,
                scale=1.0, positions=None, behind=2, inplace=False):
    c = Cache(seed, lens, Hkv, D, ps, dtype, dev, order, room=max(new, default=0), poison=False)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    total = sum(new) + behind
    def rows(H):      # shift: rows that start off 16 bytes
        return torch.empty((total, H, D + 2 * shift), dtype=dtype, device=dev).normal_(generator=g)[..., shift:shift + D]
    k, v, q = rows(Hkv), rows(Hkv), rows(Hq)
    freq = _freq(rot, dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
    before_k, before_v = c.k[0].clone(), c.v[0].clone()
    q0 = q.clone()
    use_q = freq is not None
    q_out = None if not use_q else q if inplace else torch.full_like(q, 7.0)
    got_q = cast_b200.append_paged(c.k[0], c.v[0], c.table, c.len, k, v, None if mode == "token" else cu, inv_freq=freq,
                                   positions=positions, interleaved=interleaved, rope_scale=scale,
                                   q=q if use_q else None, q_out=q_out)
    assert _lib.device_error() == 0
    assert c.len.tolist() == list(lens)
    n_rows = sum(new)
    slot = torch.cat([torch.arange(m) + n for n, m in zip(lens, new)]).to(dev) if n_rows else torch.zeros(0, device=dev)
    pos = slot if positions is None else positions[:n_rows]
    at = 0
    for b, m in enumerate(new):
        if m:
            _check_turned(c.rows(c.k[0], b, lens[b], lens[b] + m), k[at:at + m], pos[at:at + m], freq, interleaved, scale)
            assert torch.equal(c.rows(c.v[0], b, lens[b], lens[b] + m), v[at:at + m])
            n = torch.arange(lens[b], lens[b] + m, device=dev)
            pg = c.table[b].long()[n // ps]
            before_k[pg, :, n % ps] = c.k[0][pg, :, n % ps]
            before_v[pg, :, n % ps] = c.v[0][pg, :, n % ps]
        at += m
    assert torch.equal(before_k, c.k[0]) and torch.equal(before_v, c.v[0])      # nothing else was written
    if use_q:
        _check_turned(got_q[:n_rows], q0[:n_rows], pos, freq, interleaved, scale)
        rest = q0[n_rows:] if inplace else torch.full_like(q0[n_rows:], 7.0)
        assert torch.equal(got_q[n_rows:], rest)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (128, 64, True), (64, 32, False), (64, 64, True),
                                               (128, 0, False), (80, 80, False), (256, 256, False)])
@pytest.mark.parametrize("ps,order", [(16, "hnd"), (7, "nhd"), (1, "hnd")])
def test_append_rows(cuda, dtype, D, rot, interleaved, ps, order):
    _run_append(cuda, 1, [0, 15, 33, 5, 16], [17, 1, 0, 40, 16], 6, 2, D, ps, TYPES[dtype], rot, interleaved, order)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rot,interleaved", [(0, False), (64, False), (34, False), (6, True), (64, True)])
def test_append_rows_off_16_bytes(cuda, dtype, rot, interleaved):
    # rows at an odd element offset, halves that are no whole pieces: the element-wise form
    _run_append(cuda, 2, [3, 30], [9, 20], 3, 1, 64, 24, TYPES[dtype], rot, interleaved, shift=1)
    _run_append(cuda, 3, [3, 30], [9, 20], 3, 3, 50, 24, TYPES[dtype], min(rot, 50), interleaved)


@pytest.mark.parametrize("B", [1, 5, 300])
def test_append_one_token_each(cuda, B):
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 70, B).tolist()
    _run_append(cuda, 4, lens, [1] * B, 8, 2, 128, 16, torch.bfloat16, 128, mode="token")


def test_append_many_sequences_some_without_rows(cuda):
    # the search for a row's sequence goes over 3000 offsets, runs of equal ones among them
    rng = np.random.default_rng(5)
    new = (rng.integers(0, 4, 3000) * (rng.random(3000) < 0.3)).tolist()
    _run_append(cuda, 5, rng.integers(0, 20, 3000).tolist(), new, 2, 1, 64, 16, torch.float16, 64, behind=300)


def test_append_far_positions_scale_and_in_place(cuda):
    pos = torch.tensor([1 << 20, 131071, 999999, 0, -5, 77, 1000003, 2, 3, 4, 5, 6], dtype=torch.int32, device=cuda)
    _run_append(cuda, 6, [10, 20], [4, 6], 4, 2, 128, 32, torch.float32, 128, scale=1.25, positions=pos, inplace=True)


def test_append_accepted_rows_of_every_layer(cuda):
    # 70 layers (two launches), lists with none, one and all rows kept, padded with -1
    lens, packs, layers = [0, 31, 16, 5], [9, 4, 6, 12], 70
    c = Cache(7, lens, 2, 64, 16, torch.bfloat16, cuda, room=12, poison=False, layers=layers)
    g = torch.Generator(device=cuda).manual_seed(8)
    cu = np.concatenate([[0], np.cumsum(packs)]).astype(np.int32)
    hook = [torch.empty((2, int(cu[-1]), 64), dtype=torch.bfloat16, device=cuda).normal_(generator=g) for _ in range(2 * layers)]
    ks, vs = [t.transpose(0, 1) for t in hook[:layers]], [t.transpose(0, 1) for t in hook[layers:]]
    picks = [[0, 3, 8], [], [0], list(range(12))]
    keep = torch.full((4, 13), -1, dtype=torch.int32)
    for b, p in enumerate(picks):
        keep[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    want_k, want_v = [t.clone() for t in c.k], [t.clone() for t in c.v]
    for b, p in enumerate(picks):
        for j, i in enumerate(p):
            pg, r = int(c.table[b, (lens[b] + j) // 16]), (lens[b] + j) % 16
            for l in range(layers):
                want_k[l][pg, :, r], want_v[l][pg, :, r] = ks[l][cu[b] + i], vs[l][cu[b] + i]
    cast_b200.append_paged(c.k, c.v, c.table, c.len, ks, vs, torch.from_numpy(cu), keep=keep,
                           accepted=torch.tensor([len(p) for p in picks], dtype=torch.int32))
    assert _lib.device_error() == 0
    assert all(torch.equal(a, b) for a, b in zip(c.k + c.v, want_k + want_v))


def test_append_skips_what_is_out_of_range(cuda):
    c = Cache(9, [5, 5, 5, 5], 1, 64, 16, torch.bfloat16, cuda, room=1, poison=False)
    k = torch.ones(4, 1, 64, dtype=torch.bfloat16, device=cuda)
    c.table[0, 0], c.table[1, 0] = c.num, -1
    c.len[2] = 16 * c.table.shape[1]
    before = c.k[0].clone()
    cast_b200.append_paged(c.k[0], c.v[0], c.table, c.len, k, k)
    assert _lib.device_error() == _lib.CAST_DEV_BAD_LAYOUT
    before[int(c.table[3, 0]), :, 5] = 1.0
    assert torch.equal(c.k[0], before)
    # keep entries outside the pack
    cu = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=cuda)
    c = Cache(9, [5, 5, 5, 5], 1, 64, 16, torch.bfloat16, cuda, room=1, poison=False)
    before = c.k[0].clone()
    keep = torch.tensor([[1], [-1], [0], [0]], dtype=torch.int32, device=cuda)
    acc = torch.tensor([1, 1, 2, 1], dtype=torch.int32, device=cuda)
    cast_b200.append_paged(c.k[0], c.v[0], c.table, c.len, k, k, cu, keep=keep, accepted=acc)
    assert _lib.device_error() == _lib.CAST_DEV_BAD_LAYOUT
    before[int(c.table[3, 0]), :, 5] = 1.0
    assert torch.equal(c.k[0], before)


# ------------------------------------------------------------------------------------------------ decode
def _attend(q, k, v, scale, cap, slopes, dist, hide=None):
    """64-bit attention of rows q [R, Hq, D] over k / v [n, Hkv, D]: out, lse, and the bound's sums."""
    R, Hq, D = q.shape
    G = Hq // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = torch.einsum("rhd,nhd->rhn", q, k) * scale
    e = (D + 2) * 2 * U32 * torch.einsum("rhd,nhd->rhn", q.abs(), k.abs()).amax(-1, keepdim=True) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
        e = e + 4 * U32 * cap
    if slopes is not None:
        bias = slopes.double()[None, :, None] * dist
        s = s + bias
        e = e + 4 * U32 * (s.abs().amax(-1, keepdim=True) + bias.abs().amax(-1, keepdim=True))
    if hide is not None:
        s = s.masked_fill(hide[:, None], -math.inf)
    p = torch.softmax(s, -1)
    return (torch.einsum("rhn,nhd->rhd", p, v), torch.logsumexp(s, -1), e[..., 0],
            torch.einsum("rhn,nhd->rhd", p, v.abs()))


def _check_attention(got, want, e, pv, n, dtype, p_round=0.0):
    rel = (4 * e + 2.0 ** -20 + 2 * n * U32 + p_round)[..., None]
    bound = rel * pv + _half(dtype) * (want.abs() + rel * pv) + 2.0 ** -25 * (dtype == torch.float16)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()


def _run_decode(dev, seed, lens, Hq, Hkv, D, ps, dtype, order="hnd", cap=0.0, window=0, alibi=False, lse=True, scale=None,
                q_scale=1.0):
    vis = [n - window if window and n > window else 0 for n in lens]
    c = Cache(seed, lens, Hkv, D, ps, dtype, dev, order)
    for b, lo in enumerate(vis):       # keys behind the window hold poison too
        if lo:
            n = torch.arange(lo, device=dev)
            pg = c.table[b].long()[n // ps]
            c.k[0][pg, :, n % ps], c.v[0][pg, :, n % ps] = math.nan, math.inf
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    q = (torch.empty((len(lens), Hq, D), device=dev).normal_(generator=g) * q_scale).to(dtype)
    slopes = 2.0 ** (-8.0 * (torch.arange(Hq, device=dev) + 1) / Hq) if alibi else None
    L = torch.full((len(lens), Hq), 5.0, device=dev) if lse else None
    got = cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len, scale, softcap=cap, window=window,
                                           alibi_slopes=slopes, lse=L)
    assert _lib.device_error() == 0
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all() and (L is None or torch.isneginf(L[b]).all())
            continue
        k, v = c.rows(c.k[0], b, vis[b], n), c.rows(c.v[0], b, vis[b], n)
        dist = torch.arange(vis[b] - (n - 1), 1, device=dev).double()
        out, want_l, e, pv = _attend(q[b:b + 1], k, v, scale or 1 / math.sqrt(D), cap, slopes, dist)
        m = n - vis[b]
        _check_attention(got[b:b + 1], out, e, pv, m, dtype, 2.0 ** -15)     # p as two 16-bit terms
        if L is not None:
            assert ((L[b].double() - want_l[0]).abs() <= 2 * e[0] + 2.0 ** -20 + m * U32 + 4 * U32 * want_l[0].abs()).all()
    return c, q, got


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (3, 3), (7, 1), (17, 1), (40, 1), (12, 4), (16, 2)])
def test_decode_lengths_and_heads(cuda, dtype, D, Hq, Hkv):
    _run_decode(cuda, 11, [1, 0, 15, 16, 17, 31, 33, 100, 257, 1000, 0], Hq, Hkv, D, 16, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ps,order", [(1, "hnd"), (3, "nhd"), (8, "hnd"), (24, "nhd"), (64, "nhd"), (100, "hnd"), (256, "hnd")])
def test_decode_pages(cuda, dtype, ps, order):
    _run_decode(cuda, 12, [5, 130, 64, 999], 8, 2, 128, ps, TYPES[dtype], order)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ps,order", [(1, "nhd"), (5, "hnd"), (8, "hnd"), (40, "nhd")])
def test_decode_pages_of_small_heads(cuda, dtype, ps, order):
    # D = 64: steps of 32 keys (16 in 32 bits), which pages of fewer rows cut
    _run_decode(cuda, 27, [5, 130, 64, 999, 31, 32, 33], 6, 2, 64, ps, TYPES[dtype], order, window=700)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cap,window,alibi", [(20.0, 0, False), (0.0, 1, False), (0.0, 50, False), (0.0, 0, True),
                                              (30.0, 130, True), (0.0, 5000, False)])
def test_decode_score_options(cuda, dtype, cap, window, alibi):
    _run_decode(cuda, 13, [1, 49, 50, 51, 700, 129], 12, 4, 64, 24, TYPES[dtype], cap=cap, window=window, alibi=alibi,
                q_scale=3.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens", [[40000], [1], [17], [0], [3, 20000, 0, 1, 9000]])
def test_decode_few_and_long(cuda, dtype, lens):
    _run_decode(cuda, 14, lens, 32, 8, 128, 64, TYPES[dtype], scale=0.2)


@pytest.mark.parametrize("B", [129, 700])
def test_decode_more_sequences_than_threads(cuda, B):
    rng = np.random.default_rng(B)
    lens = (rng.integers(0, 60, B) * (rng.random(B) < 0.7)).tolist()
    _run_decode(cuda, 15, lens, 4, 1, 64, 16, torch.float16)


def test_decode_sees_nan_and_skips_bad_metadata(cuda):
    lens = [40, 40, 40, 40, 40, 40]
    c, q, good = _run_decode(cuda, 16, lens, 8, 2, 128, 16, torch.bfloat16)
    c.k[0][int(c.table[1, 1]), 0, 3] = math.nan      # a visible key: the rows of its head are NaN, no others
    c.len[2], c.len[3] = -1, 16 * c.table.shape[1] + 1
    c.table[4, 2] = c.num
    got = cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len)
    assert _lib.device_error() == _lib.CAST_DEV_BAD_LAYOUT
    assert got[1, :4].isnan().all() and torch.equal(got[0], good[0]) and torch.equal(got[5], good[5])
    assert not got[1, 4:].isnan().any()
    assert (got[2:4] == 0).all()


def test_decode_cache_beyond_32_bit_offsets(cuda):
    # pages behind 2^32 elements: 2^20 pages of 4096 elements, keys in the last ones
    num, Hkv, ps, D = (1 << 20) + 64, 2, 16, 128
    k = torch.empty((num, Hkv, ps, D), dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    n = 500
    ids = torch.randperm(60, device=cuda)[:-(-n // ps)] + (1 << 20)
    g = torch.Generator(device=cuda).manual_seed(17)
    q = torch.empty((1, 8, D), dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    new = torch.empty((2, n, Hkv, D), dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    table, zero = ids.int()[None].contiguous(), torch.zeros(1, dtype=torch.int32, device=cuda)
    cast_b200.append_paged(k, v, table, zero, new[0], new[1], torch.tensor([0, n], dtype=torch.int32, device=cuda))
    got = cast_b200.decode_attention_paged(q, k, v, table, zero + n)
    assert _lib.device_error() == 0
    out, _, e, pv = _attend(q, new[0], new[1], 1 / math.sqrt(D), 0, None, None)
    _check_attention(got, out, e, pv, n, torch.bfloat16, 2.0 ** -15)
    par = torch.full((3,), -1, dtype=torch.int32, device=cuda)
    par[1:] = torch.tensor([0, 1])
    qt = q.expand(3, 8, D).contiguous()
    pk = new[:, :3].contiguous()
    tree = cast_b200.varlen_tree_attention_paged(qt, k, v, table, pk[0], pk[1], [0, 3], zero + n, zero + 3, parent=par)
    for i in range(3):
        kk, vv = torch.cat((new[0], pk[0][:i + 1])), torch.cat((new[1], pk[1][:i + 1]))
        out, _, e, pv = _attend(q, kk, vv, 1 / math.sqrt(D), 0, None, None)
        _check_attention(tree[i:i + 1], out, e, pv, n + i + 1, torch.bfloat16, _half(torch.bfloat16))
    del k, v


def test_decode_tails_of_long_groups(cuda):
    # 16 sequences of 16000 keys, 8 heads: 128000 steps are 108 to a group, so the groups end in two tails; a table with
    # no room to spare. Also: the same call twice gives the same bits, and padded rows of the batch (length 0) give 0.
    lens = [16000] * 15 + [15999, 0]
    c = Cache(30, lens, 8, 128, 64, torch.bfloat16, cuda, poison=False)
    g = torch.Generator(device=cuda).manual_seed(31)
    q = torch.empty((17, 32, 128), dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    got = cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len)
    assert torch.equal(got, cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len))
    assert _lib.device_error() == 0 and (got[16] == 0).all()
    for b in (0, 3, 7, 11, 15):
        k, v = c.rows(c.k[0], b, 0, lens[b]), c.rows(c.v[0], b, 0, lens[b])
        out, _, e, pv = _attend(q[b:b + 1], k, v, 1 / math.sqrt(128), 0, None, None)
        _check_attention(got[b:b + 1], out, e, pv, lens[b], torch.bfloat16, 2.0 ** -15)


def test_decode_two_streams_with_their_own_workspaces(cuda):
    c = Cache(33, [5000, 700, 9000], 4, 128, 16, torch.float16, cuda, poison=False)
    g = torch.Generator(device=cuda).manual_seed(34)
    q = torch.empty((3, 16, 128), dtype=torch.float16, device=cuda).normal_(generator=g)
    want = cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len)
    torch.cuda.synchronize()
    n = cast_b200.decode_workspace_size(torch.float16, 3, 16, 4, 128)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [torch.empty(n, dtype=torch.uint8, device=cuda) for _ in streams]
    outs = [[torch.empty_like(q) for _ in range(5)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(5):
        for s, st in enumerate(streams):
            with torch.cuda.stream(st):
                cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, c.len, out=outs[s][i], workspace=ws[s])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for os in outs for o in os)


def test_decode_graph_streams_and_repeats(cuda):
    # captured once, replayed with other lengths, tables and contents; equal to eager calls bit for bit
    c = Cache(18, [900, 33, 1500, 7], 2, 128, 16, torch.bfloat16, cuda, room=16, poison=False)
    g = torch.Generator(device=cuda).manual_seed(19)
    q = torch.empty((4, 8, 128), dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    k, v = (torch.empty((4, 2, 128), dtype=torch.bfloat16, device=cuda).normal_(generator=g) for _ in range(2))
    freq = _freq(128, cuda)
    n = cast_b200.decode_workspace_size(torch.bfloat16, 4, 8, 2, 128)

    def step(ws, q_out, out, grown):
        cast_b200.append_paged(c.k[0], c.v[0], c.table, c.len, k, v, inv_freq=freq, q=q, q_out=q_out)
        torch.add(c.len, 1, out=grown)
        cast_b200.decode_attention_paged(q_out, c.k[0], c.v[0], c.table, grown, out=out, workspace=ws)

    bufs = [(torch.full((n,), 255, dtype=torch.uint8, device=cuda), torch.empty_like(q), torch.empty_like(q),
             torch.empty_like(c.len)) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*bufs[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*bufs[0])
    for lens in ([900, 33, 1500, 7], [12, 0, 1, 15], [901, 34, 1501, 8]):
        c.len.copy_(torch.tensor(lens, dtype=torch.int32))
        q.normal_(generator=g)
        graph.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            step(*bufs[1])
        torch.cuda.current_stream().wait_stream(side)
        step(*bufs[1])
        assert torch.equal(bufs[0][2], bufs[1][2]) and torch.equal(bufs[0][1], bufs[1][1])
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------------------------ tree
def _tree_inputs(dev, seed, S, P, Hq, Hkv, D, ps, dtype, order="hnd"):
    c = Cache(seed, S, Hkv, D, ps, dtype, dev, order)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    rng = np.random.default_rng(seed)
    total = sum(P)
    q = torch.empty((total, Hq, D), dtype=dtype, device=dev).normal_(generator=g)
    kv = torch.empty((2, Hkv, total, D), dtype=dtype, device=dev).normal_(generator=g)
    parents = [[-1] + [int(rng.integers(max(0, i - 9), i)) for i in range(1, p)] for p in P]
    cu = np.concatenate([[0], np.cumsum(P)]).astype(np.int32)
    return c, q, kv[0].transpose(0, 1), kv[1].transpose(0, 1), parents, cu


def _seen(parents):
    P = len(parents)
    m = torch.zeros(P, P, dtype=torch.bool)
    for i in range(P):
        a = i
        while a >= 0:
            m[i, a] = True
            a = parents[a]
    return m


def _check_tree(got, c, q, kp, vp, seen, cu, S, dtype, p_round):
    D = q.shape[2]
    for b, s in enumerate(S):
        rows = slice(int(cu[b]), int(cu[b + 1]))
        P = rows.stop - rows.start
        if P == 0:
            continue
        k, v = (torch.cat((c.rows(pg, b, 0, s), pk[rows])) for pg, pk in ((c.k[0], kp), (c.v[0], vp)))
        hide = torch.zeros(P, s + P, dtype=torch.bool, device=q.device)
        hide[:, s:] = ~seen[b].to(q.device)
        out, _, e, pv = _attend(q[rows], k, v, 1 / math.sqrt(D), 0, None, None, hide)
        empty = hide.all(1)
        assert (got[rows][empty] == 0).all()
        _check_attention(got[rows][~empty], out[~empty], e[~empty], pv[~empty], s + P, dtype, p_round)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ps,order", [(1, "hnd"), (2, "hnd"), (4, "nhd"), (8, "nhd"), (16, "hnd"), (24, "hnd"), (64, "nhd"),
                                      (100, "hnd"), (128, "hnd"), (384, "nhd")])
def test_tree_pages(cuda, dtype, ps, order):
    S, P = [0, 5, 127, 128, 300, 1000], [17, 1, 70, 33, 129, 3]
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 21, S, P, 8, 2, 128, ps, dt, order)
    got = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P,
                                                parent=np.concatenate(parents))
    assert _lib.device_error() == 0
    _check_tree(got, c, q, kp, vp, [_seen(p) for p in parents], cu, S, dt, 0.0 if dtype == "fp32" else _half(dt))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Hq,Hkv,D", [(3, 1, 128), (12, 4, 64), (4, 4, 128), (64, 4, 128), (7, 1, 64), (128, 1, 128)])
def test_tree_heads(cuda, dtype, Hq, Hkv, D):
    S, P = [40, 0, 200], [9, 1, 20]
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 22, S, P, Hq, Hkv, D, 16, dt)
    got = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P,
                                                parent=np.concatenate(parents))
    assert _lib.device_error() == 0
    _check_tree(got, c, q, kp, vp, [_seen(p) for p in parents], cu, S, dt, 0.0 if dtype == "fp32" else _half(dt))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Hq,Hkv,D,ps", [(3, 1, 64, 1), (10, 2, 128, 5), (8, 2, 64, 12)])
def test_tree_rows_of_odd_pages(cuda, dtype, Hq, Hkv, D, ps):
    # pages that are no multiple of 8: rows copied one by one, over several tiles and an unfinished one
    S, P = [700, 0, 129, 128], [9, 1, 130, 64]
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 28, S, P, Hq, Hkv, D, ps, dt)
    got = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P,
                                                parent=np.concatenate(parents))
    assert _lib.device_error() == 0
    _check_tree(got, c, q, kp, vp, [_seen(p) for p in parents], cu, S, dt, 0.0 if dtype == "fp32" else _half(dt))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_tree_strides_of_four_elements(cuda, dtype):
    # head strides that are multiples of 4 but not of 8: the CUDA-core form, products in 32 bits throughout
    S, P = [200, 13], [20, 65]
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 29, S, P, 8, 2, 128, 24, dt)
    wide = torch.zeros(q.shape[0], 8, 132, dtype=dt, device=cuda)
    wide[..., :128] = q
    got = cast_b200.varlen_tree_attention_paged(wide[..., :128], c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P,
                                                parent=np.concatenate(parents))
    assert _lib.device_error() == 0
    _check_tree(got, c, q, kp, vp, [_seen(p) for p in parents], cu, S, dt, 0.0)


@pytest.mark.parametrize("dtype,Hq", [("bf16", 32), ("fp32", 8)])
def test_tree_long_prefix_split_over_its_length(cuda, dtype, Hq):
    S, P = [20000, 9001], [65, 17]
    dt = TYPES[dtype]
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 23, S, P, Hq, 8, 128, 64, dt)
    got = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P,
                                                parent=np.concatenate(parents), max_pack=65, max_prefix=20000)
    assert _lib.device_error() == 0
    _check_tree(got, c, q, kp, vp, [_seen(p) for p in parents], cu, S, dt, 0.0 if dtype == "fp32" else _half(dt))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_tree_words_rows_without_keys_and_rows_behind(cuda, dtype):
    # any bits: rows that see no key at all (no prefix, no bit) become 0; rows behind the last pack are left
    S, P = [0, 50], [40, 64]
    dt = TYPES[dtype]
    c, q, kp, vp, _, cu = _tree_inputs(cuda, 24, S, [40, 67], 8, 2, 128, 16, dt)
    rng = np.random.default_rng(24)
    words = rng.integers(-2 ** 63, 2 ** 63, 107, dtype=np.int64)
    words[[0, 7, 39]] = 0
    words[50] = 0
    cu = np.array([0, 40, 104], dtype=np.int32)
    out = torch.full_like(q, 7.0)
    got = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P,
                                                torch.from_numpy(words).to(cuda), out=out)
    assert _lib.device_error() == 0 and (got[104:] == 7.0).all()
    seen = []
    for b, p in enumerate(P):
        w = torch.from_numpy(words[cu[b]:cu[b + 1]])
        seen.append(((w[:, None] >> torch.arange(p)) & 1).bool())
    _check_tree(got, c, q, kp, vp, seen, cu, S, dt, 0.0 if dtype == "fp32" else _half(dt))


def test_tree_equals_the_store_form(cuda):
    # 40 sequences x 8 KV heads are 320 units, above the two per SM up to which either launch plan splits the keys (the
    # plans cut small launches differently, and partial sums of other cuts round differently): the same tiles in the
    # same order, so the same bits
    rng = np.random.default_rng(25)
    S, P = [0, 128, 257, 1000] + rng.integers(0, 300, 36).tolist(), [64, 1, 129, 300] + rng.integers(1, 40, 36).tolist()
    c, q, kp, vp, parents, cu = _tree_inputs(cuda, 25, S, P, 32, 8, 128, 16, torch.bfloat16)
    ks = torch.zeros(40, 8, 1024, 128, dtype=torch.bfloat16, device=cuda)
    vs = torch.zeros_like(ks)
    for b, s in enumerate(S):
        ks[b, :, :s], vs[b, :, :s] = c.rows(c.k[0], b, 0, s).transpose(0, 1), c.rows(c.v[0], b, 0, s).transpose(0, 1)
    par = torch.tensor(sum(parents, []), dtype=torch.int32, device=cuda)
    pk = torch.tensor(P, dtype=torch.int32, device=cuda)
    a = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, pk, parent=par)
    b = cast_b200.varlen_tree_attention_store(q, ks, vs, kp, vp, cu, c.len, pk, parent=par)
    assert _lib.device_error() == 0 and torch.equal(a, b)


def test_tree_reports_bad_metadata(cuda):
    S, P = [100, 100, 100], [8, 8, 8]
    for dt in (torch.bfloat16, torch.float32):
        c, q, kp, vp, parents, cu = _tree_inputs(cuda, 26, S, P, 8, 2, 128, 16, dt)
        par = np.concatenate(parents)
        good = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P, parent=par)
        c.table[1, 2], c.table[1, 3] = -7, c.num
        got = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P, parent=par)
        assert _lib.device_error() == _lib.CAST_DEV_BAD_LAYOUT
        assert torch.equal(got[:8], good[:8]) and torch.equal(got[16:], good[16:])
        cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, kp, vp, cu, c.len, P, parent=par, max_prefix=99,
                                              max_pack=8)
        assert _lib.device_error() == _lib.CAST_DEV_BAD_LAYOUT


# ------------------------------------------------------------------------------------------------ together
def test_prompt_verify_accept_and_decode_on_one_cache(cuda):
    """Prompt rows appended, a draft tree verified on the pages, its accepted path appended, one token decoded: each
    attention against a contiguous 64-bit reference that never sees a page."""
    dt, Hq, Hkv, D, ps, layers = torch.bfloat16, 8, 2, 128, 16, 2
    S, P = [37, 64, 5], [12, 1, 20]
    B = len(S)
    g = torch.Generator(device=cuda).manual_seed(31)
    rnd = lambda *s: torch.empty(s, dtype=dt, device=cuda).normal_(generator=g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    width = -(-(max(S) + 30) // ps)
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(3)).int().view(B, width).to(cuda)
    kps, vps = ([torch.full((B * width, Hkv, ps, D), math.nan, dtype=dt, device=cuda) for _ in range(layers)] for _ in range(2))
    freq = _freq(D, cuda)
    cu_s, zero = i32(np.concatenate([[0], np.cumsum(S)]).tolist()), i32([0] * B)
    hist = [[[], []] for _ in range(layers)]      # contiguous rows per layer, K and V, per sequence
    for l in range(layers):
        k, v, q = rnd(sum(S), Hkv, D), rnd(sum(S), Hkv, D), rnd(sum(S), Hq, D)
        cast_b200.append_paged(kps[l], vps[l], table, zero, k, v, cu_s, inv_freq=freq, q=q)
        for b in range(B):
            rows = slice(int(cu_s[b]), int(cu_s[b + 1]))
            turned, _ = _turn(k[rows].double(), torch.arange(S[b], device=cuda), freq, False, 1.0)
            hist[l][0].append(turned.to(dt))
            hist[l][1].append(v[rows])
    length = i32(S)
    rng = np.random.default_rng(32)
    parents = [[-1] + [int(rng.integers(0, i)) for i in range(1, p)] for p in P]
    cu = np.concatenate([[0], np.cumsum(P)]).astype(np.int32)
    cu_q, par = torch.from_numpy(cu).to(cuda), i32(sum(parents, []))
    tokens = i32(rng.permutation(64)[:sum(P)].tolist())
    packs = [(rnd(sum(P), Hkv, D), rnd(sum(P), Hkv, D)) for _ in range(layers)]
    for l in range(layers):
        q = rnd(sum(P), Hq, D)
        got = cast_b200.varlen_tree_attention_paged(q, kps[l], vps[l], table, packs[l][0], packs[l][1], cu_q, length, P,
                                                    parent=par, max_pack=max(P), max_prefix=max(S))
        for b in range(B):
            rows = slice(int(cu[b]), int(cu[b + 1]))
            kk, vv = torch.cat((hist[l][0][b], packs[l][0][rows])), torch.cat((hist[l][1][b], packs[l][1][rows]))
            hide = torch.zeros(P[b], S[b] + P[b], dtype=torch.bool, device=cuda)
            hide[:, S[b]:] = ~_seen(parents[b]).to(cuda)
            out, _, e, pv = _attend(q[rows], kk, vv, 1 / math.sqrt(D), 0, None, None, hide)
            # stored keys are within one more step of the reference's rounding of the rotation
            _check_attention(got[rows], out, e + 2 * _half(dt) * 4, pv * (1 + _half(dt)), S[b] + P[b], dt, _half(dt))
    logits = torch.randn(sum(P), 64, generator=g, device=cuda)
    walk = cast_b200.walk_trees_greedy(logits, cu_q, par, tokens, max(P))
    acc = walk.accepted.tolist()
    cast_b200.append_paged(kps, vps, table, length, [p[0] for p in packs], [p[1] for p in packs], cu_q, keep=walk.keep,
                           accepted=walk.accepted)
    length = length + walk.accepted
    for l in range(layers):
        for b in range(B):
            at = (walk.keep[b, :acc[b]] + int(cu[b])).long()
            hist[l][0][b] = torch.cat((hist[l][0][b], packs[l][0][at]))
            hist[l][1][b] = torch.cat((hist[l][1][b], packs[l][1][at]))
    for l in range(layers):
        q, k, v = rnd(B, Hq, D), rnd(B, Hkv, D), rnd(B, Hkv, D)
        qr = cast_b200.append_paged(kps[l], vps[l], table, length, k, v, inv_freq=freq, q=q)
        got = cast_b200.decode_attention_paged(qr, kps[l], vps[l], table, length + 1)
        for b in range(B):
            n = S[b] + acc[b]
            turned, _ = _turn(k[b:b + 1].double(), torch.tensor([n], device=cuda), freq, False, 1.0)
            kk, vv = torch.cat((hist[l][0][b], turned.to(dt))), torch.cat((hist[l][1][b], v[b:b + 1]))
            out, _, e, pv = _attend(qr[b:b + 1], kk, vv, 1 / math.sqrt(D), 0, None, None)
            _check_attention(got[b:b + 1], out, e + 2 * _half(dt) * 4, pv, n + 1, dt, 2.0 ** -15)
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------------------------ binding
def test_binding_and_python_path_agree(cuda):
    """Arguments that need no conversion go through the binding, others (here 64-bit lengths, lists) through paged.py."""
    b = _lib.binding()
    c = Cache(41, [90, 0, 33], 2, 128, 16, torch.bfloat16, cuda, room=8, poison=False, layers=2)
    g = torch.Generator(device=cuda).manual_seed(42)
    rnd = lambda *s: torch.empty(s, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    q, k, v = rnd(3, 8, 128), rnd(3, 2, 128), rnd(3, 2, 128)
    freq = _freq(128, cuda)
    args = (c.k[0], c.v[0], c.table, c.len, k, v, None, None, None, freq, None, False, 1.0)
    first = b.append(*args, q, None)
    assert isinstance(first, torch.Tensor) and b.append(*args, None, None) is None
    kept = c.k[0].clone(), c.v[0].clone()
    slow = cast_b200.append_paged(c.k[0], c.v[0], c.table.long(), c.len.tolist(), k, v, inv_freq=freq.double(), q=q)
    assert torch.equal(first, slow) and torch.equal(kept[0], c.k[0]) and torch.equal(kept[1], c.v[0])
    lens = c.len + 1
    one = b.decode(q, c.k[0], c.v[0], c.table, lens, None, 0.0, 0, None, None, None, None)
    assert torch.equal(one, cast_b200.decode_attention_paged(q, c.k[0], c.v[0], c.table, lens.long()))
    cu, packs, par = torch.tensor([0, 2, 3, 3], dtype=torch.int32, device=cuda), [2, 1, 0], [-1, 0, -1]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    many = b.tree(q, c.k[0], c.v[0], c.table, k, v, cu, c.len, i32(packs), None, None, i32(par), 2, 90, None, None)
    slow = cast_b200.varlen_tree_attention_paged(q, c.k[0], c.v[0], c.table, k, v, cu, c.len, packs, parent=par)
    assert torch.equal(many[:3], slow[:3])
    keep, acc = i32([[0, 1], [0, -1], [-1, -1]]), i32([2, 1, 0])
    out = b.append(c.k, c.v, c.table, c.len, [k, k], [v, v], cu, keep, acc, None, None, False, 1.0, None, None)
    assert out is None
    kept = [t.clone() for t in c.k + c.v]
    cast_b200.append_paged(tuple(c.k), tuple(c.v), c.table, c.len, [k, k], [v, v], cu.tolist(), keep=keep, accepted=acc)
    assert all(torch.equal(x, y) for x, y in zip(kept, c.k + c.v)) and _lib.device_error() == 0


def test_refusals_on_the_device(cuda):
    p = torch.zeros(4, 2, 16, 96, dtype=torch.bfloat16, device=cuda)
    table, n = torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 4, 96, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(_lib.CastError, match="head dim"):
        cast_b200.decode_attention_paged(q, p, p, table, n)
    r = p[..., :64]
    q64 = q[..., :64].contiguous()
    for bad in (dict(softcap=-1.0), dict(window=-1), dict(lse=torch.zeros(1, 3, device=cuda)),
                dict(alibi_slopes=torch.zeros(3, device=cuda)), dict(out=q64.float())):
        with pytest.raises(ValueError):
            cast_b200.decode_attention_paged(q64, r, r, table, n, **bad)
    with pytest.raises(ValueError):
        cast_b200.decode_attention_paged(q64, r, r.contiguous(), table, n)          # other strides
    with pytest.raises(ValueError):
        cast_b200.decode_attention_paged(q64.float(), r, r, table, n)
    with pytest.raises(AssertionError):
        cast_b200.decode_attention_paged(q64[:, :3].contiguous(), r, r, table, n)
    k = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=cuda)
    for bad in (dict(q=q64), dict(keep=table), dict(inv_freq=torch.ones(33, device=cuda)), dict(q_out=q64),
                dict(positions=torch.zeros(2, device=cuda))):
        with pytest.raises(ValueError):
            cast_b200.append_paged(r, r, table, n, k, k, **bad)
    with pytest.raises(ValueError):
        cast_b200.append_paged(r, r, table, n, k, k[:, :1])
    with pytest.raises(ValueError):
        cast_b200.varlen_tree_attention_paged(q64, r, r, table, k, k, [0, 1], n, n)
    with pytest.raises(_lib.CastError):
        cast_b200.append_paged(r, r, table[:, :0], n, k, k)
    assert _lib.device_error() == 0
