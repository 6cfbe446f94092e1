"""Paged key-value cache: append with rotation, one-token decode attention, tree attention.

Keys and values of a layer are pages ``[num_pages, H_kv, page_size, D]`` (any page size, heads and rows in
either order: pass the permuted view); key n of sequence b is row ``n % page_size`` of page
``page_table[b, n // page_size]`` (int32). The calls read lengths and table on the device: nothing is copied to
the host, so they can be captured into a CUDA graph when ``out`` / ``q_out`` and ``workspace`` are given.

A serving step on such a cache::

    q = append_paged(k_pages, v_pages, table, length, k, v, inv_freq=inv_freq, q=q)     # slot = length[b]
    out = decode_attention_paged(q, k_pages, v_pages, table, length + 1)

and a verify round of draft trees, whose accepted rows are appended for every layer at once::

    out = varlen_tree_attention_paged(q, k_pages, v_pages, table, k_pack, v_pack, cu_q, length, pack_len,
                                      parent=trees.pack_parent, max_pack=..., max_prefix=...)   # per layer
    walk = walk_trees_greedy(...)
    append_paged(all_k_pages, all_v_pages, table, length, all_k_packs, all_v_packs, cu_q, keep=walk.keep,
                 accepted=walk.accepted)

A length or page id out of range is skipped on the device and reported by ``_lib.device_error()``.
"""
import ctypes
import math

import torch

from . import _lib
from .tree_attn import _DTYPES, _kernel_ready, _prep


def _launch(dev, fn, name, *args):
    """Calls a C entry point on dev's current stream (its last argument), with dev current."""
    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        code = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            code = fn(*args, stream)
    if code:
        _lib.check(code, name)


def _i32(t, dev, what, shape=None):
    if not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t)
    if t.dtype is not torch.int32 or t.device != dev or not t.is_contiguous():
        t = t.to(device=dev, dtype=torch.int32).contiguous()
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    return t


def _table(page_table, dev):
    if page_table.dim() != 2:
        raise ValueError("page_table must be [B, pages of a sequence]")
    if page_table.dtype is not torch.int32 or page_table.device != dev or page_table.stride(1) != 1:
        page_table = page_table.to(device=dev, dtype=torch.int32).contiguous()
    return page_table


def _pages(k_pages, v_pages, name):
    """The checked pages of one layer: [num_pages, H_kv, page_size, D], K and V alike."""
    if not k_pages.is_cuda:
        raise RuntimeError(f"cast_b200.{name} needs CUDA tensors (no CPU path)")
    if k_pages.dim() != 4 or k_pages.stride(3) != 1 or k_pages.dtype not in _DTYPES:
        raise ValueError(f"{name}: pages are [num_pages, H_kv, page_size, D] of float32, bfloat16 or float16, "
                         "dim stride 1")
    if v_pages.shape != k_pages.shape or v_pages.stride() != k_pages.stride() or v_pages.dtype != k_pages.dtype \
            or v_pages.device != k_pages.device:
        raise ValueError(f"{name}: K and V pages need one shape, one dtype, one device and the same strides")


def _ptrs(ks, vs):
    return (ctypes.c_void_p * (2 * len(ks)))(*[t.data_ptr() for kv in zip(ks, vs) for t in kv])


def append_paged(k_pages, v_pages, page_table, seq_len, k, v, cu_q=None, *, keep=None, accepted=None, inv_freq=None,
                 positions=None, interleaved=False, rope_scale=1.0, q=None, q_out=None):
    """Append new key and value rows to a paged cache, keys (and queries) rotated on the way; one launch.

    k_pages / v_pages: one layer's pages, or lists of every layer's; k / v: [total, H_kv, D], or lists. With
    seq_len [B] the lengths before the call (left as they are: the caller adds what it appended):

    * ``cu_q`` None: row b goes to slot seq_len[b] of sequence b.
    * ``cu_q`` [B + 1]: rows cu_q[b] + j go to seq_len[b] + j. Rows behind cu_q[B] are left out.
    * ``keep`` [B, w] and ``accepted`` [B] as well (a Walk's): rows cu_q[b] + keep[b, j], j < accepted[b].

    inv_freq: float32 [rotated pairs]. Pair i of a key (elements i and i + len(inv_freq), or 2i and 2i + 1 when
    ``interleaved``) turns by position * inv_freq[i] (the angle in 64 bits) and is scaled by ``rope_scale``; the
    position is the slot, or ``positions`` [total]. q: [total, H_q, D], turned likewise into ``q_out`` (a new
    tensor unless given; may be q itself), which is returned. Rows that are not appended are not written.
    """
    many = isinstance(k_pages, (list, tuple))
    kps, vps, ks, vs = (k_pages, v_pages, k, v) if many else ((k_pages,), (v_pages,), (k,), (v,))
    if not len(kps) == len(vps) == len(ks) == len(vs):
        raise ValueError("append_paged: one K and one V of pages and of new rows per layer")
    if len(kps) == 0:
        return None
    kp, k0, v0 = kps[0], ks[0], vs[0]
    for a, b in zip(kps, vps):
        _pages(a, b, "append_paged")
        if a is not kp and (a.shape != kp.shape or a.stride() != kp.stride() or a.dtype != kp.dtype or a.device != kp.device):
            raise ValueError("append_paged: every layer's pages need one shape, one dtype and the same strides")
    num_pages, H, ps, D = kp.shape
    dev = kp.device
    for t in (*ks, *vs):
        if t.dim() != 3 or t.shape != k0.shape or t.shape[1] != H or t.shape[2] != D or t.dtype != kp.dtype \
                or t.device != dev or t.stride(2) != 1:
            raise ValueError("append_paged: new rows are [total, H_kv, D] of the pages' dtype and device, dim stride 1")
    for a, b in zip(ks, vs):
        if a.stride() != k0.stride() or b.stride() != v0.stride():
            raise ValueError("append_paged: every layer's new rows need the same strides")
    total = k0.shape[0]
    table = _table(page_table, dev)
    B = table.shape[0]
    seq_len = _i32(seq_len, dev, "seq_len", (B,))
    if cu_q is not None:
        cu_q = _i32(cu_q, dev, "cu_q", (B + 1,))
    if (keep is None) != (accepted is None) or (keep is not None and cu_q is None):
        raise ValueError("append_paged: keep, accepted and cu_q go together")
    w = 0
    if keep is not None:
        keep = _i32(keep, dev, "keep")
        accepted = _i32(accepted, dev, "accepted", (B,))
        if keep.dim() != 2 or keep.shape[0] != B:
            raise ValueError("append_paged: keep must be [B, w]")
        w = keep.shape[1]
    n_freq = 0
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float32 or inv_freq.device != dev or not inv_freq.is_contiguous():
            inv_freq = inv_freq.to(device=dev, dtype=torch.float32).contiguous()
        n_freq = inv_freq.numel()
        if 2 * n_freq > D:
            raise ValueError("append_paged: inv_freq has more pairs than half a head")
    if positions is not None:
        positions = _i32(positions, dev, "positions", (total,))
    qs, Hq = None, 0
    if q is not None:
        if many or keep is not None or n_freq == 0:
            raise ValueError("append_paged: q goes with one layer and inv_freq, and not with keep")
        if q.dim() != 3 or q.shape[0] != total or q.shape[2] != D or q.dtype != kp.dtype or q.device != dev \
                or q.stride(2) != 1:
            raise ValueError("append_paged: q must be [total, H_q, D] of the pages' dtype and device, dim stride 1")
        if q_out is None:
            q_out = torch.empty_like(q)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.device != dev or q_out.stride(2) != 1:
            raise ValueError("append_paged: q_out must be like q, dim stride 1")
        Hq = q.shape[1]
        s, o = q.stride(), q_out.stride()
        qs = (ctypes.c_int64 * 4)(s[0], s[1], o[0], o[1])
    elif q_out is not None:
        raise ValueError("append_paged: q_out without q")
    sp, sk, sv = kp.stride(), k0.stride(), v0.stride()
    _launch(dev, _lib.lib().cast_paged_append, "cast_paged_append", len(kps), _ptrs(kps, vps), _ptrs(ks, vs),
            _DTYPES[kp.dtype], H, D, num_pages, ps, (ctypes.c_int64 * 6)(*sp[:3], *sp[:3]), total,
            (ctypes.c_int64 * 4)(sk[0], sk[1], sv[0], sv[1]), table.data_ptr(), table.stride(0), table.shape[1],
            seq_len.data_ptr(), B, None if cu_q is None else cu_q.data_ptr(), None if keep is None else keep.data_ptr(),
            w, None if accepted is None else accepted.data_ptr(), None if positions is None else positions.data_ptr(),
            inv_freq.data_ptr() if n_freq else None, n_freq, 1 if interleaved else 0, float(rope_scale),
            None if q is None else q.data_ptr(), None if q is None else q_out.data_ptr(), Hq, qs)
    return q_out


def decode_workspace_size(dtype, B, H_q, H_kv, D):
    """Bytes of workspace decode_attention_paged needs; independent of the lengths and of the cache."""
    return int(_lib.lib().cast_paged_decode_workspace_size(_DTYPES[dtype], B, H_q, H_kv, D))


def decode_attention_paged(q, k_pages, v_pages, page_table, seq_len, sm_scale=None, *, softcap=0.0, window=0,
                           alibi_slopes=None, out=None, lse=None, workspace=None):
    """Attention of one new token per sequence over its pages: q [B, H_q, D] -> [B, H_q, D].

    seq_len: int32 [B], the keys of each sequence, the new token's own among them (0: the row becomes 0).
    Scores are q . k * sm_scale (default 1/sqrt(D)); ``softcap`` > 0 caps them (softcap * tanh(s / softcap));
    ``alibi_slopes`` (float32 [H_q]) then adds slope * (key position - newest position); ``window`` > 0 keeps the
    last ``window`` keys. ``lse`` (float32 [B, H_q], contiguous) receives the natural log-sum-exp of the scores.
    float32, bfloat16 or float16, D 64 or 128, any H_q / H_kv. The key ranges of all sequences are split evenly
    over the GPU, whatever their lengths; results do not depend on timing.
    """
    _pages(k_pages, v_pages, "decode_attention_paged")
    dev = k_pages.device
    num_pages, H_kv, ps, D = k_pages.shape
    if q.dim() != 3 or q.shape[2] != D or q.dtype != k_pages.dtype or q.device != dev:
        raise ValueError("decode_attention_paged: q must be [B, H_q, D] of the pages' dtype and device")
    B, H_q, _ = q.shape
    assert H_q % H_kv == 0
    table = _table(page_table, dev)
    seq_len = _i32(seq_len, dev, "seq_len", (B,))
    if table.shape[0] != B:
        raise ValueError("decode_attention_paged: page_table must have one row per sequence")
    if window < 0 or not softcap >= 0.0:
        raise ValueError("decode_attention_paged: window and softcap must not be negative")
    q = _prep(q)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not _kernel_ready(out):
        raise ValueError("out must be like q: dim stride 1, row/head strides multiple of 4, 16-byte aligned base")
    if alibi_slopes is not None:
        if alibi_slopes.dtype is not torch.float32 or alibi_slopes.device != dev or not alibi_slopes.is_contiguous():
            alibi_slopes = alibi_slopes.to(device=dev, dtype=torch.float32).contiguous()
        if alibi_slopes.shape != (H_q,):
            raise ValueError("alibi_slopes must be [H_q]")
    if lse is not None and (lse.shape != (B, H_q) or lse.dtype is not torch.float32 or lse.device != dev
                            or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous float32 [B, H_q]")
    L, code = _lib.lib(), _DTYPES[q.dtype]
    n = L.cast_paged_decode_workspace_size(code, B, H_q, H_kv, D)
    if workspace is None or workspace.numel() * workspace.element_size() < n or workspace.data_ptr() % 256:
        workspace = torch.empty(n, dtype=torch.uint8, device=dev)
    sq, sp, so = q.stride(), k_pages.stride(), out.stride()
    _launch(dev, L.cast_paged_decode_attn, "cast_paged_decode_attn", q.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), code,
            (ctypes.c_int64 * 7)(sq[0], sq[1], sp[0], sp[1], sp[2], so[0], so[1]), table.data_ptr(), table.stride(0),
            table.shape[1], seq_len.data_ptr(), B, H_q, H_kv, D, num_pages, ps,
            0.0 if sm_scale is None else float(sm_scale), float(softcap), int(window),
            None if alibi_slopes is None else alibi_slopes.data_ptr(), workspace.data_ptr(), n)
    return out


def varlen_tree_attention_paged(q, k_pages, v_pages, page_table, k_pack, v_pack, cu_q, prefix_len, pack_len,
                                ancestor_mask=None, sm_scale=None, *, parent=None, max_pack=None, max_prefix=None,
                                out=None, workspace=None):
    """varlen_tree_attention_store with each request's prefix in a paged cache.

    q: [total_q, H_q, D]; request b's prefix is keys [0, prefix_len[b]) of its pages; k_pack / v_pack:
    [total_q, H_kv, D], this pass's keys and values in pack order. Output, masks and conventions as
    varlen_tree_attention. bfloat16 / float16 with D = 128 and H_q / H_kv dividing 128 run on the tensor cores
    straight from the pages, whatever their size; float32 and other head shapes on the exact CUDA-core kernel.
    max_pack / max_prefix bound pack_len and prefix_len; given, the call reads nothing back to the host.
    """
    _pages(k_pages, v_pages, "varlen_tree_attention_paged")
    dev = k_pages.device
    num_pages, H_kv, ps, D = k_pages.shape
    total_q, H_q, _ = q.shape
    assert H_q % H_kv == 0
    for t, h in ((q, H_q), (k_pack, H_kv), (v_pack, H_kv)):
        if t.shape != (total_q, h, D) or t.dtype != k_pages.dtype or t.device != dev:
            raise ValueError("q must be [total_q, H_q, D] and the packs [total_q, H_kv, D], of the pages' dtype and device")
    if (ancestor_mask is None) == (parent is None):
        raise ValueError("pass exactly one of ancestor_mask and parent")
    table = _table(page_table, dev)
    B = table.shape[0]
    cu_q = _i32(cu_q, dev, "cu_q", (B + 1,))
    prefix_len, pack_len = _i32(prefix_len, dev, "prefix_len", (B,)), _i32(pack_len, dev, "pack_len", (B,))
    if max_pack is None:
        max_pack = int(pack_len.max().item()) if B > 0 else 0
    if max_prefix is None:
        max_prefix = int(prefix_len.max().item()) if B > 0 else 0
    q, k_pack, v_pack = _prep(q), _prep(k_pack), _prep(v_pack)
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not _kernel_ready(out):
        raise ValueError("out must be like q: dim stride 1, row/head strides multiple of 4, 16-byte aligned base")
    anc_ptr, wpr, par_ptr = None, 0, None
    if ancestor_mask is not None:
        anc = torch.as_tensor(ancestor_mask, device=dev).to(torch.int64).reshape(total_q, -1).contiguous()
        anc_ptr, wpr = anc.data_ptr(), anc.shape[1]
    else:
        par = _i32(parent, dev, "parent", (total_q,))
        par_ptr = par.data_ptr()
    L, code = _lib.lib(), _DTYPES[q.dtype]
    n = L.cast_tree_attn_paged_workspace_size(code, B, total_q, H_q, H_kv, D, max_pack, max_prefix)
    if n > 0 and (workspace is None or workspace.numel() * workspace.element_size() < n or workspace.data_ptr() % 256):
        workspace = torch.empty(n, dtype=torch.uint8, device=dev)
    sq, sp, sk, sv, so = q.stride(), k_pages.stride(), k_pack.stride(), v_pack.stride(), out.stride()
    _launch(dev, L.cast_tree_attn_paged_fwd, "cast_tree_attn_paged_fwd", q.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), k_pack.data_ptr(), v_pack.data_ptr(), out.data_ptr(), code,
            (ctypes.c_int64 * 11)(sq[0], sq[1], sp[0], sp[1], sp[2], sk[0], sk[1], sv[0], sv[1], so[0], so[1]),
            table.data_ptr(), table.stride(0), table.shape[1], cu_q.data_ptr(), prefix_len.data_ptr(),
            pack_len.data_ptr(), anc_ptr, wpr, par_ptr, B, total_q, num_pages, ps, H_q, H_kv, D,
            0.0 if sm_scale is None else float(sm_scale), int(max_pack), int(max_prefix),
            workspace.data_ptr() if n > 0 else None, n)
    return out
