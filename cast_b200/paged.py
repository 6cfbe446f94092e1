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

A length or page id out of range is skipped on the device and reported by ``_lib.device_error()``; the results of that
sequence are undefined. A workspace serves one call at a time.

Each call first goes to the binding (``csrc/paged_binding.cpp``), which takes arguments that are already as the C ABI
wants them; everything else (conversions, copies, refusals) is done here.
"""
import struct
from functools import lru_cache

import torch

from . import _lib
from .tree_attn import _DTYPES


_INT_MAX = 0x7fffffff       # the C ABI's int; ctypes would pass the low 32 bits of more

# The device and the stream of a call as plain integers: the objects of torch.cuda.current_stream() take 2 us a call,
# a tenth of what a one-token step has.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _launch(index, fn, name, *args):
    """Calls a C entry point on the current stream of device `index` (its last argument), with that device current."""
    if _current_device() == index:
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _raw_stream(index))
    if code:
        _lib.check(code, name)


def _i32(t, index, what, n=None):
    """t as a contiguous int32 tensor on device `index`; n: the entries it must have."""
    if not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t)
    if t.dtype is not torch.int32 or t.get_device() != index or not t.is_contiguous():
        t = t.to(device=index, dtype=torch.int32).contiguous()
    if n is not None and t.numel() != n:
        raise ValueError(f"{what} must have {n} entries, not {tuple(t.shape)}")
    return t


def _table(page_table, index):
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
        raise ValueError("page_table must be a tensor [B, pages of a sequence]")
    if page_table.dtype is not torch.int32 or page_table.get_device() != index or page_table.stride(1) != 1:
        page_table = page_table.to(device=index, dtype=torch.int32).contiguous()
    return page_table


def _pages(k_pages, v_pages, name):
    """Checks the pages of one layer: [num_pages, H_kv, page_size, D], K and V alike. Returns what they share."""
    if not k_pages.is_cuda:
        raise RuntimeError(f"cast_b200.{name} needs CUDA tensors (no CPU path)")
    shape, stride, dtype, index = k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.get_device()
    if len(shape) != 4 or stride[3] != 1 or dtype not in _DTYPES:
        raise ValueError(f"{name}: pages are [num_pages, H_kv, page_size, D] of float32, bfloat16 or float16, "
                         "dim stride 1")
    if v_pages.shape != shape or v_pages.stride() != stride or v_pages.dtype is not dtype or v_pages.get_device() != index:
        raise ValueError(f"{name}: K and V pages need one shape, one dtype, one device and the same strides")
    num_pages, H, ps, D = shape
    if ps > _INT_MAX or H > _INT_MAX:
        raise ValueError(f"{name}: too many heads, or rows of a page")
    return (min(num_pages, _INT_MAX), H, ps, D), stride, dtype, index      # ids, and so reachable pages, are int32


def _scale(sm_scale, name):
    """The scale for the C ABI, which takes what is not positive as 1/sqrt(D): only None means that here."""
    if sm_scale is None:
        return 0.0
    if not 1e-30 <= sm_scale <= 1e30:
        raise ValueError(f"{name}: sm_scale must be positive (1e-30 to 1e30)")
    return sm_scale


def _aligned(stride, ptr):
    """What the attention kernels take: dim stride 1, row / head strides multiples of 4 (not 0), a 16-byte aligned base."""
    s0, s1, s2 = stride
    return s2 == 1 and s0 % 4 == 0 and s1 % 4 == 0 and ptr % 16 == 0 and s0 > 0 and s1 > 0


def _input(t):
    """t as the kernels take it (a copy where it is not), its strides and its address."""
    stride, ptr = t.stride(), t.data_ptr()
    if not _aligned(stride, ptr):
        t = t.contiguous()
        stride, ptr = t.stride(), t.data_ptr()
    return t, stride, ptr


def _output(out, q, shape, dtype, index):
    """The given or a new output, its strides and its address."""
    if out is None:
        out = torch.empty_like(q)
        return out, out.stride(), out.data_ptr()
    stride, ptr = out.stride(), out.data_ptr()
    if out.shape != shape or out.dtype is not dtype or out.get_device() != index or not _aligned(stride, ptr):
        raise ValueError("out must be like q: dim stride 1, row/head strides multiple of 4, 16-byte aligned base")
    return out, stride, ptr


@lru_cache(maxsize=256)
def _decode_bytes(index, *args):
    """cast_paged_decode_workspace_size on device `index` (its SM count plays a part)."""
    with torch.cuda.device(index):
        return _lib.lib().cast_paged_decode_workspace_size(*args)


def _tree_bytes(index, *args):
    if _current_device() == index:
        return _lib.lib().cast_tree_attn_paged_workspace_size(*args)
    with torch.cuda.device(index):
        return _lib.lib().cast_tree_attn_paged_workspace_size(*args)


def _workspace(workspace, n, index):
    """The caller's workspace where it is large enough, one piece and on device `index`, else a new one (None: nothing is
    needed). A view with gaps or repeats has other, or fewer, bytes behind its address than it counts."""
    if n == 0:
        return None
    if workspace is None or workspace.nbytes < n or workspace.data_ptr() % 256 or workspace.get_device() != index \
            or not workspace.is_contiguous():
        return torch.empty(n, dtype=torch.uint8, device=index)
    return workspace


_P2 = struct.Struct("2P").pack
# int64 arguments packed into bytes, which ctypes passes by address: a fourth of the time of a ctypes array
_I4, _I6, _I7, _I11 = (struct.Struct(f"{n}q").pack for n in (4, 6, 7, 11))


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
    done = (_lib._BINDING or _lib.binding()).append(k_pages, v_pages, page_table, seq_len, k, v, cu_q, keep, accepted,
                                                    inv_freq, positions, interleaved, rope_scale, q, q_out)
    if done is not NotImplemented:
        return done
    many = isinstance(k_pages, (list, tuple))
    kps, vps, ks, vs = (k_pages, v_pages, k, v) if many else ((k_pages,), (v_pages,), (k,), (v,))
    n = len(kps)
    if not n == len(vps) == len(ks) == len(vs):
        raise ValueError("append_paged: one K and one V of pages and of new rows per layer")
    if n == 0:
        return None
    (num_pages, H, ps, D), sp, dtype, index = _pages(kps[0], vps[0], "append_paged")
    shape = kps[0].shape
    rows, sk, sv = ks[0].shape, ks[0].stride(), vs[0].stride()
    if len(rows) != 3 or rows[1] != H or rows[2] != D or sk[2] != 1 or sv[2] != 1:
        raise ValueError("append_paged: new rows are [total, H_kv, D] of the pages' dtype and device, dim stride 1")
    pages, new = [], []
    for i in range(n):
        kp, vp, a, b = kps[i], vps[i], ks[i], vs[i]
        if i and (kp.shape != shape or vp.shape != shape or kp.stride() != sp or vp.stride() != sp
                  or kp.dtype is not dtype or vp.dtype is not dtype or kp.get_device() != index or vp.get_device() != index):
            raise ValueError("append_paged: every layer's pages need one shape, one dtype and the same strides")
        if a.shape != rows or b.shape != rows or a.dtype is not dtype or b.dtype is not dtype or a.get_device() != index \
                or b.get_device() != index:
            raise ValueError("append_paged: new rows are [total, H_kv, D] of the pages' dtype and device, dim stride 1")
        if i and (a.stride() != sk or b.stride() != sv):
            raise ValueError("append_paged: every layer's new rows need the same strides")
        pages += (kp.data_ptr(), vp.data_ptr())
        new += (a.data_ptr(), b.data_ptr())
    total = rows[0]
    table = _table(page_table, index)
    B, width = table.shape[0], min(table.shape[1], _INT_MAX)
    seq_len = _i32(seq_len, index, "seq_len", B)
    p_cu = p_keep = p_acc = p_pos = p_freq = p_q = p_qo = qs = None
    w = n_freq = Hq = 0
    if cu_q is not None:
        cu_q = _i32(cu_q, index, "cu_q", B + 1)
        p_cu = cu_q.data_ptr()
    if keep is not None or accepted is not None:
        if keep is None or accepted is None or cu_q is None:
            raise ValueError("append_paged: keep, accepted and cu_q go together")
        keep = _i32(keep, index, "keep")
        accepted = _i32(accepted, index, "accepted", B)
        if keep.dim() != 2 or keep.shape[0] != B:
            raise ValueError("append_paged: keep must be [B, w]")
        w, p_keep, p_acc = keep.shape[1], keep.data_ptr(), accepted.data_ptr()
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float32 or inv_freq.get_device() != index or not inv_freq.is_contiguous():
            inv_freq = inv_freq.to(device=index, dtype=torch.float32).contiguous()
        n_freq = inv_freq.numel()
        p_freq = inv_freq.data_ptr()
        if 2 * n_freq > D:
            raise ValueError("append_paged: inv_freq has more pairs than half a head")
    if positions is not None:
        positions = _i32(positions, index, "positions", total)
        p_pos = positions.data_ptr()
    if q is not None:
        if n > 1 or keep is not None or n_freq == 0:
            raise ValueError("append_paged: q goes with one layer and inv_freq, and not with keep")
        s, shape_q = q.stride(), q.shape
        if len(shape_q) != 3 or shape_q[0] != total or shape_q[2] != D or q.dtype is not dtype or q.get_device() != index or s[2] != 1:
            raise ValueError("append_paged: q must be [total, H_q, D] of the pages' dtype and device, dim stride 1")
        if q_out is None:
            q_out = torch.empty_like(q)
        o = q_out.stride()
        if q_out.shape != shape_q or q_out.dtype is not dtype or q_out.get_device() != index or o[2] != 1 \
                or (o[0] == 0 and total > 1) or (o[1] == 0 and shape_q[1] > 1):
            raise ValueError("append_paged: q_out must be like q, dim stride 1, rows and heads apart")
        Hq, p_q, p_qo, qs = shape_q[1], q.data_ptr(), q_out.data_ptr(), _I4(s[0], s[1], o[0], o[1])
    elif q_out is not None:
        raise ValueError("append_paged: q_out without q")
    ptrs = struct.Struct(f"{2 * n}P").pack if n > 1 else _P2
    _launch(index, _lib.lib().cast_paged_append, "cast_paged_append", n, ptrs(*pages), ptrs(*new), _DTYPES[dtype], H,
            D, num_pages, ps, _I6(sp[0], sp[1], sp[2], sp[0], sp[1], sp[2]), total, _I4(sk[0], sk[1], sv[0], sv[1]),
            table.data_ptr(), table.stride(0), width, seq_len.data_ptr(), B, p_cu, p_keep, w, p_acc, p_pos, p_freq,
            n_freq, interleaved, rope_scale, p_q, p_qo, Hq, qs)
    return q_out


def decode_workspace_size(dtype, B, H_q, H_kv, D):
    """Bytes of workspace decode_attention_paged needs; independent of the lengths and of the cache."""
    return int(_lib.lib().cast_paged_decode_workspace_size(_DTYPES[dtype], B, H_q, H_kv, D))


def decode_attention_paged(q, k_pages, v_pages, page_table, seq_len, sm_scale=None, *, softcap=0.0, window=0,
                           alibi_slopes=None, out=None, lse=None, workspace=None):
    """Attention of one new token per sequence over its pages: q [B, H_q, D] -> [B, H_q, D].

    seq_len: int32 [B], the keys of each sequence, the new token's own among them (0: the row becomes 0).
    Scores are q . k * sm_scale (positive; default 1/sqrt(D)); ``softcap`` > 0 caps them (softcap * tanh(s / softcap));
    ``alibi_slopes`` (float32 [H_q]) then adds slope * (key position - newest position); ``window`` > 0 keeps the
    last ``window`` keys. ``lse`` (float32 [B, H_q], contiguous) receives the natural log-sum-exp of the scores.
    float32, bfloat16 or float16, D 64 or 128, any H_q / H_kv. The key ranges of all sequences are split evenly
    over the GPU, whatever their lengths; results do not depend on timing.
    """
    done = (_lib._BINDING or _lib.binding()).decode(q, k_pages, v_pages, page_table, seq_len, sm_scale, softcap, window,
                                                    alibi_slopes, out, lse, workspace)
    if done is not NotImplemented:
        return done
    (num_pages, H_kv, ps, D), sp, dtype, index = _pages(k_pages, v_pages, "decode_attention_paged")
    shape = q.shape
    if len(shape) != 3 or shape[2] != D or q.dtype is not dtype or q.get_device() != index:
        raise ValueError("decode_attention_paged: q must be [B, H_q, D] of the pages' dtype and device")
    B, H_q, _ = shape
    assert H_q % H_kv == 0
    table = _table(page_table, index)
    rows, width = table.shape[0], min(table.shape[1], _INT_MAX)
    if rows != B:
        raise ValueError("decode_attention_paged: page_table must have one row per sequence")
    seq_len = _i32(seq_len, index, "seq_len", B)
    if window < 0 or not (softcap == 0.0 or 1e-6 <= softcap <= 1e30):
        raise ValueError("decode_attention_paged: window must not be negative, softcap 0 or 1e-6 to 1e30")
    sm_scale = _scale(sm_scale, "decode_attention_paged")
    q, sq, p_q = _input(q)
    out, so, p_out = _output(out, q, shape, dtype, index)
    p_slopes = p_lse = None
    if alibi_slopes is not None:
        if alibi_slopes.dtype is not torch.float32 or alibi_slopes.get_device() != index or not alibi_slopes.is_contiguous():
            alibi_slopes = alibi_slopes.to(device=index, dtype=torch.float32).contiguous()
        if alibi_slopes.shape != (H_q,):
            raise ValueError("alibi_slopes must be [H_q]")
        p_slopes = alibi_slopes.data_ptr()
    if lse is not None:
        if lse.shape != (B, H_q) or lse.dtype is not torch.float32 or lse.get_device() != index or not lse.is_contiguous():
            raise ValueError("lse must be a contiguous float32 [B, H_q]")
        p_lse = lse.data_ptr()
    code = _DTYPES[dtype]
    n = _decode_bytes(index, code, B, H_q, H_kv, D)
    workspace = _workspace(workspace, n, index)
    _launch(index, _lib.lib().cast_paged_decode_attn, "cast_paged_decode_attn", p_q, k_pages.data_ptr(),
            v_pages.data_ptr(), p_out, p_lse, code, _I7(sq[0], sq[1], sp[0], sp[1], sp[2], so[0], so[1]),
            table.data_ptr(), table.stride(0), width, seq_len.data_ptr(), B, H_q, H_kv, D, num_pages, ps,
            sm_scale, softcap, min(window, _INT_MAX), p_slopes,
            None if workspace is None else workspace.data_ptr(), n)
    return out


def varlen_tree_attention_paged(q, k_pages, v_pages, page_table, k_pack, v_pack, cu_q, prefix_len, pack_len,
                                ancestor_mask=None, sm_scale=None, *, parent=None, max_pack=None, max_prefix=None,
                                out=None, workspace=None):
    """varlen_tree_attention_store with each request's prefix in a paged cache.

    q: [total_q, H_q, D]; request b's prefix is keys [0, prefix_len[b]) of its pages; k_pack / v_pack:
    [total_q, H_kv, D], this pass's keys and values in pack order. Output, masks and conventions as
    varlen_tree_attention. bfloat16 / float16 with H_q / H_kv <= 128 run on the tensor cores straight from the
    pages, whatever their size; float32 on the exact CUDA-core kernel (the store form's fp32_path="exact"; its split path
    has no form on pages). D 64 or 128. max_pack / max_prefix bound pack_len and prefix_len; given, the call reads nothing
    back to the host. The keys are split for max_prefix: a bound far above the lengths costs short prefixes time.
    """
    done = (_lib._BINDING or _lib.binding()).tree(q, k_pages, v_pages, page_table, k_pack, v_pack, cu_q, prefix_len,
                                                  pack_len, ancestor_mask, sm_scale, parent, max_pack, max_prefix, out,
                                                  workspace)
    if done is not NotImplemented:
        return done
    (num_pages, H_kv, ps, D), sp, dtype, index = _pages(k_pages, v_pages, "varlen_tree_attention_paged")
    shape = q.shape
    total_q, H_q, _ = shape
    assert H_q % H_kv == 0
    if shape[2] != D or k_pack.shape != (total_q, H_kv, D) or v_pack.shape != k_pack.shape or q.dtype is not dtype \
            or k_pack.dtype is not dtype or v_pack.dtype is not dtype or q.get_device() != index or k_pack.get_device() != index \
            or v_pack.get_device() != index:
        raise ValueError("q must be [total_q, H_q, D] and the packs [total_q, H_kv, D], of the pages' dtype and device")
    if (ancestor_mask is None) == (parent is None):
        raise ValueError("pass exactly one of ancestor_mask and parent")
    table = _table(page_table, index)
    B, width = table.shape[0], min(table.shape[1], _INT_MAX)
    cu_q = _i32(cu_q, index, "cu_q", B + 1)
    prefix_len, pack_len = _i32(prefix_len, index, "prefix_len", B), _i32(pack_len, index, "pack_len", B)
    if max_pack is None:
        max_pack = int(pack_len.max().item()) if B > 0 else 0
    if max_prefix is None:
        max_prefix = int(prefix_len.max().item()) if B > 0 else 0
    if max(total_q, max_pack, max_prefix) > _INT_MAX:
        raise ValueError("varlen_tree_attention_paged: total_q, max_pack and max_prefix must be below 2^31")
    sm_scale = _scale(sm_scale, "varlen_tree_attention_paged")
    q, sq, p_q = _input(q)
    k_pack, sk, p_k = _input(k_pack)
    v_pack, sv, p_v = _input(v_pack)
    out, so, p_out = _output(out, q, shape, dtype, index)
    anc_ptr, wpr, par_ptr = None, 0, None
    if ancestor_mask is not None:
        anc = ancestor_mask
        if not isinstance(anc, torch.Tensor) or anc.dtype is not torch.int64 or anc.get_device() != index or not anc.is_contiguous():
            anc = torch.as_tensor(anc, device=torch.device("cuda", index)).to(torch.int64).contiguous()
        wpr = anc.numel() // max(total_q, 1)
        if anc.numel() != wpr * total_q:
            raise ValueError("ancestor_mask must be [total_q] or [total_q, words]")
        anc_ptr = anc.data_ptr()
    else:
        parent = _i32(parent, index, "parent", total_q)
        par_ptr = parent.data_ptr()
    code = _DTYPES[dtype]
    n = _tree_bytes(index, code, B, total_q, H_q, H_kv, D, max_pack, max_prefix)
    workspace = _workspace(workspace, n, index)
    _launch(index, _lib.lib().cast_tree_attn_paged_fwd, "cast_tree_attn_paged_fwd", p_q, k_pages.data_ptr(),
            v_pages.data_ptr(), p_k, p_v, p_out, code,
            _I11(sq[0], sq[1], sp[0], sp[1], sp[2], sk[0], sk[1], sv[0], sv[1], so[0], so[1]), table.data_ptr(),
            table.stride(0), width, cu_q.data_ptr(), prefix_len.data_ptr(), pack_len.data_ptr(), anc_ptr, wpr, par_ptr,
            B, total_q, num_pages, ps, H_q, H_kv, D, sm_scale, max_pack, max_prefix,
            None if workspace is None else workspace.data_ptr(), n)
    return out
