"""Paged KV cache on MI355X: the rows of several sequences in pages, appended to with RoPE on the way and attended exactly.

The reference's caches hold one sequence in contiguous rows (modal_rd/kv_int8.py, modal_rd/graph_decode.py); this one serves
several of unlike lengths in one call, and a sequence grows without a copy.

Layout: k_pages / v_pages [pages, Hkv, page, d] (bf16 or fp16, page a power of two >= 16, d 64 or 128; any strides between
rows, heads and pages that keep rows 16-byte aligned), table [B, W] int32 (entry w: the page of rows w * page .. of a
sequence; an entry outside 0 .. pages - 1 names no page, and its rows are neither written nor attended), lens [B] int32 (rows
of each sequence, the call's new ones among them), new [B] int32 (how many of the T token columns are real; None: all). Token j
of sequence b is row lens[b] - new[b] + j and attends the rows up to its own. All three are read by the kernels, so a captured
graph follows them.
"""
import functools

import torch

from . import _lib
from .kv_int4 import _copy, _launch_on

_ROWS = (torch.bfloat16, torch.float16)
_FAR = (1 << 31) - 1


# A step of a few tokens is one or two kernels of microseconds, so what depends on shapes, strides and dtypes alone is checked and
# laid out for the library once per such layout; addresses are looked at in every call.
def _layout(x):
    return None if x is None else (x.shape, x.stride(), x.dtype)


def _aligned(layout, rows=8):
    """Whether rows of a layout lie 16 bytes apart (rows: elements of 16 bytes), the last dimension contiguous."""
    s = layout[1]
    return s[-1] == 1 and not any(i % rows for i in s[:-1])


def _strides3(layout):
    s = layout[1]
    return _lib.i64s(s[0], s[1], s[2])


def _check_cache(what, rows, kp, vp, table, lens, new):
    """(heads, pages, page, W) of a call's cache, checked against tokens [B, heads, T, d]; arguments are layouts."""
    (shape, _, dtype), (ps, pst, pd), (vs, vst, vd) = rows, kp, vp
    if len(shape) != 4:
        raise ValueError(f"{what}: rows must be [B, heads, T, d]")
    b, d = shape[0], shape[3]
    if dtype not in _ROWS or pd != dtype or vd != dtype:
        raise ValueError(f"{what}: bf16 or fp16 rows and pages of one dtype required")
    if len(ps) != 4 or ps != vs or ps[3] != d or not ps[0] or not ps[1]:
        raise ValueError(f"{what}: k_pages and v_pages must be [pages, Hkv, page, d] with the rows' d")
    if table[2] != torch.int32 or lens[2] != torch.int32 or (new is not None and new[2] != torch.int32):
        raise ValueError(f"{what}: table, lens and new must be int32")
    if len(table[0]) != 2 or table[0][0] != b or lens[0] != (b,) or (new is not None and new[0] != (b,)):
        raise ValueError(f"{what}: table [B, W], lens [B] and new [B] must match the rows' B")
    if b > 1 and (lens[1][0] != 1 or (new is not None and new[1][0] != 1)) or (table[0][1] > 1 and table[1][1] != 1):
        raise ValueError(f"{what}: table rows, lens and new must be contiguous")
    if not (_aligned(kp) and _aligned(vp)):
        raise ValueError(f"{what}: pages need a contiguous head_dim and 16-byte aligned rows")  # they are used in place
    if max(b, shape[1], shape[2], ps[0], ps[1], table[0][1]) > _FAR:
        raise ValueError(f"{what}: sizes out of range")
    return ps[1], ps[0], ps[2], table[0][1]


def _check_rope(what, cos, sin, b, t, d, dtype):
    """(whether they have to be copied, strides, fp32) of cos, sin [B, T, d] or [T, d]."""
    if cos is None or sin is None:
        if cos is not sin:
            raise ValueError(f"{what}: cos and sin go together")
        return False, None, 0
    f32 = cos[2] == torch.float32
    if cos[2] != sin[2] or not (f32 or cos[2] == dtype):
        raise ValueError(f"{what}: cos and sin must be fp32 or of the rows' dtype")
    strides = []
    for shape, s, _ in (cos, sin):
        if len(shape) == 2:
            shape, s = (1, *shape), (0, *s)
        if len(shape) != 3 or shape[2] != d or any(n != 1 and n != m for n, m in zip(shape, (b, t))):
            raise ValueError(f"{what}: cos and sin must be [B, T, d] or [T, d]")
        strides.append((0 if shape[0] == 1 else s[0], 0 if shape[1] == 1 else s[1], s[2]))
    whole = 4 if f32 else 8
    ok = strides[0] == strides[1] and strides[0][2] == 1 and not any(i % whole for i in strides[0][:2])
    return not ok, _lib.i64s(*strides[0][:2]), int(f32)


def _whole_rope(cos, sin, b, t, d):
    """cos and sin in fresh [B, T, d] memory."""
    return tuple(_copy(x.expand(b, t, d)) for x in (cos, sin))


def _heads_last(shape, like):
    """A fresh tensor [B, h, T, d] in [B, T, h, d] memory (an output projection's order)."""
    b, h, t, d = shape
    return torch.empty_strided((b, h, t, d), (t * h * d, d, h * d, 1), dtype=like.dtype, device=like.device)


def _device_of(what, first, *tensors):
    """The index of the one ROCm device that holds every tensor (the kernels run on the current stream there)."""
    device = first.get_device()
    for x in tensors:
        if x is not None and x.get_device() != device or device < 0:
            _lib.require_gpu(first, *tensors, what=what)
            raise ValueError(f"{what}: tensors on different devices")
    return device


def _check_addresses(what, k_pages, v_pages):
    if (k_pages | v_pages) & 15:
        raise ValueError(f"{what}: pages need a contiguous head_dim and 16-byte aligned rows")


@functools.lru_cache(maxsize=512)
def _append_plan(k, v, kp, vp, table, lens, cos, sin, q, new):
    what = "paged_append"
    if v[0] != k[0] or v[2] != k[2]:
        raise ValueError(f"{what}: k and v must share a shape and dtype")
    hk, pages, page, w = _check_cache(what, k, kp, vp, table, lens, new)
    b, h, t, d = k[0]
    if h != hk or (q is not None and (len(q[0]) != 4 or q[2] != k[2] or (q[0][0], *q[0][2:]) != (b, t, d) or q[0][1] % hk)):
        raise ValueError(f"{what}: k and v [B, Hkv, T, d] and q [B, H, T, d] must match the pages")
    if q is not None and cos is None:
        raise ValueError(f"{what}: q is rotated: cos and sin required")
    copy_rope, sc, f32 = _check_rope(what, cos, sin, b, t, d, k[2])
    heads = 0 if q is None else q[0][1]
    copy = not (_aligned(k) and _aligned(v) and (q is None or _aligned(q))) or copy_rope
    sq = (_strides3(q), _lib.i64s(t * heads * d, d, heads * d)) if heads else (None, None)
    return (copy, _strides3(k), _strides3(v), *sq, sc, f32, _strides3(kp), _strides3(vp), table[1][0],
            (b, t, heads, hk, d, pages, page, w, int(k[2] is torch.float16)))


def paged_append(k, v, k_pages, v_pages, table, lens, cos=None, sin=None, q=None, new=None):
    """The new K / V rows k, v [B, Hkv, T, d] into the pages; with cos, sin ([B, T, d] or [T, d], fp32 or the rows' dtype) k is
    rotated on the way: x cos + (-x[d/2:], x[:d/2]) sin in fp32, rounded once. With q [B, H, T, d] (cos, sin required) returns q
    rotated alike, in [B, T, H, d] memory (padding columns too); else None. Rows that lie outside the table or on no page are
    not written. Two tokens of a call must not share a row."""
    what = "paged_append"
    device = _device_of(what, k, v, k_pages, v_pages, table, lens, cos, sin, q, new)
    (copy, sk, sv, sq, so, sc, f32, skp, svp, st, sizes) = _append_plan(
        _layout(k), _layout(v), _layout(k_pages), _layout(v_pages), _layout(table), _layout(lens), _layout(cos), _layout(sin),
        _layout(q), _layout(new))
    pk, pv, kp, vp = k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    pq, pc, ps = _lib.ptr(q) or 0, _lib.ptr(cos) or 0, _lib.ptr(sin) or 0
    _check_addresses(what, kp, vp)
    if k.numel() == 0:
        return None if q is None else _heads_last(q.shape, q)
    if copy or (pk | pv | pq | pc | ps) & 15:
        if cos is not None:
            cos, sin = _whole_rope(cos, sin, k.shape[0], k.shape[2], k.shape[3])
        return paged_append(_copy(k), _copy(v), k_pages, v_pages, table, lens, cos, sin, None if q is None else _copy(q), new)
    out = None if q is None else _heads_last(q.shape, q)
    _launch_on(device, _lib.lib().bb_paged_append, pk, sk, pv, sv, pq, sq, _lib.ptr(out), so, pc, ps, sc, f32, kp, skp, vp, svp,
               table.data_ptr(), st, lens.data_ptr(), _lib.ptr(new), *sizes, _lib.stream_of(k))
    return out


def _check_queries(what, q, hk):
    b, h, t, d = q[0]
    if h == 0 or hk == 0 or h % hk:
        raise ValueError(f"{what}: q [B, H, T, d] and the pages' Hkv heads must match")
    return b, h, t, d


@functools.lru_cache(maxsize=512)
def _attention_plan(q, kp, vp, table, lens, new):
    what = "paged_attention"
    hk, pages, page, w = _check_cache(what, q, kp, vp, table, lens, new)
    b, h, t, d = _check_queries(what, q, hk)
    ws = _lib.lib().bb_paged_attention_workspace(b, t, h, hk, d, page, w)
    return (not _aligned(q), _strides3(q), _strides3(kp), _strides3(vp), table[1][0],
            (b, t, h, hk, d, pages, page, w, int(q[2] is torch.float16)), _lib.i64s(t * h * d, d, h * d), ws)


def paged_attention(q, k_pages, v_pages, table, lens, scale, new=None):
    """Exact causal attention of q [B, H, T, d] over the pages: token j of a sequence attends the rows up to its own,
    lens - new + j. One token a sequence, a few drafted ones or a chunk of a prompt; sequences of unlike lengths. Returns
    [B, H, T, d] in [B, T, H, d] memory; zeros for padding and where a token attends no row, NaN for a query that is not
    finite."""
    what = "paged_attention"
    device = _device_of(what, q, k_pages, v_pages, table, lens, new)
    copy, sq, skp, svp, st, sizes, so, ws_bytes = _attention_plan(
        _layout(q), _layout(k_pages), _layout(v_pages), _layout(table), _layout(lens), _layout(new))
    pq, kp, vp = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    _check_addresses(what, kp, vp)
    if q.numel() == 0:
        return _heads_last(q.shape, q)
    if copy or pq & 15:
        return paged_attention(_copy(q), k_pages, v_pages, table, lens, scale, new)
    out = _heads_last(q.shape, q)
    ws = _lib.workspace(ws_bytes, q.device) if ws_bytes else None
    _launch_on(device, _lib.lib().bb_paged_attention, pq, sq, kp, skp, vp, svp, table.data_ptr(), st, lens.data_ptr(),
               _lib.ptr(new), *sizes, float(scale), out.data_ptr(), so, _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return out


@functools.lru_cache(maxsize=512)
def _step_plan(q, k, v, kp, vp, table, lens, cos, sin, new):
    what = "paged_step"
    hk, pages, page, w = _check_cache(what, q, kp, vp, table, lens, new)
    b, h, t, d = _check_queries(what, q, hk)
    if k[0] != (b, hk, t, d) or v[0] != k[0] or k[2] != q[2] or v[2] != q[2]:
        raise ValueError(f"{what}: k and v [B, Hkv, T, d] and q [B, H, T, d] must match the pages")
    copy_rope, sc, f32 = _check_rope(what, cos, sin, b, t, d, q[2])
    ws = _lib.lib().bb_paged_step_workspace(b, t, h, hk, d, page, w)
    return (copy_rope or not (_aligned(q) and _aligned(k) and _aligned(v)), _strides3(q), _strides3(k), _strides3(v), sc, f32,
            _strides3(kp), _strides3(vp), table[1][0], (b, t, h, hk, d, pages, page, w, int(q[2] is torch.float16)),
            _lib.i64s(t * h * d, d, h * d), ws)


def paged_step(q, k, v, k_pages, v_pages, table, lens, scale, cos=None, sin=None, new=None):
    """One step: paged_append(k, v, ..., cos, sin, q) and paged_attention of the rotated q, in one call (q and k as they are
    where cos is None). Up to 128 query vectors of a KV head (T * H / Hkv) one kernel does both, and its rotated queries are not
    rounded. Returns [B, H, T, d] in [B, T, H, d] memory."""
    what = "paged_step"
    device = _device_of(what, q, k, v, k_pages, v_pages, table, lens, cos, sin, new)
    copy, sq, sk, sv, sc, f32, skp, svp, st, sizes, so, ws_bytes = _step_plan(
        _layout(q), _layout(k), _layout(v), _layout(k_pages), _layout(v_pages), _layout(table), _layout(lens), _layout(cos),
        _layout(sin), _layout(new))
    pq, pk, pv, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    pc, ps = _lib.ptr(cos) or 0, _lib.ptr(sin) or 0
    _check_addresses(what, kp, vp)
    if q.numel() == 0:
        return _heads_last(q.shape, q)
    if copy or (pq | pk | pv | pc | ps) & 15:
        if cos is not None:
            cos, sin = _whole_rope(cos, sin, q.shape[0], q.shape[2], q.shape[3])
        return paged_step(_copy(q), _copy(k), _copy(v), k_pages, v_pages, table, lens, scale, cos, sin, new)
    out = _heads_last(q.shape, q)
    ws = _lib.workspace(ws_bytes, q.device) if ws_bytes else None
    _launch_on(device, _lib.lib().bb_paged_step, pq, sq, pk, sk, pv, sv, pc, ps, sc, f32, kp, skp, vp, svp, table.data_ptr(), st,
               lens.data_ptr(), _lib.ptr(new), *sizes, float(scale), out.data_ptr(), so, _lib.ptr(ws), ws_bytes,
               _lib.stream_of(q))
    return out
