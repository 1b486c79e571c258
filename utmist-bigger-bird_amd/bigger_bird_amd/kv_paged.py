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
from .kv_int4 import _copy, _launch_on, _one_device, _strides

_ROWS = (torch.bfloat16, torch.float16)


def _aligned(x, rows=8):
    """x [B, h, T, d] (cos, sin: [B, T, d]) with a contiguous last dimension and 16-byte aligned rows (a copy where it is not).
    rows: elements of 16 bytes."""
    s = x.stride()
    if s[-1] == 1 and x.data_ptr() % 16 == 0 and not any(i % rows for i in s[:-1]):
        return x
    return _copy(x)


def _cache(what, k_pages, v_pages, table, lens, new, shape, dtype):
    """(heads, pages, page, W) of a call's cache, checked against tokens [B, heads, T, d] of `dtype`."""
    b, _, _, d = shape
    if dtype not in _ROWS or k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise ValueError(f"{what}: bf16 or fp16 rows and pages of one dtype required")
    if k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] != d:
        raise ValueError(f"{what}: k_pages and v_pages must be [pages, Hkv, page, d] with the rows' d")
    if table.dtype != torch.int32 or lens.dtype != torch.int32 or (new is not None and new.dtype != torch.int32):
        raise ValueError(f"{what}: table, lens and new must be int32")
    if (table.ndim != 2 or table.shape[0] != b or lens.shape != (b,) or (new is not None and new.shape != (b,))):
        raise ValueError(f"{what}: table [B, W], lens [B] and new [B] must match the rows' B")
    if (b > 1 and (lens.stride(0) != 1 or (new is not None and new.stride(0) != 1))) or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{what}: table rows, lens and new must be contiguous")
    for x in (k_pages, v_pages):
        s = x.stride()
        if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or x.data_ptr() % 16:
            raise ValueError(f"{what}: pages need a contiguous head_dim and 16-byte aligned rows")  # they are written in place
    p, hk, page, _ = k_pages.shape
    return hk, p, page, table.shape[1]


def _rope(what, cos, sin, b, t, d, dtype):
    """cos, sin [B, T, d] or [T, d] as (cos, sin, strides, fp32)."""
    if cos is None or sin is None:
        if cos is not sin:
            raise ValueError(f"{what}: cos and sin go together")
        return None, None, None, 0
    f32 = cos.dtype == torch.float32
    if cos.dtype != sin.dtype or not (f32 or cos.dtype == dtype):
        raise ValueError(f"{what}: cos and sin must be fp32 or of the rows' dtype")
    if cos.ndim == 2:
        cos = cos[None]
    if sin.ndim == 2:
        sin = sin[None]
    try:
        cos, sin = (_aligned(x.expand(b, t, d), 4 if f32 else 8) for x in (cos, sin))
    except RuntimeError:
        raise ValueError(f"{what}: cos and sin must be [B, T, d] or [T, d]") from None
    if cos.stride() != sin.stride():
        cos, sin = _copy(cos), _copy(sin)
    return cos, sin, _strides(cos.stride(0), cos.stride(1)), int(f32)


def _tokens(what, x, name):
    if x.ndim != 4:
        raise ValueError(f"{what}: {name} must be [B, heads, T, d]")
    return x.shape


def _s3(x):
    s = x.stride()
    return _strides(s[0], s[1], s[2])


def _heads_last(x):
    """A fresh tensor of x's shape [B, h, T, d] in [B, T, h, d] memory (an output projection's order)."""
    b, h, t, d = x.shape
    return x.new_empty((b, t, h, d)).transpose(1, 2)


def paged_append(k, v, k_pages, v_pages, table, lens, cos=None, sin=None, q=None, new=None):
    """The new K / V rows k, v [B, Hkv, T, d] into the pages; with cos, sin ([B, T, d] or [T, d], fp32 or the rows' dtype) k is
    rotated on the way: x cos + (-x[d/2:], x[:d/2]) sin in fp32, rounded once. With q [B, H, T, d] (cos, sin required) returns q
    rotated alike, in [B, T, H, d] memory (padding columns too); else None. Rows that lie outside the table or on no page are
    not written. Two tokens of a call must not share a row."""
    what = "paged_append"
    shape = _tokens(what, k, "k")
    if v.shape != shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: k and v must share a shape and dtype")
    device = _one_device(what, k, v, k_pages, v_pages, table, lens, cos, sin, q, new)
    hk, pages, page, w = _cache(what, k_pages, v_pages, table, lens, new, shape, k.dtype)
    b, h, t, d = shape
    if h != hk or (q is not None and (q.ndim != 4 or q.dtype != k.dtype or (q.shape[0], q.shape[2], q.shape[3]) != (b, t, d)
                                      or q.shape[1] % hk)):
        raise ValueError(f"{what}: k and v [B, Hkv, T, d] and q [B, H, T, d] must match the pages")
    if q is not None and cos is None:
        raise ValueError(f"{what}: q is rotated: cos and sin required")
    cos, sin, sc, f32 = _rope(what, cos, sin, b, t, d, k.dtype)
    out = None if q is None else _heads_last(q)
    if k.numel() == 0:
        return out
    k, v = _aligned(k), _aligned(v)
    qa = None if q is None or q.shape[1] == 0 else _aligned(q)
    _launch_on(device, _lib.lib().bb_paged_append, k.data_ptr(), _s3(k), v.data_ptr(), _s3(v), _lib.ptr(qa),
               None if qa is None else _s3(qa), None if qa is None else out.data_ptr(), None if qa is None else _s3(out),
               _lib.ptr(cos), _lib.ptr(sin), sc, f32, k_pages.data_ptr(), _s3(k_pages), v_pages.data_ptr(), _s3(v_pages),
               table.data_ptr(), table.stride(0), lens.data_ptr(), _lib.ptr(new), b, t, 0 if qa is None else q.shape[1], hk, d,
               pages, page, w, int(k.dtype is torch.float16), _lib.stream_of(k))
    return out


@functools.lru_cache(maxsize=256)
def _attention_workspace(b, t, h, hk, d, page, w):
    return _lib.lib().bb_paged_attention_workspace(b, t, h, hk, d, page, w)


@functools.lru_cache(maxsize=256)
def _step_workspace(b, t, h, hk, d, page, w):
    return _lib.lib().bb_paged_step_workspace(b, t, h, hk, d, page, w)


def _queries(what, q, hk):
    b, h, t, d = q.shape
    if h == 0 or hk == 0 or h % hk:
        raise ValueError(f"{what}: q [B, H, T, d] and the pages' Hkv heads must match")
    return b, h, t, d


def paged_attention(q, k_pages, v_pages, table, lens, scale, new=None):
    """Exact causal attention of q [B, H, T, d] over the pages: token j of a sequence attends the rows up to its own,
    lens - new + j. One token a sequence, a few drafted ones or a chunk of a prompt; sequences of unlike lengths. Returns
    [B, H, T, d] in [B, T, H, d] memory; zeros for padding and where a token attends no row, NaN for a query that is not
    finite."""
    what = "paged_attention"
    shape = _tokens(what, q, "q")
    device = _one_device(what, q, k_pages, v_pages, table, lens, new)
    hk, pages, page, w = _cache(what, k_pages, v_pages, table, lens, new, shape, q.dtype)
    b, h, t, d = _queries(what, q, hk)
    out = _heads_last(q)
    if q.numel() == 0:
        return out
    q = _aligned(q)
    ws_bytes = _attention_workspace(b, t, h, hk, d, page, w)
    ws = _lib.workspace(ws_bytes, q.device) if ws_bytes else None
    _launch_on(device, _lib.lib().bb_paged_attention, q.data_ptr(), _s3(q), k_pages.data_ptr(), _s3(k_pages), v_pages.data_ptr(),
               _s3(v_pages), table.data_ptr(), table.stride(0), lens.data_ptr(), _lib.ptr(new), b, t, h, hk, d, pages, page, w,
               int(q.dtype is torch.float16), float(scale), out.data_ptr(), _s3(out), _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return out


def paged_step(q, k, v, k_pages, v_pages, table, lens, scale, cos=None, sin=None, new=None):
    """One step: paged_append(k, v, ..., cos, sin, q) and paged_attention of the rotated q, in one call (q and k as they are
    where cos is None). Up to 64 query vectors of a KV head (T * H / Hkv) one kernel does both. Returns [B, H, T, d] in
    [B, T, H, d] memory."""
    what = "paged_step"
    shape = _tokens(what, q, "q")
    device = _one_device(what, q, k, v, k_pages, v_pages, table, lens, cos, sin, new)
    hk, pages, page, w = _cache(what, k_pages, v_pages, table, lens, new, shape, q.dtype)
    b, h, t, d = _queries(what, q, hk)
    if k.shape != (b, hk, t, d) or v.shape != k.shape or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: k and v [B, Hkv, T, d] and q [B, H, T, d] must match the pages")
    cos, sin, sc, f32 = _rope(what, cos, sin, b, t, d, q.dtype)
    out = _heads_last(q)
    if q.numel() == 0:
        return out
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    ws_bytes = _step_workspace(b, t, h, hk, d, page, w)
    ws = _lib.workspace(ws_bytes, q.device) if ws_bytes else None
    _launch_on(device, _lib.lib().bb_paged_step, q.data_ptr(), _s3(q), k.data_ptr(), _s3(k), v.data_ptr(), _s3(v),
               _lib.ptr(cos), _lib.ptr(sin), sc, f32, k_pages.data_ptr(), _s3(k_pages), v_pages.data_ptr(), _s3(v_pages),
               table.data_ptr(), table.stride(0), lens.data_ptr(), _lib.ptr(new), b, t, h, hk, d, pages, page, w,
               int(q.dtype is torch.float16), float(scale), out.data_ptr(), _s3(out), _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return out
