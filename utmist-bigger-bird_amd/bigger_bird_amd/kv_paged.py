"""Paged KV cache on MI355X: the rows of several sequences in pages, appended to with RoPE on the way and attended exactly.

The reference's caches hold one sequence in contiguous rows (modal_rd/kv_int8.py, modal_rd/graph_decode.py); this one serves
several of unlike lengths in one call, and a sequence grows without a copy.

Layout: k_pages / v_pages [pages, Hkv, page, d] (bf16 or fp16, page a power of two >= 16, d 64 or 128; any strides between
rows, heads and pages that keep rows 16-byte aligned), table [B, W] int32 (entry w: the page of rows w * page .. of a
sequence; an entry outside 0 .. pages - 1 names no page, and its rows are neither written nor attended), lens [B] int32 (rows
of each sequence, the call's new ones among them), new [B] int32 (how many of the T token columns are real; None: all). Token j
of sequence b is row lens[b] - new[b] + j and attends the rows up to its own. All three are read by the kernels, so a captured
graph follows them.

`make_paged_cache` puts them under a model whose attention RDAttention is: batches of sequences, where the other caches hold one.
"""
import ctypes
import functools

import torch
from transformers import DynamicCache
from transformers.cache_utils import DynamicLayer

from . import _lib
from .kv_int4 import _copy, _launch_on

_ROWS = (torch.bfloat16, torch.float16)
_FAR = (1 << 31) - 1


# A step of a few tokens is one or two kernels of microseconds, so what depends on shapes, strides, dtypes and devices alone is
# checked and laid out for the library once per such layout (the library's arguments as the ctypes objects that they become);
# addresses are looked at in every call.
def _layouts(*tensors):
    return [x if x is None else (x.shape, x.stride(), x.dtype, x.get_device()) for x in tensors]


def _device_of(what, *layouts):
    """The index of the one ROCm device that holds every tensor (the kernels run on the current stream there)."""
    devices = {x[3] for x in layouts if x is not None}
    if -1 in devices:
        raise ValueError(f"{what} runs on the ROCm device only (got a tensor that is not on it)")
    if len(devices) != 1:
        raise ValueError(f"{what}: tensors on different devices")
    return devices.pop()


def _i64s(*vals):
    return ctypes.cast(_lib.i64s(*vals), _lib.c_i64p)


def _i32s(*vals):
    return tuple(map(ctypes.c_int, vals))


def _aligned(layout, rows=8):
    """Whether rows of a layout lie 16 bytes apart (rows: elements of 16 bytes), the last dimension contiguous."""
    s = layout[1]
    return s[-1] == 1 and not any(i % rows for i in s[:-1])


def _strides3(layout):
    s = layout[1]
    return _i64s(s[0], s[1], s[2])


def _check_cache(what, rows, kp, vp, table, lens, new):
    """(heads, pages, page, W) of a call's cache, checked against tokens [B, heads, T, d]; arguments are layouts."""
    (shape, _, dtype, _), (ps, _, pd, _), (vs, _, vd, _) = rows, kp, vp
    if len(shape) != 4:
        raise ValueError(f"{what}: rows must be [B, heads, T, d]")
    b, d = shape[0], shape[3]
    if dtype not in _ROWS or pd != dtype or vd != dtype:
        raise ValueError(f"{what}: bf16 or fp16 rows and pages of one dtype required")
    if len(ps) != 4 or ps != vs or ps[3] != d or not ps[0] or not ps[1]:
        raise ValueError(f"{what}: k_pages and v_pages must be [pages, Hkv, page, d] with the rows' d")
    if d not in (64, 128):  # (here, as rows of others have no aligned copy that the library could refuse)
        raise ValueError(f"{what}: head_dim {d} unsupported (64 or 128)")
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
    for shape, s, _, _ in (cos, sin):
        if len(shape) == 2:
            shape, s = (1, *shape), (0, *s)
        if len(shape) != 3 or shape[2] != d or any(n != 1 and n != m for n, m in zip(shape, (b, t))):
            raise ValueError(f"{what}: cos and sin must be [B, T, d] or [T, d]")
        strides.append((0 if shape[0] == 1 else s[0], 0 if shape[1] == 1 else s[1], s[2]))
    whole = 4 if f32 else 8
    ok = strides[0] == strides[1] and strides[0][2] == 1 and not any(i % whole for i in strides[0][:2])
    return not ok, _i64s(*strides[0][:2]), int(f32)


def _whole_rope(cos, sin, b, t, d):
    """cos and sin in fresh [B, T, d] memory."""
    return tuple(_copy(x.expand(b, t, d)) for x in (cos, sin))


def _heads_last(shape):
    """The strides of a tensor [B, h, T, d] in [B, T, h, d] memory (an output projection's order)."""
    b, h, t, d = shape
    return t * h * d, d, h * d, 1


def _check_addresses(what, k_pages, v_pages):
    if (k_pages | v_pages) & 15:
        raise ValueError(f"{what}: pages need a contiguous head_dim and 16-byte aligned rows")


@functools.lru_cache(maxsize=512)
def _append_plan(k, v, kp, vp, table, lens, cos, sin, q, new):
    what = "paged_append"
    device = _device_of(what, k, v, kp, vp, table, lens, cos, sin, q, new)
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
    so = _heads_last(q[0]) if q is not None else None
    sq = (_strides3(q), _i64s(*so[:3])) if heads else (None, None)
    return (device, copy, so, _strides3(k), _strides3(v), *sq, sc, f32, _strides3(kp), _strides3(vp), table[1][0],
            _i32s(b, t, heads, hk, d, pages, page, w, k[2] is torch.float16))


def paged_append(k, v, k_pages, v_pages, table, lens, cos=None, sin=None, q=None, new=None):
    """The new K / V rows k, v [B, Hkv, T, d] into the pages; with cos, sin ([B, T, d] or [T, d], fp32 or the rows' dtype) k is
    rotated on the way: x cos + (-x[d/2:], x[:d/2]) sin in fp32, rounded once (in fp16 to an infinity past 65519). With q [B, H,
    T, d] (cos, sin required) returns q rotated alike, in [B, T, H, d] memory (padding columns too); else None. Rows that lie
    outside the table or on no page are not written. Two tokens of a call must not share a row of a page."""
    what = "paged_append"
    device, copy, out_strides, sk, sv, sq, so, sc, f32, skp, svp, st, sizes = _append_plan(
        *_layouts(k, v, k_pages, v_pages, table, lens, cos, sin, q, new))
    pk, pv, kp, vp = k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    pq, pc, ps = _lib.ptr(q) or 0, _lib.ptr(cos) or 0, _lib.ptr(sin) or 0
    _check_addresses(what, kp, vp)
    if k.numel() == 0:
        return None if q is None else q.new_empty_strided(q.shape, out_strides)
    if copy or (pk | pv | pq | pc | ps) & 15:
        if cos is not None:
            cos, sin = _whole_rope(cos, sin, k.shape[0], k.shape[2], k.shape[3])
        return paged_append(_copy(k), _copy(v), k_pages, v_pages, table, lens, cos, sin, None if q is None else _copy(q), new)
    out = None if q is None else q.new_empty_strided(q.shape, out_strides)
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
    device = _device_of(what, q, kp, vp, table, lens, new)
    hk, pages, page, w = _check_cache(what, q, kp, vp, table, lens, new)
    b, h, t, d = _check_queries(what, q, hk)
    ws = _lib.lib().bb_paged_attention_workspace(b, t, h, hk, d, page, w)
    so = _heads_last(q[0])
    return (device, not _aligned(q), so, _strides3(q), _strides3(kp), _strides3(vp), table[1][0],
            _i32s(b, t, h, hk, d, pages, page, w, q[2] is torch.float16), _i64s(*so[:3]), ws)


def paged_attention(q, k_pages, v_pages, table, lens, scale, new=None):
    """Exact causal attention of q [B, H, T, d] over the pages: token j of a sequence attends the rows up to its own, lens - new
    + j. One token a sequence, a few drafted ones or a chunk of a prompt; sequences of unlike lengths. Scores, softmax and sums
    are fp32. The probabilities meet V as two terms of the rows' dtype up to 32 query vectors of a KV head (T * H / Hkv), so
    that the output's own rounding is all its error; of more vectors they are one, rounded to the dtype (0.0023 of the output's
    norm in bf16, where its rounding alone is 0.0017). Returns [B, H, T, d] in [B, T, H, d] memory; zeros for padding and where
    a token attends no row, NaN for a query that is not finite. A value of V that is not finite reaches the tokens that attend
    it alone: +inf, -inf, or NaN where both or a NaN are attended."""
    what = "paged_attention"
    device, copy, out_strides, sq, skp, svp, st, sizes, so, ws_bytes = _attention_plan(
        *_layouts(q, k_pages, v_pages, table, lens, new))
    pq, kp, vp = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    _check_addresses(what, kp, vp)
    if q.numel() == 0:
        return q.new_empty_strided(q.shape, out_strides)
    if copy or pq & 15:
        return paged_attention(_copy(q), k_pages, v_pages, table, lens, scale, new)
    out = q.new_empty_strided(q.shape, out_strides)
    ws = _lib.workspace(ws_bytes, q.device) if ws_bytes else None
    _launch_on(device, _lib.lib().bb_paged_attention, pq, sq, kp, skp, vp, svp, table.data_ptr(), st, lens.data_ptr(),
               _lib.ptr(new), *sizes, float(scale), out.data_ptr(), so, _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return out


@functools.lru_cache(maxsize=512)
def _step_plan(q, k, v, kp, vp, table, lens, cos, sin, new):
    what = "paged_step"
    device = _device_of(what, q, k, v, kp, vp, table, lens, cos, sin, new)
    hk, pages, page, w = _check_cache(what, q, kp, vp, table, lens, new)
    b, h, t, d = _check_queries(what, q, hk)
    if k[0] != (b, hk, t, d) or v[0] != k[0] or k[2] != q[2] or v[2] != q[2]:
        raise ValueError(f"{what}: k and v [B, Hkv, T, d] and q [B, H, T, d] must match the pages")
    copy_rope, sc, f32 = _check_rope(what, cos, sin, b, t, d, q[2])
    ws = _lib.lib().bb_paged_step_workspace(b, t, h, hk, d, page, w)
    so = _heads_last(q[0])
    return (device, copy_rope or not (_aligned(q) and _aligned(k) and _aligned(v)), so, _strides3(q), _strides3(k), _strides3(v),
            sc, f32, _strides3(kp), _strides3(vp), table[1][0], _i32s(b, t, h, hk, d, pages, page, w, q[2] is torch.float16),
            _i64s(*so[:3]), ws)


def paged_step(q, k, v, k_pages, v_pages, table, lens, scale, cos=None, sin=None, new=None):
    """One step: paged_append(k, v, ..., cos, sin, q) and paged_attention of the rotated q, in one call (q and k as they are
    where cos is None). Up to 128 query vectors of a KV head (T * H / Hkv) one kernel does both, and neither its rotated queries
    nor its probabilities are rounded to the rows' dtype; above they are, as paged_append and paged_attention do (0.0029 to
    0.0032 of the output's norm in bf16, and a rotated fp16 query is infinite past 65519). A row that the call writes must not
    be attended in it by another sequence, nor at another place of its own table. Returns [B, H, T, d] in [B, T, H, d]
    memory."""
    what = "paged_step"
    device, copy, out_strides, sq, sk, sv, sc, f32, skp, svp, st, sizes, so, ws_bytes = _step_plan(
        *_layouts(q, k, v, k_pages, v_pages, table, lens, cos, sin, new))
    pq, pk, pv, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    pc, ps = _lib.ptr(cos) or 0, _lib.ptr(sin) or 0
    _check_addresses(what, kp, vp)
    if q.numel() == 0:
        return q.new_empty_strided(q.shape, out_strides)
    if copy or (pq | pk | pv | pc | ps) & 15:
        if cos is not None:
            cos, sin = _whole_rope(cos, sin, q.shape[0], q.shape[2], q.shape[3])
        return paged_step(_copy(q), _copy(k), _copy(v), k_pages, v_pages, table, lens, scale, cos, sin, new)
    out = q.new_empty_strided(q.shape, out_strides)
    ws = _lib.workspace(ws_bytes, q.device) if ws_bytes else None
    _launch_on(device, _lib.lib().bb_paged_step, pq, sq, pk, sk, pv, sv, pc, ps, sc, f32, kp, skp, vp, svp, table.data_ptr(), st,
               lens.data_ptr(), _lib.ptr(new), *sizes, float(scale), out.data_ptr(), so, _lib.ptr(ws), ws_bytes,
               _lib.stream_of(q))
    return out


def _hides_rows(mask):
    """Whether a mask (None or False: none; True: one that does) hides any row from the last token, as padding on either side and
    packed sequences do and the causal mask does not. Looks at the mask's values: the host waits for them."""
    if mask is None or isinstance(mask, bool):
        return bool(mask)
    if hasattr(mask, "mask_mod"):  # a flex attention's BlockMask: a function of (batch, head, query, key)
        device = mask.kv_num_blocks.device
        t, zero = mask.seq_lengths[0], torch.zeros((), dtype=torch.int64, device=device)
        return not bool(mask.mask_mod(zero, zero, zero + t - 1, torch.arange(t, device=device)).all())
    if not torch.is_tensor(mask) or mask.ndim < 2:
        return True
    if mask.numel() == 0:
        return False
    last = mask[..., -1, :] if mask.ndim > 2 else mask
    return bool((last < 0).any() if last.dtype.is_floating_point else (last == 0).any())


class PagedKVLayer(DynamicLayer):
    """One layer's pages of a PagedCache. RDAttention attends them (`attend`, `append`); other consumers are refused, as there are
    no contiguous keys and values to hand out."""

    def __init__(self, cache, index, k_pages, v_pages):
        super().__init__()
        self.cache, self.index, self.k_pages, self.v_pages = cache, index, k_pages, v_pages
        self.dtype, self.device = k_pages.dtype, k_pages.device
        self.is_initialized = True

    def begin(self, t, padded, positions):
        """The current step's new tokens per sequence, for this layer: `t` columns (begun here, with every column real, unless
        PagedCache.extend did). `padded`: the mask that the model was given, if any (True: one that hides rows); `positions`: how
        many sequences' angles it was given."""
        return self.cache._begin(self.index, t, padded, positions)

    def append(self, k, v):
        """The step's rows k, v [B, Hkv, T, d], rotated already, into the pages."""
        c = self.cache
        paged_append(k, v, self.k_pages, self.v_pages, c.table, c.lens, new=c._new_of(k.shape[2]))

    def attend(self, q, k, v, scale, cos, sin):
        """The step's rows into the pages, k rotated by cos, sin [B or 1, T, d], and the attention of the rotated q."""
        c = self.cache
        b, _, t, _ = q.shape
        cos, sin = (x.expand(b, t, x.shape[-1]) for x in (cos, sin))
        return paged_step(q, k, v, self.k_pages, self.v_pages, c.table, c.lens, scale, cos=cos, sin=sin, new=c._new_of(t))

    def lazy_initialization(self, key_states, value_states, *args, **kwargs):
        pass

    def update(self, key_states, value_states, *args, **kwargs):
        raise ValueError("a paged cache is attended by RDAttention only (install the model's attention)")

    def get_seq_length(self, *args, **kwargs):
        """Rows of the longest sequence before the current step."""
        return max(self.cache._before())

    def get_mask_sizes(self, query_length, *args, **kwargs):
        return query_length, 0  # no mask is read: a step's tokens alone, which a model without padding needs none for

    def crop(self, tokens_to_remove):
        raise NotImplementedError("crop the whole PagedCache")

    reset = reorder_cache = batch_repeat_interleave = batch_select_indices = crop


class PagedCache(DynamicCache):
    """A model's KV cache in pages: `batch` sequences of unlike lengths share `pages` pages of `page` rows a layer.

    A forward pass is a step: its first layer takes pages for the new tokens of every sequence (as many as the input has columns,
    or what `extend` said just before, with the padding on the right), and every layer then writes and attends them.
    The lengths live on the host too, so a step's first layer copies them over and the host waits for what the GPU has queued.
    `positions(t)` are the step's position ids, needed once sequences differ in length. `truncate` takes rows back (drafted
    tokens that were not accepted), `release` empties sequences, whose pages others then take."""

    def __init__(self, config, batch, pages, page=64, rows=None, dtype=torch.bfloat16, device="cuda"):
        super().__init__(config=config)
        cfg = config.get_text_config(decoder=True)
        d = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        if page < 16 or page & (page - 1):
            raise ValueError("PagedCache: pages of a power of two of rows, at least 16")
        if batch < 1 or pages < 1 or d not in (64, 128) or dtype not in _ROWS:
            raise ValueError("PagedCache: bf16 or fp16 rows of head_dim 64 or 128, one sequence and page at least")
        self.page, self.width = page, -(-(rows or pages * page) // page)
        shape = (cfg.num_hidden_layers, 2, pages, cfg.num_key_value_heads, page, d)
        with torch.inference_mode(False):  # updated in place in either mode
            self.arena = torch.empty(shape, dtype=dtype, device=device)
            self.table = torch.full((batch, self.width), -1, dtype=torch.int32, device=device)
            self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
            self.new = torch.zeros(batch, dtype=torch.int32, device=device)
        self.lengths = [0] * batch          # rows of each sequence, the current step's among them
        self._pages = [[] for _ in range(batch)]
        self._free = list(range(pages))[::-1]
        self._step, self._left = [0] * batch, set()  # new tokens of the current step, layers that have not run it
        self._declared = False
        self.layers = [PagedKVLayer(self, i, a[0], a[1]) for i, a in enumerate(self.arena)]

    def _before(self):
        return [n - s for n, s in zip(self.lengths, self._step)] if self._left else self.lengths

    def extend(self, new):
        """Begin a step of new[b] tokens of sequence b (0: none): pages are taken for them. The next forward pass runs it; its
        input has max(new) columns or more, each sequence's tokens first."""
        new = [int(x) for x in new]
        if self._left:
            raise ValueError("PagedCache: the step before has not run through every layer (truncate takes it back)")
        if len(new) != len(self.lengths) or min(new) < 0:
            raise ValueError("PagedCache: one count of new tokens per sequence")
        after = [n + s for n, s in zip(self.lengths, new)]
        need = [-(-n // self.page) - len(p) for n, p in zip(after, self._pages)]
        if max(after) > self.width * self.page:
            raise ValueError("PagedCache: a sequence is past the rows that the cache was made for")
        if sum(x for x in need if x > 0) > len(self._free):
            raise ValueError("PagedCache: no free pages left")
        for b, x in enumerate(need):
            if x > 0:
                at = len(self._pages[b])
                self._pages[b] += [self._free.pop() for _ in range(x)]
                self.table[b, at:at + x].copy_(torch.tensor(self._pages[b][at:], dtype=torch.int32))
        self.lengths, self._step, self._left = after, new, set(range(len(self.layers)))
        self.lens.copy_(torch.tensor(after, dtype=torch.int32))
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        self._declared = True

    def _begin(self, layer, t, padded, positions):
        begun = layer in self._left
        step, before = (self._step, self._before()) if begun else ([t] * len(self.lengths), self.lengths)
        if max(step) > t:
            raise ValueError(f"PagedCache: the step has {max(step)} new tokens, the input {t} columns")
        if not begun and (len(step) > 1 and padded is not None and padded is not False or _hides_rows(padded)):
            raise ValueError("PagedCache: padding goes by extend(new tokens of each sequence) and to the right, not by a mask")
        if positions == 1 and any(s and n != max(before) for n, s in zip(before, step)):
            raise ValueError("PagedCache: sequences of unlike lengths need position_ids (positions)")
        if not begun:
            self.extend(step)
            self._declared = False
        self._left.discard(layer)
        return self._step

    def _new_of(self, t):
        return None if all(s == t for s in self._step) else self.new

    def positions(self, t=None):
        """Position ids [B, t] of a step's columns (t: as many as its longest has), of the step that extend began or the next."""
        before = torch.tensor(self._before(), device=self.lens.device)
        return before[:, None] + torch.arange(max(self._step) if t is None else t, device=self.lens.device)

    def truncate(self, lengths):
        """Keep the first lengths[b] rows of each sequence; whole pages behind them become free. A step that did not run through
        every layer is taken back with it: its rows are none that a sequence has."""
        lengths = [int(x) for x in lengths]
        if len(lengths) != len(self.lengths) or any(not 0 <= x <= n for x, n in zip(lengths, self._before())):
            raise ValueError("PagedCache: one length per sequence, of rows that it has")
        for b, n in enumerate(lengths):
            keep = -(-n // self.page)
            if keep < len(self._pages[b]):
                self.table[b, keep:len(self._pages[b])].fill_(-1)
                self._free += self._pages[b][keep:][::-1]
                del self._pages[b][keep:]
        self.lengths, self._step, self._left = lengths, [0] * len(lengths), set()
        self.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.new.zero_()

    def release(self, sequences):
        """Empty these sequences (an index or several); a step that did not run is taken back."""
        gone = {sequences} if isinstance(sequences, int) else set(sequences)
        if not gone <= set(range(len(self.lengths))):
            raise ValueError("PagedCache: no such sequence")
        self.truncate([0 if b in gone else n for b, n in enumerate(self._before())])

    def crop(self, tokens_to_remove):
        if tokens_to_remove > 0:
            raise NotImplementedError("PagedCache.crop supports negative token counts only")
        self.truncate([max(0, n + tokens_to_remove) for n in self._before()])

    def reset(self):
        self.truncate([0] * len(self.lengths))

    def nbytes(self):
        """Bytes of the pages that sequences hold, over all layers."""
        return sum(len(p) for p in self._pages) * self.arena[:, :, 0].numel() * self.arena.element_size()


def make_paged_cache(config, batch, pages, page=64, rows=None, dtype=torch.bfloat16, device="cuda"):
    """A PagedCache for `batch` sequences over `pages` pages of `page` rows in each layer (rows: the longest that a sequence may
    become; None: all pages')."""
    return PagedCache(config, batch, pages, page, rows, dtype, device)
