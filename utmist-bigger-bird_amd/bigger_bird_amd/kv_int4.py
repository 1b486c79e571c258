"""KV cache in 4 bits on MI355X: writing rows, reading them back, and exact decode over the packed rows.

The reference keeps compressed caches in formats of its own (modal_rd/turbo_kv.py); this one is new, and reaches the same
places: an HF cache layer (`make_int4_cache`, next to `make_int8_cache`) whose handles RDAttention attends with `attend`.

Format: asymmetric per token, KV head and group of 32 elements. With min and max clamped to +-65504 and NaN left out of
them, each operation in fp32: z = fp16(min), s = fp16(max((max - z) / 15, 0)), code = rint((x - z) / s) clamped to 0..15
(0 where s = 0 or x is NaN; a group of NaN alone has s = z = 0); the value is s * code + z in fp32. Byte b of a packed row
holds elements 2 b (low four bits) and 2 b + 1. A cache is codes [Hkv, capacity, d / 2] uint8 and params
[Hkv, capacity, d / 32, 2] fp16 (s, z), head-major, for K and for V: 80 bytes a row at head_dim 128, against 130 in int8
and 256 in bf16.
"""
import functools

import torch
from transformers import DynamicCache

from . import _lib
from .flash import exact_attention
from .kv_int8 import _KINDS, GROW, Int8KVLayer

# Stride arrays by their values (read-only to the library): made once per layout instead of three times a call.
_strides = functools.lru_cache(maxsize=1024)(_lib.i64s)
MAX_TOKENS = 16  # query tokens of one decode call
# Query vectors per KV head (tokens x heads) up to which a handle attends the packed rows; the kernel takes 16 a pass over the
# cache. Against reading the cache back and flash attention over it, whole calls (us) of 16 tokens at head_dim 128, over 131072
# and 16384 rows: 64 vectors of 8 KV heads 158 and 364, 40 and 57; 128 of 8 305 and 436, 72 and 65; 192 of 4 250 and 270, 54
# and 49; 256 of 4 333 and 318, 70 and 54. (Over 4096 rows the packed rows win at each of them, 24 and 33 at 256; past 128 only the
# read back's memory, 6.4 times the cache, would speak for them.)
_HANDLE_VECTORS = 128
_HEAD_DIMS = (32, 64, 128, 256)
_HALVES = (16, 32, 64, 128)  # their packed rows' bytes


def _launch_on(device, fn, *args):
    """fn(*args) with `device` (an index) current, checked (a launch goes to the current device's context)."""
    if device == torch.cuda.current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(device):
            rc = fn(*args)
    if rc:
        _lib.check(rc)


def _one_device(what, *tensors):
    """The index of the one ROCm device that holds every tensor (the kernels run on the current stream there)."""
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != device or device < 0):
            _lib.require_gpu(*tensors, what=what)
            raise ValueError(f"{what}: tensors on different devices")
    return device


def _copy(x):
    """x in fresh memory, row after row (x.contiguous() is x itself where only its address, or the stride of a dimension of
    length 1, keeps its rows from being aligned)."""
    return torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)


def _input_rows(x):
    """x [..., t, d] as [heads, t, d] with 16-byte aligned rows (a copy where it is not)."""
    x = x[None] if x.ndim == 2 else x.flatten(0, -3) if x.ndim > 3 else x
    el = x.element_size()
    if x.stride(-1) != 1 or x.data_ptr() % 16 or (x.stride(0) * el) % 16 or (x.stride(1) * el) % 16:
        x = _copy(x)
    return x


def _packed(what, q, p):
    """(heads, rows, head_dim, head stride of q in bytes, head stride of p in elements) of packed rows: q [..., t, d / 2]
    and p [..., t, d / 32, 2], the rows of a head back to back, one stride between heads."""
    if q.dtype is not torch.uint8 or p.dtype is not torch.float16:
        raise ValueError(f"{what}: codes must be uint8 and params float16")
    if q.ndim != 3:
        if q.ndim < 2 or p.ndim != q.ndim + 1 or p.shape[:-2] != q.shape[:-1]:
            raise ValueError(f"{what}: codes [..., t, d / 2] and params [..., t, d / 32, 2] must match")
        try:
            heads = q.shape[:-2].numel()  # (spelled out: -1 is ambiguous where there are no rows)
            q = q.view(heads, *q.shape[-2:]) if q.ndim > 3 else q[None]
            p = p.view(heads, *p.shape[-3:]) if p.ndim > 4 else p[None]
        except RuntimeError:
            raise ValueError(f"{what}: packed rows need one stride between heads") from None
    h, t, half = q.shape
    if half not in _HALVES or p.shape != (h, t, half // 16, 2):
        raise ValueError(f"{what}: codes [..., t, d / 2] and params [..., t, d / 32, 2] must match (d 32, 64, 128 or 256)")
    q0, q1, q2 = q.stride()
    p0, p1, p2, p3 = p.stride()
    if (q2 != 1 or p3 != 1 or (p2 != 2 and half > 16) or (t > 1 and (q1 != half or p1 != half // 8))
            or (h > 1 and (q0 < t * half or p0 < t * (half // 8)))):
        raise ValueError(f"{what}: the packed rows of a head must be contiguous and heads must not overlap")
    return (h, t, 2 * half, q0, p0) if h > 1 else (h, t, 2 * half, 0, 0)


def _packed_pair(what, kq, kp, vq, vp):
    """_packed of K, and of V (the same tuple where V is laid out as K is)."""
    k = _packed(what, kq, kp)
    if (vq.shape == kq.shape and vp.shape == kp.shape and vq.stride() == kq.stride() and vp.stride() == kp.stride()
            and vq.dtype is torch.uint8 and vp.dtype is torch.float16):
        return k, k
    return k, _packed(what, vq, vp)


def _new_packed(rows, d, device):
    """Codes and params of `rows` (the leading dimensions) rows of d elements."""
    return (torch.empty(*rows, d // 2, dtype=torch.uint8, device=device),
            torch.empty(*rows, d // 32, 2, dtype=torch.float16, device=device))


def _check_input(x):
    if x.dtype not in _KINDS:
        raise ValueError("quantize4: bf16, fp16 or fp32 input")
    if x.ndim < 2 or x.shape[-1] not in _HEAD_DIMS:
        raise ValueError("quantize4: rows [..., t, d] with d 32, 64, 128 or 256")


def _check_out(x, out, layout):
    if out[0].shape[:-1] != x.shape[:-1] or layout[2] != x.shape[-1]:
        raise ValueError("quantize4: out tensors must match x")


def quantize4(x, out=None):
    """[..., t, d] (bf16, fp16 or fp32, any strides) -> codes [..., t, d / 2] uint8, params [..., t, d / 32, 2] fp16.

    `out` = (codes, params) to write into, e.g. the rows [a, b) of a cache: (k4[:, a:b], kp[:, a:b])."""
    _check_input(x)
    device = _one_device("quantize4", x, *(out or ()))
    if out is None:
        out = _new_packed(x.shape[:-1], x.shape[-1], x.device)
    layout = _packed("quantize4", *out)
    _check_out(x, out, layout)
    if x.numel():
        _write(device, x, None, out, (None, None), layout, (0,) * 5)
    return out


def quantize4_pair(xk, xv, out_k=None, out_v=None):
    """quantize4(xk, out_k) and quantize4(xv, out_v) in one launch (a prompt's or a step's new K and V rows: one shape and
    dtype). Returns ((codes, params) of K, (codes, params) of V)."""
    _check_input(xk)
    device = _one_device("quantize4", xk, xv, *(out_k or ()), *(out_v or ()))
    if xv.shape != xk.shape or xv.dtype != xk.dtype:
        raise ValueError("quantize4: K and V rows must share a shape and dtype")
    if out_k is None:
        out_k = _new_packed(xk.shape[:-1], xk.shape[-1], xk.device)
    if out_v is None:
        out_v = _new_packed(xk.shape[:-1], xk.shape[-1], xk.device)
    k, v = _packed_pair("quantize4", *out_k, *out_v)
    _check_out(xk, out_k, k)
    if v is not k:
        _check_out(xv, out_v, v)
    if xk.numel():
        _write(device, xk, xv, out_k, out_v, k, v)
    return out_k, out_v


def _write(device, xk, xv, out_k, out_v, k, v):
    """The launch of quantize4_pair (xv None: of one tensor); k and v are the layouts of the outputs."""
    a = _input_rows(xk)
    sa, pb, sb = a.stride(), None, None
    if xv is not None:
        b = _input_rows(xv)
        pb, sb = b.data_ptr(), _strides(b.stride(0), b.stride(1))
    _launch_on(device, _lib.lib().bb_int4_quantize, a.data_ptr(), _strides(sa[0], sa[1]), pb, sb, _KINDS[a.dtype],
               a.shape[0], a.shape[1], k[2], out_k[0].data_ptr(), out_k[1].data_ptr(), _lib.ptr(out_v[0]),
               _lib.ptr(out_v[1]), _strides(k[3], k[4], v[3], v[4]), _lib.stream_of(xk))


def dequantize4(q, p, dtype):
    """codes [..., t, d / 2], params [..., t, d / 32, 2] -> [..., t, d] in dtype (bf16, fp16 or fp32; the fp32 value
    s * code + z rounded to nearest even, in fp16 infinite past 65504, which the top code of a group that spans nearly all of
    fp16's range can be). Rows [a, b) of a cache are read in place: (k4[:, a:b], kp[:, a:b])."""
    if dtype not in _KINDS:
        raise ValueError("dequantize4: bf16, fp16 or fp32 output")
    device = _one_device("dequantize4", q, p)
    k = _packed("dequantize4", q, p)
    out = torch.empty(*q.shape[:-1], k[2], dtype=dtype, device=q.device)
    if out.numel():
        _launch_on(device, _lib.lib().bb_int4_dequantize, q.data_ptr(), p.data_ptr(), None, None, _strides(k[3], k[4], 0, 0),
                   k[0], k[1], k[2], out.data_ptr(), None, _KINDS[dtype], _lib.stream_of(out))
    return out


def dequantize4_pair(k, v, dtype):
    """(dequantize4(*k, dtype), dequantize4(*v, dtype)) in one launch; k and v hold the same number of rows."""
    if dtype not in _KINDS:
        raise ValueError("dequantize4: bf16, fp16 or fp32 output")
    device = _one_device("dequantize4", *k, *v)
    lk, lv = _packed_pair("dequantize4", *k, *v)
    if lv[:3] != lk[:3]:
        raise ValueError("dequantize4: K and V must hold the same rows")
    outk = k[0].new_empty((*k[0].shape[:-1], lk[2]), dtype=dtype)
    outv = torch.empty_like(outk) if v[0].shape == k[0].shape else k[0].new_empty((*v[0].shape[:-1], lk[2]), dtype=dtype)
    if outk.numel():
        _launch_on(device, _lib.lib().bb_int4_dequantize, k[0].data_ptr(), k[1].data_ptr(), v[0].data_ptr(),
                   v[1].data_ptr(), _strides(lk[3], lk[4], lv[3], lv[4]), lk[0], lk[1], lk[2], outk.data_ptr(),
                   outv.data_ptr(), _KINDS[dtype], _lib.stream_of(outk))
    return outk, outv


def _rows16(x):
    """x [a, b, d] with a contiguous head_dim and 16-byte aligned rows (a copy where it is not)."""
    s = x.stride()
    return x if s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and x.data_ptr() % 16 == 0 else _copy(x)


@functools.lru_cache(maxsize=64)
def _workspace_bytes(rows, t, h, hk, d):
    return _lib.lib().bb_int4_decode_workspace(rows, t, h, hk, d)


@functools.lru_cache(maxsize=64)
def _one_split(vectors, d):
    """The longest cache that the library attends in one split, which needs no workspace."""
    return _lib.lib().bb_int4_decode_one_split(vectors, d)


def _decode(q, k4, kp, v4, vp, knew, vnew, n, scale, causal):
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        raise ValueError("decode_int4: bf16 or fp16 query")
    one = q.ndim == 2
    if one:
        q = q[None]
    if q.ndim != 3 or k4.ndim != 3 or v4.ndim != 3:
        raise ValueError("decode_int4: q [H, d] or [T, H, d] and caches [Hkv, capacity, ...]")
    length = n if isinstance(n, torch.Tensor) else None
    device = _one_device("decode_int4", q, k4, kp, v4, vp, knew, vnew, length)
    k, v = _packed_pair("decode_int4", k4, kp, v4, vp)
    hk, cap, d, skq, skp = k
    t, h, dq = q.shape
    if v[:3] != k[:3] or dq != d or not h or not hk or h % hk:
        raise ValueError("q [T,H,D] and the cache's Hkv heads must match")
    if length is not None and (length.dtype is not torch.int64 or length.numel() != 1):
        raise ValueError("n must be an int64 tensor of one element (it is read in place by the kernels)")
    q = _rows16(q)
    sq = q.stride()
    L = _lib.lib()
    fn, new = L.bb_int4_decode, ()
    if knew is not None:
        if one and knew.ndim == 2 and vnew.ndim == 2:
            knew, vnew = knew[:, None], vnew[:, None]
        if knew.dtype != q.dtype or vnew.dtype != q.dtype or knew.shape != (hk, t, d) or vnew.shape != (hk, t, d):
            raise ValueError("decode_int4_append: new rows must be [Hkv, T, d] (or [Hkv, d] for one token) of q's dtype")
        knew, vnew = _rows16(knew), _rows16(vnew)
        sk, sv = knew.stride(), vnew.stride()
        fn = L.bb_int4_decode_append
        new = (knew.data_ptr(), _strides(sk[0], sk[1]), vnew.data_ptr(), _strides(sv[0], sv[1]))
    out = torch.empty_like(q) if sq == (h * d, d, 1) else q.new_empty((t, h, d))
    rows = cap if length is not None else int(n)
    if rows <= _one_split(t * (h // hk), d):  # no partials
        ws, ws_bytes = None, 0
    else:
        ws_bytes = _workspace_bytes(cap, t, h, hk, d)  # for every length up to the capacity
        ws = k4.new_empty(ws_bytes)
    _launch_on(device, fn, q.data_ptr(), _strides(sq[0], sq[1]), k4.data_ptr(), kp.data_ptr(), v4.data_ptr(), vp.data_ptr(),
               _strides(skq, skp, v[3], v[4]), *new, rows, _lib.ptr(length), cap, t, h, hk,
               d, int(q.dtype is torch.float16), float(scale), int(bool(causal)), out.data_ptr(), _strides(h * d, d),
               _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return out[0] if one else out


def decode_int4(q, k4, kp, v4, vp, n, scale, causal=False):
    """Exact attention of q [H, d] (one token) or [T, H, d] (the last T tokens, at most 16), bf16 or fp16, over the first
    n rows of a 4-bit cache: codes k4 / v4 [Hkv, capacity, d / 2], params kp / vp [Hkv, capacity, d / 32, 2].

    Every token attends all n rows (as RDAttention's cached steps do), or with `causal` token t the first n - T + 1 + t.
    `n`: int, or an int64 GPU tensor of one element that the kernels read (clamped to 0 .. capacity), so that a captured
    graph stays valid while the cache grows. A token that attends no row gives zeros; a query that is not finite gives NaN.
    Returns q's shape and dtype."""
    return _decode(q, k4, kp, v4, vp, None, None, n, scale, causal)


def decode_int4_append(q, k4, kp, v4, vp, knew, vnew, n, scale, causal=False):
    """One decode step: the new K / V rows knew / vnew [Hkv, T, d] ([Hkv, d] for one token; q's dtype, any strides) are
    quantised into cache rows n - T .. n - 1 (as quantize4_pair would), and q attends as in decode_int4; n counts the
    new rows. Rows that a device-side n puts outside the cache are not written."""
    if knew is None or vnew is None:
        raise ValueError("decode_int4_append: knew and vnew required")
    return _decode(q, k4, kp, v4, vp, knew, vnew, n, scale, causal)


class Int4Handle:
    """Stands in for the K / V tensors of a decode step over an Int4KVLayer; RDAttention.exact_attention calls `attend`
    (the protocol of the reference's compressed-cache handle, modal_rd/turbo_kv.py:129-141)."""

    def __init__(self, layer, shape):
        self.turbo, self.shape = layer, shape

    def attend(self, q, scale):
        """q [1, H, t, d] -> [1, H, t, d] attention of every query over the layer's whole cache. The step's new rows, when
        the layer still holds them, are quantised by the same call (decode_int4_append). More queries than a few passes
        take attend the cache read back."""
        layer = self.turbo
        groups = q.shape[1] // layer.store_k.q.shape[0]
        if q.shape[2] > MAX_TOKENS or q.shape[2] * groups > _HANDLE_VECTORS:
            k, v = layer.read_back(q.dtype)
            return exact_attention(q[0], k, v, num_heads=q.shape[1], kv_groups=groups, scale=scale)[None]
        cache = (*layer.store_k.packed(), *layer.store_v.packed())
        rows = q[0].transpose(0, 1)
        pending = layer._pending
        if pending is not None and pending[0].shape[1] == rows.shape[0] and pending[2] == layer.n - rows.shape[0]:
            out = decode_int4_append(rows, *cache, pending[0], pending[1], layer.n, scale)
            layer._pending = None
        else:
            layer._flush()
            out = decode_int4(rows, *cache, layer.n, scale)
        return out.transpose(0, 1)[None]


class _Int4Rows:
    """One cached tensor (K or V): codes [Hkv, capacity, d / 2] and params [Hkv, capacity, d / 32, 2]; rows [0, n) are
    valid (n is kept by the owning layer). Capacity comes in GROW-row steps past what is needed."""

    def __init__(self, hkv, d, rows, device):
        if d not in _HEAD_DIMS:
            raise ValueError("quantize4: rows [..., t, d] with d 32, 64, 128 or 256")
        self.q, self.p = _new_packed((hkv, rows + GROW), d, device)

    @property
    def capacity(self):
        return self.q.shape[1]

    def packed(self):
        return self.q, self.p

    def takes(self, x):
        """Whether rows x [Hkv, t, d] fit this store."""
        return x.shape[0] == self.q.shape[0] and x.shape[2] == 2 * self.q.shape[2] and x.get_device() == self.q.get_device()

    def ensure(self, n, need):
        """Make room for rows [n, need), keeping rows [0, n)."""
        if need <= self.capacity:
            return
        old_q, old_p = self.q, self.p
        self.q = old_q.new_empty(old_q.shape[0], need + GROW, old_q.shape[2])
        self.p = old_p.new_empty(old_p.shape[0], need + GROW, *old_p.shape[2:])
        self.q[:, :n].copy_(old_q[:, :n])
        self.p[:, :n].copy_(old_p[:, :n])

    def rows(self, a, b):
        return self.q[:, a:b], self.p[:, a:b]

    def dequantized(self, n, dtype):
        """[1, Hkv, n, d] in `dtype`."""
        return dequantize4(*self.rows(0, n), dtype)[None]

    def nbytes(self, n):
        return n * self.q.shape[0] * (self.q.shape[2] + 2 * self.p[0, 0].numel())


class Int4KVLayer(Int8KVLayer):
    """HF cache layer with 4-bit K/V storage, batch size 1; the protocol of Int8KVLayer:

    * prefill (the first update): the K/V are quantised into fresh row stores and the full-precision inputs are returned;
    * later updates quantise the new rows (K and V in one launch) into spare capacity and return the dequantised cache,
      or, for a step of at most `attend_tokens` tokens behind cached ones (or of one token) whose consumer opts in (cache
      kwargs {"bb_attend": True}) on a bf16 or fp16 model with head_dim 64 or 128, Int4Handle stand-ins for decode_int4;
    * assigning `keys` / `values` (kv_evict compacting the cache) re-quantises the given rows;
    * `crop(-r)` drops the last r rows.
    """

    attend_tokens = MAX_TOKENS

    def _flush(self):
        """Quantise a step's rows still held for the fused decode (the handle was not attended)."""
        if self._pending is not None:
            self._write(*self._pending)
            self._pending = None  # only now: a write that fails keeps the rows

    def _write(self, kr, vr, row):
        end = row + kr.shape[1]
        quantize4_pair(kr, vr, self.store_k.rows(row, end), self.store_v.rows(row, end))

    @staticmethod
    def _heads(x):
        """[1, Hkv, t, d] -> [Hkv, t, d]."""
        if x.ndim != 4 or x.shape[0] != 1:
            raise NotImplementedError("Int4KVLayer is batch-size-1 only")
        return x[0]

    def _fill(self, x):
        rows = self._heads(x)
        h, t, d = rows.shape
        store = _Int4Rows(h, d, t, x.device)
        quantize4(rows, store.rows(0, t))
        return store

    def update(self, key_states, value_states, cache_kwargs=None, *args, **kwargs):
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        self._flush()
        kr, vr = self._heads(key_states), self._heads(value_states)
        h, t, d = kr.shape
        if self.store_k is None:
            sk, sv = _Int4Rows(h, d, t, kr.device), _Int4Rows(h, d, t, kr.device)
            quantize4_pair(kr, vr, sk.rows(0, t), sv.rows(0, t))
            self.store_k, self.store_v, self.n = sk, sv, t  # only now: rows that are refused leave the layer empty
            return key_states, value_states
        if vr.shape != kr.shape or not (self.store_k.takes(kr) and self.store_v.takes(vr)):
            raise ValueError("Int4KVLayer: K and V rows must have the cache's heads, head_dim and device, and be as many")
        start, end = self.n, self.n + t
        self.store_k.ensure(start, end)
        self.store_v.ensure(start, end)
        wants_handle = isinstance(cache_kwargs, dict) and cache_kwargs.get("bb_attend", False)
        # a handle's queries attend every row; several tokens that are the whole cache are a prompt, attended causally
        if (self.fused and wants_handle and 1 <= t <= self.attend_tokens and (start or t == 1) and d in (64, 128)
                and kr.dtype in (torch.bfloat16, torch.float16) and vr.dtype == kr.dtype):
            # quantised when the handle is attended (or by _flush before any other use of the cache)
            self._pending, self.n = (kr, vr, start), end
            handle = Int4Handle(self, (1, h, end, d))
            return handle, handle
        self._write(kr, vr, start)
        self.n = end
        k, v = self.read_back(self.dtype)
        return k[None], v[None]

    def read_back(self, dtype):
        """The cached K and V [Hkv, n, d] in `dtype`, one launch."""
        self._flush()
        return dequantize4_pair(self.store_k.rows(0, self.n), self.store_v.rows(0, self.n), dtype)

    def reset(self):
        """Every row zero, in place, as DynamicLayer's (whose own form would zero the dequantised copies)."""
        self._pending = None
        for store in (self.store_k, self.store_v):
            if store is not None:
                for part in store.rows(0, self.n):
                    part.zero_()

    def batch_repeat_interleave(self, repeats):
        raise NotImplementedError("Int4KVLayer is batch-size-1 only")

    def batch_select_indices(self, indices):
        raise NotImplementedError("Int4KVLayer is batch-size-1 only")


def make_int4_cache(config, fused=True):
    """A DynamicCache whose layers are Int4KVLayer. `fused=False` never hands out decode handles, even to consumers that
    ask for them."""
    cache = DynamicCache(config=config)
    layers = []
    for _ in range(config.get_text_config(decoder=True).num_hidden_layers):
        layer = Int4KVLayer()
        layer.fused = fused
        layers.append(layer)
    cache.layers = layers
    return cache
