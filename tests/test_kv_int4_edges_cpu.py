"""4-bit KV cache without a GPU: the host's layouts, limits and the cache layer's bookkeeping at their edges."""
import math

import pytest
import torch

from bigger_bird_amd import kv_int4

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _at(x, elements):
    """x's values, contiguous, `elements` elements past an aligned address."""
    buf = torch.empty(x.numel() + elements, dtype=x.dtype, device=x.device)
    return buf[elements:].view(x.shape).copy_(x)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rows_are_copied_to_an_aligned_place(dtype):
    """Contiguous tensors at any address, and odd strides of dimensions of length 1, which torch counts as contiguous too."""
    gen = torch.Generator().manual_seed(3)
    cases = [_at(torch.randn(shape, generator=gen).to(dtype), o) for o in (1, 2, 3) for shape in
             ((5, 128), (2, 5, 64), (3, 2, 5, 32), (1, 1, 128))]
    cases += [torch.randn(1, 1, 131, generator=gen).to(dtype)[..., :128], torch.randn(1, 7, 132, generator=gen).to(dtype)[:, :1, :128]]
    for x in cases:
        y = kv_int4._input_rows(x)
        el = y.element_size()
        assert y.ndim == 3 and torch.equal(y, x.reshape(-1, *x.shape[-2:]))
        assert y.data_ptr() % 16 == 0 and y.stride(-1) == 1 and not any(s * el % 16 for s in y.stride()[:2])
        if dtype is not FP32 and x.ndim == 3:
            y = kv_int4._rows16(x)
            assert torch.equal(y, x) and y.data_ptr() % 16 == 0 and y.stride(-1) == 1 and not any(s % 8 for s in y.stride()[:2])
    x = torch.zeros(2, 5, 128, dtype=dtype)
    assert kv_int4._input_rows(x).data_ptr() == x.data_ptr(), "aligned rows are taken where they are"


def _layer(hk=2, n=5, d=64, dtype=BF16, monkeypatch=None):
    """A layer that holds n rows, on the CPU (its stores are never launched on)."""
    layer = kv_int4.Int4KVLayer()
    layer.lazy_initialization(torch.zeros(1, hk, n, d, dtype=dtype), None)
    layer.store_k, layer.store_v, layer.n = kv_int4._Int4Rows(hk, d, n, "cpu"), kv_int4._Int4Rows(hk, d, n, "cpu"), n
    return layer


def test_refused_write_keeps_the_pending_rows(monkeypatch):
    """Rows behind a handle stay with the layer until a write of them has succeeded."""
    layer = _layer()
    x = torch.randn(1, 2, 1, 64).to(BF16)
    layer.update(x, x, {"bb_attend": True})
    pending, calls = layer._pending, []
    assert pending is not None and layer.n == 6

    def refuse(*a):
        raise RuntimeError("out of memory")

    monkeypatch.setattr(kv_int4, "quantize4_pair", refuse)
    with pytest.raises(RuntimeError):
        layer.nbytes()
    assert layer._pending is pending and layer.n == 6
    monkeypatch.setattr(kv_int4, "quantize4_pair", lambda *a: calls.append(a))
    layer.nbytes()
    assert layer._pending is None and len(calls) == 1
    assert torch.equal(calls[0][0], x[0]) and calls[0][2][0].data_ptr() == layer.store_k.q[:, 5:].data_ptr()


@pytest.mark.parametrize("k,v", [((1, 3, 1, 64), (1, 3, 1, 64)), ((1, 2, 1, 128), (1, 2, 1, 128)), ((1, 2, 1, 64), (1, 2, 1, 128)),
                                 ((1, 2, 1, 64), (1, 1, 1, 64)), ((1, 2, 1, 64), (1, 2, 2, 64))])
@pytest.mark.parametrize("attend", [True, False])
def test_rows_of_another_shape_are_refused_at_once(k, v, attend):
    """A step whose rows do not fit the cache is refused by the update, before the layer counts them."""
    layer = _layer()
    with pytest.raises(ValueError, match="rows"):
        layer.update(torch.zeros(k, dtype=BF16), torch.zeros(v, dtype=BF16), {"bb_attend": attend})
    assert layer.n == 5 and layer._pending is None and layer.store_k.capacity == 5 + kv_int4.GROW


def test_handles_need_rows_before_the_step(monkeypatch):
    """A handle's queries attend every row. That is a cached step; several tokens that are the whole cache are a prompt, which
    RDAttention attends causally from K and V themselves."""
    layer = _layer()
    monkeypatch.setattr(kv_int4, "quantize4_pair", lambda *a: None)
    monkeypatch.setattr(kv_int4, "dequantize4_pair", lambda k, v, dtype: (torch.zeros(*k[0].shape[:2], 64),) * 2)
    for held, t, handle in ((5, 3, True), (5, 1, True), (0, 3, False), (0, 1, True)):
        layer.crop(-100)
        layer.n = held
        x = torch.zeros(1, 2, t, 64, dtype=BF16)
        k, v = layer.update(x, x, {"bb_attend": True})
        assert isinstance(k, kv_int4.Int4Handle) == handle and layer.n == held + t, (held, t)
        if not handle:
            assert k.shape == v.shape == (1, 2, held + t, 64) and layer._pending is None


@pytest.mark.parametrize("lead", [(0,), (2, 0), (1, 8, 0), (2, 0, 5), (0, 2, 5), (3, 2, 2, 0)])
def test_layouts_without_rows(lead):
    """No rows, or no heads, in any number of dimensions."""
    q, p = kv_int4._new_packed(lead, 128, "cpu")
    h, t, d, _, _ = kv_int4._packed("quantize4", q, p)
    assert (h, t, d) == (math.prod(lead[:-1]), lead[-1], 128)


@pytest.mark.parametrize("heads,rows,write,read", [
    (8, 2 ** 26, False, True), (64, 2 ** 23, False, True), (8, 2 ** 26 - 32, True, True), (1, 2 ** 28 - 16, True, True),
    (1, 2 ** 28, False, False), (2, 2 ** 28, False, False)])
def test_limits_over_several_heads(heads, rows, write, read):
    """A write takes less than 2^36 elements over all heads and less than 2^35 a head, a read back less than 2^35 a head, whatever
    the heads. (A size that is taken meets the refusal of a misaligned pointer behind that check: nothing is launched.)"""
    from bigger_bird_amd import _lib

    L, at = _lib.lib(), 1 << 20
    sx, sc = _lib.i64s(rows * 128, 128), _lib.i64s(rows * 64, rows * 8, rows * 64, rows * 8)
    for taken, call in ((write, lambda: L.bb_int4_quantize(at + 8, sx, None, None, 0, heads, rows, 128, at, at, None, None, sc, None)),
                        (read, lambda: L.bb_int4_dequantize(at, at, None, None, sc, heads, rows, 128, at + 8, None, 0, None))):
        with pytest.raises(ValueError, match="aligned" if taken else "out of range"):
            _lib.check(call())


def test_reset_zeroes_the_rows_in_place(monkeypatch):
    """DynamicLayer.reset: every cached value is zero, the length and the buffers stay; rows behind a handle are rows like any."""
    layer = _layer()
    for store in (layer.store_k, layer.store_v):
        store.q.fill_(0x5A)
        store.p.fill_(2.0)
    x = torch.ones(1, 2, 2, 64, dtype=BF16)
    layer.update(x, x, {"bb_attend": True})
    buffers = [y.data_ptr() for s in (layer.store_k, layer.store_v) for y in s.packed()]
    layer.reset()
    assert layer.n == 7 and layer._pending is None
    assert buffers == [y.data_ptr() for s in (layer.store_k, layer.store_v) for y in s.packed()]
    for store in (layer.store_k, layer.store_v):
        assert not store.q[:, :7].any() and not store.p[:, :7].any()
    kv_int4.Int4KVLayer().reset()  # a layer that holds nothing


def test_reset_of_a_layer_with_one_store():
    """Between the assignments of keys and values (kv_evict's) a layer can hold one of the two."""
    layer = _layer()
    layer.store_v = None
    layer.store_k.q.fill_(0x5A)
    layer.reset()
    assert layer.n == 5 and not layer.store_k.q[:, :5].any()
