"""4-bit KV cache without a GPU: the plain form's properties, the C ABI's and the Python surface's refusals (all before any
launch), and the cache layer's bookkeeping of refused calls."""
import ctypes

import pytest
import torch

import int4_plain as plain
from bigger_bird_amd import _lib, decode_int4, dequantize4, make_int4_cache, quantize4
from bigger_bird_amd.kv_int4 import Int4KVLayer

FAKE = 1 << 20  # an aligned address that no refused call reads


def test_plain_form_bounds():
    """Every value is off by at most half a scale, and by what the fp16 roundings of s and z take at the ends (15 steps of
    2^-11 s each, 2^-11 |z|); packing and unpacking agree; the two ends of a group are codes 0 and 15."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(3, 50, 128, generator=gen) * torch.exp(torch.randn(128, generator=gen))
    code, s, z = plain.quantize(x)
    q, p = plain.pack(code, s, z)
    assert torch.equal(plain.codes(q).double(), code)
    v, spread = plain.values(q, p)
    zz = z.repeat_interleave(32, -1).abs()
    assert ((v - x.double()).abs() <= spread * (0.5 + 15 * 2.0 ** -11) + zz * 2.0 ** -11 + 1e-7).all()
    g = code.unflatten(-1, (-1, 32))
    assert (g.amin(-1) == 0).all() and (g.amax(-1) == 15).all()


def test_plain_attention_is_softmax_attention():
    gen = torch.Generator().manual_seed(2)
    k, v = torch.randn(2, 40, 64, generator=gen), torch.randn(2, 40, 64, generator=gen)
    kq, vq = plain.pack(*plain.quantize(k)), plain.pack(*plain.quantize(v))
    q = torch.randn(3, 4, 64, generator=gen)
    kd, vd = (plain.values(*x)[0].repeat_interleave(2, 0) for x in (kq, vq))
    mask = torch.arange(40) <= torch.arange(37, 40)[:, None]
    for causal in (False, True):
        want = torch.nn.functional.scaled_dot_product_attention(
            q.double().transpose(0, 1), kd, vd, attn_mask=mask if causal else None, scale=0.3).transpose(0, 1)
        got, tol = plain.attend(q, *kq, *vq, 40, 0.3, causal)
        assert (got - want).abs().max() < 1e-12 and (tol > 0).all()


def _refused(rc, text):
    assert rc == -1
    with pytest.raises(ValueError, match=text):
        _lib.check(rc)


def _decode(**kw):
    a = dict(q=FAKE, sq=(1024, 128), kq=FAKE, kp=FAKE, vq=FAKE, vp=FAKE, sc=(64000, 8000, 64000, 8000), n=1000, n_dev=None,
             cap=1000, T=1, H=8, Hkv=2, D=128, f16=0, scale=0.1, causal=0, out=FAKE, so=(1024, 128), ws=FAKE,
             ws_bytes=1 << 30)
    a.update(kw)
    for key in ("sq", "sc", "so"):
        a[key] = None if a[key] is None else _lib.i64s(*a[key])
    return tuple(a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "null"), (dict(vq=None), "null"), (dict(kp=None), "null"), (dict(sc=None), "null"),
    (dict(kq=FAKE + 8), "aligned"), (dict(vp=FAKE + 2), "aligned"), (dict(sc=(64000, 8001, 64000, 8000)), "aligned"),
    (dict(sc=(64008, 8000, 64000, 8000)), "aligned"), (dict(H=7), "must match"), (dict(Hkv=0), "must match"),
    (dict(D=32), "head_dim 32"), (dict(D=256), "head_dim 256"), (dict(T=0), "1 to 16"), (dict(T=17), "1 to 16"),
    (dict(n=0), "empty"), (dict(n=-1), "empty"), (dict(cap=0), "empty"), (dict(n=1001), "capacity"),
    (dict(n=3, T=4), "at least as long"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(q=FAKE + 8), "aligned"), (dict(sq=(1024, 132)), "aligned"), (dict(out=FAKE + 4), "aligned"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=100), "workspace"),
    (dict(n=1 << 34, cap=1 << 34, sc=(0, 0, 0, 0)), "out of range"), (dict(n_dev=FAKE, cap=2 ** 63 - 1), "out of range"),
    (dict(n_dev=FAKE, ws_bytes=100), "workspace")])
def test_decode_refusals(kw, text):
    _refused(_lib.lib().bb_int4_decode(*_decode(**kw), None), text)


@pytest.mark.parametrize("new,text", [
    ((None, (1, 8), FAKE, (8, 8)), "null"), ((FAKE, None, FAKE, (8, 8)), "null"),
    ((FAKE + 2, (8, 8), FAKE, (8, 8)), "aligned"), ((FAKE, (8, 4), FAKE, (8, 8)), "aligned"),
    ((FAKE, (8, 8), FAKE, (9, 8)), "aligned")])
def test_append_refusals(new, text):
    a = _decode()
    k, sk, v, sv = (x if not isinstance(x, tuple) else _lib.i64s(*x) for x in new)
    _refused(_lib.lib().bb_int4_decode_append(*a[:7], k, sk, v, sv, *a[7:], None), text)


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(D=48), "head_dim 48"), (dict(kind=3), "element kind"), (dict(x=FAKE + 4), "aligned"),
    (dict(sx=(132, 128)), "aligned"), (dict(rows=1 << 40), "out of range"), (dict(rows=-1), "out of range"),
    (dict(heads=1, rows=(0xffffff + 1) * 16), "out of range"), (dict(heads=70000), "out of range"),
    (dict(vq=None), "null"), (dict(sc=(8, 8, 16, 8)), "aligned")])
def test_write_and_read_refusals(kw, text):
    a = dict(x=FAKE, sx=(1280, 128), kind=0, heads=2, rows=10, D=128, q=FAKE, p=FAKE, vq=FAKE, vp=FAKE,
             sc=(640, 80, 640, 80))
    a.update(kw)
    sx, sc = _lib.i64s(*a["sx"]), _lib.i64s(*a["sc"])
    L = _lib.lib()
    _refused(L.bb_int4_quantize(a["x"], sx, FAKE, sx, a["kind"], a["heads"], a["rows"], a["D"], a["q"], a["p"], a["vq"],
                                a["vp"], sc, None), text)
    if "x" in kw or "sx" in kw:
        return
    _refused(L.bb_int4_dequantize(a["q"], a["p"], a["vq"], a["vp"], sc, a["heads"], a["rows"], a["D"], FAKE, FAKE,
                                  a["kind"], None), text)


def test_empty_writes_launch_nothing():
    L = _lib.lib()
    sx, sc = _lib.i64s(128, 128), _lib.i64s(64, 8, 64, 8)
    assert L.bb_int4_quantize(FAKE, sx, FAKE, sx, 0, 2, 0, 128, FAKE, FAKE, FAKE, FAKE, sc, None) == 0
    assert L.bb_int4_dequantize(FAKE, FAKE, None, None, sc, 0, 5, 128, FAKE, None, 0, None) == 0


def test_workspace_grows_with_the_call():
    L = _lib.lib()
    assert L.bb_int4_decode_workspace(0, 1, 8, 2, 128) == 0 and L.bb_int4_decode_workspace(10, 1, 0, 2, 128) == 0
    small, large = (L.bb_int4_decode_workspace(n, 1, 32, 8, 128) for n in (1000, 131072))
    assert 0 < small < large <= 256 * 1024 * 1024
    for t, d in ((1, 128), (1, 64), (4, 128), (16, 64)):  # one split: nothing to merge
        one = L.bb_int4_decode_one_split(t * 4, d)
        assert one >= 256 and L.bb_int4_decode_workspace(one, t, 32, 8, d) == 0
        assert L.bb_int4_decode_workspace(one + 1, t, 32, 8, d) > 0
    sizes = [L.bb_int4_decode_workspace(n, 2, 12, 4, 64) for n in range(1, 40000, 37)]
    assert sizes == sorted(sizes), "a workspace for the capacity serves every length"
    assert L.bb_int4_decode_workspace(131072, 4, 32, 8, 128) >= 4 * large // 2


def test_python_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="ROCm device"):
        quantize4(torch.zeros(2, 4, 128))
    with pytest.raises(ValueError, match="ROCm device"):
        dequantize4(torch.zeros(2, 4, 64, dtype=torch.uint8), torch.zeros(2, 4, 4, 2, dtype=torch.float16), torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm device"):
        decode_int4(torch.zeros(8, 128, dtype=torch.bfloat16), *[torch.zeros(2, 4, 64, dtype=torch.uint8),
                    torch.zeros(2, 4, 4, 2, dtype=torch.float16)] * 2, 4, 0.1)
    with pytest.raises(ValueError, match="d 32, 64, 128 or 256"):
        quantize4(torch.zeros(2, 4, 100))


def test_layer_refusals_leave_it_empty():
    layer = Int4KVLayer()
    for x, kind in ((torch.zeros(2, 2, 5, 64), NotImplementedError), (torch.zeros(1, 2, 5, 64), ValueError),
                    (torch.zeros(1, 2, 5, 80), ValueError)):
        with pytest.raises(kind):
            layer.update(x, x)
        assert layer.get_seq_length() == 0 and layer.store_k is None
    for call in (layer.batch_repeat_interleave, layer.batch_select_indices):
        with pytest.raises(NotImplementedError):
            call(2)


def test_make_int4_cache():
    from transformers import LlamaConfig

    cfg = LlamaConfig(vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=3, num_attention_heads=2,
                      num_key_value_heads=1)
    cache = make_int4_cache(cfg, fused=False)
    assert len(cache.layers) == 3 and all(isinstance(x, Int4KVLayer) and not x.fused for x in cache.layers)
    assert cache.get_seq_length() == 0


def test_ctypes_signatures_match_the_header():
    """The parameter counts that ctypes declares for the 4-bit entry points are those of the header."""
    import re
    from pathlib import Path

    text = re.sub(r"/\*.*?\*/", "", (Path(__file__).resolve().parents[1] / "include" / "bb_attn.h").read_text(), flags=re.S)
    for name, args in re.findall(r"\b(bb_int4_[a-z0-9_]+)\s*\(([^)]*)\)", text):
        assert len(args.split(",")) == len(_lib.SIGNATURES[name][1]), name
    assert ctypes.sizeof(ctypes.c_size_t) == 8
