"""Paged KV cache without a GPU: the C ABI's argument checks (before any launch), the sizes that it asks for, and the plain forms
that the GPU tests compare with."""
import ctypes

import pytest
import torch

import paged_plain as plain
from bigger_bird_amd import _lib, paged_append, paged_attention, paged_step

P16 = ctypes.c_void_p(16)


def _s(*v):
    return _lib.i64s(*v)


def _attention(**over):
    a = dict(q=P16, sq=_s(4096, 128, 4096), k=P16, sk=_s(65536, 8192, 128), v=P16, sv=_s(65536, 8192, 128), table=P16, st=4,
             lens=P16, fresh=None, B=2, T=1, H=32, Hkv=8, D=128, pages=10, page=64, W=4, is_f16=0, scale=1.0, out=P16,
             so=_s(4096, 128, 4096), ws=None, ws_bytes=0, stream=None)
    a.update(over)
    L = _lib.lib()
    return L.bb_paged_attention(*a.values()), L.bb_last_error().decode()


def _append(**over):
    a = dict(k=P16, skn=_s(1024, 128, 1024), v=P16, svn=_s(1024, 128, 1024), q=P16, sq=_s(4096, 128, 4096), q_out=P16,
             sqo=_s(4096, 128, 4096), cos=P16, sin=P16, sc=_s(128, 128), f32=0, kp=P16, sk=_s(65536, 8192, 128), vp=P16,
             sv=_s(65536, 8192, 128), table=P16, st=4, lens=P16, fresh=None, B=2, T=1, H=32, Hkv=8, D=128, pages=10, page=64,
             W=4, is_f16=0, stream=None)
    a.update(over)
    L = _lib.lib()
    return L.bb_paged_append(*a.values()), L.bb_last_error().decode()


def _step(**over):
    a = dict(q=P16, sq=_s(4096, 128, 4096), k=P16, skn=_s(1024, 128, 1024), v=P16, svn=_s(1024, 128, 1024), cos=P16, sin=P16,
             sc=_s(128, 128), f32=0, kp=P16, sk=_s(65536, 8192, 128), vp=P16, sv=_s(65536, 8192, 128), table=P16, st=4,
             lens=P16, fresh=None, B=2, T=1, H=32, Hkv=8, D=128, pages=10, page=64, W=4, is_f16=0, scale=1.0, out=P16,
             so=_s(4096, 128, 4096), ws=None, ws_bytes=0, stream=None)
    a.update(over)
    L = _lib.lib()
    return L.bb_paged_step(*a.values()), L.bb_last_error().decode()


CACHE = [
    (dict(table=None), "null argument"),
    (dict(lens=None), "null argument"),
    (dict(B=0), "must match"),
    (dict(H=12), "must match"),
    (dict(D=96), "head_dim 96 unsupported"),
    (dict(page=8), "pages of 8 rows unsupported"),
    (dict(page=48), "pages of 48 rows unsupported"),
    (dict(W=0), "empty table"),
    (dict(W=1 << 25), "out of range"),
    (dict(sk=_s(65536, 8192, 100)), "16-byte aligned rows"),
    (dict(sv=_s(-65536, 8192, 128)), "16-byte aligned rows"),
    (dict(sv=_s(65536, 8192, 1 << 27)), "out of range"),
    (dict(sk=_s(1 << 31, 8192, 128)), "out of range"),
    (dict(page=1 << 20, W=1, sk=_s(1 << 27, 1 << 27, 1024)), "out of range"),
    (dict(fresh=ctypes.c_void_p(18)), "misaligned lengths"),
]


@pytest.mark.parametrize("over,msg", CACHE + [
    (dict(q=None), "null argument"),
    (dict(H=0), "must match"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(scale=float("nan")), "scale must be positive"),
    (dict(sq=_s(4096, 130, 4096)), "16-byte alignment"),
    (dict(out=ctypes.c_void_p(8)), "16-byte alignment"),
    (dict(W=64), "workspace of"),
    (dict(B=60000, H=32 * 1024, Hkv=1024, W=4096), "out of range"),
])
def test_attention_refusals(over, msg):
    rc, err = _attention(**over)
    assert rc == -1 and msg in err, err


@pytest.mark.parametrize("over,msg", [(o, m) for o, m in CACHE if "H" not in o] + [
    (dict(k=None), "null argument"),
    (dict(q=None), "null argument"),
    (dict(cos=None), "null argument"),
    (dict(cos=None, sin=None), "cos and sin required"),
    (dict(sc=_s(128, 4)), "cos and sin rows must be 16-byte aligned"),
    (dict(sc=_s(2, 128), f32=1), "cos and sin rows must be 16-byte aligned"),
    (dict(skn=_s(1024, 4, 1024)), "16-byte alignment"),
    (dict(T=1 << 30), "too many rows"),
    (dict(T=(1 << 22) + 1, B=1, H=112), "too many rows"),  # 2^29 rows of 8 lanes and more: more threads than a launch has
])
def test_append_refusals(over, msg):
    rc, err = _append(**over)
    assert rc == -1 and msg in err, err


@pytest.mark.parametrize("over,msg", CACHE + [
    (dict(v=None), "null argument"),
    (dict(scale=-1.0), "scale must be positive"),
    (dict(T=64), "workspace of"),  # more vectors than the step's kernel takes: the rotated queries need room
    (dict(sin=None), "null argument"),
])
def test_step_refusals(over, msg):
    rc, err = _step(**over)
    assert rc == -1 and msg in err, err


def test_workspaces():
    L = _lib.lib()
    # a table of one split's rows: no partials
    assert L.bb_paged_attention_workspace(4, 1, 32, 8, 128, 64, 4) == 0
    long_ = L.bb_paged_attention_workspace(1, 1, 32, 8, 128, 64, 2048)
    assert 0 < long_ < 16 << 20
    # the partials go by the workgroups aimed at, not by the table's width
    assert L.bb_paged_attention_workspace(1, 1, 32, 8, 128, 64, 1 << 20) == long_
    assert L.bb_paged_step_workspace(1, 1, 32, 8, 128, 64, 2048) == long_
    # a chunk's step keeps the rotated queries
    assert (L.bb_paged_step_workspace(2, 512, 32, 8, 128, 64, 2048)
            >= L.bb_paged_attention_workspace(2, 512, 32, 8, 128, 64, 2048) + 2 * 512 * 32 * 128 * 2)
    for bad in [(0, 1, 32, 8, 128, 64, 4), (1, 1, 30, 8, 128, 64, 4), (1, 1, 32, 8, 96, 64, 4), (1, 1, 32, 8, 128, 64, 0)]:
        assert L.bb_paged_attention_workspace(*bad) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device only"):
        paged_attention(x, pages, pages, table, lens, 1.0)
    with pytest.raises(ValueError, match="ROCm device only"):
        paged_append(x, x, pages, pages, table, lens)
    with pytest.raises(ValueError, match="ROCm device only"):
        paged_step(x, x, x, pages, pages, table, lens, 1.0)


def test_plain_form_is_attention_over_contiguous_rows():
    g = torch.Generator().manual_seed(0)
    page, n = 16, 37
    kp, vp = (torch.randn(7, 2, page, 64, generator=g).double() for _ in "kv")
    table = torch.tensor([[5, 0, 3]], dtype=torch.int32)
    q = torch.randn(1, 4, 2, 64, generator=g).double()
    out, tol = plain.attend(q, kp, vp, table, [n], 0.125, None, 0.0)
    k, v = (x[[5, 0, 3]].transpose(0, 1).reshape(2, 48, 64)[:, :n].repeat_interleave(2, 0) for x in (kp, vp))
    x = (q[0] @ k.transpose(1, 2)) * 0.125
    x[:, 0, n - 1] = -torch.inf
    assert torch.allclose(out[0], torch.softmax(x, -1) @ v, atol=1e-12) and (tol >= 0).all()
    # a page that the table does not name is not attended
    table[0, 1] = 9
    out, _ = plain.attend(q, kp, vp, table, [n], 0.125, None, 0.0)
    x[:, :, 16:32] = -torch.inf
    assert torch.allclose(out[0], torch.softmax(x, -1) @ v, atol=1e-12)


# ---------------------------------------------------------------- the cache's lengths and pages
def _cache(batch=3, pages=10, page=16, rows=None, layers=2):
    from transformers import LlamaConfig

    from bigger_bird_amd import make_paged_cache

    cfg = LlamaConfig(vocab_size=32, hidden_size=256, intermediate_size=64, num_hidden_layers=layers, num_attention_heads=4,
                      num_key_value_heads=2)
    return make_paged_cache(cfg, batch, pages, page, rows, device="cpu")


def _run(cache, t, padded=False, positions=1):
    """A forward pass's part in the bookkeeping: every layer begins the step of t columns."""
    for layer in cache.layers:
        layer.begin(t, padded, positions)


def _consistent(cache):
    held = [p for seq in cache._pages for p in seq]
    assert sorted(held + cache._free) == list(range(cache.arena.shape[2]))  # every page once
    for b, pages in enumerate(cache._pages):
        assert len(pages) == -(-cache.lengths[b] // cache.page)
        assert cache.table[b].tolist() == pages + [-1] * (cache.width - len(pages))
    assert cache.lens.tolist() == cache.lengths


def test_cache_steps():
    c = _cache()
    assert c.get_seq_length() == 0 and c.arena.shape == (2, 2, 10, 2, 16, 64) and len(c.layers) == 2
    _run(c, 20)
    _consistent(c)
    assert c.lengths == [20] * 3 and len(c._free) == 4 and c.get_seq_length() == 20 and c._new_of(20) is None
    _run(c, 1)
    assert c.lengths == [21] * 3
    c.extend([0, 12, 1])
    assert c.get_seq_length() == 21 and c.positions().tolist() == [list(range(21, 33))] * 3
    with pytest.raises(ValueError, match="has not run"):
        c.extend([1, 1, 1])
    with pytest.raises(ValueError, match="12 new tokens, the input 5 columns"):
        c.layers[0].begin(5, False, 3)
    _run(c, 13, padded=True)
    assert c.lengths == [21, 33, 22] and c._new_of(13).tolist() == [0, 12, 1] and c.get_seq_length() == 33
    _consistent(c)
    with pytest.raises(ValueError, match="need position_ids"):
        _run(c, 1)
    assert c.lengths == [21, 33, 22]  # refused before anything changed
    _run(c, 1, positions=3)
    assert c.positions(2).tolist() == [[22, 23], [34, 35], [23, 24]]
    _consistent(c)


def test_cache_refusals_change_nothing():
    c = _cache(batch=2, pages=3, page=16, rows=32)
    with pytest.raises(ValueError, match="by a mask"):
        _run(c, 5, padded=True)
    with pytest.raises(ValueError, match="past the rows"):
        c.extend([33, 0])
    with pytest.raises(ValueError, match="no free pages"):
        c.extend([17, 17])
    for bad in ([1], [1, -1]):
        with pytest.raises(ValueError, match="one count"):
            c.extend(bad)
    assert c.lengths == [0, 0] and len(c._free) == 3 and not c._left
    _consistent(c)
    c.extend([17, 16])
    _run(c, 17, positions=2)
    with pytest.raises(ValueError, match="no free pages"):
        _run(c, 1, positions=2)
    assert c.lengths == [17, 16]
    _consistent(c)
    for kw in (dict(page=8), dict(page=48), dict(pages=0), dict(batch=0)):
        with pytest.raises(ValueError, match="PagedCache"):
            _cache(**kw)
    with pytest.raises(ValueError, match="RDAttention only"):
        c.update(torch.zeros(2, 2, 1, 64), torch.zeros(2, 2, 1, 64), 0)


def test_cache_truncate_and_release():
    c = _cache(batch=3, pages=9, page=16)
    c.extend([40, 33, 16])
    _run(c, 40, positions=3)
    c.truncate([32, 33, 0])
    assert c.lengths == [32, 33, 0] and len(c._free) == 4
    _consistent(c)
    for bad in ([33, 33, 0], [32, 33, -1], [32]):
        with pytest.raises(ValueError, match="one length"):
            c.truncate(bad)
    for bad in (3, -1, [0, 3]):
        with pytest.raises(ValueError, match="no such sequence"):
            c.release(bad)
    assert c.lengths == [32, 33, 0]
    c.release(1)
    assert c.lengths == [32, 0, 0] and len(c._free) == 7
    _consistent(c)
    c.extend([0, 90, 5])  # a step that does not run is taken back
    c.truncate([32, 0, 0])
    _consistent(c)
    c.crop(-3)
    assert c.lengths == [29, 0, 0]
    with pytest.raises(NotImplementedError):
        c.crop(3)
    c.release([0, 2])
    assert c.nbytes() == 0 and len(c._free) == 9
    c.reset()
    _consistent(c)


def test_rdattention_refuses_what_a_paged_cache_cannot_do():
    from types import SimpleNamespace

    from bigger_bird_amd import RDAttention

    c = _cache(batch=2)
    lin = torch.nn.Linear(256, 256, bias=False)
    kv = torch.nn.Linear(256, 128, bias=False)
    base = SimpleNamespace(config=SimpleNamespace(num_attention_heads=4, num_key_value_heads=2), layer_idx=0, head_dim=64,
                           scaling=0.125, q_proj=lin, k_proj=kv, v_proj=kv, o_proj=lin)
    pe = torch.ones(1, 3, 64), torch.zeros(1, 3, 64)
    with pytest.raises(ValueError, match="holds no gradients"):
        RDAttention(base)(torch.zeros(2, 3, 256), pe, None, c)
    with torch.no_grad():
        with pytest.raises(ValueError, match="kv_evict"):
            RDAttention(base, kv_evict=True)(torch.zeros(2, 3, 256), pe, None, c)
        with pytest.raises(ValueError, match="2 sequences, the input has 3"):
            RDAttention(base)(torch.zeros(3, 3, 256), pe, None, c)
        with pytest.raises(ValueError, match="by a mask"):
            RDAttention(base)(torch.zeros(2, 3, 256), pe, torch.zeros(2, 1, 3, 3), c)
    assert c.lengths == [0, 0]
