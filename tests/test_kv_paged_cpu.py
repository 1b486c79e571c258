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
