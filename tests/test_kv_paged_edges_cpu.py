"""Paged KV cache without a GPU, at its edges: steps that are taken back, masks, and calls that are refused before a launch."""
import ctypes

import pytest
import torch
from torch.nn.attention.flex_attention import create_block_mask

from bigger_bird_amd import _lib
from bigger_bird_amd.kv_paged import _append_plan, _attention_plan, _step_plan
from test_kv_paged_cpu import P16, _append, _attention, _cache, _consistent, _run, _s, _step

P16_ODD = ctypes.c_void_p(24)


def _two(lengths=(20, 10)):
    c = _cache(batch=2, pages=9, page=16)
    c.extend(lengths)
    _run(c, max(lengths), positions=2)
    return c


@pytest.mark.parametrize("begun", [False, True])
def test_a_step_that_did_not_run_leaves_no_rows(begun):
    """release and crop while a step is under way (not run at all, or by the first layer only) count the rows before it alone: the
    step's were not written in every layer."""
    for take, want in ((lambda c: c.release(0), [0, 10]), (lambda c: c.crop(-1), [19, 9]), (lambda c: c.crop(0), [20, 10]),
                       (lambda c: c.release([]), [20, 10]), (lambda c: c.truncate([20, 7]), [20, 7]),
                       (lambda c: c.reset(), [0, 0])):
        c = _two()
        c.extend([3, 24])
        if begun:
            c.layers[0].begin(24, False, 2)
        take(c)
        assert c.lengths == want and not c._left and c.new.tolist() == [0, 0]
        assert c.get_seq_length() == max(want) and c.positions(1).tolist() == [[n] for n in want]
        _consistent(c)
        _run(c, 1, positions=2)  # and the next step goes on from there
        assert c.lengths == [n + 1 for n in want]
        _consistent(c)


def test_truncate_refuses_rows_that_were_not_written():
    c = _two()
    c.extend([3, 24])
    for bad in ([21, 10], [20, 34]):
        with pytest.raises(ValueError, match="rows that it has"):
            c.truncate(bad)
    assert c._left and c.lengths == [23, 34]  # refused before anything changed
    _consistent(c)
    _run(c, 24, positions=2)
    c.truncate([21, 34])
    assert c.lengths == [21, 34]
    _consistent(c)


# ---------------------------------------------------------------- the C ABI's checks
@pytest.mark.parametrize("over,msg", [
    (dict(out=P16_ODD), "16-byte alignment"),
    (dict(so=_s(4096, 130, 4096)), "16-byte alignment"),
    (dict(scale=0.0), "scale must be positive"),
    (dict(B=1, T=128, H=1 << 15, Hkv=1), "lengths out of range"),
])
def test_a_step_of_many_vectors_is_refused_before_it_writes(over, msg):
    """64 tokens of four heads a KV head are two launches, the append and the attention: what the second refuses is refused before
    the first (which there is no GPU for here, so that its error would be another)."""
    rc, err = _step(**{**dict(T=64, ws=P16, ws_bytes=1 << 40), **over})
    assert rc == -1 and msg in err, err


def test_no_workspace_for_a_call_that_is_refused():
    L = _lib.lib()
    assert L.bb_paged_step_workspace(1, 64, 32, 8, 128, 64, 4) == 64 * 32 * 128 * 2
    for bad in [(1, 128, 1 << 15, 1, 128, 64, 4), (1, 64, 32, 8, 96, 64, 4), (1, 64, 30, 8, 128, 64, 4), (1, 64, 32, 8, 128, 64, 0)]:
        assert L.bb_paged_attention_workspace(*bad) == 0 and L.bb_paged_step_workspace(*bad) == 0


@pytest.mark.parametrize("sizes", [dict(B=1 << 15, T=1 << 30, H=65534, Hkv=1), dict(B=65535, T=(1 << 31) - 1, H=(1 << 31) - 1, Hkv=1)])
def test_more_rows_than_64_bits_count(sizes):
    rc, err = _append(**sizes)
    assert rc == -1 and "too many rows" in err, err


@pytest.mark.parametrize("sizes", [dict(B=64, T=4096, W=32768), dict(B=64, T=4096, W=1 << 22), dict(B=60000, T=1, W=1 << 22)])
def test_a_wide_table_is_no_reason_to_refuse(sizes):
    """How many sequences a call may have does not go by the rows that its table has room for."""
    rc, err = _attention(**sizes)
    assert rc == -1 and "workspace of" in err, err
    rc, err = _step(**{**sizes, "scale": 0.0, "ws": P16, "ws_bytes": 1 << 50})
    assert rc == -1 and "scale must be positive" in err, err
    a = dict(B=64, T=1, H=32, Hkv=8, D=128, page=64, W=4) | sizes
    L = _lib.lib()
    assert 0 < L.bb_paged_attention_workspace(*a.values()) <= L.bb_paged_step_workspace(*a.values())
    rc, err = _attention(**{**sizes, "B": 65535, "T": 1 << 13})  # but by its own tiles
    assert rc == -1 and "out of range" in err, err


# ---------------------------------------------------------------- the Python calls' checks
def _layout(*shape, stride=None, dtype=torch.bfloat16):
    """What the plans go by, of a tensor that could lie on the first GPU."""
    x = torch.empty_strided(shape, stride, dtype=dtype, device="meta") if stride else torch.empty(shape, dtype=dtype, device="meta")
    return x.shape, x.stride(), x.dtype, 0


@pytest.mark.parametrize("d,wide", [(100, 104), (96, 96), (32, 32), (256, 256), (65, 72)])
def test_other_head_dims_are_refused_by_the_plans(d, wide):
    """Rows of 100 elements in pages padded to 104 cannot be copied to aligned rows: they are refused before that is tried."""
    pages = _layout(3, 2, 16, d, stride=(2 * 16 * wide, 16 * wide, wide, 1))
    table, lens = _layout(1, 2, dtype=torch.int32), _layout(1, dtype=torch.int32)
    q, k = _layout(1, 4, 1, d), _layout(1, 2, 1, d)
    for call in (lambda: _attention_plan(q, pages, pages, table, lens, None),
                 lambda: _append_plan(k, k, pages, pages, table, lens, None, None, None, None),
                 lambda: _step_plan(q, k, k, pages, pages, table, lens, None, None, None)):
        with pytest.raises(ValueError, match=f"head_dim {d} unsupported"):
            call()


# ---------------------------------------------------------------- masks
def _masks(t):
    causal = torch.ones(1, 1, t, t, dtype=torch.bool).tril()
    bias = torch.where(causal, 0.0, torch.finfo(torch.float32).min)
    left, right, packed = causal.clone(), causal.clone(), causal.clone()
    left[..., :2] = False
    right[..., t - 1] = False
    packed[..., t // 2:, :t // 2] = False
    padded = torch.ones(1, t, dtype=torch.long)
    padded[0, 0] = 0
    blocks = [create_block_mask(f, 1, None, t, t, device="cpu") for f in
              (lambda b, h, i, j: j <= i, lambda b, h, i, j: (j <= i) & (padded[b, j] != 0))]
    plain = [blocks[0], torch.ones(1, 1, 0, 0, dtype=torch.bool), causal, bias, bias.to(torch.bfloat16),
             torch.ones(1, t, dtype=torch.long), torch.ones(1, t, dtype=torch.bool)]
    hiding = [blocks[1], left, right, packed, torch.where(left, 0.0, -float("inf")), torch.where(right, 0.0, torch.finfo(torch.float32).min),
              padded, padded.bool(), object()]
    return plain, hiding


def test_a_mask_that_hides_rows_of_one_sequence_is_refused():
    """A mask is not read by the attention. One sequence takes the causal mask that some attention implementations always make, and
    is refused one that hides any of its rows from its last token; a step that extend began goes by its counts."""
    plain_masks, hiding = _masks(6)
    for mask in plain_masks:
        c = _cache(batch=1)
        for layer in c.layers:
            layer.begin(6, mask, 1)
        assert c.lengths == [6] and not c._left
    for mask in (*hiding, True):
        c = _cache(batch=1)
        with pytest.raises(ValueError, match="by a mask"):
            c.layers[0].begin(6, mask, 1)
        assert c.lengths == [0] and not c._left
        c.extend([4])
        for layer in c.layers:
            layer.begin(6, mask, 1)
        assert c.lengths == [4]
    c = _cache(batch=2)  # several sequences: any mask, as before
    for mask in (*plain_masks, *hiding):
        with pytest.raises(ValueError, match="by a mask"):
            c.layers[0].begin(6, mask, 1)


def test_rdattention_hands_the_mask_on():
    from types import SimpleNamespace

    from bigger_bird_amd import RDAttention

    lin, kv = torch.nn.Linear(256, 256, bias=False), torch.nn.Linear(256, 128, bias=False)
    base = SimpleNamespace(config=SimpleNamespace(num_attention_heads=4, num_key_value_heads=2), layer_idx=0, head_dim=64,
                           scaling=0.125, q_proj=lin, k_proj=kv, v_proj=kv, o_proj=lin)
    pe = torch.ones(1, 6, 64), torch.zeros(1, 6, 64)
    plain_masks, hiding = _masks(6)
    with torch.no_grad():
        for mask in hiding:
            c = _cache(batch=1)
            with pytest.raises(ValueError, match="by a mask"):
                RDAttention(base)(torch.zeros(1, 6, 256), pe, mask, c)
            assert c.lengths == [0]
        for mask in plain_masks:  # taken, up to the rows' dtype (fp32 here), which the step refuses on any device
            with pytest.raises(ValueError, match="ROCm device only"):
                RDAttention(base)(torch.zeros(1, 6, 256), pe, mask, _cache(batch=1))
