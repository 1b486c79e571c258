"""Paged KV cache (bigger_bird_amd.kv_paged) on the GPU against the plain 64-bit forms of tests/paged_plain.py: rows and layouts,
ragged and empty sequences, pages that end inside a tile or that the table does not name, values that are not finite, captured
steps, streams and refusals."""
import pytest
import torch

import paged_plain as plain
from bigger_bird_amd import paged_append, paged_attention, paged_step
from paged_plain import HALF_STEP

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
STREAM_VECTORS, STEP_VECTORS = 32, 128  # T * H / Hkv up to which the streaming kernel takes an attention, a step


def _say(*a):
    print("case", *a, flush=True)


def _heads(gen, b, h, t, d, dtype, dev, scale=1.0):
    """[b, h, t, d] as projections leave them: views of [b, t, h * d]."""
    return (torch.randn(b, t, h * d, generator=gen, device=dev) * scale).to(dtype).view(b, t, h, d).transpose(1, 2)


def _pages(gen, p, hk, page, d, dtype, dev, layout="heads"):
    """Random pages: [p, hk, page, d] contiguous, rows before heads in memory, or K and V of a pool that alternates."""
    if layout == "rows":
        return [torch.randn(p, page, hk, d, generator=gen, device=dev).to(dtype).transpose(1, 2) for _ in "kv"]
    if layout == "pool":
        return list(torch.randn(p, 2, hk, page, d, generator=gen, device=dev).to(dtype).unbind(1))
    if layout == "padded":
        return [torch.randn(p, hk + 1, page, d + 8, generator=gen, device=dev).to(dtype)[:, 1:, :, :d] for _ in "kv"]
    return [torch.randn(p, hk, page, d, generator=gen, device=dev).to(dtype) for _ in "kv"]


def _table(gen, lens, page, dev, spare=2, width=None):
    """A table with a page of its own for every row, in random order, and the number of pages; entries past a sequence's rows
    name no page."""
    need = [max(0, -(-max(0, n) // page)) for n in lens]
    width = width or max(1, max(need) + 1)
    order = torch.randperm(sum(need) + spare, generator=gen, device=dev).int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        n = min(n, width)
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def _int(v, dev):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device=dev)


def _angles(gen, b, t, d, dtype, dev):
    a = torch.rand(b, t, d, generator=gen, device=dev) * 6.28
    return a.cos().to(dtype), a.sin().to(dtype)


def _p_step(dtype, streams):
    """Rounding of a probability as an operand: two terms in the streaming kernel, one in the tiles'."""
    return HALF_STEP[dtype] ** (2 if streams else 1)


def _check(got, want, tol, dtype):
    tol = tol + HALF_STEP[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == FP16 else 0.0)
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    worst = (err - tol).argmax()
    assert (err <= tol).all(), f"error {err.flatten()[worst].item():.3e}, tolerance there {tol.flatten()[worst].item():.3e}"


def _attend_case(b_lens, new, T, H, hk, d, page, dtype, dev, layout="heads", seed=0, width=None, holes=False):
    gen = torch.Generator(device=dev).manual_seed(seed)
    table, p = _table(gen, b_lens, page, dev, width=width)
    if holes:
        table.view(-1)[::3] = torch.tensor([-1, p, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev).repeat(
            table.numel())[:len(table.view(-1)[::3])]
    kp, vp = _pages(gen, p, hk, page, d, dtype, dev, layout)
    q = _heads(gen, len(b_lens), H, T, d, dtype, dev)
    return q, kp, vp, table, _int(b_lens, dev), _int(new, dev)


# (lens, new, T, H, Hkv, d, page, dtype)
ATTEND = [
    ([1], None, 1, 8, 2, 128, 16, BF16),
    ([257], None, 1, 32, 4, 64, 16, BF16),
    ([0, 1, 16, 17, 1000, 0, 63], None, 1, 32, 8, 128, 16, BF16),
    ([0, 1, 16, 17, 1000, 0, 63], None, 1, 8, 8, 64, 32, FP16),
    ([9001, 3, 40003], None, 1, 32, 8, 128, 64, BF16),           # several splits of one sequence next to short ones
    ([30011], None, 1, 3, 1, 64, 128, FP16),
    ([131, 70, 2, 4, 0], [3, 1, 2, 0, 3], 3, 8, 2, 128, 16, FP16),  # padding, an idle sequence, rows before the first
    ([500, 2], None, 4, 20, 4, 128, 16, BF16),                      # 20 vectors; tokens without rows
    ([4097], None, 8, 16, 4, 64, 16, BF16),                         # 32 vectors, several splits
    ([700], None, 33, 4, 4, 128, 16, BF16),                         # 33 vectors: one more than the streaming kernel takes
    ([700, 40, 0, 90], [60, 7, 0, 60], 60, 8, 2, 64, 16, FP16),     # padded chunks
    ([300, 129, 64], [300, 129, 64], 300, 8, 2, 128, 32, BF16),     # whole prompts, two tiles of vectors
    ([1025], [1025], 1025, 4, 4, 128, 256, FP16),                   # one query head a KV head
    ([9000, 5000], None, 65, 32, 8, 128, 64, BF16),                 # few rows over long caches: splits of tiles
    ([9000], None, 257, 10, 2, 64, 16, BF16),                       # five query heads a KV head
    ([2100], None, 70, 16, 1, 128, 64, FP16),
]


@pytest.mark.parametrize("lens,new,T,H,hk,d,page,dtype", ATTEND)
def test_attention(lens, new, T, H, hk, d, page, dtype, dev):
    _say("attend", lens, new, T, H, hk, d, page, dtype)
    args = _attend_case(lens, new, T, H, hk, d, page, dtype, dev)
    got = paged_attention(*args[:5], d ** -0.5, new=args[5])
    assert got.shape == (len(lens), H, T, d) and got.dtype == dtype and got.transpose(1, 2).is_contiguous()
    want, tol = plain.attend(*args[:5], d ** -0.5, new, _p_step(dtype, T * H // hk <= STREAM_VECTORS))
    _check(got, want, tol, dtype)
    assert torch.equal(got, paged_attention(*args[:5], d ** -0.5, new=args[5]))  # the same bits again
    for b, n in enumerate(lens):
        for j in range(T):
            if plain.seen(lens, new, T, args[3].shape[1] * page, b, j) == 0:
                assert (got[b, :, j] == 0).all()


@pytest.mark.parametrize("T,H", [(1, 8), (3, 8), (40, 8)])
@pytest.mark.parametrize("layout", ["rows", "pool", "padded"])
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16)])
def test_attention_layouts(T, H, layout, d, dtype, dev):
    """Pages whose rows, heads or K and V alternate in memory, a table that is part of a wider one, queries of other strides."""
    _say("layouts", T, H, layout, d, dtype)
    lens = [517, 33, 200]
    q, kp, vp, table, ln, _ = _attend_case(lens, None, T, H, 4, d, 16, dtype, dev, layout)
    wide = torch.full((3, table.shape[1] + 7), 2 ** 30, dtype=torch.int32, device=dev)
    wide[:, 3:3 + table.shape[1]] = table
    want, tol = plain.attend(q, kp, vp, table, lens, d ** -0.5, None, _p_step(dtype, T * H // 4 <= STREAM_VECTORS))
    for x in (q, q.contiguous(), q.transpose(1, 2).contiguous().transpose(1, 2)[..., :], torch.cat([q, q], -1)[..., :d],
              torch.cat([q[..., :1], q], -1)[..., 1:]):
        _check(paged_attention(x, kp, vp, wide[:, 3:3 + table.shape[1]], ln, d ** -0.5), want, tol, dtype)


@pytest.mark.parametrize("T,H,hk", [(1, 8, 2), (5, 8, 2), (70, 8, 2), (300, 4, 4)])
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16)])
def test_unnamed_pages_are_not_attended(T, H, hk, d, dtype, dev):
    _say("unnamed pages", T, H, hk, d, dtype)
    lens = [2000, 333, 48, 16]
    args = _attend_case(lens, None, T, H, hk, d, 16, dtype, dev, holes=True)
    args[3][3] = -5  # a sequence without any page
    got = paged_attention(*args[:5], d ** -0.5)
    want, tol = plain.attend(*args[:5], d ** -0.5, None, _p_step(dtype, T * H // hk <= STREAM_VECTORS))
    _check(got, want, tol, dtype)
    assert (got[3] == 0).all()


@pytest.mark.parametrize("T", [1, 40])
def test_lengths_past_the_table_and_below_zero(T, dev):
    _say("lengths out of range", T)
    q, kp, vp, table, lens, _ = _attend_case([64, 64, 64, 64], None, T, 8, 2, 128, 16, BF16, dev, width=4)
    for vals, new in (([65, 1000, 2 ** 31 - 1, -1], None), ([70, 64, -2 ** 31, 3], [T + 5, 2 ** 31 - 1, 1, -3])):
        got = paged_attention(q, kp, vp, table, _int(vals, dev), 0.1, new=_int(new, dev))
        want, tol = plain.attend(q, kp, vp, table, vals, 0.1, new, _p_step(BF16, T * 4 <= STREAM_VECTORS))
        _check(got, want, tol, BF16)


@pytest.mark.parametrize("T,G", [(4, 2), (4, 8), (70, 4), (300, 1)])
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16)])
def test_values_that_are_not_finite(T, G, d, dtype, dev):
    """What lies behind a sequence, on pages that it does not own and in rows that a token does not attend never reaches it;
    what it attends does, and a query that is not finite is NaN in its own row only."""
    _say("not finite", T, G, d, dtype)
    n, hk = 407, 2
    q, kp, vp, table, lens, _ = _attend_case([n, n], None, T, hk * G, hk, d, 16, dtype, dev)
    own = torch.zeros(kp.shape[0], 16, dtype=torch.bool, device=dev)
    for b in range(2):
        for r in range(n):
            own[table[b, r // 16].item(), r % 16] = True
    for x in (kp, vp):
        x.masked_fill_(~own[:, None, :, None], float("nan"))
    p_step = _p_step(dtype, T * G <= STREAM_VECTORS)
    want, tol = plain.attend(q, kp, vp, table, lens, d ** -0.5, None, p_step)
    _check(paged_attention(q, kp, vp, table, lens, d ** -0.5), want, tol, dtype)
    # the last token's row: the tokens before it do not attend it
    at = table[0, (n - 1) // 16].item(), slice(None), (n - 1) % 16
    for x, bad in ((vp, float("inf")), (vp, float("nan")), (kp, float("nan")), (kp, float("inf"))):
        old = x[at].clone()
        x[at] = bad
        got = paged_attention(q, kp, vp, table, lens, d ** -0.5)
        x[at] = old
        assert not torch.isfinite(got[0, :, T - 1].float()).any()
        got[0, :, T - 1] = want[0, :, T - 1].to(dtype)
        _check(got, want, tol, dtype)
    q2 = q.clone()
    q2[1, 1, T // 2, 5] = float("nan")
    q2[1, 0, 0] = float("inf")
    got = paged_attention(q2, kp, vp, table, lens, d ** -0.5)
    assert torch.isnan(got[1, 1, T // 2]).all() and torch.isnan(got[1, 0, 0]).all()
    got[1, 1, T // 2], got[1, 0, 0] = want[1, 1, T // 2].to(dtype), want[1, 0, 0].to(dtype)
    _check(got, want, tol, dtype)


@pytest.mark.parametrize("T", [1, 40])
def test_scores_of_any_size(T, dev):
    """A softmax whose scores all lie far below zero or far apart; scores that are all -inf have none."""
    _say("score sizes", T)
    q, kp, vp, table, lens, _ = _attend_case([300], None, T, 4, 2, 64, 16, BF16, dev)
    p_step = _p_step(BF16, T * 2 <= STREAM_VECTORS)
    one = torch.ones_like(q)
    for size in (2.0 ** -60, 2.0 ** 20, 2.0 ** 50, 2.0 ** 100):
        kp[:] = -size  # every score the same: the mean of the values
        want, tol = plain.attend(one, kp, vp, table, lens, 1.0, None, p_step)
        _check(paged_attention(one, kp, vp, table, lens, 1.0), want, tol * 0 + want.abs() * 2.0 ** -6 + 2.0 ** -7, BF16)
    kp[:] = -float("inf")
    assert torch.isnan(paged_attention(one, kp, vp, table, lens, 1.0).float()).all()


APPEND = [
    ([1], None, 1, 8, 2, 128, 16, BF16),
    ([70, 5, 0, 33], [9, 5, 0, 1], 9, 8, 2, 128, 16, BF16),
    ([100, 3], [40, 40], 40, 5, 5, 64, 32, FP16),  # rows before the first are not written
    ([1111], None, 1111, 32, 8, 128, 64, BF16),
    ([90, 2000], None, 3, 16, 1, 64, 16, FP16),
]


def _expected_rows(k, v, cos, sin, lens, new, kp, vp, table, page):
    """(page, row) of each written token, and its K (64 bits) and V rows [tokens, Hkv, d]."""
    at = plain.append_rows(lens, new, k.shape[2], table.cpu(), kp.shape[0], page)
    kk = plain.rotate(k, cos[:, None], sin[:, None]) if cos is not None else k.double()
    b, j, pg, r = (torch.tensor(x, device=k.device) for x in zip(*at))
    return (pg, r), kk[b, :, j], v[b, :, j]


def _check_append(before, after, at, kk, vv, dtype, rotated):
    kp, vp = after
    same = torch.ones(kp.shape[0], kp.shape[2], dtype=torch.bool, device=kp.device)
    same[at] = False
    for old, now in zip(before, after):  # the rest of the pages is as it was, bit for bit
        assert torch.equal(old.transpose(1, 2)[same].view(torch.int16), now.transpose(1, 2)[same].view(torch.int16))
    assert torch.equal(vp.transpose(1, 2)[at], vv)
    got = kp.transpose(1, 2)[at].double()
    if not rotated:
        assert torch.equal(got, kk)
        return
    # two products and a sum in fp32 (three roundings of 2^-24 of at most sqrt 2 times the pair's size), rounded once
    size = kk.abs() + kk.norm(dim=-1, keepdim=True)
    tol = 4 * 2.0 ** -24 * size + HALF_STEP[dtype] * kk.abs() * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype == FP16 else 0.0)
    assert ((got - kk).abs() <= tol).all()


@pytest.mark.parametrize("rot", [None, "own", "fp32"])
@pytest.mark.parametrize("lens,new,T,H,hk,d,page,dtype", APPEND)
def test_append(lens, new, T, H, hk, d, page, dtype, rot, dev):
    _say("append", lens, new, T, H, hk, d, page, dtype, rot)
    gen = torch.Generator(device=dev).manual_seed(T)
    table, p = _table(gen, lens, page, dev)
    for layout in ("heads", "rows", "pool", "padded"):
        kp, vp = _pages(gen, p, hk, page, d, dtype, dev, layout)
        k, v, q = (_heads(gen, len(lens), h, T, d, dtype, dev) for h in (hk, hk, H))
        cos, sin = _angles(gen, len(lens), T, d, FP32 if rot == "fp32" else dtype, dev) if rot else (None, None)
        before = kp.clone(), vp.clone()
        out = paged_append(k, v, kp, vp, table, _int(lens, dev), cos=cos, sin=sin, q=q if rot else None, new=_int(new, dev))
        at, kk, vv = _expected_rows(k, v, cos, sin, lens, new, kp, vp, table, page)
        _check_append(before, (kp, vp), at, kk, vv, dtype, rot is not None)
        if rot:
            want = plain.rotate(q, cos[:, None], sin[:, None])
            tol = 4 * 2.0 ** -24 * (want.abs() + want.norm(dim=-1, keepdim=True)) + HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -10)
            assert out.shape == q.shape and out.transpose(1, 2).is_contiguous()
            assert ((out.double() - want).abs() <= tol + (2.0 ** -25 if dtype == FP16 else 0.0)).all()
        else:
            assert out is None


def test_append_broadcast_angles_and_odd_layouts(dev):
    """cos and sin [T, d] for every sequence; rows at unaligned addresses and transposed; entries that name no page."""
    _say("append layouts")
    gen = torch.Generator(device=dev).manual_seed(3)
    lens, T, hk, d, page = [40, 40, 21], 6, 3, 64, 16
    table, p = _table(gen, lens, page, dev)
    table[1, 2] = p + 3  # rows 32 .. 39 of the second sequence are on no page
    kp, vp = _pages(gen, p, hk, page, d, BF16, dev)
    k = torch.randn(3, hk, d, T, generator=gen, device=dev).to(BF16).transpose(2, 3)
    v = torch.randn(3, hk, T, d + 1, generator=gen, device=dev).to(BF16)[..., 1:]
    cos, sin = (x[0] for x in _angles(gen, 1, T, d, FP32, dev))
    before = kp.clone(), vp.clone()
    paged_append(k, v, kp, vp, table, _int(lens, dev), cos=cos, sin=sin)
    at, kk, vv = _expected_rows(k, v, cos.expand(3, T, d), sin.expand(3, T, d), lens, None, kp, vp, table, page)
    assert len(at[0]) == 12
    _check_append(before, (kp, vp), at, kk, vv, BF16, True)


STEP = [
    ([1], None, 1, 8, 2, 128, 16, BF16),
    ([5000, 1, 17, 256, 0], None, 1, 32, 8, 128, 16, BF16),
    ([257, 4099], None, 1, 8, 8, 64, 64, FP16),
    ([900, 30, 2, 64], [4, 1, 4, 0], 4, 16, 4, 128, 16, FP16),   # padding, rows before the first, an idle sequence
    ([500], None, 8, 32, 8, 128, 32, BF16),                       # 32 vectors
    ([33, 600], [33, 20], 33, 6, 2, 64, 16, BF16),                # 99 vectors, several tiles of the streaming kernel
    ([128, 77], [128, 77], 128, 8, 2, 128, 16, BF16),             # a prompt: more than the step's kernel takes
    ([3000], None, 40, 16, 4, 64, 256, FP16),
]


@pytest.mark.parametrize("rot", [None, "own", "fp32"])
@pytest.mark.parametrize("lens,new,T,H,hk,d,page,dtype", STEP)
def test_step(lens, new, T, H, hk, d, page, dtype, rot, dev):
    _say("step", lens, new, T, H, hk, d, page, dtype, rot)
    gen = torch.Generator(device=dev).manual_seed(T + 11)
    table, p = _table(gen, lens, page, dev)
    kp, vp = _pages(gen, p, hk, page, d, dtype, dev, "pool" if T == 4 else "heads")
    at = plain.append_rows(lens, new, T, table.cpu(), p, page)
    for _, _, pg, r in at:  # what the new rows replace is not attended, whatever it is
        kp[pg, :, r] = float("nan")
        vp[pg, :, r] = float("inf")
    k, v, q = (_heads(gen, len(lens), h, T, d, dtype, dev) for h in (hk, hk, H))
    cos, sin = _angles(gen, len(lens), T, d, FP32 if rot == "fp32" else dtype, dev) if rot else (None, None)
    before = kp.clone(), vp.clone()
    got = paged_step(q, k, v, kp, vp, table, _int(lens, dev), d ** -0.5, cos=cos, sin=sin, new=_int(new, dev))
    if at:
        _check_append(before, (kp, vp), *_expected_rows(k, v, cos, sin, lens, new, kp, vp, table, page), dtype, rot is not None)
    one_kernel = T * H // hk <= STEP_VECTORS
    qr = plain.rotate(q, cos[:, None], sin[:, None]) if rot else q
    # the rotated query: in two 16-bit terms where one kernel does all, else rounded; fp32's roundings are in the bound's d + 10
    q_step = 0.0 if not rot else HALF_STEP[dtype] ** (2 if one_kernel else 1) + (2.0 ** -20 if dtype == FP16 else 0.0)
    want, tol = plain.attend(qr, kp, vp, table, lens, d ** -0.5, new, _p_step(dtype, one_kernel), q_step)
    _check(got, want, tol, dtype)


def test_step_is_append_and_attention(dev):
    """The pages after a step are those after an append, bit for bit, and without a rotation so is the attention."""
    _say("step against its parts")
    gen = torch.Generator(device=dev).manual_seed(1)
    lens, T, hk, d = [700, 45, 1], 2, 4, 128
    table, p = _table(gen, lens, 16, dev)
    kp, vp = _pages(gen, p, hk, 16, d, BF16, dev)
    k, v, q = (_heads(gen, 3, h, T, d, BF16, dev) for h in (hk, hk, 16))
    cos, sin = _angles(gen, 3, T, d, BF16, dev)
    ln = _int(lens, dev)
    for turn in ({}, dict(cos=cos, sin=sin)):
        a, b = (kp.clone(), vp.clone()), (kp.clone(), vp.clone())
        out = paged_step(q, k, v, *a, table, ln, 0.1, **turn)
        qr = paged_append(k, v, *b, table, ln, q=q if turn else None, **turn)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        if not turn:
            assert qr is None and torch.equal(out, paged_attention(q, *b, table, ln, 0.1))


def test_sequences_share_pages(dev):
    """Two sequences with the same first pages (a shared prompt) and their own last ones."""
    _say("shared pages")
    q, kp, vp, table, lens, _ = _attend_case([200, 170], None, 1, 8, 2, 128, 16, BF16, dev)
    table[1, :6] = table[0, :6]
    want, tol = plain.attend(q, kp, vp, table, [200, 170], 0.1, None, _p_step(BF16, True))
    _check(paged_attention(q, kp, vp, table, lens, 0.1), want, tol, BF16)


def test_pages_past_4_gib(dev):
    """Pages whose byte offsets pass 2^32 (only the pages that are used are touched), K and V of one pool."""
    _say("pages past 4 GiB")
    pool = torch.empty(24000, 2, 8, 64, 128, dtype=BF16, device=dev)  # 6.3 GB
    gen = torch.Generator(device=dev).manual_seed(2)
    kp, vp = pool[:, 0], pool[:, 1]
    table = torch.tensor([[23999, 5, 16500], [20001, 16384, -1]], dtype=torch.int32, device=dev)
    for e in table.view(-1).tolist():
        if e >= 0:
            pool[e] = torch.randn(2, 8, 64, 128, generator=gen, device=dev).to(BF16)
    lens = [150, 128]
    for T in (1, 40):
        q, k, v = (_heads(gen, 2, h, T, 128, BF16, dev) for h in (32, 8, 8))
        got = paged_step(q, k, v, kp, vp, table, _int(lens, dev), 0.09)
        at, kk, vv = _expected_rows(k, v, None, None, lens, None, kp, vp, table, 64)
        assert torch.equal(kp.transpose(1, 2)[at].double(), kk) and torch.equal(vp.transpose(1, 2)[at], vv)
        want, tol = plain.attend(q, kp, vp, table, lens, 0.09, None, _p_step(BF16, T * 4 <= STEP_VECTORS))
        _check(got, want, tol, BF16)


def test_many_sequences(dev):
    """More (sequence, tile) pairs than a wave's lanes, in both kernels."""
    _say("many sequences")
    gen = torch.Generator(device=dev).manual_seed(4)
    lens = [int(x) for x in torch.randint(0, 400, (150,), generator=torch.Generator().manual_seed(5))]
    for T, H, hk in ((1, 4, 2), (140, 4, 2)):
        q, kp, vp, table, ln, _ = _attend_case(lens, None, T, H, hk, 64, 32, BF16, dev)
        new = [min(T, max(0, n)) for n in lens]
        got = paged_attention(q, kp, vp, table, ln, 0.125, new=_int(new, dev))
        want, tol = plain.attend(q, kp, vp, table, lens, 0.125, new, _p_step(BF16, T * H // hk <= STREAM_VECTORS))
        _check(got, want, tol, BF16)


@pytest.mark.parametrize("b,long,T,H,hk", [(70, 9000, 1, 4, 2), (70, 5000, 3, 8, 2), (66, 4000, 40, 2, 2), (1100, 3000, 1, 2, 1)])
def test_many_sequences_of_unlike_lengths(b, long, T, H, hk, dev):
    """One long sequence, which is split, among many short or empty ones; the call, its step and replays of both in a graph."""
    _say("many sequences of unlike lengths", b, T)
    gen = torch.Generator(device=dev).manual_seed(6)
    lens = [(7 * i) % 40 if i % 3 else 0 for i in range(b)]
    lens[b // 2] = long
    new = [min(T, n) for n in lens]
    q, kp, vp, table, ln, _ = _attend_case(lens, None, T, H, hk, 64, 16, BF16, dev)
    k, v = (_heads(gen, b, hk, T, 64, BF16, dev) for _ in "kv")
    nw = _int(new, dev)
    streams = T * H // hk <= STREAM_VECTORS
    want, tol = plain.attend(q, kp, vp, table, lens, 0.125, new, _p_step(BF16, streams))
    _check(paged_attention(q, kp, vp, table, ln, 0.125, new=nw), want, tol, BF16)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        paged_attention(q, kp, vp, table, ln, 0.125, new=nw)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = paged_attention(q, kp, vp, table, ln, 0.125, new=nw)
        stepped = paged_step(q, k, v, kp, vp, table, ln, 0.125, new=nw)
    for turn in range(3):  # the long sequence moves
        lens[b // 2 - turn], lens[b // 2 - turn - 1] = lens[b // 2 - turn - 1], lens[b // 2 - turn]
        table[[b // 2 - turn, b // 2 - turn - 1]] = table[[b // 2 - turn - 1, b // 2 - turn]]
        new = [min(T, n) for n in lens]
        ln.copy_(_int(lens, dev))
        nw.copy_(_int(new, dev))
        before = paged_attention(q, kp, vp, table, ln, 0.125, new=nw)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, before)
        if streams:  # (of 40 vectors the step is the streaming kernel's, the attention the tiles')
            assert torch.equal(stepped, paged_attention(q, kp, vp, table, ln, 0.125, new=nw))
        want, tol = plain.attend(q, kp, vp, table, lens, 0.125, new, _p_step(BF16, T * H // hk <= STEP_VECTORS))
        _check(stepped, want, tol, BF16)


@pytest.mark.parametrize("T", [1, 50])
def test_captured_steps_follow_the_cache(T, dev):
    """Two captured graphs over one cache, replayed in turn while the lengths and the table grow, with eager work between: every
    replay is the eager step's bits."""
    _say("captured steps", T)
    gen = torch.Generator(device=dev).manual_seed(6)
    B, H, hk, d, page, W = 3, 8, 2, 128, 16, 400
    pool = torch.randn(2, B * W, hk, page, d, generator=gen, device=dev).to(BF16)
    twin = pool.clone()
    full = torch.randperm(B * W, generator=gen, device=dev).int().view(B, W)
    table, lens, new = torch.full_like(full, -1), _int([0] * B, dev), _int([T] * B, dev)
    graphs = []
    for _ in range(2):
        q, k, v = (_heads(gen, B, h, T, d, BF16, dev) for h in (H, hk, hk))
        cos, sin = _angles(gen, B, T, d, BF16, dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            paged_step(q, k, v, *pool, table, lens, 0.1, cos=cos, sin=sin, new=new)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_step(q, k, v, *pool, table, lens, 0.1, cos=cos, sin=sin, new=new)
        graphs.append((g, out, (q, k, v, cos, sin)))
    n = [0, 0, 0]
    for i, grow in enumerate(([5, 60, 0], [1, 1, 1], [3000, 20, 1], [1, 1, 1], [7, 3000, 5000], [1, 1, 1])):
        n = [a + b for a, b in zip(n, grow)]
        lens.copy_(_int(n, dev))
        new.copy_(_int([min(T, x) for x in grow], dev))
        for b in range(B):
            table[b, :-(-n[b] // page)] = full[b, :-(-n[b] // page)]
        g, out, (q, k, v, cos, sin) = graphs[i % 2]
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen, device=dev))
        g.replay()
        want = paged_step(q, k, v, *twin, table, lens, 0.1, cos=cos, sin=sin, new=new)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pool, twin)


def test_another_stream_and_steps_back_to_back(dev):
    """Steps on a side stream that nothing waits between: each reads what the one before wrote."""
    _say("streams")
    gen = torch.Generator(device=dev).manual_seed(8)
    table, p = _table(gen, [600, 600], 16, dev)
    base = _pages(gen, p, 2, 16, 64, FP16, dev)
    rows = [tuple(_heads(gen, 2, h, 1, 64, FP16, dev) for h in (8, 2, 2)) for _ in range(40)]
    lens = [_int([500 + i, 300 + i], dev) for i in range(40)]
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        kp, vp = (x.clone() for x in base)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            outs = [paged_step(*x, kp, vp, table, n, 0.125) for x, n in zip(rows, lens)]
        torch.cuda.synchronize()
        results.append((torch.stack(outs), kp, vp))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_nothing_to_do(dev):
    _say("empty calls")
    pages = torch.zeros(2, 2, 16, 64, dtype=BF16, device=dev)
    for b, t in ((0, 1), (2, 0)):
        x, q = torch.zeros(b, 2, t, 64, dtype=BF16, device=dev), torch.zeros(b, 4, t, 64, dtype=BF16, device=dev)
        table, lens = torch.zeros(b, 1, dtype=torch.int32, device=dev), torch.zeros(b, dtype=torch.int32, device=dev)
        assert paged_attention(q, pages, pages, table, lens, 1.0).shape == q.shape
        assert paged_step(q, x, x, pages, pages, table, lens, 1.0).shape == q.shape
        assert paged_append(x, x, pages, pages, table, lens) is None


def test_refusals(dev):
    _say("refusals")
    q, kp, vp, table, lens, _ = _attend_case([40, 9], None, 2, 8, 2, 128, 16, BF16, dev)
    k = torch.zeros(2, 2, 2, 128, dtype=BF16, device=dev)
    cos = torch.ones(2, 2, 128, dtype=BF16, device=dev)
    for msg, fn in [
        ("bf16 or fp16 rows and pages", lambda: paged_attention(q.float(), kp, vp, table, lens, 1.0)),
        ("bf16 or fp16 rows and pages", lambda: paged_attention(q.half(), kp, vp, table, lens, 1.0)),
        ("bf16 or fp16 rows and pages", lambda: paged_attention(q, kp, vp.half(), table, lens, 1.0)),
        ("must be", lambda: paged_attention(q[0], kp, vp, table, lens, 1.0)),
        ("with the rows' d", lambda: paged_attention(q[..., :64], kp, vp, table, lens, 1.0)),
        ("with the rows' d", lambda: paged_attention(q, kp, vp[:-1], table, lens, 1.0)),
        ("must match", lambda: paged_attention(q[:, :7], kp, vp, table, lens, 1.0)),
        ("must match", lambda: paged_attention(q, kp, vp, table[:1], lens, 1.0)),
        ("must match", lambda: paged_attention(q, kp, vp, table, lens[:1], 1.0)),
        ("must match", lambda: paged_attention(q, kp, vp, table, lens, 1.0, new=lens[:1])),
        ("must be int32", lambda: paged_attention(q, kp, vp, table.long(), lens, 1.0)),
        ("must be int32", lambda: paged_attention(q, kp, vp, table, lens.long(), 1.0)),
        ("must be contiguous", lambda: paged_attention(q, kp, vp, table, lens.repeat(2)[::2], 1.0)),
        ("must be contiguous", lambda: paged_attention(q, kp, vp, table.repeat(1, 2)[:, ::2], lens, 1.0)),
        ("aligned rows", lambda: paged_attention(q, kp.transpose(2, 3).contiguous().transpose(2, 3), vp, table, lens, 1.0)),
        ("aligned rows", lambda: paged_attention(q, torch.cat([kp, kp[..., :4]], -1)[..., :128], vp, table, lens, 1.0)),
        ("scale must be positive", lambda: paged_attention(q, kp, vp, table, lens, 0.0)),
        ("pages of 8 rows", lambda: paged_attention(q, kp[:, :, :8], vp[:, :, :8], table, lens, 1.0)),
        ("share a shape and dtype", lambda: paged_append(k, k[:, :, :1], kp, vp, table, lens)),
        ("cos and sin required", lambda: paged_append(k, k, kp, vp, table, lens, q=q)),
        ("go together", lambda: paged_append(k, k, kp, vp, table, lens, cos=cos)),
        ("fp32 or of the rows' dtype", lambda: paged_append(k, k, kp, vp, table, lens, cos=cos.half(), sin=cos.half())),
        ("must be \\[B, T, d\\]", lambda: paged_append(k, k, kp, vp, table, lens, cos=cos[:, :, :64], sin=cos[:, :, :64])),
        ("must match", lambda: paged_append(k[:, :1], k[:, :1], kp, vp, table, lens)),
        ("must match", lambda: paged_append(k, k, kp, vp, table, lens, cos=cos, sin=cos, q=q[:, :, :1])),
        ("must match", lambda: paged_step(q, k, k[:, :1], kp, vp, table, lens, 1.0)),
        ("must match", lambda: paged_step(q, k.half(), k, kp, vp, table, lens, 1.0)),
        ("scale must be positive", lambda: paged_step(q, k, k, kp, vp, table, lens, -1.0)),
        ("ROCm device only", lambda: paged_attention(q, kp, vp, table.cpu(), lens, 1.0)),
    ]:
        before = kp.clone()
        with pytest.raises(ValueError, match=msg):
            fn()
        assert torch.equal(before.view(torch.int16), kp.view(torch.int16))


# ---------------------------------------------------------------- under a model
def _model(dev, arm, dtype=BF16, kv_heads=2, **kw):
    from transformers import LlamaConfig, LlamaForCausalLM

    from bigger_bird_amd import install

    cfg = LlamaConfig(vocab_size=512, hidden_size=1024, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=kv_heads, max_position_embeddings=4096, rope_theta=500000.0, attn_implementation="sdpa")
    torch.manual_seed(0)
    m = LlamaForCausalLM(cfg).eval().to(dev, dtype)
    return install(m, arm, **kw)


class _Outputs:
    """Every layer's attention output (the input of o_proj) of each call."""

    def __init__(self, model):
        self.calls = []
        for layer in model.model.layers:
            layer.self_attn.o_proj.register_forward_pre_hook(lambda m, a: self.calls.append(a[0].detach().clone()))

    def take(self):
        out, self.calls = self.calls, []
        return out


def _alike(got, want, what):
    """Two runs of one model in 16 bits, the attention of one by other kernels: the bar of the module's other tests."""
    err = (got.float() - want.float()).abs()
    assert err.max().item() <= 2e-2 and err.mean().item() <= 2e-3, f"{what}: max {err.max().item():.3e} mean {err.mean().item():.3e}"


@pytest.mark.parametrize("arm,dtype", [("dense_rd", BF16), ("rd", BF16), ("rd", FP16)])
def test_model_batch_against_single_sequences(arm, dtype, dev):
    """Prompts of unlike lengths in one padded batch, then steps of one token and of several, against each sequence alone on the
    16-bit cache: every layer's attention output. (A step of several tokens behind cached ones goes token by token there.)"""
    _say("model", arm, dtype)
    from transformers import DynamicCache

    from bigger_bird_amd import make_paged_cache

    model = _model(dev, arm, dtype, **({} if arm == "dense_rd" else dict(sink=64, window=512, vertical=128, exact_tail=64)))
    taken = _Outputs(model)
    lens = [1000, 300, 17]
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 512, (3, 1000), generator=g).to(dev)
    later = torch.randint(0, 512, (3, 5), generator=g).to(dev)
    with torch.no_grad():
        alone = []
        for b, n in enumerate(lens):
            cache = DynamicCache(config=model.config)
            model(input_ids=ids[b:b + 1, :n], past_key_values=cache, use_cache=True)
            steps = [taken.take()]
            for i in range(5):
                model(input_ids=later[b:b + 1, i:i + 1], past_key_values=cache, use_cache=True)
                steps.append(taken.take())
            alone.append(steps)
        cache = make_paged_cache(model.config, 3, 120, page=16, dtype=dtype, device=dev)
        for part in cache.arena.flatten(0, 1):
            part.fill_(float("nan"))  # what memory held before
        cache.extend(lens)
        model(input_ids=ids, position_ids=cache.positions(1000), past_key_values=cache, use_cache=True)
        got = taken.take()
        for b, n in enumerate(lens):
            for i in range(2):
                _alike(got[i][b, :n], alone[b][0][i][0], f"prompt {b} layer {i}")
                assert (got[i][b, n:] == 0).all()
        assert cache.lengths == lens
        for i in range(2):  # one token each
            model(input_ids=later[:, i:i + 1], position_ids=cache.positions(1), past_key_values=cache, use_cache=True)
            got = taken.take()
            for b in range(3):
                for j in range(2):
                    _alike(got[j][b], alone[b][1 + i][j][0], f"step {i} of {b} layer {j}")
        cache.extend([3, 0, 2])  # several tokens of some sequences
        model(input_ids=later[:, 2:5], position_ids=cache.positions(3), past_key_values=cache, use_cache=True)
        got = taken.take()
        for b, m in ((0, 3), (2, 2)):
            for i in range(m):
                for j in range(2):
                    _alike(got[j][b, i], alone[b][3 + i][j][0, 0], f"token {i} of {b} layer {j}")
        assert cache.lengths == [1005, 302, 21]
        # the drafted tokens of the first are taken back, the third makes room: its pages go to the second
        cache.truncate([1002, 302, 21])
        cache.release(2)
        cache.extend([1, 3, 0])
        ids2 = torch.stack([later[0, 2:5], later[1, 2:5], later[2, 2:5]])
        model(input_ids=ids2, position_ids=cache.positions(3), past_key_values=cache, use_cache=True)
        got = taken.take()
        for j in range(2):
            _alike(got[j][0, 0], alone[0][3][j][0, 0], "after truncate")
            for i in range(3):
                _alike(got[j][1, i], alone[1][3 + i][j][0, 0], "after release")
            assert (got[j][0, 1:] == 0).all() and (got[j][2] == 0).all()


def test_model_generate(dev):
    """Hugging Face's generate over a paged cache: prompts of one length, greedy, the tokens of each alone on the 16-bit cache as
    far as the logits' order is clear of 16-bit differences."""
    _say("generate")
    from transformers import DynamicCache

    from bigger_bird_amd import make_paged_cache

    model = _model(dev, "dense_rd")
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(2)).to(dev)
    with torch.no_grad():
        cache = make_paged_cache(model.config, 2, 20, page=16, device=dev)
        got = model.generate(ids, past_key_values=cache, do_sample=False, max_new_tokens=12, pad_token_id=0)
        assert got.shape == (2, 52) and cache.lengths == [51, 51]
        for b in range(2):
            one = DynamicCache(config=model.config)
            out = model(input_ids=ids[b:b + 1], past_key_values=one, use_cache=True)
            for i in range(12):
                logits = out.logits[0, -1].float()
                token = got[b, 40 + i]
                assert logits[token] >= logits.max() - 0.05
                out = model(input_ids=token.view(1, 1), past_key_values=one, use_cache=True)


def test_model_refusals_on_a_paged_cache(dev):
    _say("model refusals")
    from bigger_bird_amd import make_paged_cache

    model = _model(dev, "dense_rd")
    ids = torch.zeros(2, 8, dtype=torch.long, device=dev)
    cache = make_paged_cache(model.config, 2, 20, page=16, device=dev)
    mask = torch.ones(2, 8, dtype=torch.long, device=dev)
    mask[1, :3] = 0
    with torch.no_grad():
        with pytest.raises(ValueError, match="not by a mask"):
            model(input_ids=ids, attention_mask=mask, past_key_values=cache, use_cache=True)
        assert cache.lengths == [0, 0]
        cache.extend([8, 5])
        model(input_ids=ids, position_ids=cache.positions(8), past_key_values=cache, use_cache=True)
        with pytest.raises(ValueError, match="need position_ids"):
            model(input_ids=ids[:, :1], past_key_values=cache, use_cache=True)
    with pytest.raises(ValueError, match="holds no gradients"):
        model(input_ids=ids, past_key_values=cache, use_cache=True)
