"""4-bit KV cache on the GPU: the sums' precision, rows that are not finite or far below zero, layouts that a copy has to put right,
and the cache layer where a step is refused, against the 64-bit forms of tests/int4_plain.py."""
import pytest
import torch

import int4_plain as plain
from bigger_bird_amd.kv_int4 import (decode_int4, decode_int4_append, dequantize4, dequantize4_pair, quantize4,
                                     quantize4_pair)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _say(*a):
    print("case", *a, flush=True)


def test_sums_keep_their_bits(dev):
    """512 KV heads are one split however long the cache, so each of its four waves adds up a quarter of 16384 keys in a chain. The
    scores are nearly equal, which makes the outputs small against the sums they come from.

    Tolerance, on 2-norms over a head. A wave's chain for a column is m = 2 * 4096 / 32 products (two 16-bit terms, 32 keys each); a
    rounding to nearest is off by ulp / sqrt(12) rms with an ulp of at most 2^-23 of the sum so far, which grows evenly to
    a = sum_j p_j s_j c_j / 4: sqrt(m / 36) * 2^-23 * a rms, and twice that for four waves with independent roundings. The minima's
    sums are as large in shorter chains; the two terms and the scores' roundings are below 2^-25 of a at random and average out
    over the keys. Four times the first term covers them. The output's own rounding is known and taken apart."""
    _say("sums", 512, 16384)
    gen = torch.Generator(device=dev).manual_seed(21)
    hk, n, d = 512, 16384, 128
    cache = []
    for _ in range(2):
        codes = torch.randint(0, 256, (hk, n, d // 2), generator=gen, device=dev, dtype=torch.uint8)
        s = 0.25 + 0.1 * torch.rand(hk, n, d // 32, generator=gen, device=dev)
        cache += [codes, torch.stack([s, -7.5 * s], -1).half()]
    q = (0.2 * torch.randn(1, hk, d, generator=gen, device=dev)).half()
    got = decode_int4(q, *cache, n, d ** -0.5)[0].double()
    rms = (2 * 4096 / 32 / 36) ** 0.5 * 2.0 ** -23 / 2
    for h in (0, 1, 100, 255, 256, 511):
        k4, kp, v4, vp = (x[h] for x in cache)
        p = torch.softmax(plain.values(k4, kp)[0] @ q[0, h].double() * d ** -0.5, 0)
        v, s = plain.values(v4, vp)
        want, a = p @ v, p @ (s * plain.codes(v4).double())
        rounding = want.half().double() - want
        limit = (rounding.norm() ** 2 + (4 * rms * a.norm()) ** 2) ** 0.5
        off = (got[h] - want).norm()
        print(f"head {h}: off {off / want.norm():.2e}, rounding {rounding.norm() / want.norm():.2e}, "
              f"limit {limit / want.norm():.2e}", flush=True)
        assert off <= 1.02 * limit


def _cache(gen, hk, n, cap, d, dev):
    """Packed K and V of n rows, the spare rows behind them of NaN params."""
    out = []
    for _ in range(2):
        q4 = torch.randint(0, 256, (hk, cap, d // 2), generator=gen, device=dev, dtype=torch.uint8)
        p4 = torch.full((hk, cap, d // 32, 2), float("nan"), device=dev, dtype=FP16)
        x = torch.randn(hk, n, d, generator=gen, device=dev) * torch.exp(0.7 * torch.randn(hk, 1, d, generator=gen, device=dev))
        q4[:, :n], p4[:, :n] = plain.pack(*plain.quantize(x))
        out += [q4, p4]
    return out


# one split and several; up to 4 vectors of a KV head, and more
SHAPES = [(500, 1, 8, 2, 128), (500, 4, 8, 2, 64), (4000, 1, 8, 2, 64), (4000, 1, 8, 2, 128), (4000, 3, 16, 2, 128),
          (5000, 2, 20, 2, 64)]


@pytest.mark.parametrize("n,T,H,Hkv,d", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_nonfinite_query_gives_nan(n, T, H, Hkv, d, dtype, dev):
    """A NaN or an infinity of either sign in one query is a NaN row, as in the formula, with a host and a device length, and no
    other row changes; a token that attends no row stays zeros whatever its query holds."""
    _say("nonfinite", n, T, H, Hkv, d, dtype)
    gen = torch.Generator(device=dev).manual_seed(n + T)
    cache = _cache(gen, Hkv, n, n + 3, d, dev)
    q = torch.randn(T, H, d, generator=gen, device=dev).to(dtype)
    want = decode_int4(q, *cache, n, 0.1, causal=True)
    assert torch.isfinite(want.float()).all()
    for bad in (float("nan"), float("inf"), -float("inf")):
        q2 = q.clone()
        q2[T - 1, 3, 5] = bad
        for length in (n, torch.tensor([n], device=dev)):
            got = decode_int4(q2, *cache, length, 0.1, causal=True)
            assert got[T - 1, 3].isnan().all(), bad
            if length is n:
                got[T - 1, 3] = want[T - 1, 3]
                assert torch.equal(got, want)
        if T > 1:
            q2[0, 1, 7] = bad
            got = decode_int4(q2, *cache, torch.tensor([T - 1], device=dev), 0.1, causal=True)
            assert (got[0] == 0).all() and got[T - 1, 3].isnan().all()
        assert (decode_int4(q2, *cache, torch.tensor([0], device=dev), 0.1) == 0).all()


@pytest.mark.parametrize("n,T,H,Hkv,d", SHAPES)
def test_infinite_scores(n, T, H, Hkv, d, dev):
    """Keys at which every product is positive: an infinite element makes every score +inf or -inf, which is NaN either way."""
    _say("infinite scores", n, T, H, Hkv, d)
    gen = torch.Generator(device=dev).manual_seed(n)
    k, v = (torch.rand(Hkv, n, d, generator=gen, device=dev) + 0.5 for _ in range(2))
    cache = (*plain.pack(*plain.quantize(k)), *plain.pack(*plain.quantize(v)))
    q = torch.ones(T, H, d, device=dev, dtype=BF16)
    q[T - 1, 0] *= float("inf")
    q[T - 1, 1] *= -float("inf")
    got = decode_int4(q, *cache, n, 0.1)
    assert got[T - 1, :2].isnan().all()
    got[T - 1, :2] = 0
    assert torch.isfinite(got.float()).all()


@pytest.mark.parametrize("n,T,H,Hkv,d", SHAPES)
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_scores_far_from_zero(n, T, H, Hkv, d, sign, dev):
    """Scores of about -1e32 and 1e32, finite in fp32. Keys that are all alike score the same, so the output is V's mean; with one
    key that scores higher by more than any rounding it is that key's V row. Both hold to the output's rounding and to the sums'
    of probabilities that are exactly 1: 2^-17 of a V scale times 15 for the two terms, and 2^-20 of the largest sum (s c + |z|) for
    the fp32 sums and scales. Rows next to them with ordinary queries stay within int4_plain's bound (not bit for bit: a wave moves
    all its vectors' running maxima when one of them rises, and then their roundings are others)."""
    _say("far", n, T, H, Hkv, d, sign)
    gen = torch.Generator(device=dev).manual_seed(n + 1)
    k = (torch.rand(Hkv, 1, d, generator=gen, device=dev) + 0.5).expand(Hkv, n, d).clone()
    v = torch.randn(Hkv, n, d, generator=gen, device=dev)
    q = torch.randn(T, H, d, generator=gen, device=dev).to(BF16)
    far = torch.zeros(T, H, dtype=torch.bool, device=dev)
    far[:, 1::2] = True
    q2 = torch.where(far[..., None], torch.full_like(q, sign * 1e30), q)
    vq = plain.pack(*plain.quantize(v))
    vv, vs = plain.values(*vq)
    top = (vs * 15 + vq[1][..., 1].double().abs().repeat_interleave(32, -1)).amax((0, 1))
    for planted in (None, 0, n // 2, n - 1):
        if planted is not None:
            k[:, planted] *= 1.5 if sign > 0 else 0.5
        cache = (*plain.pack(*plain.quantize(k)), *vq)
        near, near_tol = plain.attend(q, *cache, n, 0.1)
        for length in (n, torch.tensor([n], device=dev)):
            got = decode_int4(q2, *cache, length, 0.1)
            near_err = (got.double() - near).abs()
            assert (near_err <= near_tol + 2.0 ** -8 * (near.abs() + near_tol))[~far].all()
            want = (vv.mean(1) if planted is None else vv[:, planted]).repeat_interleave(H // Hkv, 0)
            tol = 2.0 ** -8 * want.abs() + 2.0 ** -17 * 15 * vs.amax() + 2.0 ** -20 * top
            err = (got.double() - want).abs()
            assert (err <= tol)[far].all(), (planted, err[far].max().item())
        if planted is not None:
            k[:, planted] /= 1.5 if sign > 0 else 0.5


def _at(x, elements):
    """x's values, contiguous, `elements` elements past an aligned address."""
    buf = torch.empty(x.numel() + elements, dtype=x.dtype, device=x.device)
    return buf[elements:].view(x.shape).copy_(x)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_contiguous_rows_at_any_address(dtype, dev):
    """Rows, queries and new rows that are contiguous but start between 16-byte addresses give what aligned ones give."""
    _say("addresses", dtype)
    gen = torch.Generator(device=dev).manual_seed(4)
    for shape in ((9, 128), (3, 9, 64), (2, 3, 9, 32), (1, 1, 256)):
        x, y = (torch.randn(shape, generator=gen, device=dev).to(dtype) for _ in range(2))
        want = [*quantize4(x), *quantize4(y)]
        for o in (1, 3):
            assert all(map(torch.equal, quantize4(_at(x, o)), want[:2]))
            (kq, kp), (vq, vp) = quantize4_pair(_at(x, o), _at(y, 2), None, None)
            assert all(map(torch.equal, (kq, kp, vq, vp), want))
    if dtype is FP32:
        return
    for T, H, Hkv, d in ((1, 8, 2, 128), (3, 8, 2, 64)):
        n = 700
        cache = _cache(gen, Hkv, n, n + 3, d, dev)
        q = torch.randn(T, H, d, generator=gen, device=dev).to(dtype)
        k, v = (torch.randn(Hkv, T, d, generator=gen, device=dev).to(dtype) for _ in range(2))
        want = decode_int4(q, *cache, n, 0.1)
        for o in (1, 3):
            assert torch.equal(decode_int4(_at(q, o), *cache, n, 0.1), want)
        a, b = ([x.clone() for x in cache] for _ in range(2))
        assert torch.equal(decode_int4_append(_at(q, 1), *a, _at(k, 3), _at(v, 1), n + T, 0.1),
                           decode_int4_append(q, *b, k, v, n + T, 0.1))
        assert all(torch.equal(x[:, :n + T], y[:, :n + T]) for x, y in zip(a, b))


@pytest.mark.parametrize("t", [1, 2, 16, 40])
def test_prompt_after_a_crop_to_nothing_is_causal(t, dev):
    """A layer cropped to no rows takes a new prompt: RDAttention attends it causally, as it does any t == n, however short."""
    _say("crop to nothing", t)
    from types import SimpleNamespace

    from bigger_bird_amd import RDAttention
    from bigger_bird_amd.kv_int4 import Int4KVLayer

    H, Hkv, d = 8, 2, 64
    base = SimpleNamespace(config=SimpleNamespace(num_attention_heads=H, num_key_value_heads=Hkv), layer_idx=0, head_dim=d,
                           scaling=d ** -0.5, q_proj=None, k_proj=None, v_proj=None, o_proj=None)
    attn, layer = RDAttention(base, sink=64, window=16384, vertical=512, exact_tail=256), Int4KVLayer()
    gen = torch.Generator(device=dev).manual_seed(t)
    q, k, v = (torch.randn(1, h, t, d, generator=gen, device=dev).to(BF16) for h in (H, Hkv, Hkv))
    layer.update(torch.randn_like(k).repeat(1, 1, 30, 1), torch.randn_like(v).repeat(1, 1, 30, 1))
    layer.crop(-30 * t)
    assert layer.get_seq_length() == 0
    kk, vv = layer.update(k, v, {"bb_attend": True})
    out = attn.exact_attention(q, kk, vv, t, t)
    cache = (*plain.pack(*plain.quantize(k[0])), *plain.pack(*plain.quantize(v[0])))
    want, _ = plain.attend(q[0].transpose(0, 1), *cache, t, d ** -0.5, True)
    # K and V rounded to bf16 (2^-8 each: a score of |q| |k| d^-0.5 sums, a value), probabilities and output in bf16
    kd, vd = (plain.values(*cache[i:i + 2])[0].abs() for i in (0, 2))
    dx = 2.0 ** -8 * d ** -0.5 * torch.matmul(q[0].double().abs().view(Hkv, -1, d), kd.transpose(1, 2)).max()
    assert (out[0].transpose(0, 1).double() - want).abs().max() <= (2 * dx + 3 * 2.0 ** -8) * vd.max()
    assert layer.get_seq_length() == t


@pytest.mark.parametrize("shape", [(0, 128), (1, 8, 0, 64), (2, 0, 5, 128), (3, 2, 2, 0, 32)])
def test_no_rows_in_any_number_of_dimensions(shape, dev):
    _say("no rows", shape)
    x = torch.zeros(shape, device=dev)
    k, v = quantize4_pair(x, x)
    one = quantize4(x, k)
    assert one[0].shape == (*shape[:-1], shape[-1] // 2) and one[1].shape == (*shape[:-1], shape[-1] // 32, 2)
    assert dequantize4(*one, BF16).shape == shape and all(y.shape == shape for y in dequantize4_pair(k, v, FP32))


def test_cache_without_heads_is_refused(dev):
    _say("no heads")
    q = torch.zeros(1, 8, 128, device=dev, dtype=BF16)
    none = quantize4(torch.zeros(0, 5, 128, device=dev))
    with pytest.raises(ValueError, match="must match"):
        decode_int4(q, *none, *none, 5, 0.1)
    with pytest.raises(ValueError, match="must match"):
        decode_int4(q[:, :0], *none, *none, 5, 0.1)


@pytest.mark.parametrize("T,G,d,dtype", [(1, 1, 128, BF16), (2, 4, 64, FP16), (5, 1, 128, BF16)])
def test_512_and_more_kv_heads_are_one_split(T, G, d, dtype, dev):
    """More KV heads than workgroups at once: one split and no workspace past the lengths where short caches end."""
    _say("heads", T, G, d, dtype)
    from bigger_bird_amd import _lib

    gen = torch.Generator(device=dev).manual_seed(T)
    hk, n = 520, 2003
    assert n > _lib.lib().bb_int4_decode_one_split(T * G, d) and _lib.lib().bb_int4_decode_workspace(n, T, hk * G, hk, d) == 0
    cache = _cache(gen, hk, n, n + 1, d, dev)
    q = torch.randn(T, hk * G, d, generator=gen, device=dev).to(dtype)
    for length in (n, torch.tensor([n], device=dev)):
        got = decode_int4(q, *cache, length, d ** -0.5, causal=True).double()
        for h in (0, 7, 259, 519):
            heads = slice(h * G, h * G + G)
            want, tol = plain.attend(q[:, heads], *(x[h:h + 1] for x in cache), n, d ** -0.5, True)
            tol = tol + (2.0 ** -8 if dtype is BF16 else 2.0 ** -11) * (want.abs() + tol) + (2.0 ** -25 if dtype is FP16 else 0)
            assert ((got[:, heads] - want).abs() <= tol).all(), h


def test_rows_past_32_bit_offsets_to_the_rounding(dev):
    """One KV head with 70 million rows (4.5 GB of codes) that are zero but for planted ones, whose constant K rows score 17 and
    whose V rows are read past 2^32 bytes. The other rows add exactly 1 each to the sums and nothing to the outputs, so what
    is off is the output's half step; 2^-17 of a V scale times 15 and the fp32 sums' 2^-20 of s c + |z|, times the probability; and
    the probability itself by 17 log2(e) roundings of 2^-23 relative in the score and a few in the exponentials: 2^-17."""
    _say("70M rows")
    n, H, d = 70_000_003, 4, 128
    k4, v4 = (torch.zeros(1, n, d // 2, dtype=torch.uint8, device=dev) for _ in range(2))
    kp, vp = (torch.zeros(1, n, d // 32, 2, dtype=FP16, device=dev) for _ in range(2))
    q = torch.ones(1, H, d, device=dev, dtype=BF16)
    x = torch.full((1, 1, d), 16.0, device=dev, dtype=BF16)
    y = torch.arange(d, device=dev, dtype=FP32).to(BF16)[None, None]
    yq = plain.pack(*plain.quantize(y))
    yv, ys = (t[0, 0] for t in plain.values(*yq))
    size = 15 * ys + yq[1][0, 0, :, 1].double().abs().repeat_interleave(32)
    weight = torch.tensor(17.0, dtype=torch.float64).exp().item()
    for planted, at in enumerate((n - 4, n - 1, 5), 1):
        out = None
        if at == n - 1:
            out = decode_int4_append(q, k4, kp, v4, vp, x, y, n, 17.0 / 2048)
        else:
            quantize4_pair(x, y, (k4[:, at:at + 1], kp[:, at:at + 1]), (v4[:, at:at + 1], vp[:, at:at + 1]))
            out = decode_int4(q, k4, kp, v4, vp, n, 17.0 / 2048)
        p = planted * weight / (planted * weight + n - planted)
        want = p * yv
        tol = 2.0 ** -8 * want + p * (2.0 ** -17 * 15 * ys + 2.0 ** -20 * size) + 2.0 ** -17 * want
        assert ((out[0].double() - want).abs() <= tol).all(), planted
