"""4-bit KV cache (bigger_bird_amd.kv_int4) on the GPU against the plain 64-bit forms of tests/int4_plain.py: the write and
the read back bit for bit, the decode within bounds derived from its arithmetic, the cache layer inside RDAttention."""
from types import SimpleNamespace

import pytest
import torch

import int4_plain as plain
from bigger_bird_amd import RDAttention, bigger_bird_flash, install, kv_int4
from bigger_bird_amd.kv_int4 import (GROW, Int4Handle, Int4KVLayer, decode_int4, decode_int4_append, dequantize4,
                                     dequantize4_pair, make_int4_cache, quantize4, quantize4_pair)

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}


def _say(*a):
    print("case", *a, flush=True)


def _rows(gen, hk, t, d, dtype, dev):
    """[hk, t, d] rows as a projection leaves them: a view of [t, hk * d]; channels of unlike size."""
    x = torch.randn(t, hk * d, generator=gen, device=dev)
    x *= torch.exp(0.7 * torch.randn(hk * d, generator=gen, device=dev))
    return x.to(dtype).view(t, hk, d).transpose(0, 1)


def _cache(gen, hk, n, cap, d, dev):
    """Packed K or V rows; the rows from n on hold NaN params and any codes."""
    q4 = torch.randint(0, 256, (hk, cap, d // 2), generator=gen, device=dev, dtype=torch.uint8)
    p4 = torch.full((hk, cap, d // 32, 2), float("nan"), device=dev, dtype=FP16)
    if n:
        q4[:, :n], p4[:, :n] = plain.pack(*plain.quantize(_rows(gen, hk, n, d, BF16, dev)))
    return q4, p4


def _check_decode(got, q, cache, n, scale, causal):
    want, tol = plain.attend(q, *cache, n, scale, causal)
    # the output's rounding: half a step relative to the value, and for fp16 values below 2^-14, which are multiples of 2^-24
    # whatever their size, 2^-25 absolute
    tol = tol + HALF_STEP[q.dtype] * (want.abs() + tol) + (2.0 ** -25 if q.dtype == FP16 else 0.0)
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert (err <= tol).all(), f"max err {err.max().item():.3e}, tolerance there {tol.flatten()[err.argmax()].item():.3e}"
    return err


# ---------------------------------------------------------------- write and read back
@pytest.mark.parametrize("hk,t,d,dtype", [(8, 1, 128, BF16), (8, 65, 128, BF16), (16, 811, 64, FP16), (3, 37, 32, FP32),
                                          (5, 129, 256, BF16), (2, 1000, 128, FP32), (1, 3, 64, BF16)])
def test_write_and_read_back_bitwise(hk, t, d, dtype, dev):
    _say("write", hk, t, d, dtype)
    gen = torch.Generator(device=dev).manual_seed(t * d)
    k, v = _rows(gen, hk, t, d, dtype, dev), _rows(gen, hk, t, d, dtype, dev)
    cap, a = t + 11, 4
    stores = [(torch.full((hk, cap, d // 2), 0xA5, dtype=torch.uint8, device=dev),
               torch.full((hk, cap, d // 32, 2), 7.0, dtype=FP16, device=dev)) for _ in range(2)]
    at = [(q[:, a:a + t], p[:, a:a + t]) for q, p in stores]
    quantize4_pair(k, v, *at)
    for x, (q4, p4) in zip((k, v), stores):
        wq, wp = plain.pack(*plain.quantize(x))
        assert torch.equal(q4[:, a:a + t], wq) and torch.equal(p4[:, a:a + t], wp)
        for other in (slice(0, a), slice(a + t, cap)):  # rows around the written ones stay
            assert (q4[:, other] == 0xA5).all() and (p4[:, other] == 7.0).all()
        q1, p1 = quantize4(x)  # a fresh pair of tensors, one tensor a launch
        assert torch.equal(q1, wq) and torch.equal(p1, wp)
    for out in (BF16, FP16, FP32):
        got = dequantize4_pair(*at, out)
        for y, (q4, p4) in zip(got, at):
            want = plain.values(q4, p4)[0].to(FP32).to(out)
            assert y.dtype == out and torch.equal(y, want) and torch.equal(dequantize4(q4, p4, out), want)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_write_special_values(dtype, dev):
    """Constant groups, zeros, values whose scale is subnormal or zero in fp16, values past fp16's range, infinities and NaN,
    a large offset with a small spread, exact halves between codes: each in one group, its neighbours unaffected."""
    _say("special", dtype)
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(24, 128, generator=gen)
    x[0, :32] = 1.25
    x[1, 32:64] = 0.0
    x[2, :32] *= 1e-6
    x[3, :32] *= 1e-9
    x[4, :32] = 1e-7
    x[5, 64:96] *= 6e4
    x[6, 3] = float("inf")
    x[6, 40] = -float("inf")
    x[7, 3] = float("nan")
    x[8, :] = float("nan")
    x[9, :32] += 1000.0
    x[10, :32] = torch.arange(32) / 2.0 * 15 / 15.5
    x[11, :32] = torch.cat([torch.arange(31) / 2.0, torch.tensor([15.0])])  # s = 1: halves tie to even
    x[12, :32] = -1.0003
    x[13, :16], x[13, 16:32] = 3.0e38, -3.0e38
    x[14, :32] = 65504.0 + torch.arange(32) * 64
    x = x.to(dtype).to(dev)[None]
    q4, p4 = quantize4(x)
    wq, wp = plain.pack(*plain.quantize(x))
    assert torch.equal(q4, wq) and torch.equal(p4, wp)
    assert torch.isfinite(dequantize4(q4, p4, FP32)).all()


def test_write_near_halves(dev):
    """Quotients next to a border between two codes, one fp32 step to either side: the code is that of the division."""
    _say("near halves")
    gen = torch.Generator().manual_seed(9)
    s = (torch.rand(4000, generator=gen) * 3 + 1e-3).half().float()
    x = torch.zeros(4000, 32)
    x[:, 31] = 15 * s  # z = 0, and s again up to its rounding
    real = ((x[:, 31].double() / 15).float()).half().float()
    for i in range(30):
        k = i // 2
        b = (real.double() * (k + 0.5)).float()
        x[:, i] = torch.nextafter(b, torch.full_like(b, 1e9 if i % 2 else -1e9)) if i < 28 else b
    x = x.to(dev)[None]
    q4, p4 = quantize4(x)
    wq, wp = plain.pack(*plain.quantize(x))
    assert torch.equal(p4, wp) and torch.equal(q4, wq)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_write_many_groups_bitwise(dtype, dev):
    """Four million groups: scales whose fp32 quotient lies on a border of fp16 are rounded twice, as the format says, and so
    are the values read back."""
    _say("many groups", dtype)
    gen = torch.Generator(device=dev).manual_seed(14)
    for _ in range(4):
        x = _rows(gen, 8, 32768, 128, dtype, dev)
        q4, p4 = quantize4(x)
        wq, wp = plain.pack(*plain.quantize(x))
        assert torch.equal(p4, wp) and torch.equal(q4, wq)
        for out in (BF16, FP16):
            assert torch.equal(dequantize4(q4, p4, out), plain.values(q4, p4)[0].to(FP32).to(out))


def test_write_strides(dev):
    """Layouts other than the projections': head-major, a non-contiguous head_dim, misaligned rows, 2-D and 4-D inputs."""
    _say("strides")
    gen = torch.Generator(device=dev).manual_seed(3)
    base = torch.randn(2, 3, 70, 136, generator=gen, device=dev).to(BF16)
    for x in (base[0, :, :, :128], base[0, :, :, 3:131], base[0].transpose(-1, -2)[:, :64, :].transpose(-1, -2)[..., :64],
              base[1, 2, :, 8:], base[..., :64], base[:, :, ::7, 4:68], base[:1, 1:, 5:6, :32]):
        q4, p4 = quantize4(x)
        wq, wp = plain.pack(*plain.quantize(x))
        assert torch.equal(q4, wq) and torch.equal(p4, wp), (x.shape, x.stride())
        want = plain.values(wq, wp)[0].to(BF16)
        assert torch.equal(dequantize4(q4, p4, BF16), want)


# ---------------------------------------------------------------- decode
DECODE = [
    # n, T, H, Hkv, d, dtype, causal
    (1, 1, 32, 8, 128, BF16, False), (2, 2, 8, 8, 64, FP16, True), (15, 1, 8, 1, 64, BF16, False),
    (16, 16, 4, 1, 128, FP16, True), (17, 1, 6, 2, 128, FP16, False), (63, 3, 8, 2, 128, BF16, True),
    (64, 1, 8, 2, 64, FP16, False), (65, 5, 5, 1, 64, BF16, True), (127, 1, 4, 4, 128, BF16, False),
    (128, 4, 16, 4, 64, BF16, True), (129, 1, 16, 1, 128, FP16, False), (255, 2, 16, 2, 64, FP16, False),
    (256, 1, 32, 4, 64, BF16, False), (257, 1, 32, 4, 64, BF16, False), (257, 16, 32, 8, 128, BF16, True),
    (511, 7, 3, 1, 128, BF16, True), (1000, 1, 24, 8, 128, FP16, False), (1025, 4, 32, 8, 64, FP16, True),
    (4099, 1, 32, 8, 64, FP16, False), (8111, 1, 32, 16, 128, BF16, False), (20011, 1, 32, 32, 128, FP16, False),
    (20011, 8, 8, 2, 128, BF16, True), (33000, 4, 32, 8, 128, BF16, True), (131072, 1, 32, 8, 128, BF16, False),
    (131071, 3, 8, 4, 128, FP16, True), (700, 1, 32, 1, 128, BF16, False), (301, 2, 600, 600, 64, BF16, True),
    (769, 1, 8, 2, 128, BF16, False), (1537, 1, 4, 1, 64, FP16, False), (5003, 16, 24, 1, 64, BF16, True),
]


@pytest.mark.parametrize("n,T,H,Hkv,d,dtype,causal", DECODE)
def test_decode_matches_plain(n, T, H, Hkv, d, dtype, causal, dev):
    _say("decode", n, T, H, Hkv, d, dtype, causal)
    gen = torch.Generator(device=dev).manual_seed(n + T)
    cap = n + 37
    cache = (*_cache(gen, Hkv, n, cap, d, dev), *_cache(gen, Hkv, n, cap, d, dev))
    q = (2 * torch.randn(T, H, d, generator=gen, device=dev)).to(dtype)
    got = decode_int4(q, *cache, n, d ** -0.5, causal=causal)
    assert got.dtype == dtype and got.shape == q.shape
    err = _check_decode(got, q, cache, n, d ** -0.5, causal)
    print(f"max err {err.max().item():.3e}", flush=True)
    length = torch.tensor([n], device=dev)
    on_dev = decode_int4(q, *cache, length, d ** -0.5, causal=causal)
    _check_decode(on_dev, q, cache, n, d ** -0.5, causal)
    if T == 1:
        assert torch.equal(decode_int4(q[0], *cache, n, d ** -0.5)[None], got)


@pytest.mark.parametrize("n,T,H,Hkv,d,dtype,causal", [
    (1, 1, 32, 8, 128, BF16, False), (7, 7, 8, 2, 64, FP16, True), (256, 1, 8, 2, 128, BF16, False),
    (257, 1, 32, 4, 64, BF16, False), (513, 4, 32, 8, 128, BF16, True), (1024, 16, 32, 8, 128, FP16, True),
    (2050, 3, 6, 2, 64, FP16, False), (4099, 1, 32, 8, 64, FP16, False), (16385, 1, 32, 16, 128, BF16, False),
    (131072, 1, 32, 8, 128, BF16, False)])
def test_append_is_write_then_decode(n, T, H, Hkv, d, dtype, causal, dev):
    _say("append", n, T, H, Hkv, d, dtype, causal)
    gen = torch.Generator(device=dev).manual_seed(n)
    cap = n + 5
    cache = (*_cache(gen, Hkv, n - T, cap, d, dev), *_cache(gen, Hkv, n - T, cap, d, dev))
    q = torch.randn(T, H, d, generator=gen, device=dev).to(dtype)
    knew, vnew = _rows(gen, Hkv, T, d, dtype, dev), _rows(gen, Hkv, T, d, dtype, dev)
    apart = [x.clone() for x in cache]
    quantize4_pair(knew, vnew, (apart[0][:, n - T:n], apart[1][:, n - T:n]), (apart[2][:, n - T:n], apart[3][:, n - T:n]))
    want = decode_int4(q, *apart, n, d ** -0.5, causal=causal)
    for length in (n, torch.tensor([n], device=dev)):
        mine = [x.clone() for x in cache]
        got = decode_int4_append(q, *mine, knew, vnew, length, d ** -0.5, causal=causal)
        for x, y in zip(mine, apart):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), "the cache's bytes, spare rows included"
        if length is n:
            assert torch.equal(got, want)
        _check_decode(got, q, apart, n, d ** -0.5, causal)
    if T == 1:  # the one-token form
        mine = [x.clone() for x in cache]
        assert torch.equal(decode_int4_append(q[0], *mine, knew[:, 0], vnew[:, 0], n, d ** -0.5), want[0])


@pytest.mark.parametrize("d,dtype,scale_up", [(128, BF16, 40.0), (64, FP16, 40.0), (128, FP16, 200.0)])
def test_decode_large_scores(d, dtype, scale_up, dev):
    """Scores up to thousands, rising along the keys (the running maximum moves in every chunk), and probabilities that
    underflow."""
    _say("large scores", d, dtype, scale_up)
    gen = torch.Generator(device=dev).manual_seed(8)
    n, H, Hkv = 3001, 8, 2
    k = torch.randn(Hkv, n, d, generator=gen, device=dev) * torch.linspace(0.1, scale_up, n, device=dev)[None, :, None]
    v = _rows(gen, Hkv, n, d, BF16, dev)
    cache = (*plain.pack(*plain.quantize(k)), *plain.pack(*plain.quantize(v)))
    q = torch.randn(2, H, d, generator=gen, device=dev).to(dtype)
    for order in (torch.arange(n, device=dev), torch.arange(n - 1, -1, -1, device=dev)):
        mixed = tuple(x[:, order].contiguous() for x in cache)
        _check_decode(decode_int4(q, *mixed, n, d ** -0.5, causal=True), q, mixed, n, d ** -0.5, True)


def test_decode_small_and_large_scales(dev):
    """V scales that are subnormal in fp16 and near its largest value; outputs stay finite and as exact as the type."""
    _say("scales")
    gen = torch.Generator(device=dev).manual_seed(18)
    n, H, Hkv, d = 700, 8, 2, 128
    for size in (3e-6, 1e-4, 3e4):
        k, v = _rows(gen, Hkv, n, d, BF16, dev), torch.randn(Hkv, n, d, generator=gen, device=dev) * size
        cache = (*quantize4(k.contiguous()), *quantize4(v.clamp(-6e4, 6e4)))
        for dtype in (BF16, FP16):
            q = torch.randn(1, H, d, generator=gen, device=dev).to(dtype)
            _check_decode(decode_int4(q, *cache, n, d ** -0.5), q, cache, n, d ** -0.5, False)


@pytest.mark.parametrize("T,H,Hkv,d", [(1, 8, 2, 128), (4, 8, 2, 64), (3, 16, 2, 128)])
def test_decode_nonfinite_query_stays_with_its_row(T, H, Hkv, d, dev):
    _say("nonfinite query", T, H, Hkv, d)
    gen = torch.Generator(device=dev).manual_seed(6)
    n = 500
    cache = (*_cache(gen, Hkv, n, n + 3, d, dev), *_cache(gen, Hkv, n, n + 3, d, dev))
    q = torch.randn(T, H, d, generator=gen, device=dev).to(BF16)
    want = decode_int4(q, *cache, n, 0.1)
    for bad in (float("nan"), float("inf")):
        q2 = q.clone()
        q2[T - 1, 3, 5] = bad
        got = decode_int4(q2, *cache, n, 0.1)
        got[T - 1, 3] = want[T - 1, 3]
        assert torch.equal(got, want)


@pytest.mark.parametrize("d,lengths", [(64, (1, 2, 3, 31, 33, 127, 128, 129, 255, 513, 1535)),
                                       (128, (1, 2, 3, 31, 33, 63, 65, 129, 191, 255, 767))])
@pytest.mark.parametrize("heads", [(4, 2), (16, 2)])
def test_decode_every_tail(d, lengths, heads, dev):
    """Lengths that end inside a step, a chunk and a piece of params, in one split: narrow and wide kernel, host and device
    length, with a new last row."""
    _say("tails", d, heads)
    gen = torch.Generator(device=dev).manual_seed(d)
    H, Hkv = heads
    cache = (*_cache(gen, Hkv, 1600, 1601, d, dev), *_cache(gen, Hkv, 1600, 1601, d, dev))
    q = torch.randn(1, H, d, generator=gen, device=dev).to(FP16)
    k, v = _rows(gen, Hkv, 1, d, FP16, dev), _rows(gen, Hkv, 1, d, FP16, dev)
    for n in lengths:
        _check_decode(decode_int4(q, *cache, n, d ** -0.5), q, cache, n, d ** -0.5, False)
        mine = [x.clone() for x in cache]
        got = decode_int4_append(q, *mine, k, v, torch.tensor([n], device=dev), d ** -0.5)
        _check_decode(got, q, mine, n, d ** -0.5, False)
        want = plain.pack(*plain.quantize(v))
        assert torch.equal(mine[2][:, n - 1:n], want[0]) and torch.equal(mine[3][:, n - 1:n], want[1])
        assert torch.equal(mine[2][:, n:], cache[2][:, n:]) and torch.equal(mine[0][:, :n - 1], cache[0][:, :n - 1])


def test_decode_device_length_clamped_and_empty(dev):
    """A device-side length of 0 (or below) attends nothing: zeros, nothing read; past the capacity it is the capacity. With
    `causal`, the first tokens of a length below T attend nothing. Appended rows outside the cache are not written."""
    _say("device lengths")
    gen = torch.Generator(device=dev).manual_seed(2)
    cap, H, Hkv, d, T = 300, 8, 2, 128, 4
    cache = (*_cache(gen, Hkv, cap, cap, d, dev), *_cache(gen, Hkv, cap, cap, d, dev))
    q = torch.randn(T, H, d, generator=gen, device=dev).to(BF16)
    knew, vnew = _rows(gen, Hkv, T, d, BF16, dev), _rows(gen, Hkv, T, d, BF16, dev)
    length = torch.zeros(1, dtype=torch.int64, device=dev)
    for n in (0, -5):
        length.fill_(n)
        assert (decode_int4(q, *cache, length, 0.1) == 0).all()
    length.fill_(cap + 9)
    _check_decode(decode_int4(q, *cache, length, 0.1, causal=True), q, cache, cap, 0.1, True)
    length.fill_(2)
    got = decode_int4(q, *cache, length, 0.1, causal=True)
    assert (got[:2] == 0).all()
    _check_decode(got, q, cache, 2, 0.1, True)
    for n in (2, cap + 2, cap + 50):  # rows n - T .. n - 1 that lie in the cache, and no others
        mine = [x.clone() for x in cache]
        length.fill_(n)
        decode_int4_append(q, *mine, knew, vnew, length, 0.1)
        lo, hi = max(0, n - T), min(n, cap)
        for x, y, new, part in ((mine[0], cache[0], knew, 0), (mine[1], cache[1], knew, 1), (mine[2], cache[2], vnew, 0),
                                (mine[3], cache[3], vnew, 1)):
            want = y.clone()
            if lo < hi:
                want[:, lo:hi] = plain.pack(*plain.quantize(new))[part][:, lo - (n - T):hi - (n - T)]
            assert torch.equal(x, want), n


@pytest.mark.parametrize("T,d,dtype", [(1, 128, BF16), (3, 64, FP16)])
def test_captured_step_follows_the_length(T, d, dtype, dev):
    """A captured step (length += T, append, attend) replayed while the cache grows, eager work and synchronisations between
    the replays: every replay equals the eager step bit for bit, cache bytes included."""
    _say("graph", T, d, dtype)
    gen = torch.Generator(device=dev).manual_seed(31)
    n0, steps, H, Hkv = 250, 5, 8, 2
    cap = n0 + steps * T + 40
    cache = (*_cache(gen, Hkv, n0, cap, d, dev), *_cache(gen, Hkv, n0, cap, d, dev))
    eager = [x.clone() for x in cache]
    qs = torch.randn(steps, T, H, d, generator=gen, device=dev).to(dtype)
    ks = [_rows(gen, Hkv, T, d, dtype, dev).contiguous() for _ in range(steps)]
    vs = [_rows(gen, Hkv, T, d, dtype, dev).contiguous() for _ in range(steps)]
    q, k, v = qs[0].clone(), ks[0].clone(), vs[0].clone()
    length = torch.tensor([n0], device=dev)
    scratch = [x.clone() for x in cache]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up on copies
        decode_int4_append(q, *scratch, k, v, length + T, d ** -0.5, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        length.add_(T)
        out = decode_int4_append(q, *cache, k, v, length, d ** -0.5, causal=True)
    for i in range(steps):
        q.copy_(qs[i])
        k.copy_(ks[i])
        v.copy_(vs[i])
        graph.replay()
        torch.cuda.synchronize()
        n = n0 + (i + 1) * T
        assert length.item() == n
        want = decode_int4_append(qs[i], *eager, ks[i], vs[i], torch.tensor([n], device=dev), d ** -0.5, causal=True)
        assert torch.equal(out, want), f"replay {i}"
        for x, y in zip(cache, eager):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), f"cache after replay {i}"


@pytest.mark.parametrize("T,H,Hkv,d,dtype", [(1, 8, 2, 128, BF16), (4, 8, 2, 128, FP16), (3, 20, 2, 64, BF16)])
def test_two_captured_steps_with_partials(T, H, Hkv, d, dtype, dev):
    """Two steps captured over caches of several splits, in one memory pool, replayed in turn while both lengths grow, the live
    splits with them: every replay equals the eager step bit for bit, cache bytes included."""
    _say("two graphs", T, H, Hkv, d, dtype)
    gen = torch.Generator(device=dev).manual_seed(53)
    steps, graphs = 4, []
    for n0, cap, filled in ((900, 5000, 4900), (2550, 2700, 2550)):
        cache = (*_cache(gen, Hkv, filled, cap, d, dev), *_cache(gen, Hkv, filled, cap, d, dev))
        q = torch.randn(T, H, d, generator=gen, device=dev).to(dtype)
        k, v = (_rows(gen, Hkv, T, d, dtype, dev).contiguous() for _ in range(2))
        scratch = [x.clone() for x in cache]
        eager = [x.clone() for x in cache]
        length = torch.tensor([n0], device=dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm-up on copies
            decode_int4_append(q, *scratch, k, v, length + T, d ** -0.5)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            length.add_(T)
            out = decode_int4_append(q, *cache, k, v, length, d ** -0.5)
        graphs.append((graph, cache, eager, q, k, v, length, out, n0))
    for i in range(steps):
        for graph, cache, eager, q, k, v, length, out, n0 in graphs:
            for x in (q, k, v):
                x.copy_(torch.randn(x.shape, generator=gen, device=dev))
            jump = 400 if n0 == 900 else 0  # rows that the cache holds already
            length.add_(jump)
            graph.replay()
            torch.cuda.synchronize()
            n = n0 + (i + 1) * (T + jump)
            assert length.item() == n
            want = decode_int4_append(q, *eager, k, v, torch.tensor([n], device=dev), d ** -0.5)
            _check_decode(out, q, eager, n, d ** -0.5, False)
            assert torch.equal(out, want), f"replay {i}"
            for x, y in zip(cache, eager):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), f"cache after replay {i}"


def test_two_streams_at_once(dev):
    """Calls on two streams, each with its own cache, interleaved: every result as alone, and the same on every call."""
    _say("streams")
    gen = torch.Generator(device=dev).manual_seed(41)
    H, Hkv, d = 32, 8, 128
    work = []
    for n in (9001, 30000):
        cache = (*_cache(gen, Hkv, n, n, d, dev), *_cache(gen, Hkv, n, n, d, dev))
        q = torch.randn(1, H, d, generator=gen, device=dev).to(BF16)
        work.append((q, cache, n, decode_int4(q, *cache, n, d ** -0.5)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(10):
        for s, (q, cache, n, _) in zip(streams, work):
            with torch.cuda.stream(s):
                outs.append(decode_int4(q, *cache, n, d ** -0.5))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, work[i % 2][3])


def test_cache_past_32_bit_offsets(dev):
    """One KV head with 70 million rows (4.5 GB of codes): rows written, read back and attended past 2^32 bytes. All rows are
    zero but two planted ones, so the softmax has a closed form."""
    _say("70M rows")
    n, H, d = 70_000_003, 4, 128
    k4, v4 = (torch.zeros(1, n, d // 2, dtype=torch.uint8, device=dev) for _ in range(2))
    kp, vp = (torch.zeros(1, n, d // 32, 2, dtype=FP16, device=dev) for _ in range(2))
    q = torch.ones(1, H, d, device=dev, dtype=BF16)
    x = torch.full((1, 1, d), 16.0, device=dev, dtype=BF16)
    y = torch.arange(d, device=dev, dtype=FP32).to(BF16)[None, None]
    far = n - 4
    quantize4_pair(x, y, (k4[:, far:far + 1], kp[:, far:far + 1]), (v4[:, far:far + 1], vp[:, far:far + 1]))
    back = dequantize4_pair((k4[:, far - 1:far + 2], kp[:, far - 1:far + 2]), (v4[:, far - 1:far + 2], vp[:, far - 1:far + 2]),
                            FP32)
    assert (back[0][0, 1] == 16).all() and (back[0][0, ::2] == 0).all() and (back[1][0, ::2] == 0).all()
    yv = back[1][0, 1].double()
    scale = 17.0 / 2048  # a score of 17 at the planted key, 0 elsewhere
    for step in (False, True):
        if step:
            out = decode_int4_append(q, k4, kp, v4, vp, x, y, n, scale)
            w = torch.tensor(17.0, dtype=torch.float64).exp()
            p = 2 * w / (2 * w + n - 2)
        else:
            out = decode_int4(q, k4, kp, v4, vp, n, scale)
            w = torch.tensor(17.0, dtype=torch.float64).exp()
            p = w / (w + n - 1)
        want = (p * yv.cpu())[None].expand(H, d)
        # bf16 rounding of the output and of the probabilities, and fp32 sums over 2.7e5 keys a split
        assert ((out[0].double().cpu() - want).abs() <= want * (2.0 ** -7 + 2 ** -8) + 0.05).all()


# ---------------------------------------------------------------- the cache layer and RDAttention
def _attn(H, Hkv, d):
    base = SimpleNamespace(config=SimpleNamespace(num_attention_heads=H, num_key_value_heads=Hkv), layer_idx=0,
                           head_dim=d, scaling=d ** -0.5, q_proj=None, k_proj=None, v_proj=None, o_proj=None)
    return RDAttention(base, sink=64, window=16384, vertical=512, exact_tail=256)


def test_layer_appends_across_growth_and_crop(dev):
    _say("layer appends")
    g = torch.Generator().manual_seed(1)
    k = torch.randn(1, 2, 700, 64, generator=g).to(dev)
    v = torch.randn(1, 2, 700, 64, generator=g).to(dev)
    layer = Int4KVLayer()
    pk, pv = layer.update(k[..., :100, :], v[..., :100, :])
    assert torch.equal(pk, k[..., :100, :]) and torch.equal(pv, v[..., :100, :]), "prefill returns full precision"
    buffers = {layer.store_k.q.data_ptr()}
    for i in range(100, 700, 3):
        got_k, got_v = layer.update(k[..., i:i + 3, :], v[..., i:i + 3, :])
        buffers.add(layer.store_k.q.data_ptr())
    assert len(buffers) >= 1 + (700 - 100 - GROW) // GROW, "appends must have crossed several reallocations"
    want_k, want_v = (plain.values(*plain.pack(*plain.quantize(x)))[0].to(FP32) for x in (k, v))
    assert layer.get_seq_length() == 700 and got_k.shape == (1, 2, 700, 64)
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)
    assert layer.nbytes() == 2 * 700 * 2 * (32 + 8)
    layer.crop(-50)
    assert layer.get_seq_length() == 650 and torch.equal(layer.keys, want_k[..., :650, :])
    layer.update(k[..., :1, :], v[..., :1, :])
    assert torch.equal(layer.keys[..., 650:, :], want_k[..., :1, :])
    assert torch.equal(layer.values[..., :650, :], want_v[..., :650, :])
    layer.keys, layer.values = k[..., 10:40, :], v[..., 10:40, :]  # kv_evict's assignment
    assert layer.get_seq_length() == 30 and torch.equal(layer.keys, want_k[..., 10:40, :])
    with pytest.raises(NotImplementedError):
        layer.crop(3)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (FP16, 64)])
def test_layer_steps_through_rd_attention(dtype, d, dev):
    """Prompt, steps of one and of several tokens, a chunk too long for a handle, a crop, a further step: what RDAttention
    gives equals plain attention over the values of the layer's rows, and the rows equal a one-shot write."""
    _say("layer steps", dtype, d)
    H, Hkv = 16, 4
    attn, layer = _attn(H, Hkv, d), Int4KVLayer()
    gen = torch.Generator(device=dev).manual_seed(12)
    total = 600
    k, v = (torch.randn(1, Hkv, total, d, generator=gen, device=dev).to(dtype) for _ in range(2))
    layer.update(k[..., :500, :], v[..., :500, :])
    n = 500
    for t in (1, 1, 4, 1, 16, 40, 2):
        q = torch.randn(1, H, t, d, generator=gen, device=dev).to(dtype)
        kk, vv = layer.update(k[..., n:n + t, :], v[..., n:n + t, :], {"bb_attend": True})
        n += t
        assert isinstance(kk, Int4Handle) == (t <= Int4KVLayer.attend_tokens) and kk.shape == (1, Hkv, n, d)
        with torch.inference_mode():
            out = attn.exact_attention(q, kk, vv, t, n)
        assert layer._pending is None and out.shape == (1, H, t, d)
        cache = (*layer.store_k.rows(0, n), *layer.store_v.rows(0, n))
        if t <= Int4KVLayer.attend_tokens:
            _check_decode(out[0].transpose(0, 1), q[0].transpose(0, 1), cache, n, d ** -0.5, False)
        else:
            want, _ = plain.attend(q[0].transpose(0, 1), *cache, n, d ** -0.5)
            assert (out[0].transpose(0, 1).double() - want).abs().max() < 2e-2  # the flash kernel's bar over 16-bit values
        if t == 16:
            layer.crop(-3)
            n -= 3
            k = torch.cat([k[..., :n, :], k[..., n + 3:, :]], -2)
            v = torch.cat([v[..., :n, :], v[..., n + 3:, :]], -2)
    for got, x in ((layer.keys, k), (layer.values, v)):
        assert torch.equal(got, plain.values(*plain.pack(*plain.quantize(x[..., :n, :])))[0].to(FP32).to(dtype))


def test_layer_pending_rows_on_every_path(dev):
    """Rows handed out behind a handle are quantised on every other path that looks at the cache first."""
    _say("pending")
    g = torch.Generator(device=dev).manual_seed(8)
    H, Hkv, d = 8, 2, 128
    k, v = (torch.randn(1, Hkv, 310, d, generator=g, device=dev).to(BF16) for _ in range(2))
    want_k, want_v = (plain.values(*plain.pack(*plain.quantize(x)))[0].to(FP32).to(BF16) for x in (k, v))
    layer = Int4KVLayer()
    layer.update(k[..., :300, :], v[..., :300, :])
    hk, _ = layer.update(k[..., 300:302, :], v[..., 300:302, :], {"bb_attend": True})
    assert isinstance(hk, Int4Handle) and layer._pending is not None
    assert torch.equal(layer.keys, want_k[..., :302, :]) and layer._pending is None
    layer.update(k[..., 302:303, :], v[..., 302:303, :], {"bb_attend": True})
    assert layer.nbytes() == 2 * 303 * Hkv * (64 + 16) and layer._pending is None
    layer.update(k[..., 303:306, :], v[..., 303:306, :], {"bb_attend": True})
    layer.update(k[..., 306:310, :], v[..., 306:310, :], {"bb_attend": True})
    q = torch.randn(1, H, 1, d, generator=g, device=dev).to(BF16)
    out = hk.attend(q, d ** -0.5)  # a stale handle, with another number of queries than pending rows
    assert layer._pending is None
    assert torch.equal(layer.values, want_v) and torch.equal(layer.keys, want_k)
    cache = (*layer.store_k.rows(0, 310), *layer.store_v.rows(0, 310))
    _check_decode(out[0].transpose(0, 1), q[0].transpose(0, 1), cache, 310, d ** -0.5, False)
    with pytest.raises(ValueError):
        layer.update(k[..., :1, :], v[..., :1, :], {"bb_attend": True})[0].attend(q.float(), 0.1)
    assert torch.equal(layer.keys[..., 310:, :], want_k[..., :1, :]), "a refused attend loses no row"


def test_handle_with_many_vectors_reads_the_cache_back(dev):
    """16 tokens of 16 query heads over one KV head: more vectors than the handle gives to the decode kernel."""
    _say("many vectors")
    g = torch.Generator(device=dev).manual_seed(9)
    H, d, n = 16, 128, 400
    layer = Int4KVLayer()
    k, v = (torch.randn(1, 1, n, d, generator=g, device=dev).to(BF16) for _ in range(2))
    layer.update(k[..., :n - 16, :], v[..., :n - 16, :])
    handle, _ = layer.update(k[..., n - 16:, :], v[..., n - 16:, :], {"bb_attend": True})
    assert isinstance(handle, Int4Handle)
    q = torch.randn(1, H, 16, d, generator=g, device=dev).to(BF16)
    more = torch.randn(1, H, 20, d, generator=g, device=dev).to(BF16)  # more tokens than a call of the kernel takes
    for qq in (q, more):
        t = qq.shape[2]
        out = _attn(H, 1, d).exact_attention(qq, handle, handle, t, n)
        assert layer._pending is None and out.shape == (1, H, t, d)
        cache = (*layer.store_k.rows(0, n), *layer.store_v.rows(0, n))
        want, _ = plain.attend(qq[0].transpose(0, 1), *cache, n, d ** -0.5)
        assert (out[0].transpose(0, 1).double() - want).abs().max() < 2e-2  # the flash kernel's bar over 16-bit values


KW = dict(sink=8, window=96, vertical=24, n_route=16, exact_tail=24, block_m=16, block_n=16)


@pytest.mark.parametrize("installed", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_model_generates_on_the_4bit_cache(installed, dtype, dev, monkeypatch):
    """A small model decoding on the 4-bit cache, with RDAttention (fused handles, once per layer and step) and with the
    stock HF module (dequantised tensors): prefill logits identical to a DynamicCache, and each decode step's logits equal
    to those of the same model on a 16-bit cache that holds the 4-bit values, within the flash and decode kernels' rounding
    (0.05, the bar of the int8 cache's test)."""
    _say("model", installed, dtype)
    from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

    cfg = LlamaConfig(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=8192,
                      attn_implementation="sdpa")
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).to(dev, dtype).eval()
    if installed:
        install(model, "rd", **KW)
    ids = torch.randint(0, 512, (1, 406), generator=torch.Generator().manual_seed(4)).to(dev)
    calls = []
    real = Int4Handle.attend
    monkeypatch.setattr(Int4Handle, "attend", lambda h, q, s: calls.append(1) or real(h, q, s))
    packed, plain16 = make_int4_cache(model.config), DynamicCache(config=model.config)
    with torch.inference_mode():
        a = model(ids[:, :400], past_key_values=packed, use_cache=True).logits
        b = model(ids[:, :400], past_key_values=plain16, use_cache=True).logits
        assert torch.equal(a, b), "prefill logits must be identical"
        for i in range(400, 406):
            for mine, theirs in zip(packed.layers, plain16.layers):  # the 16-bit cache takes the 4-bit values
                theirs.keys, theirs.values = mine.keys.clone(), mine.values.clone()
            a = model(ids[:, i:i + 1], past_key_values=packed, use_cache=True).logits
            b = model(ids[:, i:i + 1], past_key_values=plain16, use_cache=True).logits
            # the step's own row is 4-bit here and 16-bit there: one key of 400
            assert (a.float() - b.float()).abs().max().item() < 0.05
    assert all(x.get_seq_length() == 406 for x in packed.layers)
    assert len(calls) == (12 if installed else 0)


def test_composes_with_kv_evict(dev):
    _say("evict")
    from transformers import LlamaConfig, LlamaForCausalLM

    cfg = LlamaConfig(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=8192,
                      attn_implementation="sdpa")
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).to(dev, BF16).eval()
    install(model, "rd", kv_evict=True, **KW)
    ids = torch.randint(0, 512, (1, 400), generator=torch.Generator().manual_seed(4)).to(dev)
    cache = make_int4_cache(model.config)
    with torch.inference_mode():
        model(ids, past_key_values=cache, use_cache=True)
        m = KW["sink"] + KW["window"] + 4 * KW["vertical"]
        assert all(x.get_seq_length() == m for x in cache.layers)
        out = model(ids[:, :1], past_key_values=cache, use_cache=True,
                    cache_position=torch.tensor([400], device=dev)).logits
    assert torch.isfinite(out.float()).all() and all(x.get_seq_length() == m + 1 for x in cache.layers)


def test_write_attend_read_together(dev):
    """The operators as a serving loop uses them: a prompt written, steps appended and attended, a draft verified causally,
    rejected rows dropped and written over, and the whole cache read back for a dense chunk of 16-bit attention."""
    _say("together")
    gen = torch.Generator(device=dev).manual_seed(77)
    H, Hkv, d, cap = 32, 8, 128, 2048
    k4, v4 = (torch.empty(Hkv, cap, d // 2, dtype=torch.uint8, device=dev) for _ in range(2))
    kp, vp = (torch.full((Hkv, cap, d // 32, 2), float("nan"), dtype=FP16, device=dev) for _ in range(2))
    k, v = _rows(gen, Hkv, cap, d, BF16, dev), _rows(gen, Hkv, cap, d, BF16, dev)
    n = 1500
    quantize4_pair(k[:, :n], v[:, :n], (k4[:, :n], kp[:, :n]), (v4[:, :n], vp[:, :n]))
    cache = (k4, kp, v4, vp)
    for T, kept in ((1, 1), (1, 1), (4, 2), (4, 4), (1, 1), (8, 1), (1, 1)):
        q = torch.randn(T, H, d, generator=gen, device=dev).to(BF16)
        out = decode_int4_append(q, *cache, k[:, n:n + T], v[:, n:n + T], n + T, d ** -0.5, causal=True)
        _check_decode(out, q, cache, n + T, d ** -0.5, True)
        n += kept
    kd, vd = dequantize4_pair((k4[:, :n], kp[:, :n]), (v4[:, :n], vp[:, :n]), BF16)
    for got, x in ((kd, k), (vd, v)):
        assert torch.equal(got, plain.values(*plain.pack(*plain.quantize(x[:, :n])))[0].to(FP32).to(BF16))
    q = torch.randn(H, 64, d, generator=gen, device=dev).to(BF16)
    none = torch.empty((H, 1, 0), dtype=torch.int32, device=dev)
    dense = bigger_bird_flash(q, kd, vd, none, front=0, window=n, num_heads=H, kv_groups=H // Hkv, scale=d ** -0.5)
    one = decode_int4(q[:, -1].contiguous(), *cache, n, d ** -0.5)
    assert (dense[:, -1].float() - one.float()).abs().max() < 2e-2  # the last row of both attends all keys


def test_refusals_on_the_gpu(dev):
    _say("refusals")
    q4, p4 = quantize4(torch.randn(2, 10, 128, device=dev))
    q = torch.randn(1, 8, 128, device=dev).to(BF16)
    good = (q4, p4, q4.clone(), p4.clone())
    for n, match in ((0, "empty cache"), (11, "capacity")):
        with pytest.raises(ValueError, match=match):
            decode_int4(q, *good, n, 0.1)
    with pytest.raises(ValueError, match="at least as long"):
        decode_int4(q.expand(4, 8, 128), *good, 3, 0.1)
    with pytest.raises(ValueError, match="1 to 16"):
        decode_int4(q.expand(17, 8, 128), *[x.repeat(1, 3, *[1] * (x.ndim - 2)) for x in good], 20, 0.1)
    with pytest.raises(ValueError, match="scale"):
        decode_int4(q, *good, 10, 0.0)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        decode_int4(q.float(), *good, 10, 0.1)
    with pytest.raises(ValueError, match="must match"):
        decode_int4(q[:, :7], *good, 10, 0.1)
    with pytest.raises(ValueError, match="must match"):
        decode_int4(q, q4, p4, q4[:, :9], p4[:, :9], 9, 0.1)
    with pytest.raises(ValueError, match="contiguous"):
        decode_int4(q, q4[:, ::2], p4[:, ::2], q4[:, ::2], p4[:, ::2], 5, 0.1)
    with pytest.raises(ValueError, match="uint8"):
        decode_int4(q, q4.to(torch.int8), p4, q4, p4, 5, 0.1)
    with pytest.raises(ValueError, match="int64"):
        decode_int4(q, *good, torch.tensor([5], device=dev, dtype=torch.int32), 0.1)
    with pytest.raises(ValueError, match="head_dim 32"):
        s4, t4 = quantize4(torch.randn(2, 10, 32, device=dev))
        decode_int4(q[..., :32], s4, t4, s4, t4, 10, 0.1)
    with pytest.raises(ValueError, match="new rows"):
        decode_int4_append(q, *good, q4.new_zeros(2, 1, 128), q4.new_zeros(2, 1, 128), 10, 0.1)
    with pytest.raises(ValueError, match="required"):
        decode_int4_append(q, *good, None, None, 10, 0.1)
    with pytest.raises(ValueError, match="runs on the ROCm device"):
        decode_int4(q, *[x.cpu() for x in good], 10, 0.1)
    with pytest.raises(ValueError, match="must match x"):
        quantize4(torch.randn(2, 10, 64, device=dev), (q4, p4))
    with pytest.raises(ValueError, match="same rows"):
        dequantize4_pair((q4, p4), (q4[:, :5], p4[:, :5]), BF16)
    with pytest.raises(ValueError, match="output"):
        dequantize4(q4, p4, torch.float64)
    with pytest.raises(ValueError, match="input"):
        quantize4(torch.zeros(2, 10, 128, device=dev, dtype=torch.float64))
    empty = quantize4(torch.zeros(2, 0, 128, device=dev))
    assert empty[0].shape == (2, 0, 64) and dequantize4(*empty, BF16).shape == (2, 0, 128)
    assert kv_int4.MAX_TOKENS == 16
