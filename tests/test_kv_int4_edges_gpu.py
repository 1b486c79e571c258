"""4-bit KV cache on the GPU: the sums' precision, rows that are not finite or far below zero, layouts that a copy has to put right,
and the cache layer where a step is refused, against the 64-bit forms of tests/int4_plain.py."""
import pytest
import torch

import int4_plain as plain
from bigger_bird_amd.kv_int4 import decode_int4

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
