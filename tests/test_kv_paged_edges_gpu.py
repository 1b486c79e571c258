"""Paged KV cache on the GPU at its edges: where a value that is not finite lies, scores and queries near the types' ends, calls that
are refused, against the plain 64-bit forms of tests/paged_plain.py."""
import pytest
import torch

import paged_plain as plain
from bigger_bird_amd import paged_attention
from test_kv_paged_gpu import BF16, FP16, STREAM_VECTORS, _attend_case, _check, _heads, _int, _p_step, _pages, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [407, 3000])
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16)])
def test_a_value_that_is_not_finite_wherever_it_lies(n, d, dtype, dev):
    """70 tokens, 280 vectors; each of their rows in turn holds infinities and NaN, so that every wave comes to load one: the tokens
    before it do not attend it, those from it on do."""
    _say("one value", n, d, dtype)
    T, H, hk = 70, 8, 2
    q, kp, vp, table, lens, _ = _attend_case([n], None, T, H, hk, d, 64, dtype, dev)
    want, tol = plain.attend(q, kp, vp, table, [n], d ** -0.5, None, _p_step(dtype, T * H // hk <= STREAM_VECTORS))
    for j in range(T):
        r = n - T + j
        at = table[0, r // 64].item(), slice(None), r % 64
        old = vp[at].clone()
        vp[at] = float("nan") if j % 2 else float("inf")
        got = paged_attention(q, kp, vp, table, lens, d ** -0.5)
        vp[at] = old
        if j:
            _check(got[:, :, :j], want[:, :, :j], tol[:, :, :j], dtype)
        assert not torch.isfinite(got[:, :, j:].float()).any()


@pytest.mark.parametrize("B", [40, 70])  # up to 64 sequences each workgroup finds its work; more are laid out before
@pytest.mark.parametrize("T", [1, 40])
def test_tables_of_many_rows(B, T, dev):
    """A table of 2^28 rows, the most there may be, over sequences of a few hundred that share their pages."""
    _say("wide tables", B, T)
    gen = torch.Generator(device=dev).manual_seed(B + T)
    kp, vp = _pages(gen, 12, 8, 64, 64, BF16, dev)
    one = torch.full((1, 1 << 22), -1, dtype=torch.int32, device=dev)
    one[0, :12] = torch.randperm(12, generator=gen, device=dev).int()
    lens = [(97 * i) % 700 for i in range(B)]
    new = [min(T, n) for n in lens]
    q = _heads(gen, B, 8, T, 64, BF16, dev)
    table = one.expand(B, -1)
    got = paged_attention(q, kp, vp, table, _int(lens, dev), 0.125, new=_int(new, dev))
    want, tol = plain.attend(q, kp, vp, table[:, :12], lens, 0.125, new, _p_step(BF16, T <= STREAM_VECTORS))
    _check(got, want, tol, BF16)
