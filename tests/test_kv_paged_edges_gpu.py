"""Paged KV cache on the GPU at its edges: where a value that is not finite lies, scores and queries near the types' ends, calls that
are refused, against the plain 64-bit forms of tests/paged_plain.py."""
import pytest
import torch

import paged_plain as plain
from bigger_bird_amd import paged_attention
from test_kv_paged_gpu import BF16, FP16, STREAM_VECTORS, _attend_case, _check, _p_step, _say

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
