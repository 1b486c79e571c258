"""Paged KV cache on the GPU at its edges: where a value that is not finite lies, scores and queries near the types' ends, calls that
are refused, against the plain 64-bit forms of tests/paged_plain.py."""
import pytest
import torch

import paged_plain as plain
from bigger_bird_amd import paged_append, paged_attention, paged_step
from paged_plain import HALF_STEP
from test_kv_paged_gpu import (BF16, FP16, FP32, STEP_VECTORS, STREAM_VECTORS, _attend_case, _check, _heads, _int, _model, _p_step,
                               _pages, _say, _table)

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


@pytest.mark.parametrize("T,H,hk", [(1, 8, 2), (8, 8, 2), (20, 8, 2)])  # one block of 16 vectors, 32 of them, three tiles of 32
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("rot", [FP16, FP32])
def test_rotated_queries_past_what_fp16_holds(T, H, hk, d, rot, dev):
    """Pairs of 50000 turned by 45 degrees are 70711, and angles with a factor (as scaled RoPE has them) make them larger; a query
    that is not finite is NaN still, beside them."""
    _say("large queries", T, H, d, rot)
    gen = torch.Generator(device=dev).manual_seed(T)
    lens = [700, 65]
    table, p = _table(gen, lens, 16, dev)
    kp, vp = _pages(gen, p, hk, 16, d, FP16, dev)
    q, k, v = (_heads(gen, 2, h, T, d, FP16, dev) for h in (H, hk, hk))
    q[0, ::2] = q[0, ::2].sign() * 50000  # one sequence's every second head; the others are as they were
    cos = torch.full((2, T, d), 0.70710678, device=dev).to(rot)
    sin = cos.clone()
    if rot == FP32:
        cos[0], sin[0] = cos[0] * 300, sin[0] * 300
        k[0] /= 300
    q[1, 1, T - 1, 3] = float("nan")
    got = paged_step(q, k, v, kp, vp, table, _int(lens, dev), 2.0 ** -24, cos=cos, sin=sin)
    assert torch.isnan(got[1, 1, T - 1]).all()
    got[1, 1, T - 1], q[1, 1, T - 1] = 0, 0
    qr = plain.rotate(q, cos[:, None], sin[:, None])
    assert (qr.abs().amax(-1)[0, ::2] > 65519).any()
    want, tol = plain.attend(qr, kp, vp, table, lens, 2.0 ** -24, None, _p_step(FP16, True), HALF_STEP[FP16] ** 2 + 2.0 ** -20)
    got[1, 1, T - 1] = want[1, 1, T - 1].half()
    _check(got, want, tol, FP16)


@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("size", [1.109375, 1.3359375])
@pytest.mark.parametrize("dtype,exponents", [(BF16, (0, 20, 26, 28, 33, 60, 100)), (FP16, (0, 14, 22, 24, 26, 28))])
def test_large_scores_of_any_mantissa(T, size, dtype, exponents, dev):
    """Scores of 64 * size * 2^e and their negatives, whose product with scale log2(e) is not exact: all the same, so that the output
    is the mean of the values, and falling by 64 * 2^(e - 5) a row, where the first row takes all for scores of 2^20 and more.

    Tolerance: a probability is 2^x for all rows alike, its rounding as an operand of HALF_STEP in the numerator only; sums of 400
    terms in fp32; the output's rounding."""
    _say("large scores", T, size, dtype)
    q, kp, vp, table, lens, _ = _attend_case([400], None, T, 4, 2, 64, 16, dtype, dev)
    row = torch.arange(16, device=dev)
    for e in exponents:
        a, b = (2.0 ** (e // 2), 2.0 ** (e - e // 2)) if dtype == FP16 else (1.0, 2.0 ** e)
        for sign in (1.0, -1.0):
            qq = torch.full_like(q, sign * a)
            kp[:] = size * b
            want, _ = plain.attend(qq, kp, vp, table, [400], 1.0, None, 0.0)
            mean, _ = plain.attend(qq, kp, vp.abs(), table, [400], 1.0, None, 0.0)
            _check(paged_attention(qq, kp, vp, table, lens, 1.0), want, (HALF_STEP[dtype] + 400 * 2.0 ** -23) * mean, dtype)
        if e < 20:
            continue
        # the first page's rows size, size - 1/32, .., the rest lower than all of them
        kp[:] = b / 2
        kp[table[0, 0].item()] = ((size - row / 32) * b).to(dtype)[:, None]
        first = vp[table[0, 0].item(), :, 0].double()[None, :, None].repeat_interleave(2, 1).expand(1, 4, T, 64)
        _check(paged_attention(torch.full_like(q, a), kp, vp, table, lens, 1.0), first, HALF_STEP[dtype] * first.abs(), dtype)


def _infinite_values(q, kp, vp, table, lens, T, page, dtype, gen):
    """Infinities and NaN into some columns of V, at rows that tokens attend: +inf, -inf and NaN alone, +inf and -inf together and
    two of a sign; a row early in the sequence, in the middle, among the last T, and one whose scores are far below the others'."""
    inf, nan = float("inf"), float("nan")
    at = lambda b, r: (table[b, r // page].item(), slice(None), r % page)
    for b, n in enumerate(lens):
        if not n:
            continue
        rows = [0, n // 3, n // 2, max(0, n - 2), n - 1]
        kp[at(b, rows[1])] = -3 * q[b, ::q.shape[1] // kp.shape[1], 0]  # for the first head's first token: scores far below
        for c, marks in enumerate(([(0, inf)], [(1, -inf)], [(2, nan)], [(3, inf), (0, -inf)], [(4, inf), (2, inf)], [(4, -inf)],
                                   [(1, inf), (4, nan)], [(0, -inf), (3, -inf)])):
            for r, x in marks:
                page_, _, row = at(b, rows[r])
                vp[page_, :, row, 7 * c + 1] = x


def _attend_infinities(q, kp, vp, table, lens, scale, new, p_step):
    """plain.attend of the finite values, and over it what attended infinities and NaN come to: a softmax's probabilities are all
    positive, so +inf, -inf, or NaN where there are both or a NaN. (Looked up in V itself: torch's softmax in 64 bits on the GPU
    gives 0 for e^-95, and 0 times an infinity is not what the formula says.)"""
    finite = torch.where(torch.isfinite(vp), vp, 0)
    want, tol = plain.attend(q, kp, finite, table, lens, scale, new, p_step)
    B, H, T, d = q.shape
    hk, page = vp.shape[1], vp.shape[2]
    up, down = (torch.zeros(B, hk, T, d, dtype=torch.bool, device=q.device) for _ in "+-")
    for b in range(B):
        v, _ = plain.rows_of(vp, table, b, lens[b])
        is_up, is_down = (torch.isnan(v) | (v == x) for x in (float("inf"), -float("inf")))
        for j in range(T):
            n = plain.seen(lens, new, T, table.shape[1] * page, b, j)
            up[b, :, j], down[b, :, j] = is_up[:, :n].any(1), is_down[:, :n].any(1)
    up, down = (x.repeat_interleave(H // hk, 1) for x in (up, down))
    want[up], want[down], want[up & down] = float("inf"), -float("inf"), float("nan")
    return want, tol


def _check_with_infinities(got, want, tol, dtype):
    assert torch.isinf(want).any() and torch.isnan(want).any()
    whole = torch.isfinite(want)
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert (f(got) == f(want)).all(), (f.__name__, (f(got) != f(want)).nonzero()[:5].tolist())
    zero = torch.zeros_like(want)
    _check(torch.where(whole, got, 0), torch.where(whole, want, zero), tol, dtype)


@pytest.mark.parametrize("lens,T,H,hk", [([300, 47, 0], 1, 8, 2), ([300, 47, 9], 4, 8, 2), ([9001, 70], 1, 4, 1), ([700, 45], 8, 12, 3),
                                         ([300, 90], 40, 8, 2), ([700], 300, 4, 4), ([5000], 70, 8, 2)])
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, FP16), (64, BF16), (128, FP16)])
def test_infinite_values_that_are_attended(lens, T, H, hk, d, dtype, dev):
    """A column that attends +inf is +inf, with -inf too or NaN it is NaN, in every kernel and however small the probability; the
    other columns are not touched. In the step the last rows come in as new ones."""
    _say("infinite values", lens, T, H, hk, d, dtype)
    gen = torch.Generator(device=dev).manual_seed(T)
    new = [min(T, n) for n in lens]
    q, kp, vp, table, ln, nw = _attend_case(lens, new, T, H, hk, d, 16, dtype, dev)
    _infinite_values(q, kp, vp, table, lens, T, 16, dtype, gen)
    scale = 2 * d ** -0.5
    for step in (False, True):
        streams = T * H // hk <= (STEP_VECTORS if step else STREAM_VECTORS)
        want, tol = _attend_infinities(q, kp, vp, table, lens, scale, new, _p_step(dtype, streams))
        if step:
            k, v = (torch.zeros(len(lens), hk, T, d, dtype=dtype, device=dev) for _ in "kv")
            for b, n in enumerate(lens):
                for j in range(new[b]):
                    r = n - new[b] + j
                    page, row = table[b, r // 16].item(), r % 16
                    k[b, :, j], v[b, :, j] = kp[page, :, row], vp[page, :, row]
                    kp[page, :, row], vp[page, :, row] = 0, float("nan")
            got = paged_step(q, k, v, kp, vp, table, ln, scale, new=nw)
        else:
            got = paged_attention(q, kp, vp, table, ln, scale, new=nw)
        _check_with_infinities(got, want, tol, dtype)


def test_rows_without_an_aligned_copy_are_refused(dev):
    _say("head_dim 100")
    pages = torch.zeros(3, 2, 16, 104, dtype=BF16, device=dev)[..., :100]
    table, lens = _int([[0, 1]], dev), _int([20], dev)
    q, k = torch.zeros(1, 4, 1, 100, dtype=BF16, device=dev), torch.zeros(1, 2, 1, 100, dtype=BF16, device=dev)
    for call in (lambda: paged_attention(q, pages, pages, table, lens, 1.0), lambda: paged_append(k, k, pages, pages, table, lens),
                 lambda: paged_step(q, k, k, pages, pages, table, lens, 1.0)):
        with pytest.raises(ValueError, match="head_dim 100 unsupported"):
            call()


def test_model_masks_of_one_sequence(dev):
    """With eager attention a model always makes a causal mask: one sequence runs, prompt, chunk and token, as without one; a padded
    prompt is refused, and run by its count after extend."""
    _say("masks of one sequence")
    from bigger_bird_amd import make_paged_cache

    model = _model(dev, "dense_rd")
    ids = torch.randint(0, 512, (1, 60), generator=torch.Generator().manual_seed(3)).to(dev)
    mask = torch.ones(1, 40, dtype=torch.long, device=dev)
    outs = []
    with torch.no_grad():
        for kind in ("sdpa", "eager"):
            model.config._attn_implementation = kind
            cache = make_paged_cache(model.config, 1, 20, page=16, device=dev)
            outs.append([model(input_ids=ids[:, a:b], past_key_values=cache, use_cache=True).logits
                         for a, b in ((0, 40), (40, 59), (59, 60))])
            assert cache.lengths == [60]
            for side in (slice(0, 3), slice(37, 40)):
                cache, padded = make_paged_cache(model.config, 1, 20, page=16, device=dev), mask.clone()
                padded[:, side] = 0
                with pytest.raises(ValueError, match="not by a mask"):
                    model(input_ids=ids[:, :40], attention_mask=padded, past_key_values=cache, use_cache=True)
                assert cache.lengths == [0]
            cache.extend([37])
            got = model(input_ids=ids[:, :40], attention_mask=padded, past_key_values=cache, use_cache=True).logits
            assert cache.lengths == [37] and torch.equal(got[:, :37], outs[0][0][:, :37])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("layout", ["heads", "rows", "pool", "padded"])
@pytest.mark.parametrize("T,H,hk", [(1, 8, 2), (6, 8, 2), (90, 8, 2)])
@pytest.mark.parametrize("d,dtype,page", [(128, BF16, 16), (64, FP16, 64)])
def test_infinite_values_in_any_layout_beside_unnamed_pages(layout, T, H, hk, d, dtype, page, dev):
    """The rows that infinities are looked up in are those of the table's pages, with the pages' strides, up to each token's own."""
    _say("infinite values", layout, T, d, dtype, page)
    gen = torch.Generator(device=dev).manual_seed(T + page)
    lens, T_new = [1500, 200], [T, max(1, T // 2)]
    q, kp, vp, table, ln, nw = _attend_case(lens, T_new, T, H, hk, d, page, dtype, dev, layout)
    own = torch.zeros(kp.shape[0], page, dtype=torch.bool, device=dev)
    for b, n in enumerate(lens):
        for r in range(n):
            own[table[b, r // page].item(), r % page] = True
    vp.masked_fill_(~own[:, None, :, None], float("-inf"))  # what no sequence holds
    table[0, 3], table[1, 1] = -1, 2 ** 30
    for b, n in enumerate(lens):
        for c, (r, x) in enumerate(((0, float("inf")), (n // 2, float("-inf")), (n - 1, float("inf")), (n - 1, float("nan")),
                                    (3 * page + 1 if b == 0 else page + 1, float("inf")))):  # the last on a page that is not named
            e = int(table[b, r // page])
            if 0 <= e < vp.shape[0]:
                vp[e, :, r % page, 9 * c + 2] = x
    want, tol = _attend_infinities(q, kp, vp, table, lens, d ** -0.5, T_new, _p_step(dtype, T * H // hk <= STREAM_VECTORS))
    got = paged_attention(q, kp, vp, table, ln, d ** -0.5, new=nw)
    _check_with_infinities(got, want, tol, dtype)
