"""The paged cache's operators in plain 64-bit torch, for the tests (CPU or GPU tensors)."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rows_of(pages, table, b, n):
    """(rows [Hkv, n, d] of sequence b in 64 bits, whether each of them is on a page); rows of no page are zeros."""
    p, hk, page, d = pages.shape
    out = torch.zeros(hk, n, d, dtype=torch.float64, device=pages.device)
    on = torch.zeros(n, dtype=torch.bool, device=pages.device)
    for w in range(-(-n // page)):
        e = int(table[b, w])
        if 0 <= e < p:
            m = min(page, n - w * page)
            out[:, w * page:w * page + m] = pages[e, :, :m].double()
            on[w * page:w * page + m] = True
    return out, on


def seen(lens, new, T, cap, b, j):
    """Rows that token j of sequence b attends."""
    fresh = T if new is None else min(max(int(new[b]), 0), T)
    n = int(lens[b])
    return min(max(n - fresh + j + 1, 0), min(max(n, 0), cap)) if j < fresh else 0


def rotate(x, cos, sin):
    """x [..., T, d] with cos, sin [..., T, d], 64 bits."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    h = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., h:], x[..., :h]], -1) * sin


def append_rows(lens, new, T, table, pages, page):
    """[(b, j, page, row in it)] of the tokens that are written."""
    out = []
    for b in range(len(lens)):
        fresh = T if new is None else min(max(int(new[b]), 0), T)
        for j in range(fresh):
            r = int(lens[b]) - fresh + j
            if 0 <= r < table.shape[1] * page and 0 <= int(table[b, r // page]) < pages:
                out.append((b, j, int(table[b, r // page]), r % page))
    return out


def attend(q, kp, vp, table, lens, scale, new, p_step, q_step=0.0):
    """q [B, H, T, d] (any float type) over the pages in 64 bits: (out, bound).

    The bound is what a kernel that works in fp32 with 16-bit matrix operands may be off before its output is rounded:
      * a score is a sum of d products in fp32, at most d + 8 roundings of 2^-24 of sum |q| |k|, and the scaling another two;
        a query kept in 16-bit terms is off by q_step of itself, which moves the score by q_step sum |q| |k|. The exponential is
        off by as much as the score, and by 2^-22 for the instruction and its argument's rounding (an argument of size up to
        |score - max| <= 256 where the probability is not negligible: 256 * 2^-24 more); numerator and denominator both;
      * a probability's rounding as an operand, p_step, and in fp16 2^-25 absolute where it is subnormal (the sum of
        probabilities is at least 1, as the largest is); numerator only;
      * sums over keys in fp32: chains of at most 4096 terms, 2^-24 each, numerator and denominator."""
    B, H, T, d = q.shape
    hk, page = kp.shape[1], kp.shape[2]
    G, cap = H // hk, table.shape[1] * page
    out = torch.zeros(B, H, T, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    tiny = 2.0 ** -25 if kp.dtype == torch.float16 else 0.0
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        k, on = rows_of(kp, table, b, n)
        v, _ = rows_of(vp, table, b, n)
        for j in range(T):
            m = seen(lens, new, T, cap, b, j)
            keep = on[:m].nonzero()[:, 0]
            if not len(keep):
                continue
            qq = q[b, :, j].double().view(hk, G, d)
            kk, vv = k[:, keep], v[:, keep]
            x = qq @ kk.transpose(1, 2) * scale
            size = (qq.abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True) * scale
            p = torch.softmax(x, -1)
            dx = size * ((d + 10) * 2.0 ** -24 + q_step) + 2.0 ** -22 + 256 * 2.0 ** -24 + 4096 * 2.0 ** -24
            pv = p @ vv.abs()
            out[b, :, j] = (p @ vv).view(H, d)
            tol[b, :, j] = (pv * (2 * dx + p_step) + tiny * vv.abs().sum(1, keepdim=True)).reshape(H, d)
    return out, tol
