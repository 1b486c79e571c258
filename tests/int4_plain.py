"""The 4-bit cache format and its attention in plain 64-bit torch, for the tests (CPU or GPU tensors)."""
import torch


def quantize(x):
    """x [..., t, d] (any float type) -> codes [..., t, d] (0..15), s and z [..., t, d / 32], all float64: the format's fp32
    and fp16 roundings, every quantity in 64 bits between them."""
    r32 = lambda y: y.to(torch.float32).double()  # noqa: E731
    w = x.double().unflatten(-1, (-1, 32))
    nan = torch.isnan(w)
    lo = torch.where(nan, torch.inf, w).amin(-1)
    hi = torch.where(nan, -torch.inf, w).amax(-1)
    some = lo <= hi
    lo, hi = (torch.where(some, y.clamp(-65504.0, 65504.0), 0.0) for y in (lo, hi))
    z = lo.to(torch.float16).double()
    s = r32(r32(hi - z) / 15).clamp_min(0).to(torch.float16).double()
    safe = torch.where(s > 0, s, torch.ones_like(s))
    code = torch.round(r32(r32(w - z[..., None]) / safe[..., None])).clamp(0, 15)
    code = torch.where((s[..., None] > 0) & ~nan, code, torch.zeros_like(code))
    return code.flatten(-2), s, z


def pack(code, s, z):
    """codes and params as the cache holds them."""
    c = code.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack([s, z], -1).to(torch.float16)


def codes(q):
    """The codes [..., d] of packed rows [..., d / 2]."""
    return torch.stack([q & 15, q >> 4], -1).flatten(-2)


def values(q, p):
    """The values of packed rows in 64 bits, and the group scales spread over the elements."""
    c = codes(q).double()
    s = p[..., 0].double().repeat_interleave(32, -1)
    return c * s + p[..., 1].double().repeat_interleave(32, -1), s


def attend(q, k4, kp, v4, vp, n, scale, causal=False):
    """q [T, H, d] over the first n rows of a packed cache, in 64 bits: (out [T, H, d], bound [T, H, d]).

    The bound is what a kernel that works in fp32 with 16-bit matrix operands may be off before its output is rounded:
      * a probability times a V scale as two operands of 8 significant bits each is off by 2^-17 of itself at most (the first
        operand's rest is at most 2^-8 of the power of two below the number, and rounding a rest of that size is off by 2^-9 of
        it), and meets codes of 0..15: 2^-17 * 15 < 2^-16 * 8, times sum_j p_j s_j;
      * a score is a sum over d of products q (16 + code) s and q z in fp32: at most 64 roundings of 2^-24 of their absolute
        sum (31 s + |z|) |q| scale, the probabilities then are off by as much (exp), and the fp32 exponential and the sums
        over keys (chains of at most 4096) by 4096 * 2^-24 relative;
      * the output is off by the probabilities' error times sum_j p_j |v_j| twice (numerator and denominator)."""
    T, H, d = q.shape
    hk = k4.shape[0]
    G = H // hk
    out = torch.zeros(T, H, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for g in range(hk):
        k, ks = values(k4[g, :n], kp[g, :n])
        v, vs = values(v4[g, :n], vp[g, :n])
        kabs = 31 * ks + kp[g, :n, :, 1].double().abs().repeat_interleave(32, -1)
        for t in range(T):
            m = n - T + 1 + t if causal else n
            if m <= 0:
                continue
            qq = q[t, g * G:(g + 1) * G].double()
            x = (qq @ k[:m].T) * scale
            p = torch.softmax(x, -1)
            dx = 64 * 2.0 ** -24 * scale * (qq.abs() @ kabs[:m].T).amax(-1, keepdim=True) + 4096 * 2.0 ** -24
            out[t, g * G:(g + 1) * G] = p @ v[:m]
            tol[t, g * G:(g + 1) * G] = 2.0 ** -16 * 8 * (p @ vs[:m]) + 2 * dx * (p @ v[:m].abs())
    return out, tol
