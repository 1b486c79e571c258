"""The 4-bit KV cache operators as a program calls them, their plain forms and their values in 64 bits.

A case is a plain dict with a "kind":

  write   quantize4_pair: K and V rows of a prompt (or of a follow-up) into the rows of a 4-bit cache, read back
  read    dequantize4_pair: the cached K and V rows as 16-bit or fp32 tensors
  attend  decode_int4: one to sixteen query tokens over the cached rows
  step    decode_int4_append: the step's new K and V rows into the cache, and its query tokens over all rows

The format. A row of d elements is d / 32 groups. Per group, on values clamped to +-65504: z = fp16(min),
s = fp16(max((max - z) / 15, 0)), code = rint((x - z) / s) clamped to 0 .. 15 (0 where s = 0), each operation in fp32;
the value is s * code + z in fp32. Byte b of a packed row holds element 2 b (low four bits) and 2 b + 1. A cache is
codes [Hkv, capacity, d / 2] uint8 and params [Hkv, capacity, d / 32, 2] fp16 (s, z) for K, and the same for V.
"""
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "utmist-bigger-bird_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"
SPARE = 256  # rows a cache keeps ready behind the valid ones


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a 128K-token prompt of an 8-KV-head model goes to the cache (the context length of bench.py)
        dict(name="write_128k", kind="write", n=0, t=131072, hk=8, d=128, dtype="bf16"),
        # a short prompt of odd length on an fp16 model with 64-wide heads
        dict(name="write_8k_fp16_d64", kind="write", n=0, t=8111, hk=16, d=64, dtype="fp16"),
        # a follow-up of a few dozen tokens behind a cached conversation
        dict(name="write_65", kind="write", n=4097, t=65, hk=8, d=128, dtype="bf16"),
        # a chunk of a prompt attends the whole cache in 16 bits, so the cache is read back
        dict(name="read_128k", kind="read", n=131072, hk=8, d=128, dtype="bf16"),
        # a short cache of odd length, read back on an fp16 model
        dict(name="read_4k_fp16_d64", kind="read", n=4099, hk=8, d=64, dtype="fp16"),
        # one token over a long cache (the shape of bench.py's decode leg)
        dict(name="attend_128k", kind="attend", n=131072, t=1, hk=8, g=4, d=128, dtype="bf16", causal=False),
        # a model with as many KV heads as query heads, fp16, odd length
        dict(name="attend_20k_fp16_mha", kind="attend", n=20011, t=1, hk=32, g=1, d=128, dtype="fp16", causal=False),
        # one token over a few cached rows, eight query heads per KV head, 64-wide heads: latency counts
        dict(name="attend_257_d64", kind="attend", n=257, t=1, hk=4, g=8, d=64, dtype="bf16", causal=False),
        # four drafted tokens verified in one pass, each attending up to its own row
        dict(name="verify4_32k", kind="attend", n=32768, t=4, hk=8, g=4, d=128, dtype="bf16", causal=True),
        # a whole decode step over a long cache
        dict(name="step_128k", kind="step", n=131072, t=1, hk=8, g=4, d=128, dtype="bf16", causal=False),
        # a decode step over a medium cache, two query heads per KV head
        dict(name="step_8k_g2", kind="step", n=8111, t=1, hk=16, g=2, d=128, dtype="bf16", causal=False),
        # a decode step over a short fp16 cache with 64-wide heads
        dict(name="step_4k_fp16_d64", kind="step", n=4099, t=1, hk=8, g=4, d=64, dtype="fp16", causal=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "step", "step"])
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([128, 128, 64])
    if kind in ("write", "read"):
        hk = rng.choice([1, 2, 4, 5, 8])
        rows = _log(rng, 1, 131072)
        dtype = rng.choice([dtype, dtype, "fp32"]) if rows * hk <= 524288 else dtype
        if kind == "read":
            return dict(kind=kind, n=rows, hk=hk, d=d, dtype=dtype)
        return dict(kind=kind, n=rng.choice([0, rng.randrange(1, 5000)]), t=rows, hk=hk, d=d, dtype=dtype)
    hk, g = rng.choice([(8, 4), (8, 4), (16, 2), (32, 1), (4, 8), (2, 3), (1, 16)])
    t = rng.choice([1, 1, 1, 2, 3, 4, 8, 16])
    n = _log(rng, 1, 131072 * 8 // max(hk, 8) // -(-t * g // 16))
    t = min(n, t)
    return dict(kind=kind, n=n, t=t, hk=hk, g=g, d=d, dtype=dtype, causal=rng.choice([False, True]))


# ---------------------------------------------------------------- inputs
def _rows(gen, hk, t, d, dtype):
    """K or V rows as projections leave them: a [hk, t, d] view of [t, hk * d], channels of unlike size, a few large."""
    size = torch.exp(0.5 * torch.randn(hk * d, generator=gen, device=DEV))
    size[torch.randint(0, hk * d, (max(1, hk * d // 64),), generator=gen, device=DEV)] *= 6.0
    x = torch.randn(t, hk * d, generator=gen, device=DEV)
    x *= size
    return x.to(dtype).view(t, hk, d).transpose(0, 1)


def _cache(gen, hk, n, d):
    """A cache holding n rows of K or V; the spare rows behind them hold whatever memory held."""
    codes = torch.randint(0, 256, (hk, n + SPARE, d // 2), generator=gen, device=DEV, dtype=torch.uint8)
    params = torch.full((hk, n + SPARE, d // 32, 2), float("nan"), device=DEV, dtype=torch.float16)
    if n:
        codes[:, :n], params[:, :n] = _pack(_rows(gen, hk, n, d, torch.bfloat16))
    return codes, params


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, hk, d, dtype = case["kind"], case["hk"], case["d"], DTYPES[case["dtype"]]
    n = case["n"]
    s = dict(case, k=_cache(gen, hk, n + (case["t"] if kind == "write" else 0), d))
    s["v"] = _cache(gen, hk, n + (case["t"] if kind == "write" else 0), d)
    if kind in ("write", "step"):
        s["knew"], s["vnew"] = _rows(gen, hk, case["t"], d, dtype), _rows(gen, hk, case["t"], d, dtype)
    if kind in ("attend", "step"):
        s["q"] = torch.randn(case["t"], hk * case["g"], d, generator=gen, device=DEV).to(dtype)
        s["scale"] = d ** -0.5
    s["dtype"] = dtype
    return s


# ---------------------------------------------------------------- plain forms
def _pack(x):
    """x [hk, t, d] -> codes [hk, t, d / 2], params [hk, t, d / 32, 2]."""
    g = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32))
    z = g.amin(-1, keepdim=True).half()
    top = g.amax(-1, keepdim=True) - z.float()
    s = (top.double() / 15).float().clamp_min(0.0).half()  # quotients in 64 bits, rounded to fp32 once
    code = ((g - z.float()).double() / s.double()).float().round().clamp(0, 15)
    code = torch.where(s > 0, code, 0.0).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([s, z], -1)


def _unpack(codes, params):
    """The fp32 values [hk, t, d] of packed rows."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).float()
    p = params.float()
    return (p[..., 0:1] * c + p[..., 1:2]).flatten(-2)


def _attend(q, k, v, scale, causal):
    """q [t, H, d], k / v [hk, n, d] fp32 values -> [t, H, d] in q's type."""
    t, h, d = q.shape
    hk, n = k.shape[:2]
    qg = q.float().view(t, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)  # [hk, g t, d]
    x = torch.matmul(qg, k.transpose(1, 2)).mul_(scale).view(hk, -1, t, n)
    if causal:
        late = torch.arange(n, device=q.device) > torch.arange(n - t, n, device=q.device)[:, None]
        x = x.masked_fill(late, -float("inf"))
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(x.view(hk, -1, n), v).view(hk, -1, t, d) / x.sum(-1, keepdim=True)
    return o.permute(2, 0, 1, 3).reshape(t, h, d).to(q.dtype)


def _rows_of(cache, a, b):
    return cache[0][:, a:b], cache[1][:, a:b]


# ---------------------------------------------------------------- one pass
def run(s):
    kind, n, k, v = s["kind"], s["n"], s["k"], s["v"]
    if own:
        import bigger_bird_amd as bb

        if kind == "write":
            at = _rows_of(k, n, n + s["t"]), _rows_of(v, n, n + s["t"])
            bb.quantize4_pair(s["knew"], s["vnew"], *at)
            return bb.dequantize4_pair(*at, s["dtype"])
        if kind == "read":
            return bb.dequantize4_pair(_rows_of(k, 0, n), _rows_of(v, 0, n), s["dtype"])
        if kind == "attend":
            return bb.decode_int4(s["q"], *k, *v, n, s["scale"], causal=s["causal"])
        out = bb.decode_int4_append(s["q"], *k, *v, s["knew"], s["vnew"], n, s["scale"], causal=s["causal"])
        new = _rows_of(k, n - s["t"], n), _rows_of(v, n - s["t"], n)
        return out, *bb.dequantize4_pair(*new, s["dtype"])
    if kind in ("write", "step"):
        a = n if kind == "write" else n - s["t"]
        new = _rows_of(k, a, a + s["t"]), _rows_of(v, a, a + s["t"])
        new[0][0][:], new[0][1][:] = _pack(s["knew"])
        new[1][0][:], new[1][1][:] = _pack(s["vnew"])
        values = tuple(_unpack(*x).to(s["dtype"]) for x in new)
        if kind == "write":
            return values
    kf, vf = _unpack(*_rows_of(k, 0, n)), _unpack(*_rows_of(v, 0, n))
    if kind == "read":
        return kf.to(s["dtype"]), vf.to(s["dtype"])
    out = _attend(s["q"], kf, vf, s["scale"], s["causal"])
    return out if kind == "attend" else (out, *values)


# ---------------------------------------------------------------- 64 bits
def _values64(codes, params):
    """The values of packed rows in 64 bits, by arithmetic on the bytes."""
    b = codes.to(torch.float64)
    high = torch.floor(b / 16)
    c = torch.empty(*b.shape[:-1], b.shape[-1] * 2, dtype=torch.float64, device=b.device)
    c[..., 0::2] = b - 16 * high
    c[..., 1::2] = high
    s = params[..., 0].to(torch.float64).repeat_interleave(32, -1)
    z = params[..., 1].to(torch.float64).repeat_interleave(32, -1)
    return c * s + z


def _quantised64(x):
    """The values that x [t, d] has once written: the format's roundings, each quantity held in 64 bits between them."""
    def r32(y):
        return y.to(torch.float32).to(torch.float64)

    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for a in range(0, x.shape[-1], 32):
        w = x[:, a:a + 32].to(torch.float64)
        w = torch.minimum(torch.maximum(w, torch.full_like(w, -65504.0)), torch.full_like(w, 65504.0))
        lo, hi = w.min(1, keepdim=True).values, w.max(1, keepdim=True).values
        z = lo.to(torch.float16).to(torch.float64)
        s = r32(r32(hi - z) / 15)
        s = torch.where(s > 0, s, torch.zeros_like(s)).to(torch.float16).to(torch.float64)
        c = torch.round(r32(r32(w - z) / torch.where(s > 0, s, torch.ones_like(s))))
        c = torch.where(s > 0, torch.minimum(torch.maximum(c, torch.zeros_like(c)), torch.full_like(c, 15.0)),
                        torch.zeros_like(c))
        out[:, a:a + 32] = c * s + z
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind, n, t, hk = s["kind"], s["n"], s.get("t"), s["hk"]
    if kind == "read":
        return tuple(torch.stack([_values64(c[0][h, :n], c[1][h, :n]) for h in range(hk)]) for c in (s["k"], s["v"]))
    new = None
    if kind in ("write", "step"):
        new = tuple(torch.stack([_quantised64(x[h]) for h in range(hk)]) for x in (s["knew"], s["vnew"]))
        if kind == "write":
            return new
    g = s["g"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for h in range(hk):
        kv = [_values64(c[0][h, :n], c[1][h, :n]) for c in (s["k"], s["v"])]
        if new is not None:
            kv[0][n - t:], kv[1][n - t:] = new[0][h], new[1][h]
        for i in range(t):
            seen = n - t + 1 + i if s["causal"] else n
            for j in range(h * g, h * g + g):
                x = (kv[0][:seen] @ s["q"][i, j].to(torch.float64)) * s["scale"]
                w = torch.exp(x - x.max())
                out[i, j] = (w @ kv[1][:seen]) / w.sum()
    return out if kind == "attend" else (out, *new)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, hk, d, n = case["kind"], case["hk"], case["d"], case["n"]
    t = case.get("t", 0)
    el = 4 if case["dtype"] == "fp32" else 2
    packed = 2 * hk * (d // 2 + d // 8)  # bytes of one cached position: K and V, codes and params
    values = 2 * hk * d * el
    if kind == "write":
        return {"bytes": t * (2 * values + packed), "flops": 0}
    if kind == "read":
        return {"bytes": n * (packed + values), "flops": 0}
    h = hk * case["g"]
    io = 2 * t * h * d * el + n * packed
    if kind == "step":
        io += t * 2 * values  # the new rows come in, and their values go out
    return {"bytes": io, "flops": 4 * t * h * n * d}
