"""The paged KV cache operators as a program calls them, their plain forms and their values in 64 bits.

A case is a plain dict with a "kind":

  append  paged_append: the new K and V rows of several sequences into their pages, K and Q rotated to their positions
  attend  paged_attention: the last tokens of each sequence (one, a few drafted ones, a chunk of a prompt) over its pages
  step    paged_step: the new rows into the pages, and their tokens over all rows

The layout. k_pages / v_pages [pages, hk, page, d]; table [b, width] int32 names the page of rows w * page .. of a sequence;
lens [b] int32 counts the rows of each sequence, the call's new ones among them; new [b] int32 says how many of the t token
columns are real (the rest is padding, attends nothing and is written nowhere). Token j of a sequence is row
lens - new + j, and attends the rows up to its own.
"""
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "utmist-bigger-bird_amd"))

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"
THETA = 500000.0


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a prompt of odd length goes to fresh pages of an 8-KV-head model
        dict(name="append_8k", kind="append", b=1, t=8111, n=8111, hk=8, g=4, d=128, page=64, dtype="bf16", rot="bf16"),
        # one token each of 64 short conversations, small pages: latency counts
        dict(name="append_64x1", kind="append", b=64, t=1, n=40, hk=8, g=4, d=128, page=16, dtype="bf16", rot="bf16"),
        # follow-ups of unlike lengths on an fp16 model with 64-wide heads and as many KV heads as query heads
        dict(name="append_6x513_fp16_d64", kind="append", b=6, t=513, n=900, hk=16, g=1, d=64, page=32, dtype="fp16", rot="fp32"),
        # one token over one long cache (the context length of bench.py)
        dict(name="attend_1x128k", kind="attend", b=1, t=1, n=131072, hk=8, g=4, d=128, page=64, dtype="bf16"),
        # one token each of 32 conversations of unlike lengths, small pages
        dict(name="attend_32x8k", kind="attend", b=32, t=1, n=8192, hk=8, g=4, d=128, page=16, dtype="bf16"),
        # one token over a few rows, eight query heads per KV head, 64-wide heads: latency counts
        dict(name="attend_257_d64", kind="attend", b=1, t=1, n=257, hk=4, g=8, d=64, page=16, dtype="bf16"),
        # up to four drafted tokens of eight sequences verified in one pass, fp16, two query heads per KV head
        dict(name="verify_8x16k_fp16", kind="attend", b=8, t=4, n=16384, hk=16, g=2, d=128, page=128, dtype="fp16"),
        # a few dozen tokens of a follow-up over a long cache: few query rows, much to read
        dict(name="chunk_65_128k", kind="attend", b=1, t=65, n=131072, hk=8, g=4, d=128, page=64, dtype="bf16"),
        # the last chunk of a 32K-token prompt that is worked off in pieces
        dict(name="chunk_4k_32k", kind="attend", b=1, t=4096, n=32768, hk=8, g=4, d=128, page=64, dtype="bf16"),
        # four whole prompts of unlike lengths, right-padded, on an fp16 model with 64-wide heads
        dict(name="prompts_4x2k_fp16_d64", kind="attend", b=4, t=2048, n=2048, hk=8, g=4, d=64, page=16, dtype="fp16"),
        # a decode step of 16 conversations of unlike lengths
        dict(name="step_16x8k", kind="step", b=16, t=1, n=8111, hk=8, g=4, d=128, page=64, dtype="bf16", rot="bf16"),
        # a decode step of one sequence over a short fp16 cache with 64-wide heads
        dict(name="step_4k_fp16_d64", kind="step", b=1, t=1, n=4099, hk=8, g=4, d=64, page=16, dtype="fp16", rot="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "step", "step"])
    dtype = rng.choice(["bf16", "fp16"])
    hk, g = rng.choice([(8, 4), (8, 4), (16, 2), (32, 1), (4, 8), (2, 3), (1, 16)])
    case = dict(kind=kind, hk=hk, g=g, d=rng.choice([128, 128, 64]), page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype)
    b = case["b"] = _log(rng, 1, 64)
    if kind == "append":
        t = case["t"] = _log(rng, 1, 8192 // b)
        return dict(case, n=t + rng.choice([0, rng.randrange(1, 200)]), rot=rng.choice([dtype, "fp32"]))
    if kind == "attend" and rng.random() < 0.4:  # chunks of prompts
        t = _log(rng, 5, 4096 // b)
        n = t + rng.choice([0, _log(rng, 1, min(1 << 30, 4096 * 28672 * 32 // (b * hk * g)) // t)])
        return dict(case, t=t, n=min(n, max(t, 131072 * 8 // max(hk, 8) // b)))
    t = case["t"] = rng.choice([1, 1, 1, 2, 3, 4, 8])
    case["n"] = max(t, _log(rng, 1, 131072 * 8 // max(hk, 8) // b))
    return case if kind == "attend" else dict(case, rot=rng.choice([dtype, "fp32"]))


def _lengths(case):
    """(rows, new tokens) of each sequence: the first has all t tokens and n rows, the others spread below."""
    rows, new = [], []
    for i in range(case["b"]):
        f, h = (i * 0.6180339887) % 1.0, (i * 0.7548776662) % 1.0
        new.append(case["t"] - int((case["t"] - 1) * f))
        rows.append(new[-1] + int((case["n"] - case["t"]) * (1.0 - 0.9 * h)))
    return rows, new


# ---------------------------------------------------------------- inputs
def _rows(gen, b, h, t, d, dtype):
    """Q, K or V as projections leave them: a [b, h, t, d] view of [b, t, h * d], channels of unlike size."""
    size = torch.exp(0.4 * torch.randn(h * d, generator=gen, device=DEV))
    x = torch.randn(b, t, h * d, generator=gen, device=DEV)
    x *= size
    return x.to(dtype).view(b, t, h, d).transpose(1, 2)


def _angles(rows, new, t, d, dtype):
    """cos and sin [b, t, d] of the tokens' positions, as a model's rotary embedding hands them out."""
    first = torch.tensor(rows, device=DEV, dtype=torch.float64) - torch.tensor(new, device=DEV, dtype=torch.float64)
    pos = first[:, None] + torch.arange(t, device=DEV, dtype=torch.float64)
    freq = THETA ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    a = pos[:, :, None] * freq
    a = torch.cat([a, a], -1)
    return a.cos().to(dtype), a.sin().to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    b, t, hk, d, page, dtype = (case[x] for x in ("b", "t", "hk", "d", "page", "dtype"))
    h, dtype = hk * case["g"], DTYPES[dtype]
    rows, new = _lengths(case)
    width = -(-case["n"] // page)
    pages = sum(-(-r // page) for r in rows) + 3  # a few are free
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    w = torch.arange(width, device=DEV)
    count = torch.tensor([-(-r // page) for r in rows], device=DEV)
    start = count.cumsum(0) - count
    at = torch.where(w < count[:, None], start[:, None] + w, pages - 1)  # the free places of the table name some free page
    s = dict(case, table=order[at].contiguous(), scale=d ** -0.5)
    s["lens"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
    s["new"] = torch.tensor(new, dtype=torch.int32, device=DEV) if min(new) < t else None
    s["k_pages"], s["v_pages"] = (torch.randn(pages, hk, page, d, generator=gen, device=DEV).mul_(1.1).to(dtype) for _ in "kv")
    s["q"] = _rows(gen, b, h, t, d, dtype)
    if case["kind"] != "attend":
        s["k"], s["v"] = _rows(gen, b, hk, t, d, dtype), _rows(gen, b, hk, t, d, dtype)
        s["cos"], s["sin"] = _angles(rows, new, t, d, DTYPES[case["rot"]])
    return s


# ---------------------------------------------------------------- plain forms
def _new(s):
    return s["new"] if s["new"] is not None else torch.full_like(s["lens"], s["t"])


def _rotate(x, cos, sin):
    """fp32 values of x [b, h, t, d] rotated to the positions of cos / sin [b, t, d]."""
    x = x.float()
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos.float()[:, None] + turned * sin.float()[:, None]


def _put(pages, x, s):
    """x [b, hk, t, d] into the rows of its tokens."""
    new = _new(s).long()
    j = torch.arange(s["t"], device=DEV)
    real = j < new[:, None]
    row = (s["lens"].long() - new)[:, None] + j
    entry = s["table"].long().gather(1, (row // s["page"]).clamp_max(s["table"].shape[1] - 1))
    pages[entry[real], :, (row % s["page"])[real]] = x.transpose(1, 2)[real].to(pages.dtype)


def _attend(q, s):
    b, h, t, d = q.shape
    hk = s["hk"]
    k, v = (x[s["table"].long()].transpose(1, 2).reshape(b, hk, -1, d).float() for x in (s["k_pages"], s["v_pages"]))
    n, new = k.shape[2], _new(s)
    j = torch.arange(t, device=DEV)
    seen = torch.where(j < new[:, None], (s["lens"] - new)[:, None] + j + 1, 0)  # [b, t] rows that a token attends
    late = torch.arange(n, device=DEV) >= seen[:, :, None]
    x = torch.matmul(q.float().reshape(b, hk, -1, d), k.transpose(2, 3)).view(b, h, t, n).mul_(s["scale"])
    x.masked_fill_(late[:, None], -float("inf"))
    x.sub_(x.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    v = v.masked_fill((torch.arange(n, device=DEV) >= s["lens"][:, None])[:, None, :, None], 0.0)
    o = torch.matmul(x.view(b, hk, -1, n), v).view(b, h, t, d)
    return torch.where(total > 0, o / total, 0.0).to(q.dtype)


# ---------------------------------------------------------------- one pass
def run(s):
    kind, q = s["kind"], s["q"]
    pages = s["k_pages"], s["v_pages"]
    if own:
        import bigger_bird_amd as bb

        if kind == "attend":
            return bb.paged_attention(q, *pages, s["table"], s["lens"], s["scale"], new=s["new"])
        turn = dict(cos=s["cos"], sin=s["sin"], new=s["new"])
        if kind == "append":
            return bb.paged_append(s["k"], s["v"], *pages, s["table"], s["lens"], q=q, **turn), *pages
        return bb.paged_step(q, s["k"], s["v"], *pages, s["table"], s["lens"], s["scale"], **turn), *pages
    if kind == "attend":
        return _attend(q, s)
    q = _rotate(q, s["cos"], s["sin"])
    _put(pages[0], _rotate(s["k"], s["cos"], s["sin"]), s)
    _put(pages[1], s["v"], s)
    if kind == "append":
        return q.to(s["q"].dtype), *pages
    return _attend(q, s).to(s["q"].dtype), *pages


# ---------------------------------------------------------------- 64 bits
def _turned64(x, cos, sin):
    """x [t, d] rotated as pairs (x_i, x_{i + d/2}), in 64 bits."""
    x, cos, sin = x.to(torch.float64), cos.to(torch.float64), sin.to(torch.float64)
    m = x.shape[1] // 2
    out = torch.empty_like(x)
    out[:, :m] = x[:, :m] * cos[:, :m] - x[:, m:] * sin[:, :m]
    out[:, m:] = x[:, m:] * cos[:, m:] + x[:, :m] * sin[:, m:]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind, b, t, hk, g, page = (s[x] for x in ("kind", "b", "t", "hk", "g", "page"))
    rows, new = _lengths(case)
    table = s["table"].tolist()
    kp, vp = s["k_pages"].to(torch.float64), s["v_pages"].to(torch.float64)
    q = s["q"].to(torch.float64)
    if kind != "attend":
        for i in range(b):
            cos, sin = s["cos"][i], s["sin"][i]
            for h in range(hk * g):
                q[i, h] = _turned64(q[i, h], cos, sin)
            where = [divmod(rows[i] - new[i] + j, page) for j in range(new[i])]
            at = torch.tensor([table[i][w] for w, _ in where], device=DEV), torch.tensor([r for _, r in where], device=DEV)
            for h in range(hk):
                kp[at[0], h, at[1]] = _turned64(s["k"][i, h], cos, sin)[:new[i]]
                vp[at[0], h, at[1]] = s["v"][i, h, :new[i]].to(torch.float64)
    if kind == "append":
        return q, kp, vp
    out = torch.zeros_like(q)
    for i in range(b):
        mine = torch.tensor(table[i][:-(-rows[i] // page)], device=DEV)
        for h in range(hk):
            k, v = (x[mine, h].reshape(-1, x.shape[3])[:rows[i]] for x in (kp, vp))
            for a in range(0, new[i], 512):  # blocks of tokens
                e = min(new[i], a + 512)
                last = rows[i] - new[i] + e
                x = (q[i, h * g:(h + 1) * g, a:e] @ k[:last].T) * s["scale"]
                own_row = rows[i] - new[i] + torch.arange(a, e, device=DEV)
                x = x.masked_fill(torch.arange(last, device=DEV) > own_row[:, None], -float("inf"))
                w = torch.exp(x - x.max(-1, keepdim=True).values)
                out[i, h * g:(h + 1) * g, a:e] = (w @ v[:last]) / w.sum(-1, keepdim=True)
    return out if kind == "attend" else (out, kp, vp)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, hk, g, d = case["kind"], case["hk"], case["g"], case["d"]
    rows, new = _lengths(case)
    tokens = sum(new)
    row = 2 * hk * d * 2  # bytes of one position: K and V
    rot = 2 * d * (4 if case.get("rot") == "fp32" else 2)
    q = hk * g * d * 2
    if kind == "append":
        return {"bytes": tokens * (2 * row + 2 * q + rot), "flops": 0}
    pairs = sum(m * (r - m) + m * (m + 1) // 2 for r, m in zip(rows, new))
    io = 2 * tokens * q + sum(rows) * row
    if kind == "step":
        io += tokens * (row + rot)  # the new rows come in (as pages they are counted with the rest, written)
    return {"bytes": io, "flops": 4 * hk * g * d * pairs}
