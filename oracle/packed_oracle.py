"""Attention over packed sequences and over a paged cache in float64 (torch on the CPU), for the tests: the definition, its
gradients by the formulas, for each result the magnitudes that rounding errors are bounded by, and the 8-bit numbers of a cache."""
from __future__ import annotations

import math

import torch

GROUP = 32
LOWEST = {torch.bfloat16: -117, torch.float16: -15}
HIGHEST = {torch.bfloat16: 120, torch.float16: 8}


def one(q, k, v, start, causal, scale, dO=None):
    """A sequence's head: q [n,D] at the positions from ``start`` on, k and v [m,D].  Returns ``(values, sizes)``, dicts of o and, with dO, dq,
    dk, dv.  ``sizes[name]`` is (a, b, c): a the magnitude that a relative rounding of the last contraction's 16-bit operand meets, b what a
    relative error of dO . o meets, c what an absolute error of that operand meets."""
    q, k, v = (t.double() for t in (q, k, v))
    s = q @ k.T * scale
    if causal:
        s = s.masked_fill(torch.arange(k.shape[0]) > start + torch.arange(q.shape[0])[:, None], -math.inf)
    top = s.amax(-1, keepdim=True) if k.shape[0] else torch.zeros(q.shape[0], 1).double()
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    seen = (s > -math.inf).double()
    values, sizes = {"o": p @ v}, {"o": (p @ v.abs(), 0 * (p @ v), seen @ v.abs())}
    if dO is not None:
        g = dO.double()
        ds = p * (g @ v.T - (g * values["o"]).sum(-1, keepdim=True))
        values |= {"dq": ds @ k * scale, "dk": ds.T @ q * scale, "dv": p.T @ g}
        off = (g.abs() * sizes["o"][0]).sum(-1, keepdim=True)  # what a relative error of dO . o is of
        sizes["dq"] = (ds.abs() @ k.abs() * scale, off * (p @ k.abs()) * scale, seen @ k.abs() * scale)
        sizes["dk"] = (ds.abs().T @ q.abs() * scale, (p * off).T @ q.abs() * scale, seen.T @ q.abs() * scale)
        sizes["dv"] = (p.T @ g.abs(), 0 * values["dv"], seen.T @ g.abs())
    return values, sizes


def packed(q, k, v, offsets, causal, dO=None, scale=None):
    """``[T,H,D]`` tensors; ``offsets`` a list."""
    T, H, D = q.shape
    G = H // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    shapes = {"o": q.shape} if dO is None else {"o": q.shape, "dq": q.shape, "dk": k.shape, "dv": v.shape}
    values = {n: torch.zeros(s, dtype=torch.float64) for n, s in shapes.items()}
    sizes = {n: [torch.zeros(s, dtype=torch.float64) for _ in range(3)] for n, s in shapes.items()}
    for b, e in zip(offsets, offsets[1:]):
        for h in range(H if e > b else 0):
            part, size = one(q[b:e, h], k[b:e, h // G], v[b:e, h // G], 0, causal, scale, None if dO is None else dO[b:e, h])
            for n, x in part.items():
                head = h if n in ("o", "dq") else h // G
                values[n][b:e, head] += x
                for i in range(3):
                    sizes[n][i][b:e, head] += size[n][i]
    return values, sizes


def paged(q, k, v, lengths, offsets, scale=None):
    """q [T,H,D]; k, v: lists of a sequence's [m,H,D] numbers as the cache holds them."""
    T, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    value, size = torch.zeros(q.shape, dtype=torch.float64), [torch.zeros(q.shape, dtype=torch.float64) for _ in range(3)]
    for i, (b, e) in enumerate(zip(offsets, offsets[1:])):
        for h in range(H if e > b and lengths[i] > 0 else 0):
            hk = h // (H // k[i].shape[1])
            x, y = one(q[b:e, h], k[i][:, hk], v[i][:, hk], lengths[i] - (e - b), True, scale)
            value[b:e, h] = x["o"]
            for j in range(3):
                size[j][b:e, h] = y["o"][j]
    return value, size


def limit(want, size, dtype):
    """How far a result may be off.  u = eps / 2 is a rounding to 16 bits: one of the last contraction's operand (a) and one of the result; dO . o is
    formed with an o that has both (2 u b).  What float32 contractions of up to 128 products, the exponentials and the sums over keys and heads
    add is below 2^-14 (a + b).  fp16 numbers below 2^-14 are rounded in steps of 2^-24: 2^-25 (1 + c)."""
    a, b, c = size
    u = torch.finfo(dtype).eps / 2
    off = u * a + 2 * u * b + (u * u + 2.0 ** -14) * (a + b) + u * want.abs()
    return off + 2.0 ** -25 * (1.0 + c) if dtype == torch.float16 else off + 2.0 ** -120


def e4m3_values():
    """The 256 numbers of the format: sign, four bits of exponent with bias 7, three of the fraction; 0x7f and 0xff are NaN."""
    out = []
    for code in range(256):
        e, f = code >> 3 & 15, code & 7
        x = math.nan if e == 15 and f == 7 else math.ldexp(8 + f, e - 10) if e else math.ldexp(f, -9)
        out.append(-x if code & 128 else x)
    return torch.tensor(out, dtype=torch.float64)


def quantise(x):
    """``[...,D]`` 16-bit numbers as 8-bit codes and exponent codes, by the definition: of the format's numbers the nearest one counts, and of
    two the one with an even code."""
    low, high = LOWEST[x.dtype], HIGHEST[x.dtype]
    table = e4m3_values()[:127]  # 0 .. 448, ascending
    y = x.double()
    groups = -(-y.shape[-1] // GROUP)
    codes = torch.empty(x.shape, dtype=torch.uint8)
    scales = torch.empty(*x.shape[:-1], groups, dtype=torch.uint8)
    for g in range(groups):
        part = y[..., g * GROUP:(g + 1) * GROUP]
        most = torch.where(part.isfinite(), part.abs(), 0.0).amax(-1)
        e = torch.full(most.shape, low)
        for _ in range(high - low):
            e = e + ((most > 448 * torch.pow(2.0, e.double())) & (e < high)).long()
        z = part.abs() * torch.pow(2.0, -e.double())[..., None]
        top = torch.where(e == high, 240.0, 448.0)[..., None]
        z = torch.minimum(z, top)
        above = torch.searchsorted(table, z.nan_to_num(0.0).contiguous()).clamp(max=126)
        below = (above - 1).clamp(min=0)
        near = (table[above] - z) - (z - table[below])
        code = torch.where((near < 0) | ((near == 0) & (above % 2 == 0)), above, below) + 128 * torch.signbit(part).long()
        codes[..., g * GROUP:(g + 1) * GROUP] = torch.where(part.isfinite(), code, 127).to(torch.uint8)
        scales[..., g] = (e + 127).to(torch.uint8)
    return codes, scales


def dequantise(codes, scales):
    """float64 values of codes [...,D] and exponent codes [...,groups]."""
    power = torch.pow(2.0, scales.double() - 127).repeat_interleave(GROUP, -1)[..., :codes.shape[-1]]
    return e4m3_values()[codes.long()] * power


def rows(pages, scales, table, length, size):
    """What a cache [pages,H,size,D] holds of a sequence, float64 [length,H,D]; pages that it has not read as zeros."""
    out = torch.zeros(length, pages.shape[1], pages.shape[3], dtype=torch.float64)
    for x in range(length):
        page = int(table[x // size])
        if 0 <= page < pages.shape[0]:
            row = pages[page, :, x % size]
            out[x] = row.double() if scales is None else dequantise(row.view(torch.uint8), scales[page, :, x % size].view(torch.uint8))
    return out
