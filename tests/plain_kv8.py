"""Plain 64-bit statements of the 8-bit cache's operators, and seeded cases of them."""

from __future__ import annotations

import math
import random

import torch

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
LARGEST, LEAST, MOST = 448.0, -64, 64


def exponent_of(x: torch.Tensor) -> torch.Tensor:
    """The least e (held to -64..64) with max |x| <= 448 * 2^e over the last axis of 64-bit ``x``, by comparison."""
    top = x.abs().amax(-1)
    e = torch.full(top.shape, LEAST, dtype=torch.int64)
    for step in range(LEAST, MOST):
        e += (top > LARGEST * 2.0 ** step).long()
    return e


def rounded(z: torch.Tensor) -> torch.Tensor:
    """64-bit numbers to e4m3, ties to even: four significant bits, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(z / step) * step).clamp(-LARGEST, LARGEST)


def quantise(x: torch.Tensor) -> tuple:
    """(codes as 64-bit numbers, scale bytes) of rows of ``x``; a row that is not finite: zeros and 255."""
    x = x.double().cpu()
    finite = torch.isfinite(x).all(-1)
    safe = torch.where(finite[..., None], x, torch.zeros_like(x))
    e = exponent_of(safe)
    codes = rounded(safe / torch.exp2(e.double())[..., None])
    return codes, torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def cache_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What an 8-bit cache stands for, in 64 bits."""
    b = scales.view(torch.uint8).cpu().double()
    up = torch.where(b == 255, torch.full_like(b, math.nan), torch.exp2(b - 127))
    return codes.view(torch.uint8).cpu().view(CODES).double() * up[..., None]


def norm_rotate(x: torch.Tensor, weight, eps: float, table) -> torch.Tensor:
    """[N, heads, D] normalised per head and rotated in halves of the first 2 * table.shape[1] elements, 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if table is not None:
        half = table.shape[1]
        c, s = table[..., 0].double()[:, None], table[..., 1].double()[:, None]
        a, b = x[..., :half], x[..., half : 2 * half]
        x = torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * half :]), -1)
    return x


def attention(q, k, v, start: int, scale: float, window: int, keep_first: int) -> tuple:
    """(out, sum of weight * |value|, floor) [n, heads, D] of queries at positions start.. over 64-bit keys and values
    [L, kv heads, D].  floor: what half-precision weights below 2^-14 of the largest contribution can lose.  Such a
    weight is off by at most 2^-25 of the largest p_j 2^(b_j), which is at most max_j p_j max(top_j / 224, 2^-64)
    (top_j: the largest |element| of value j, whose code is 224 or more unless the scale is the least one), and is multiplied by a code |d_j| <= 448 |v_j| / top_j."""
    n, heads, _ = q.shape
    groups = heads // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    pos = torch.arange(start, start + n)[:, None]
    key = torch.arange(k.shape[0])[None]
    seen = key <= pos
    if window:
        seen &= (pos - key < window) | (key < keep_first)
    out, size, floor = [], [], []
    for h in range(heads):
        t = (q[:, h] @ k[:, h // groups].t()) * scale
        w = torch.softmax(t.masked_fill(~seen, -math.inf), -1)
        values = v[:, h // groups]
        # a key that is not seen has no part, whatever it holds
        finite = torch.where(torch.isfinite(values), values, torch.zeros_like(values))
        bad = (seen[:, :, None] & ~torch.isfinite(values)[None]).any(1)
        o = w @ finite
        out.append(torch.where(bad, torch.full_like(o, math.nan), o))
        size.append(w @ finite.abs())
        top = finite.abs().amax(-1)
        share = torch.where(top[:, None] > 0, finite.abs() / top.clamp(min=1e-300)[:, None], torch.zeros_like(finite))
        floor.append(2.0 ** -25 * (w * (top / 224).clamp(min=2.0 ** -64)).amax(-1, keepdim=True) * (448 * (seen.double() @ share)))
    return torch.stack(out, 1), torch.stack(size, 1), torch.stack(floor, 1)


def pool(lengths, nkv: int, dim: int, page: int, seed: int, spread: float = 1.0, spare: int = 3, values=None) -> dict:
    """An 8-bit cache on the CPU that holds ``lengths`` positions per entry in scattered pages.  Every other slot, the
    spare pages included, holds large codes under a NaN scale.  ``values``: [(k, v)] per entry [length, nkv, dim]."""
    host, g = random.Random(seed), torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    ids = list(range(pages))
    host.shuffle(ids)
    width = max(counts + [1]) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    k_codes = torch.full((pages, nkv, page, dim), 448.0).to(CODES)
    v_codes = k_codes.clone()
    k_scales = torch.full((pages, nkv, page), 255, dtype=torch.uint8)
    v_scales = k_scales.clone()
    at, held = 0, []
    for e, n in enumerate(lengths):
        table[e, : counts[e]] = torch.tensor(ids[at : at + counts[e]], dtype=torch.int32)
        at += counts[e]
        both = []
        for which, (codes, scales) in enumerate(((k_codes, k_scales), (v_codes, v_scales))):
            if values is None:
                x = torch.randn((n, nkv, dim), generator=g, dtype=torch.float64) * torch.exp(spread * torch.randn((n, nkv, 1), generator=g, dtype=torch.float64))
            else:
                x = values[e][which].double()
            c, s = quantise(x)
            for i in range(n):
                p, slot = int(table[e, i // page]), i % page
                codes.view(torch.uint8)[p, :, slot] = c[i].float().to(CODES).view(torch.uint8)
                scales[p, :, slot] = s[i]
            both.append(c * torch.where(s == 255, torch.tensor(math.nan, dtype=torch.float64), torch.exp2(s.double() - 127))[..., None])
        held.append(tuple(both))
    return {"k_cache": k_codes, "v_cache": v_codes, "k_scale": k_scales.view(SCALES), "v_scale": v_scales.view(SCALES),
            "table": table, "held": held, "pages": pages}
