"""The 8-bit cache's operators against 64-bit statements of them.

Bounds.  A stored number is off by at most half a step of e4m3: 2^-4 of it, or 2^-10 of the scale below
2^-6.  Attention: weights are rounded to half precision (2^-11 of each, and below 2^-14 of the largest
contribution by what ``plain_kv8.attention`` derives as floor), scores and sums are 32-bit (a score of some tens
is off by about 2^-18), and the output is rounded to bfloat16 (2^-8): with A = (2^-11 + 2^-12) * sum of
weight * |value| + floor an output (portions with heads of 64 and 128: weights rounded to bfloat16, A = (2^-8 + 2^-12) * sum) is within A + 2^-8 (|out| + A).  (The floor belongs to it: where one key has
nearly all the weight and an element of its value is zero, that element consists of what is rounded there.
Below bfloat16's normal numbers half a step is 2^-134, whatever the value.)"""

from __future__ import annotations

import math

import pytest
import torch

import plain_kv8 as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
CACHES = ("k_cache", "v_cache", "k_scale", "v_scale")


@pytest.fixture(scope="module")
def native():
    from forge_engine_b200.ops import native as module

    module.require_cuda()
    module.lib()
    return module


def status_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def to_device(cache: dict) -> tuple:
    return tuple(cache[name].view(torch.uint8).to(DEV).view(cache[name].dtype) for name in CACHES)


def empty_caches(pages, nkv, page, dim) -> tuple:
    codes = [torch.zeros((pages, nkv, page, dim), dtype=torch.uint8, device=DEV).view(plain.CODES) for _ in range(2)]
    return (*codes, *(torch.zeros((pages, nkv, page), dtype=torch.uint8, device=DEV).view(plain.SCALES) for _ in range(2)))


def special_rows(dim: int, g) -> torch.Tensor:
    """Vectors where a scale is at an edge: zeros, one element, powers of two times 448, the type's extremes."""
    rows = [torch.zeros(dim), torch.zeros(dim), torch.full((dim,), 448.0), torch.full((dim,), 449.0), torch.randn(dim, generator=g) * 1e-30,
            torch.randn(dim, generator=g) * 1e30, torch.randn(dim, generator=g) * 2.0 ** -70, torch.randn(dim, generator=g) * 1e-40,
            torch.exp(6 * torch.randn(dim, generator=g)), torch.full((dim,), 3.3e38)]
    rows[1][dim // 2] = -0.875
    rows[8][::2] *= -1
    return torch.stack(rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,nkv,page", [(16, 3, 4), (48, 1, 5), (64, 2, 16), (96, 2, 1), (128, 8, 16), (256, 2, 32)])
def test_write_and_read_back(native, dtype, dim, nkv, page) -> None:
    """Plain writing is exact: the same codes and scales as the 64-bit statement, and an exact read in both types."""
    g = torch.Generator().manual_seed(dim + page)
    special = special_rows(dim, g)
    n = 3 * len(special)
    k, v = (torch.randn((n, nkv, dim), generator=g) * torch.exp(3 * torch.randn((n, nkv, 1), generator=g)) for _ in range(2))
    k[: len(special), nkv - 1] = special
    v[len(special) : 2 * len(special), 0] = special
    k, v = k.to(dtype), v.to(dtype)
    k[n - 1, 0, 3] = math.inf
    v[n - 2, nkv - 1, dim - 1] = math.nan
    # two entries whose tokens alternate, from positions in the middle of a page
    entry = torch.arange(n) % 2
    pos = page // 2 + torch.arange(n) // 2
    width = int(pos.max()) // page + 2
    table = torch.randperm(2 * width, generator=g).to(torch.int32).view(2, width)
    caches = empty_caches(2 * width, nkv, page, dim)
    status = status_word()
    # column slices of a wider row, as a projection leaves them
    wide = torch.cat((torch.full((n, 8), 7.0, dtype=dtype), k.flatten(1), v.flatten(1), torch.zeros((n, 4), dtype=dtype)), 1).to(DEV)
    ks, vs = wide[:, 8 : 8 + nkv * dim], wide[:, 8 + nkv * dim : 8 + 2 * nkv * dim]
    places = ints(pos.tolist()), ints(entry.tolist())
    native.kv8_write(ks, vs, *places, *caches, table.to(DEV), status)
    assert int(status.item()) == 0
    page_of, slot = table[entry, pos // page].long(), pos % page
    touched = torch.zeros((2 * width, page), dtype=torch.bool)
    touched[page_of, slot] = True
    for x, codes, scales in ((k, caches[0], caches[2]), (v, caches[1], caches[3])):
        want_codes, want_scales = plain.quantise(x)
        got = codes.view(torch.uint8).cpu().view(plain.CODES)[page_of, :, slot].double()
        assert torch.equal(scales.view(torch.uint8).cpu()[page_of, :, slot], want_scales)
        assert torch.equal(got, want_codes)
        # nothing else was written
        assert int(codes.view(torch.uint8).cpu().transpose(1, 2)[~touched].count_nonzero()) == 0
        assert int(scales.view(torch.uint8).cpu().transpose(1, 2)[~touched].count_nonzero()) == 0
    for out_dtype in (torch.bfloat16, torch.float32):
        outs = [torch.empty((n, nkv, dim), dtype=out_dtype, device=DEV) for _ in range(2)]
        native.kv8_read(*caches, table.to(DEV), *places, *outs, status)
        for x, codes, scales, out in ((k, caches[0], caches[2], outs[0]), (v, caches[1], caches[3], outs[1])):
            want = plain.cache_values(codes, scales)[page_of, :, slot]
            assert torch.equal(torch.nan_to_num(out.cpu().double(), nan=-1.0), torch.nan_to_num(want, nan=-1.0))
    assert int(status.item()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,rot,nq,nkv", [(128, 128, 32, 8), (64, 64, 14, 2), (96, 96, 6, 3), (256, 64, 4, 1), (32, 8, 5, 5), (16, 16, 1, 1), (128, 0, 8, 8)])
@pytest.mark.parametrize("tokens", [1, 5, 700])
def test_write_normalised_and_rotated(native, dtype, dim, rot, nq, nkv, tokens) -> None:
    page, eps = 16, 1e-6
    g = torch.Generator().manual_seed(dim * 7 + tokens)
    x = (torch.randn((tokens, (nq + 2 * nkv) * dim), generator=g) * 2).to(dtype)
    weights = [torch.exp(0.3 * torch.randn(dim, generator=g)) for _ in range(2)]
    pos = torch.arange(tokens) + 5000
    table = None
    if rot:
        angle = pos.double()[:, None] * 1e4 ** (-torch.arange(0, rot, 2).double() / rot)
        table = torch.stack((angle.cos(), angle.sin()), -1).float()
    width = 5000 // page + tokens // page + 2
    pages = torch.randperm(width, generator=g).to(torch.int32)[None]
    caches = empty_caches(width, nkv, page, dim)
    status = status_word()
    xd = x.to(DEV)
    q, k, v = xd.split((nq * dim, nkv * dim, nkv * dim), dim=1)
    q_out = torch.empty((tokens, nq * dim), dtype=torch.bfloat16, device=DEV)
    native.kv8_write(k, v, ints(pos.tolist()), ints([0] * tokens), *caches, pages.to(DEV), status, q=q, q_out=q_out,
                     q_norm=weights[0].to(DEV), k_norm=weights[1].to(DEV), eps=eps, table=None if table is None else table.to(DEV))
    assert int(status.item()) == 0 and torch.equal(xd.cpu(), x)
    heads = x.double().view(tokens, nq + 2 * nkv, dim)
    want_q = plain.norm_rotate(heads[:, :nq], weights[0], eps, table)
    got_q = q_out.cpu().double().view(tokens, nq, dim)
    # rounding to bfloat16 once; 32-bit norm and rotation before it are off by less than 2^-18 of the pair
    size = want_q.abs().amax(-1, keepdim=True)
    assert bool(((got_q - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -18 * size).all())
    page_of, slot = pages[0, pos // page].long(), pos % page
    for want, codes, scales in ((plain.norm_rotate(heads[:, nq : nq + nkv], weights[1], eps, table), caches[0], caches[2]),
                                (heads[:, nq + nkv :], caches[1], caches[3])):
        got = plain.cache_values(codes, scales)[page_of, :, slot]
        scale = torch.exp2(scales.view(torch.uint8).cpu().double() - 127)[page_of, :, slot][..., None]
        top = want.abs().amax(-1, keepdim=True)
        assert bool((top <= 448 * scale * (1 + 2.0 ** -18)).all()) and bool((top * (1 + 2.0 ** -18) > 224 * scale).all())
        bound = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * scale) + 2.0 ** -17 * top
        assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,rot,nkv,norm", [(128, 128, 8, True), (128, 128, 8, False), (64, 0, 4, True), (96, 40, 3, True), (256, 64, 2, True), (16, 16, 5, True)])
def test_keys_take_the_codes_of_exact_arithmetic(native, dtype, dim, rot, nkv, norm) -> None:
    """Norm, rotation and quantisation in 64 bits give the same codes and scales, element by element: a 32-bit error never
    carries a key over the middle between two codes.  (64-bit rounding is 2^-29 of a 32-bit one: of these half a million
    to four million elements none lies that close to a middle.)"""
    tokens, page, eps = 4096, 16, 2.0 ** -20
    g = torch.Generator().manual_seed(dim + rot)
    x = (torch.randn((tokens, 2 * nkv * dim), generator=g) * torch.exp(torch.randn((tokens, 1), generator=g))).to(dtype)
    weight = torch.exp(0.3 * torch.randn(dim, generator=g)) if norm else None
    table = None
    if rot:
        angle = torch.rand((tokens, rot // 2), generator=g).double() * 2 * math.pi
        table = torch.stack((angle.cos(), angle.sin()), -1).float()
    pages = torch.arange(tokens // page, dtype=torch.int32)[None]
    caches = empty_caches(tokens // page, nkv, page, dim)
    status = status_word()
    k, v = x.to(DEV).split((nkv * dim, nkv * dim), dim=1)
    native.kv8_write(k, v, ints(range(tokens)), ints([0] * tokens), *caches, pages.to(DEV), status, k_norm=None if weight is None else weight.to(DEV),
                     eps=eps, table=None if table is None else table.to(DEV))
    assert int(status.item()) == 0
    heads = x.double().view(tokens, 2 * nkv, dim)
    want, scales = plain.quantise(plain.norm_rotate(heads[:, :nkv], weight, eps, table))
    got = caches[0].view(torch.uint8).cpu().view(plain.CODES).transpose(1, 2).reshape(tokens, nkv, dim).double()
    assert torch.equal(caches[2].view(torch.uint8).cpu().transpose(1, 2).reshape(tokens, nkv), scales)
    assert int((got != want).sum()) == 0


def test_write_queries_only_and_places_that_are_not_there(native) -> None:
    dim, nkv, page = 64, 2, 4
    g = torch.Generator().manual_seed(3)
    caches = empty_caches(6, nkv, page, dim)
    table = torch.tensor([[0, 5, -1], [6, 1, 2]], dtype=torch.int32, device=DEV)
    x = torch.randn((4, 3 * dim), generator=g).to(DEV)
    q_out = torch.full((4, 3 * dim), 9.0, dtype=torch.bfloat16, device=DEV)
    status = status_word()
    native.kv8_write(None, None, ints([0] * 4), ints([0] * 4), *caches, table, status, q=x, q_out=q_out)
    assert torch.equal(q_out, x.to(torch.bfloat16)) and int(status.item()) == 0
    kv = torch.randn((1, nkv * dim), generator=g).to(DEV)
    outs = [torch.full((1, nkv, dim), 5.0, device=DEV) for _ in range(2)]
    for pos, entry, bit in ((8, 0, 2), (0, 1, 2), (12, 1, 4), (-1, 0, 4), (0, 2, 4), (0, -1, 4), (2 ** 31 - 1, 1, 4)):
        for call in ("write", "read"):
            status.zero_()
            if call == "write":
                native.kv8_write(kv, kv, ints([pos]), ints([entry]), *caches, table, status)
            else:
                native.kv8_read(*caches, table, ints([pos]), ints([entry]), *outs, status)
                assert float(outs[0].abs().sum() + outs[1].abs().sum()) == 0.0
            assert int(status.item()) == bit, (pos, entry, call)
    assert all(int(c.view(torch.uint8).count_nonzero()) == 0 for c in caches)
    # nothing to do is done
    none = torch.empty((0, nkv * dim), device=DEV)
    native.kv8_write(none, none, ints([]), ints([]), *caches, table, status_word())
    native.kv8_read(*caches, table, ints([]), ints([]), *(torch.empty((0, nkv, dim), device=DEV) for _ in range(2)), status_word())


def attend(native, cache, requests, q, window, keep, scale, extra_rows=2, plan=None, caches=None):
    """(out on the CPU, status) of one call; ``q`` holds ``extra_rows`` rows more than the entries have."""
    nkv, page, dim = (cache["k_cache"].shape[i] for i in (1, 2, 3))
    heads = q.shape[1] // dim
    caches = to_device(cache) if caches is None else caches
    status = status_word()
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    ends = [0]
    for _, n in requests:
        ends.append(ends[-1] + n)
    plan = native.kv8_plan(requests, heads, nkv, dim, window, keep) if plan is None else plan
    native.attention_kv8(q.to(DEV), *caches, cache["table"].to(DEV), ints(ends), ints(s for s, _ in requests), len(requests),
                         max(n for _, n in requests), heads, window, keep, scale, out, status, plan)
    out = out.cpu()
    assert bool((out[ends[-1] :] == 7.0).all())
    return out, int(status.item())


def check_attention(cache, requests, q, out, window, keep, scale, large_scores=False) -> None:
    """``large_scores``: scores of many hundreds, whose own rounding counts.  A product of 16 terms on the tensor cores
    aligns them and the sum so far to the largest of the 17 and keeps no more than 23 bits below it, so with
    T = scale * log2(e) * sum |q_i k_i| a score (in log2 units) is off by at most (D / 16) * 17 * 2^-23 * T; a weight
    and the sum that divides it each change by ln 2 times that."""
    dim = cache["k_cache"].shape[3]
    at = 0
    for e, (start, n) in enumerate(requests):
        if n == 0:
            continue
        k, v = cache["held"][e]
        want, size, floor = plain.attention(q[at : at + n].view(n, -1, dim), k[: start + n], v[: start + n], start, scale, window, keep)
        got = out[at : at + n].double().view(n, -1, dim)
        at += n
        brain = dim in (64, 128) and n * (want.shape[1] // k.shape[1]) > 16
        a = (2.0 ** -8 + 2.0 ** -12) * size if brain else (2.0 ** -11 + 2.0 ** -12) * size + floor
        if large_scores:
            spread = torch.einsum("nkgd,lkd->nkgl", q[at - n : at].double().view(n, k.shape[1], -1, dim).abs(), k[: start + n].abs())
            spread = spread.amax(-1).flatten(1)[..., None] * scale / math.log(2)
            a = a + 2 * math.log(2) * (dim // 16) * 17 * 2.0 ** -23 * spread * (size + floor)
        off = (got - want).abs() - (a + torch.clamp(2.0 ** -8 * (want.abs() + a), min=2.0 ** -134))
        same = torch.equal(torch.isnan(got), torch.isnan(want))
        assert same, e
        worst = float(torch.nan_to_num(off, nan=-1.0).max())
        assert worst <= 0.0, e


SIZES = [
    # dim, heads, kv heads, page, (cached, new) per entry
    (128, 32, 8, 16, [(0, 1)]),
    (128, 32, 8, 16, [(700, 1), (63, 1), (64, 1), (0, 1), (1000, 4), (127, 2)]),
    (128, 40, 8, 16, [(513, 3), (5, 3)]),
    (64, 16, 1, 8, [(300, 1), (255, 1)]),
    (64, 4, 4, 64, [(1500, 1), (0, 16), (31, 7)]),
    (256, 4, 2, 4, [(90, 1), (200, 8)]),
    (96, 6, 2, 5, [(77, 1), (140, 5)]),
    (16, 8, 2, 1, [(40, 1), (7, 4)]),
    (48, 3, 1, 3, [(50, 1), (0, 5)]),
    (112, 7, 7, 16, [(50, 16), (129, 1)]),
    # portions
    (128, 32, 8, 16, [(0, 5)]),
    (128, 8, 2, 16, [(0, 300)]),
    (128, 32, 8, 16, [(700, 40), (3, 17), (1100, 1)]),
    (128, 10, 2, 16, [(130, 129), (0, 0), (0, 77)]),
    (128, 7, 1, 32, [(500, 61)]),
    (64, 12, 4, 16, [(0, 257), (64, 64), (999, 100)]),
    (64, 16, 1, 4, [(400, 33)]),
    (256, 2, 2, 16, [(100, 70)]),
    (96, 6, 2, 5, [(77, 40), (0, 100)]),
    (32, 4, 1, 16, [(1000, 65)]),
    (16, 8, 2, 1, [(40, 30)]),
    (80, 4, 2, 16, [(0, 90)]),
]


@pytest.mark.parametrize("window,keep", [(0, 0), (50, 0), (128, 4), (1, 0), (300, 70)])
@pytest.mark.parametrize("dim,heads,nkv,page,requests", SIZES)
def test_attention(native, dim, heads, nkv, page, requests, window, keep) -> None:
    seed = dim + heads * 3 + page + window
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, seed)
    g = torch.Generator().manual_seed(seed)
    tokens = sum(n for _, n in requests)
    q = (torch.randn((tokens + 2, heads * dim), generator=g) * 2).to(torch.bfloat16)
    scale = dim ** -0.5
    out, status = attend(native, cache, requests, q, window, keep, scale)
    assert status == 0
    check_attention(cache, requests, q, out, window, keep, scale)


@pytest.mark.parametrize("dim,requests", [(128, [(900, 1), (333, 1), (10, 1)]), (128, [(700, 3), (90, 4), (64, 1)]), (48, [(300, 1), (200, 4)]), (96, [(300, 2), (200, 3)]), (64, [(700, 200), (90, 40)]), (128, [(700, 200), (90, 40), (64, 1)]),
                                          (32, [(700, 90)])])
def test_attention_cut_into_pieces(native, dim, requests) -> None:
    """Every cut of the keys gives the same attention; a plan made for shorter entries still sees all keys."""
    heads, nkv, page = 8, 2, 16
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, dim)
    g = torch.Generator().manual_seed(4)
    q = (torch.randn((sum(n for _, n in requests) + 2, heads * dim), generator=g) * 2).to(torch.bfloat16)
    for spans in ((1, 16, 1, 16, 1, 16, 8), (2, 8, 2, 8, 3, 8, 12), (3, 4, 3, 4, 2, 2, 8), (1, 2, 1, 2, 1, 2, 8), (100, 1, 100, 1, 100, 1, 8)):
        for window, keep in ((0, 0), (200, 20)):
            out, status = attend(native, cache, requests, q, window, keep, dim ** -0.5, plan=spans)
            assert status == 0
            check_attention(cache, requests, q, out, window, keep, dim ** -0.5)


@pytest.mark.parametrize("dim", [128, 64, 96])
def test_attention_with_scales_of_every_size(native, dim) -> None:
    """Keys and values whose scales differ by many powers of two, vectors of zeros among them, and one huge key that
    only the last queries see."""
    heads, nkv, page, requests = 8, 2, 16, [(300, 1), (200, 60), (0, 130)]
    g = torch.Generator().manual_seed(dim)
    values = []
    for s, n in requests:
        k, v = (torch.randn((s + n, nkv, dim), generator=g, dtype=torch.float64) for _ in range(2))
        v *= torch.exp2(torch.randint(-40, 40, (s + n, nkv, 1), generator=g).double())
        k *= torch.exp2(torch.randint(-20, 2, (s + n, nkv, 1), generator=g).double())
        v[::7] = 0
        k[3::11] = 0
        v[s + n - 1] *= 2.0 ** 20
        values.append((k, v))
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5, values=values)
    q = (torch.randn((sum(n for _, n in requests) + 2, heads * dim), generator=g)).to(torch.bfloat16)
    for factor in (1.0, 2.0 ** -30, 2.0 ** 6):
        scaled = (q.float() * factor).to(torch.bfloat16)
        out, status = attend(native, cache, requests, scaled, 0, 0, dim ** -0.5)
        assert status == 0
        check_attention(cache, requests, scaled, out, 0, 0, dim ** -0.5, large_scores=factor > 1)


@pytest.mark.parametrize("dim", [128, 64, 96])
@pytest.mark.parametrize("up,down", [(75, -72), (-71, 71), (100, -73), (-90, 71)])
def test_queries_far_from_one(native, dim, up, down) -> None:
    """Queries beyond the scales a cached vector can have, against keys at the other end."""
    heads, nkv, page, requests = 8, 2, 16, [(100, 1), (70, 4), (60, 50)]
    g = torch.Generator().manual_seed(dim)
    values = [tuple(torch.randn((s + n, nkv, dim), generator=g, dtype=torch.float64) * f for f in (2.0 ** down, 1.0)) for s, n in requests]
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5, values=values)
    q = (torch.randn((sum(n for _, n in requests) + 2, heads * dim), generator=g, dtype=torch.float64) * 2.0 ** up).to(torch.bfloat16)
    scale = dim ** -0.5 * 2.0 ** -(up + down)
    out, status = attend(native, cache, requests, q, 0, 0, scale)
    assert status == 0
    check_attention(cache, requests, q, out, 0, 0, scale)


@pytest.mark.parametrize("dim,requests", [(128, [(90, 1), (100, 4), (0, 1)]), (128, [(20, 100), (0, 70)]), (64, [(20, 150)]), (32, [(20, 40)])])
@pytest.mark.parametrize("window,keep", [(0, 0), (30, 2)])
def test_what_is_not_finite_reaches_only_who_sees_it(native, dim, requests, window, keep) -> None:
    heads, nkv, page = 8, 2, 16
    g = torch.Generator().manual_seed(dim)
    values = []
    for s, n in requests:
        k, v = (torch.randn((s + n, nkv, dim), generator=g, dtype=torch.float64) for _ in range(2))
        k[(s + n) // 2, 0, 3] = math.nan
        v[max(0, s + n - 2), 1, 0] = math.inf
        values.append((k, v))
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5, values=values)
    q = torch.randn((sum(n for _, n in requests) + 2, heads * dim), generator=g).to(torch.bfloat16)
    q[0, 5] = math.nan
    out, _ = attend(native, cache, requests, q, window, keep, dim ** -0.5)
    at = 0
    for e, (s, n) in enumerate(requests):
        for i in range(n):
            for h in range(heads):
                kvh = h // (heads // nkv)
                bad = (s + n) // 2 if kvh == 0 else max(0, s + n - 2)
                sees = bad <= s + i and (not window or s + i - bad < window or bad < keep)
                got = out[at + i].view(heads, dim)[h]
                assert bool(torch.isnan(got).all()) == (sees or (at + i == 0 and h == 0)), (e, i, h)
                assert bool(torch.isfinite(got).all()) != bool(torch.isnan(got).all())
        at += n


def test_missing_pages_are_flagged_and_passed_pages_are_not(native) -> None:
    dim, heads, nkv, page = 64, 4, 2, 16
    for requests in ([(200, 1)], [(200, 30)]):
        cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 1)
        q = torch.randn((sum(n for _, n in requests) + 2, heads * dim)).to(torch.bfloat16)
        cache["table"][0, 2] = -1                    # positions 32..47
        out, status = attend(native, cache, requests, q, 100, 20, dim ** -0.5)
        assert status == 0                           # outside the window of every query, behind the kept ones
        check_attention(cache, requests, q, out, 100, 20, dim ** -0.5)
        _, status = attend(native, cache, requests, q, 0, 0, dim ** -0.5)
        assert status == 2
        _, status = attend(native, cache, requests, q, 100, 33, dim ** -0.5)
        assert status == 2
        cache["table"][0, 2] = cache["pages"]
        _, status = attend(native, cache, requests, q, 0, 0, dim ** -0.5)
        assert status == 2


def test_bad_token_counts_touch_nothing(native) -> None:
    dim, heads, nkv, page = 64, 4, 2, 16
    cache = plain.pool([20, 20], nkv, dim, page, 1)
    caches = to_device(cache)
    q = torch.randn((4, heads * dim)).to(torch.bfloat16).to(DEV)
    for ends, starts in (([0, 5, 6], [0, 0]), ([-1, 2, 3], [0, 0]), ([3, 1, 1], [0, 0]), ([0, 1, 2], [-5, -1])):
        for plan in ((1, 2, 1, 2, 1, 2, 2), (4, 1, 4, 1, 4, 1, 2)):
            out, status = torch.full_like(q, 7.0), status_word()
            native.attention_kv8(q, *caches, cache["table"].to(DEV), ints(ends), ints(starts), 1, 5, heads, 0, 0, 1.0, out, status, plan)
            assert int(status.item()) == 4 and bool((out == 7.0).all())


@pytest.mark.parametrize("dim", [64, 32])
@pytest.mark.parametrize("requests", [[(5, 1), (0, 1)], [(40, 30)]])
def test_scales_lie_anywhere(native, dim, requests) -> None:
    """Scales are bytes: pages of one token of one head, and views that begin at an odd address."""
    heads, nkv, page = 2, 1, 1
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 2)
    caches = list(to_device(cache))
    for i in (2, 3):
        room = torch.zeros(caches[i].numel() + 1, dtype=torch.uint8, device=DEV)
        room[1:] = caches[i].view(torch.uint8).flatten()
        caches[i] = room[1:].view(caches[i].shape).view(plain.SCALES)
        assert caches[i].data_ptr() % 4 == 1
    q = torch.randn((sum(n for _, n in requests) + 2, heads * dim), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    out, status = attend(native, cache, requests, q, 0, 0, dim ** -0.5, caches=caches)
    assert status == 0
    check_attention(cache, requests, q, out, 0, 0, dim ** -0.5)
    # written and read back there
    kv = torch.randn((1, dim)).to(DEV)
    word, at = status_word(), ints([3])
    native.kv8_write(kv, kv, at, ints([0]), *caches, cache["table"].to(DEV), word)
    outs = [torch.empty((1, nkv, dim), device=DEV) for _ in range(2)]
    native.kv8_read(*caches, cache["table"].to(DEV), at, ints([0]), *outs, word)
    codes, scales = plain.quantise(kv.cpu()[:, None])
    assert int(word.item()) == 0
    assert all(torch.equal(o.cpu().double(), codes * torch.exp2(scales.double() - 127)[..., None]) for o in outs)


@pytest.mark.parametrize("requests", [[(200, 1)], [(200, 30)]])
@pytest.mark.parametrize("window,keep", [(2 ** 40, 0), (2 ** 32 + 5, 3), (2 ** 31 - 1, 2 ** 31 - 1), (20, 2 ** 31 - 1), (20, 2 ** 32 + 1)])
def test_windows_and_kept_tokens_past_every_position(native, requests, window, keep) -> None:
    dim, heads, nkv, page = 64, 4, 2, 16
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 1)
    q = torch.randn((sum(n for _, n in requests) + 2, heads * dim), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    out, status = attend(native, cache, requests, q, window, keep, dim ** -0.5)
    assert status == 0
    check_attention(cache, requests, q, out, 0, 0, dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 32])
@pytest.mark.parametrize("entry,most", [(3, 1), (5, 3), (30, 20)])
def test_an_entry_of_more_tokens_than_said_is_told(native, dim, entry, most) -> None:
    """The call is sized by ``max_new``; an entry beyond it sets the status bit and nothing of it is written, cut or not."""
    heads, nkv, page = 4, 2, 16
    cache = plain.pool([300], nkv, dim, page, 1)
    caches, table = to_device(cache), cache["table"].to(DEV)
    q = torch.randn((entry + 8, heads * dim)).to(torch.bfloat16).to(DEV)
    for plan in ((1, 3, 1, 3, 1, 3, 2), (4, 1, 4, 1, 4, 1, 2)):
        out, status = torch.full_like(q, 7.0), status_word()
        native.attention_kv8(q, *caches, table, ints([0, entry]), ints([300 - entry]), 1, most, heads, 0, 0, 1.0, out, status, plan)
        assert int(status.item()) == 4 and bool((out == 7.0).all())


def test_a_portion_behind_a_long_context_among_many_single_tokens(native) -> None:
    """Row tiles are counted over the portions alone: more entries than a warp looks at in a step, portions in front, in the
    middle and last, empty entries between; the pieces' buffer grows with the portions, not with the entries."""
    dim, heads, nkv, page = 128, 8, 2, 16
    requests = [(7, 9)] + [(30 + i, 1) for i in range(40)] + [(1500, 150), (0, 0), (3, 3)] + [(60, 1)] * 30 + [(700, 70)]
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5)
    q = (torch.randn((sum(n for _, n in requests) + 2, heads * dim), generator=torch.Generator().manual_seed(2)) * 2).to(torch.bfloat16)
    made = native.kv8_plan(requests, heads, nkv, dim, 0, 0)
    assert made[6] == 6                          # 1 + 3 + 2
    for cut in (made, (1, 4, 1, 4, 2, 8, 6)):
        out, status = attend(native, cache, requests, q, 0, 0, dim ** -0.5, plan=cut)
        assert status == 0
        check_attention(cache, requests, q, out, 0, 0, dim ** -0.5)
    assert native.kv8_lib(dim)[1](len(requests), 150, nkv, 4, 4, 4, 6, 8) == 6 * nkv * 8 * 256 * (dim + 2)


@pytest.mark.parametrize("dim", [64, 32, 128])
def test_three_hundred_heads_on_one(native, dim) -> None:
    """One token's rows fill more than a row tile."""
    requests, heads = [(40, 1), (130, 2), (0, 1)], 300
    cache = plain.pool([s + n for s, n in requests], 1, dim, 16, 3)
    q = torch.randn((6, heads * dim), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    out, status = attend(native, cache, requests, q, 0, 0, dim ** -0.5)
    assert status == 0
    check_attention(cache, requests, q, out, 0, 0, dim ** -0.5)


def test_written_read_and_attended_together(native) -> None:
    """A prompt in two portions, then single tokens, each written and attended, on a stream of its own; the cache read
    back is what the attention saw."""
    dim, heads, nkv, page = 128, 8, 2, 16
    g = torch.Generator().manual_seed(9)
    total = 150 + 41 + 3
    x = (torch.randn((total, (heads + 2 * nkv) * dim), generator=g)).to(DEV)
    pages = -(-total // page)
    table = torch.randperm(pages, generator=g).to(torch.int32)[None].to(DEV)
    caches = empty_caches(pages, nkv, page, dim)
    status = status_word()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(side):
        at = 0
        for n in (150, 41, 1, 1, 1):
            rows = x[at : at + n]
            q, k, v = rows.split((heads * dim, nkv * dim, nkv * dim), dim=1)
            q_out = torch.empty((n, heads * dim), dtype=torch.bfloat16, device=DEV)
            native.kv8_write(k, v, ints(range(at, at + n)), ints([0] * n), *caches, table, status, q=q, q_out=q_out)
            out = torch.empty_like(q_out)
            native.attention_kv8(q_out, *caches, table, ints([0, n]), ints([at]), 1, n, heads, None, 0, dim ** -0.5, out, status,
                                 native.kv8_plan([(at, n)], heads, nkv, dim))
            outs.append(out)
            at += n
        back = [torch.empty((total, nkv, dim), dtype=torch.float32, device=DEV) for _ in range(2)]
        native.kv8_read(*caches, table, ints(range(total)), ints([0] * total), *back, status)
    side.synchronize()
    assert int(status.item()) == 0
    k, v = (b.cpu().double() for b in back)
    want_k, scales = plain.quantise(x[:, heads * dim : (heads + nkv) * dim].view(total, nkv, dim))
    assert torch.equal(k, want_k * torch.exp2(scales.double() - 127)[..., None])
    q = x[:, : heads * dim].to(torch.bfloat16).cpu()
    cache = {"k_cache": caches[0], "held": [(k, v)]}
    check_attention(cache, [(0, total)], q, torch.cat(outs).cpu(), 0, 0, dim ** -0.5)


def test_two_captured_graphs_and_eager_calls_between(native) -> None:
    """Two captured calls replayed side by side on two streams, with eager calls between, keep apart: the pieces of a cut
    entry lie in the call's own buffer."""
    dim, heads, nkv, page = 128, 8, 2, 16
    cases = []
    for seed, requests in ((1, [(900, 1), (400, 60)]), (2, [(800, 2), (1000, 33)])):
        cache = plain.pool([s + n for s, n in requests], nkv, dim, page, seed)
        g = torch.Generator().manual_seed(seed)
        q = torch.randn((sum(n for _, n in requests), heads * dim), generator=g).to(torch.bfloat16)
        ends = [0]
        for _, n in requests:
            ends.append(ends[-1] + n)
        args = (q.to(DEV), *to_device(cache), cache["table"].to(DEV), ints(ends), ints(s for s, _ in requests), len(requests),
                max(n for _, n in requests), heads, 0, 0, dim ** -0.5)
        cases.append((cache, requests, q, args, torch.zeros(q.shape, dtype=torch.bfloat16, device=DEV), status_word()))
    plan = (2, 8, 2, 8, 2, 8, 4)
    graphs, streams = [], []
    for cache, requests, q, args, out, status in cases:
        native.attention_kv8(*args, out, status, plan)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            native.attention_kv8(*args, out, status, plan)
        graphs.append(graph)
        streams.append(torch.cuda.Stream())
        out.zero_()
    torch.cuda.synchronize()
    eager = [torch.zeros_like(c[4]) for c in cases]
    for _ in range(5):
        for i, (graph, stream) in enumerate(zip(graphs, streams)):
            with torch.cuda.stream(stream):
                graph.replay()
            native.attention_kv8(*cases[i][3], eager[i], cases[i][5], plan)
    torch.cuda.synchronize()
    for (cache, requests, q, _, out, status), other in zip(cases, eager):
        assert int(status.item()) == 0 and torch.equal(out, other)
        check_attention(cache, requests, q, out.cpu(), 0, 0, dim ** -0.5)
