"""The 8-bit cache's operators where single calls came out wrong, and the head sizes between 128 and 256.  Bounds and
plain statements: ``test_gpu_kv8.py``, ``plain_kv8.py``."""

from __future__ import annotations

import math

import pytest
import torch

import plain_kv8 as plain
from test_gpu_kv8 import DEV, attend, check_attention, empty_caches, ints, native, status_word  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def rows_of(requests, heads: int, dim: int, seed: int, extra: int = 2) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((sum(n for _, n in requests) + extra, heads * dim), generator=g) * 2).to(torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("scale", [2.0 ** -20, 2.0 ** -31, 1e-30, 1e-44, 1e-60])
def test_small_scales_and_queries_of_zeros(native, dim, scale) -> None:  # noqa: F811
    """A scale of any size gives rows of zeros and others the mean of the values they see, masked keys left out."""
    heads, nkv, page, requests = 8, 2, 16, [(30, 1), (50, 4), (5, 70), (200, 40)]
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, dim)
    q = rows_of(requests, heads, dim, 3)
    q[::2] = 0
    q[1::4, dim : 2 * dim] = 0
    for window, keep in ((0, 0), (40, 3)):
        out, status = attend(native, cache, requests, q, window, keep, scale)
        assert status == 0
        check_attention(cache, requests, q, out, window, keep, scale)


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("dim,requests", [(128, [(90, 1), (20, 2)]), (128, [(90, 4), (5, 3)]), (96, [(90, 1), (50, 4)]), (96, [(90, 30)]),
                                          (48, [(90, 1), (50, 4), (20, 30)]), (64, [(90, 30)])])
def test_queries_that_are_infinite_give_nan(native, dim, requests, value) -> None:  # noqa: F811
    """An infinite element of a query makes its head's output NaN, also where every score is minus infinity; no other
    row notices."""
    heads, nkv, page = 8, 2, 16
    g = torch.Generator().manual_seed(dim)
    values = []
    for s, n in requests:
        k, v = (torch.randn((s + n, nkv, dim), generator=g, dtype=torch.float64) for _ in range(2))
        k[:, :, 5] = -math.copysign(1.0, value) * (1 + k[:, :, 5].abs())
        values.append((k, v))
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5, values=values)
    q = rows_of(requests, heads, dim, 4)
    bad = torch.zeros((q.shape[0], heads), dtype=torch.bool)
    at = 0
    for _, n in requests:
        bad[at, 1] = bad[at + n - 1, heads - 1] = True
        at += n
    q.view(-1, heads, dim)[:, :, 5][bad] = value
    for plan in (None, (1, 2, 1, 2, 1, 2, 8)):
        out, status = attend(native, cache, requests, q, 0, 0, dim ** -0.5, plan=plan)
        got = out[:at].view(at, heads, dim)
        assert status == 0 and bool(torch.isnan(got[bad[:at]]).all()) and bool(torch.isfinite(got[~bad[:at]]).all())


def zero_values(which: str, length: int) -> torch.Tensor:
    """Which of a request's values are zero."""
    at = torch.arange(length)
    return {"every other": at % 2 == 0, "first half": at < length // 2, "second half": at >= length // 2, "all but one": at != length // 3}[which]


@pytest.mark.parametrize("which", ["every other", "first half", "second half", "all but one"])
@pytest.mark.parametrize("dim,requests", [(128, [(900, 1), (333, 2)]), (128, [(700, 4)]), (48, [(700, 1), (200, 4)]), (96, [(700, 60)]),
                                          (128, [(700, 60)])])
def test_zeros_beside_the_largest_values_count(native, dim, requests, which) -> None:  # noqa: F811
    """Values of zeros, whose scale is the least there is, beside values whose scale is near the largest: each key counts in
    the sum that divides, whatever its value's scale."""
    heads, nkv, page = 8, 2, 16
    g = torch.Generator().manual_seed(dim)
    values = []
    for s, n in requests:
        k, v = (torch.randn((s + n, nkv, dim), generator=g, dtype=torch.float64) for _ in range(2))
        v *= 2.0 ** 70
        v[zero_values(which, s + n)] = 0
        values.append((k, v))
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5, values=values)
    assert {int(x) for x in cache["v_scale"].view(torch.uint8).unique()} >= {63} and int(cache["v_scale"].view(torch.uint8)[cache["v_scale"].view(torch.uint8) < 255].max()) >= 190
    q = rows_of(requests, heads, dim, 4)
    for plan in (None, (1, 16, 1, 16, 1, 16, 8), (100, 1, 100, 1, 100, 1, 8)):
        out, status = attend(native, cache, requests, q, 0, 0, dim ** -0.5, plan=plan)
        assert status == 0
        check_attention(cache, requests, q, out, 0, 0, dim ** -0.5)


@pytest.mark.parametrize("rot", [8, 16])
def test_hundreds_of_heads_some_not_finite(native, rot) -> None:  # noqa: F811
    """More heads than a writing warp has rounds to note which it takes again: keys that are not finite stay so."""
    dim, nkv, page, tokens = 256, 1200, 16, 300
    g = torch.Generator().manual_seed(rot)
    row = torch.randn((1, nkv * dim), generator=g)
    bad = [0, 5, 300, 511, 700, 902, 1100, 1199]
    for i, head in enumerate(bad):
        row[0, head * dim + (37 * i) % dim] = (math.inf, -math.inf, math.nan)[i % 3]
    angle = torch.rand((1, rot // 2), generator=g).double()
    table = torch.stack((angle.cos(), angle.sin()), -1).float()
    pages = -(-tokens // page)
    caches = empty_caches(pages, nkv, page, dim)
    status = status_word()
    rows = row.to(DEV).expand(tokens, -1)
    native.kv8_write(rows, rows, ints(range(tokens)), ints([0] * tokens), *caches, ints(range(pages)).view(1, pages), status,
                     table=table.expand(tokens, -1, -1).contiguous().to(DEV))
    assert int(status.item()) == 0
    heads = row.view(1, nkv, dim)
    finite = torch.where(torch.isfinite(heads).all(-1, keepdim=True), heads, torch.full_like(heads, math.nan))
    for x, codes, scales in ((plain.norm_rotate(finite, None, 0.0, table), caches[0], caches[2]), (heads.double(), caches[1], caches[3])):
        want_codes, want_scales = plain.quantise(x[0])
        got_scales = scales.view(torch.uint8).transpose(1, 2).reshape(pages * page, nkv)[:tokens]
        got_codes = codes.view(torch.uint8).transpose(1, 2).reshape(pages * page, nkv, dim)[:tokens]
        assert torch.equal(got_scales, want_scales.to(DEV).expand(tokens, -1))
        want = want_codes.float().to(plain.CODES).view(torch.uint8).to(DEV)
        # a zero has two signs
        assert bool(((got_codes == want) | (((got_codes | want) & 0x7F) == 0)).all())


KINDS = {"few": [(300, 1), (40, 2)], "single": [(300, 4), (17, 3)], "portion": [(260, 70), (5, 30)]}


@pytest.mark.parametrize("dim", [64, 128, 96, 48])
@pytest.mark.parametrize("planned", [("few",), ("single",), ("portion",), ("few", "portion"), ("single", "portion"), ("few", "single"), ()])
def test_entries_outside_the_plan_are_told(native, dim, planned) -> None:  # noqa: F811
    """An entry of a kind that the plan has not got sets the status bit and is left as it was; the others are right.  With
    fillers the same without the bit."""
    heads, nkv, page = 8, 2, 16
    requests = [r for pair in zip(*KINDS.values()) for r in pair]
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5)
    caches = tuple(cache[name].view(torch.uint8).to(DEV).view(cache[name].dtype) for name in ("k_cache", "v_cache", "k_scale", "v_scale"))
    q = rows_of(requests, heads, dim, 4)
    inside = [r for kind in planned for r in KINDS[kind]]
    ends = [0]
    for _, n in requests:
        ends.append(ends[-1] + n)
    made = native.kv8_plan(inside, heads, nkv, dim)
    for plan in (made, *(tuple(2 if i in (0, 2, 4) else 2 * (made[i] > 0) if i in (1, 3, 5) else made[i] for i in range(7)) for _ in made[1::2])):
        for fillers in (False, True):
            out, status = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV), status_word()
            native.attention_kv8(q.to(DEV), *caches, cache["table"].to(DEV), ints(ends), ints(s for s, _ in requests), len(requests), 70, heads,
                                 None, 0, dim ** -0.5, out, status, plan, fillers=fillers)
            assert int(status.item()) == (0 if fillers else 32)
            for e, request in enumerate(requests):
                rows = out[ends[e] : ends[e + 1]].cpu()
                if request in inside:
                    one = {**cache, "held": [cache["held"][e]]}
                    check_attention(one, [request], q[ends[e] : ends[e + 1]], rows, 0, 0, dim ** -0.5)
                elif planned or fillers or request not in KINDS["few"]:
                    assert bool((rows == 7.0).all()), request


@pytest.mark.parametrize("dim", [64, 96])
@pytest.mark.parametrize("spans", [1, 3])
def test_row_tiles_beyond_the_plan_are_told(native, dim, spans) -> None:  # noqa: F811
    """A plan with fewer row tiles than the entries have: the first ones are right, nothing else is written, and the status
    says so - unless the others are fillers."""
    heads, nkv, page, requests = 8, 2, 16, [(100, 70), (0, 300), (30, 90)]
    rows_of_tile = 256 if dim == 64 else 64
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, 5)
    caches = tuple(cache[name].view(torch.uint8).to(DEV).view(cache[name].dtype) for name in ("k_cache", "v_cache", "k_scale", "v_scale"))
    q = rows_of(requests, heads, dim, 4)
    ends = [0, 70, 370, 460]
    tiles = [-(-n * heads // nkv // rows_of_tile) for _, n in requests]
    first = tiles[0] + tiles[1]
    for units, bit in ((first, 32), (tiles[0] + 1, 32), (sum(tiles), 0), (sum(tiles) + 5, 0)):
        for fillers in (False, True):
            out, status = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV), status_word()
            native.attention_kv8(q.to(DEV), *caches, cache["table"].to(DEV), ints(ends), ints(s for s, _ in requests), 3, 300, heads, None, 0,
                                 dim ** -0.5, out, status, (1, 0, 1, 0, 1 if spans > 1 else 100, spans, units), fillers=fillers)
            assert int(status.item()) == (0 if fillers else bit)
            out = out.cpu()
            whole = sum(1 for i in range(3) if sum(tiles[: i + 1]) <= units)
            check_attention({**cache, "held": cache["held"][:whole]}, requests[:whole], q, out, 0, 0, dim ** -0.5)
            # of the entry that is cut off, the tokens of the tiles that are there
            written = ends[whole] + (units - sum(tiles[:whole])) * rows_of_tile * nkv // heads if whole < 3 else 460
            assert bool((out[written:] == 7.0).all())


def test_more_tokens_than_said_are_told_by_a_plan_of_portions(native) -> None:  # noqa: F811
    """``max_new`` says that there is no portion, the plan that there is nothing else: nothing fits, and the status says so."""
    dim, heads, nkv, page = 64, 8, 2, 16
    cache = plain.pool([300], nkv, dim, page, 1)
    caches = tuple(cache[name].view(torch.uint8).to(DEV).view(cache[name].dtype) for name in ("k_cache", "v_cache", "k_scale", "v_scale"))
    q = rows_of([(0, 40)], heads, dim, 2).to(DEV)
    out, status = torch.full_like(q, 7.0), status_word()
    native.attention_kv8(q, *caches, cache["table"].to(DEV), ints([0, 40]), ints([260]), 1, 3, heads, None, 0, 1.0, out, status,
                         native.kv8_plan([(260, 40)], heads, nkv, dim))
    assert int(status.item()) == 4 and bool((out == 7.0).all())


# head sizes above 128 that are not 256: stretches of 128 and what is left of 64, 32 and 16 columns
LARGE_DIMS = [144, 160, 176, 192, 208, 224, 240]


@pytest.mark.parametrize("dim", LARGE_DIMS)
def test_head_sizes_between_128_and_256(native, dim) -> None:  # noqa: F811
    """Few rows, 9 to 16 rows and portions, uncut and cut, with and without a window."""
    heads, nkv, page, requests = 8, 2, 16, [(300, 1), (150, 2), (260, 4), (31, 3), (140, 40), (0, 70), (0, 1)]
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, dim)
    q = rows_of(requests, heads, dim, 3)
    for plan in (None, (1, 4, 1, 4, 1, 4, 12), (2, 2, 2, 2, 2, 2, 12), (100, 1, 100, 1, 100, 1, 12)):
        for window, keep in ((0, 0), (70, 20)):
            out, status = attend(native, cache, requests, q, window, keep, dim ** -0.5, plan=plan)
            assert status == 0
            check_attention(cache, requests, q, out, window, keep, dim ** -0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", LARGE_DIMS)
def test_writing_and_reading_head_sizes_between_128_and_256(native, dim, dtype) -> None:  # noqa: F811
    """Norm, partial rotation, codes, scales and the way back; keys and values alone take the exact codes."""
    tokens, nq, nkv, page, eps = 37, 3, 2, 16, 2.0 ** -20
    for rot in (dim, 24, 0):
        g = torch.Generator().manual_seed(dim + rot)
        x = (torch.randn((tokens, (nq + 2 * nkv) * dim), generator=g) * 2).to(dtype)
        weights = [torch.exp(0.3 * torch.randn(dim, generator=g)) for _ in range(2)] if rot else [None, None]
        table = None
        if rot:
            angle = torch.rand((tokens, rot // 2), generator=g).double() * 2 * math.pi
            table = torch.stack((angle.cos(), angle.sin()), -1).float()
        pages = -(-tokens // page)
        caches = empty_caches(pages, nkv, page, dim)
        status, table_of = status_word(), ints(range(pages)).view(1, pages)
        places = ints(range(tokens)), ints([0] * tokens)
        q, k, v = x.to(DEV).split((nq * dim, nkv * dim, nkv * dim), dim=1)
        q_out = torch.empty((tokens, nq * dim), dtype=torch.bfloat16, device=DEV)
        on = [None if w is None else w.to(DEV) for w in weights]
        native.kv8_write(k, v, *places, *caches, table_of, status, q=q, q_out=q_out, q_norm=on[0], k_norm=on[1], eps=eps,
                         table=None if table is None else table.to(DEV))
        outs = [torch.empty((tokens, nkv, dim), dtype=torch.float32, device=DEV) for _ in range(2)]
        native.kv8_read(*caches, table_of, *places, *outs, status)
        assert int(status.item()) == 0
        split = x.double().view(tokens, nq + 2 * nkv, dim)
        want_q = plain.norm_rotate(split[:, :nq], weights[0], eps, table)
        size = want_q.abs().amax(-1, keepdim=True)
        got_q = q_out.cpu().double().view(tokens, nq, dim)
        # rounding to bfloat16 once; 32-bit norm and rotation before it are off by less than 2^-18 of the pair
        assert bool(((got_q - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -18 * size).all())
        for want, got in ((plain.norm_rotate(split[:, nq : nq + nkv], weights[1], eps, table), outs[0]), (split[:, nq + nkv :], outs[1])):
            codes, scales = plain.quantise(want)
            assert torch.equal(got.cpu().double(), codes * torch.exp2(scales.double() - 127)[..., None])


@pytest.mark.parametrize("dim,requests", [(64, [(500, 1), (333, 70), (7, 200)]), (128, [(77, 3), (500, 90), (0, 33)])])
@pytest.mark.parametrize("page", [1, 5, 48])
@pytest.mark.parametrize("window,keep", [(0, 0), (130, 9)])
def test_pages_of_any_size_and_queries_inside_wider_rows(native, dim, requests, page, window, keep) -> None:  # noqa: F811
    """Pages that end inside a key tile, and queries that are columns of a projection, eight bytes from where 16 would be."""
    heads, nkv = 8, 2
    cache = plain.pool([s + n for s, n in requests], nkv, dim, page, dim + page)
    q = rows_of(requests, heads, dim, 3)
    wide = torch.full((q.shape[0], heads * dim + 24), 9.0, dtype=torch.bfloat16)
    wide[:, 4 : 4 + heads * dim] = q
    caches = tuple(cache[name].view(torch.uint8).to(DEV).view(cache[name].dtype) for name in ("k_cache", "v_cache", "k_scale", "v_scale"))
    ends = [0]
    for _, n in requests:
        ends.append(ends[-1] + n)
    for plan in (native.kv8_plan(requests, heads, nkv, dim, window, keep), (1, 3, 1, 3, 2, 3, 12)):
        out, status = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV), status_word()
        native.attention_kv8(wide.to(DEV)[:, 4 : 4 + heads * dim], *caches, cache["table"].to(DEV), ints(ends), ints(s for s, _ in requests),
                             len(requests), max(n for _, n in requests), heads, window, keep, dim ** -0.5, out, status, plan)
        assert int(status.item()) == 0 and bool((out[ends[-1] :] == 7.0).all())
        check_attention(cache, requests, q, out.cpu(), window, keep, dim ** -0.5)


@pytest.mark.parametrize("dim,nkv", [(128, 8), (256, 4), (48, 8)])
def test_caches_past_32_bit_offsets(native, dim, nkv) -> None:  # noqa: F811
    """Pages that lie more than 2^32 bytes into a cache, beside pages at its start: written, read back and attended."""
    heads, page = 2 * nkv, 64
    pages = 2 ** 32 // (nkv * page * dim) + 100
    codes = [torch.empty((pages, nkv, page, dim), dtype=torch.uint8, device=DEV).view(plain.CODES) for _ in range(2)]
    scales = [torch.empty((pages, nkv, page), dtype=torch.uint8, device=DEV).view(plain.SCALES) for _ in range(2)]
    caches = (*codes, *scales)
    requests = [(150, 1), (100, 60)]
    table = ints([pages - 1, 0, pages - 7, pages - 2, 3, pages - 50]).view(2, 3)
    g = torch.Generator().manual_seed(dim)
    held = []
    status = status_word()
    for e, (s, n) in enumerate(requests):
        x = torch.randn((s + n, 2 * nkv * dim), generator=g)
        k, v = x.to(DEV).split((nkv * dim, nkv * dim), dim=1)
        places = ints(range(s + n)), ints([e] * (s + n))
        native.kv8_write(k, v, *places, *caches, table, status)
        outs = [torch.empty((s + n, nkv, dim), device=DEV) for _ in range(2)]
        native.kv8_read(*caches, table, *places, *outs, status)
        both = []
        for t, out in zip(x.view(s + n, 2 * nkv, dim).split((nkv, nkv), dim=1), outs):
            c, b = plain.quantise(t)
            both.append(c * torch.exp2(b.double() - 127)[..., None])
            assert torch.equal(out.cpu().double(), both[-1])
        held.append(tuple(both))
    assert int(status.item()) == 0
    q = rows_of(requests, heads, dim, 3)
    for plan in (None, (1, 2, 1, 2, 1, 2, 8)):
        out, told = attend(native, {"k_cache": codes[0], "table": table}, requests, q, 0, 0, dim ** -0.5, plan=plan, caches=caches)
        assert told == 0
        check_attention({"k_cache": codes[0], "held": held}, requests, q, out, 0, 0, dim ** -0.5)
