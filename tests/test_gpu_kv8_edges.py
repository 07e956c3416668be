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
