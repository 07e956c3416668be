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
