"""The 8-bit cache on the CPU: what its operators refuse, and the plan of its attention."""

from __future__ import annotations

import pytest
import torch

import plain_kv8 as plain
from forge_engine_b200.errors import CUDAUnavailableError, UnsupportedShapeError
from forge_engine_b200.ops import native

N, HEADS, NKV, DIM, PAGE, PAGES = 6, 4, 2, 32, 8, 5


def caches(dim=DIM, nkv=NKV, page=PAGE, pages=PAGES):
    codes = [torch.zeros((pages, nkv, page, dim), dtype=torch.uint8).view(plain.CODES) for _ in range(2)]
    return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"),
                    (*codes, *(torch.zeros((pages, nkv, page), dtype=torch.uint8).view(plain.SCALES) for _ in range(2)))))


def places():
    return dict(positions=torch.zeros(N, dtype=torch.int32), token_entry=torch.zeros(N, dtype=torch.int32),
                block_table=torch.zeros((2, 3), dtype=torch.int32), status=torch.zeros(1, dtype=torch.int32))


def write_args(**other):
    return {**caches(), **places(), "k": torch.zeros((N, NKV * DIM)), "v": torch.zeros((N, NKV * DIM)), **other}


def read_args(**other):
    return {**caches(), **places(), "k_out": torch.zeros((N, NKV, DIM)), "v_out": torch.zeros((N, NKV, DIM)), **other}


def attention_args(**other):
    args = {**caches(), "q": torch.zeros((N, HEADS * DIM), dtype=torch.bfloat16), "block_table": torch.zeros((2, 3), dtype=torch.int32),
            "cu_tokens": torch.tensor([0, 1, 6], dtype=torch.int32), "starts": torch.zeros(2, dtype=torch.int32), "n_entries": 2,
            "max_new": 5, "num_q_heads": HEADS, "window": None, "keep_first": 0, "scale": 1.0,
            "out": torch.zeros((N, HEADS * DIM), dtype=torch.bfloat16), "status": torch.zeros(1, dtype=torch.int32), "plan": (1, 1, 1, 1, 1, 1, 1)}
    return {**args, **other}


CACHE_FAULTS = [
    dict(k_cache=torch.zeros((PAGES, NKV, PAGE, DIM), dtype=torch.bfloat16)),
    dict(v_cache=torch.zeros((PAGES, NKV, PAGE, DIM), dtype=torch.uint8)),
    dict(k_scale=torch.zeros((PAGES, NKV, PAGE))),
    dict(v_scale=caches(page=4)["v_scale"]),
    dict(v_cache=caches(dim=64)["v_cache"]),
    caches(dim=24), caches(dim=272), caches(dim=8),
    dict(block_table=torch.zeros((2, 3), dtype=torch.int64)),
    dict(block_table=torch.zeros(6, dtype=torch.int32)),
    dict(status=torch.zeros(1)),
]


@pytest.mark.parametrize("call,args", [(native.kv8_write, write_args), (native.kv8_read, read_args), (native.attention_kv8, attention_args)])
def test_caches_that_are_none(call, args) -> None:
    for fault in CACHE_FAULTS:
        with pytest.raises(UnsupportedShapeError):
            call(**args(**fault))
    # nothing runs without a device
    with pytest.raises(CUDAUnavailableError):
        call(**args())


@pytest.mark.parametrize("fault", [
    dict(k=None), dict(v=None), dict(k=None, v=None), dict(k=torch.zeros((N, NKV * DIM + 1))), dict(k=torch.zeros((N + 1, NKV * DIM))),
    dict(v=torch.zeros((N, NKV * DIM), dtype=torch.bfloat16)), dict(k=torch.zeros((N, NKV * DIM), dtype=torch.float16), v=torch.zeros((N, NKV * DIM), dtype=torch.float16)),
    dict(k=torch.zeros((NKV * DIM, N)).t()),
    dict(positions=torch.zeros(N, dtype=torch.int64)), dict(token_entry=torch.zeros(N - 1, dtype=torch.int32)),
    dict(q=torch.zeros((N, HEADS * DIM))), dict(q_out=torch.zeros((N, HEADS * DIM), dtype=torch.bfloat16)),
    dict(q=torch.zeros((N, HEADS * DIM)), q_out=torch.zeros((N, HEADS * DIM))),
    dict(q=torch.zeros((N, HEADS * DIM + 4)), q_out=torch.zeros((N, HEADS * DIM + 4), dtype=torch.bfloat16)),
    dict(q=torch.zeros((N, HEADS * DIM), dtype=torch.bfloat16), q_out=torch.zeros((N, HEADS * DIM), dtype=torch.bfloat16)),
    dict(k_norm=torch.zeros(DIM - 1)), dict(k_norm=torch.zeros(DIM, dtype=torch.bfloat16)), dict(q_norm=torch.zeros((1, DIM))),
    dict(table=torch.zeros((N, DIM, 2))), dict(table=torch.zeros((N, 2, 2))), dict(table=torch.zeros((N - 1, 8, 2))), dict(table=torch.zeros((N, 8))),
])
def test_write_refuses(fault) -> None:
    with pytest.raises(UnsupportedShapeError):
        native.kv8_write(**write_args(**fault))


@pytest.mark.parametrize("fault", [
    dict(k_out=torch.zeros((N, NKV, DIM), dtype=torch.bfloat16)), dict(k_out=torch.zeros((N, NKV * DIM))), dict(v_out=torch.zeros((N + 1, NKV, DIM))),
    dict(k_out=torch.zeros((N, NKV, DIM), dtype=torch.float16), v_out=torch.zeros((N, NKV, DIM), dtype=torch.float16)),
    dict(positions=torch.zeros(N + 1, dtype=torch.int32)), dict(token_entry=torch.zeros(N)),
])
def test_read_refuses(fault) -> None:
    with pytest.raises(UnsupportedShapeError):
        native.kv8_read(**read_args(**fault))


@pytest.mark.parametrize("fault", [
    dict(num_q_heads=3), dict(num_q_heads=0), dict(num_q_heads=8), dict(q=torch.zeros((N, HEADS * DIM))), dict(out=torch.zeros((N, HEADS * DIM))),
    dict(out=torch.zeros((N + 1, HEADS * DIM), dtype=torch.bfloat16)), dict(q=torch.zeros((HEADS * DIM, N), dtype=torch.bfloat16).t()),
    dict(n_entries=3), dict(n_entries=-1), dict(max_new=-1), dict(window=-1), dict(keep_first=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(cu_tokens=torch.zeros(2, dtype=torch.int32)), dict(cu_tokens=torch.zeros(3, dtype=torch.int64)), dict(starts=torch.zeros(1, dtype=torch.int32)),
    dict(block_table=torch.zeros((1, 3), dtype=torch.int32)),
])
def test_attention_refuses(fault) -> None:
    with pytest.raises(UnsupportedShapeError):
        native.attention_kv8(**attention_args(**fault))


def test_quantising_restates_the_type() -> None:
    """The 64-bit statement against torch's own conversion to e4m3."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn((200, 32), generator=g) * torch.exp(4 * torch.randn((200, 1), generator=g))
    codes, scales = plain.quantise(x)
    e = scales.double() - 127
    assert torch.equal(codes, (x.double() * torch.exp2(-e)[:, None]).float().to(plain.CODES).double())
    assert bool((codes.abs().amax(-1) >= 224).all())
    assert scales[0] == plain.quantise(x[:1] * 2)[1] - 1


@pytest.mark.parametrize("window,keep", [(0, 0), (100, 0), (1000, 10)])
@pytest.mark.parametrize("entries", [[(0, 1)], [(5000, 1), (0, 1), (300, 2)], [(0, 2048)], [(32768, 1)], [(10, 0), (4000, 700), (9, 1)], [(7, 0)], []])
def test_plans_cover_every_key(entries, window, keep) -> None:
    for heads, nkv, dim in ((32, 8, 128), (4, 4, 64), (16, 1, 96)):
        plan = native.kv8_plan(entries, heads, nkv, dim, window, keep)
        groups = heads // nkv
        kinds = [(lambda r: 0 < r <= 8, plan[:2]), (lambda r: 8 < r <= 16, plan[2:4]), (lambda r: r > 16, plan[4:6])]
        for is_kind, (span, spans) in kinds:
            mine = [start + n for start, n in entries if is_kind(n * groups)]
            assert (spans > 0) == bool(mine) and span >= 1 and (not spans or spans // (spans & -spans) in (1, 3))
            if mine and not window:
                assert span * spans * native.KV8_TILE >= max(mine)
        rows_of = 256 if dim in (64, 128) else 64
        assert plan[6] >= sum(-(-n * groups // rows_of) for _, n in entries if n * groups > 16)


def test_plans_take_any_pairs_once() -> None:
    want = native.kv8_plan([(700, 1), (3, 40)], 32, 8, 128)
    assert native.kv8_plan(iter([[700, 1], [3, 40]]), 32, 8, 128) == want
    assert native.kv8_plan(((700, 1), (3, 40)), 32, 8, 128, None, 0) == want
    # a context that grows by a token at a time changes its plan at most four times while it doubles
    assert len({native.kv8_plan([(n, 1)], 32, 8, 128) for n in range(4096, 8192)}) <= 5


@pytest.mark.parametrize("scale", [float("inf"), 1e39])
def test_attention_refuses_scales_beyond_32_bits(scale) -> None:
    with pytest.raises(UnsupportedShapeError):
        native.attention_kv8(**attention_args(scale=scale))


@pytest.mark.parametrize("tiles", [49152, 49153, 60000, 65535, 65536])
def test_row_tiles_are_rounded_within_what_a_call_takes(tiles) -> None:
    """A plan's count of row tiles is rounded up, but not beyond what the kernels take while the true count is within it."""
    units = native.kv8_plan([(0, 4 * tiles)], 16, 1, 96, 128)[6]
    assert units >= tiles and (units <= 65535) == (tiles <= 65535)
