"""The 8-bit cache in the cache manager and the settings, on the CPU."""

from __future__ import annotations

import pytest
import torch

from forge_engine_b200.cache.manager import CacheManager, CacheNeeds, PagedKVSpec
from forge_engine_b200.config import EngineConfig
from forge_engine_b200.engine.runner import check_cache
from forge_engine_b200.errors import ConfigError


def manager(*specs, **more):
    return CacheManager([CacheNeeds(kv=s) for s in specs], page_size=4, num_pages=6, max_requests=2, dtype=torch.bfloat16, device="cpu", **more)


def test_storage_and_views() -> None:
    eight, wide = PagedKVSpec(2, 32, eight_bit=True), PagedKVSpec(2, 32)
    cache = manager(eight, wide, eight)
    assert len(cache.groups) == 2 and cache.groups[0].units == [0, 2]
    view = cache.view(2)
    assert view.kv[0].shape == (7, 2, 4, 32) and view.kv[0].dtype == torch.float8_e4m3fn
    assert view.scales[1].shape == (7, 2, 4) and view.scales[1].dtype == torch.float8_e8m0fnu
    assert cache.view(1).scales is None and cache.view(1).kv[0].dtype == torch.bfloat16
    assert cache.bytes_per_token() == 2 * (2 * 2 * 33) + 2 * 64 * 2
    # what runs own does not overlap
    cache.view(0).scales[0].view(torch.uint8).fill_(3)
    assert int(cache.view(2).scales[0].view(torch.uint8).sum()) == 0 and int(cache.view(0).scales[1].view(torch.uint8).sum()) == 0
    with pytest.raises(ValueError):
        manager(PagedKVSpec(2, 32, v_head_dim=16, eight_bit=True))


def test_windows_release_pages_as_before() -> None:
    cache = manager(PagedKVSpec(1, 16, window=5, eight_bit=True))
    cache.begin_request("a")
    cache.reserve("a", 12)
    cache.advance("a", 12)
    assert cache.request("a").tables[0].pages[:2] == [-1, -1] and cache.free_pages() == [5]
    with pytest.raises(ValueError):
        cache.read("a", 0)
    cache.check_consistency()


def test_read_of_a_wide_cache() -> None:
    cache = manager(PagedKVSpec(2, 16))
    cache.begin_request("a")
    cache.reserve("a", 10)
    k, v = cache.kv_of_run(0)
    for at in range(10):
        page = cache.request("a").tables[0].pages[at // 4]
        k[page, :, at % 4] = at
        v[page, :, at % 4] = -at
    cache.advance("a", 10)
    got_k, got_v = cache.read("a", 0, first=2, count=7, dtype=torch.float32)
    assert got_k.dtype == torch.float32 and got_k[:, 0, 0].tolist() == list(range(2, 9)) and got_v[:, 1, 3].tolist() == [-x for x in range(2, 9)]
    assert cache.read("a", 0)[0].shape == (10, 2, 16) and cache.read("a", 0, first=10)[0].shape == (0, 2, 16)
    for first, count in ((-1, 1), (0, 11), (11, None), (3, -1)):
        with pytest.raises(ValueError):
            cache.read("a", 0, first=first, count=count)


def test_settings() -> None:
    assert EngineConfig(cache_dtype="float8").cache_dtype == "float8" and EngineConfig().cache_dtype is None
    for bad in (dict(cache_dtype="int8"), dict(cache_dtype="float8", dtype="float32")):
        with pytest.raises(ValueError):
            EngineConfig(**bad)
    eight, wide = CacheNeeds(kv=PagedKVSpec(1, 16, eight_bit=True)), CacheNeeds(kv=PagedKVSpec(1, 16))
    check_cache([wide, None], None)
    check_cache([eight, CacheNeeds(), None], "float8")
    for needs in ([eight, wide], [None], [CacheNeeds()]):
        with pytest.raises(ConfigError):
            check_cache(needs, "float8")


def test_parts_are_built_and_views_made_by_position_as_before() -> None:
    """What the 8-bit cache added to the parts' interfaces comes after what was there."""
    from forge_engine_b200.parts.base import BuildContext, CacheView

    timer, status = object(), object()
    ctx = BuildContext(torch.bfloat16, "cpu", status, timer)
    assert ctx.timer is timer and ctx.status is status and ctx.cache_dtype is None
    state, own, states = object(), object(), {"a": 1}
    view = CacheView(None, 0, True, state, own, states)
    assert view.state is state and view.own_state is own and view.states is states and view.scales is None


def attention_layer(scale: float, position=None, cache_dtype="float8", dtype=torch.bfloat16):
    from forge_engine_b200.config.specs import AttentionSpec, NoPositionSpec
    from forge_engine_b200.parts.attention import GQAttention
    from forge_engine_b200.parts.base import BuildContext

    spec = AttentionSpec(32, 4, 2, 16, False, 1e-6, False, scale, position or NoPositionSpec(), None)
    weights = {name: torch.zeros(info.shape, dtype=dtype) for name, info in GQAttention.weight_shapes(spec).items()}
    return GQAttention(spec, weights, BuildContext(dtype, torch.device("cpu"), None, cache_dtype=cache_dtype))


def test_layers_whose_scale_the_kernels_refuse_are_refused_at_build() -> None:
    """A layer that multiplies its scores by nothing positive runs over a wide cache alone: the model says so when it is
    built, not in its first step."""
    for scale, takes in ((0.25, True), (1.0, True), (0.0, False), (-0.25, False), (float("inf"), False), (float("nan"), False)):
        layer = attention_layer(scale)
        assert layer.eight_bit == takes and layer.cache_needs().kv.eight_bit == takes
        if not takes:
            with pytest.raises(ConfigError):
                check_cache([layer.cache_needs()], "float8")
    assert not attention_layer(0.25, dtype=torch.float32).eight_bit and not attention_layer(0.25, cache_dtype=None).eight_bit


def test_a_layer_over_a_wide_cache_does_not_ask_its_position_encoding_when_built(monkeypatch) -> None:
    from forge_engine_b200.parts.base import PositionEncoding

    monkeypatch.setattr(PositionEncoding, "rotary", lambda self: pytest.fail("asked"))
    assert not attention_layer(0.25, cache_dtype=None).eight_bit
