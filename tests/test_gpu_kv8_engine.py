"""The engine over an 8-bit cache: the whole path against the plain implementation with its keys and values rounded the
same way, replayed steps against eager ones, and what the cache manager hands back.

Bounds.  The engine's keys and values come from bfloat16 products and differ from the plain ones by about 2^-9 of
themselves.  Such a number rounds to another code with a probability of about 2^-9 over a step of 2^-3.5, 2 %, and is
then off by that step, 9 %: 1.3 % root mean square where a bfloat16 cache has 0.2 %.  One of a layer's products of
several gets six times as noisy; twice the bfloat16 engine's bounds (3e-2 of the largest logit, total variation 0.02) are
allowed."""

from __future__ import annotations

import math

import pytest
import torch

import plain_kv8
import plain_qwen3 as plain
from helpers import make_model_folder, random_ids, run_trace

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def rounded(x: torch.Tensor) -> torch.Tensor:
    """What an 8-bit cache makes of vectors along the last axis."""
    codes, scales = plain_kv8.quantise(x)
    return (codes * torch.exp2(scales.double() - 127)[..., None]).to(x.dtype)


@pytest.fixture(scope="module", params=["TINY_A", "TINY_B", "TINY_C", "TINY_D"])
def folder(request, tmp_path_factory):
    raw = dict(getattr(plain, request.param), eos_token_id=None)
    path = tmp_path_factory.mktemp("kv8") / request.param
    cfg, weights = make_model_folder(path, raw, 5)
    return path, cfg, weights


def runner_of(path, **more):
    from forge_engine_b200.engine import ModelRunner

    return ModelRunner.from_folder(path, dtype="bfloat16", page_size=16, num_pages=64, max_requests=4, cache_dtype="float8", **more)


def attention_of_rounded(x, weights, prefix, cfg, window=None):
    """``plain.attention`` with keys and values as an 8-bit cache holds them."""
    length, nq, nkv, d = x.shape[0], cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim

    def heads(name, count):
        bias = weights[f"{prefix}.{name}.bias"] if cfg.attention_bias else None
        return plain.linear(x, weights[f"{prefix}.{name}.weight"], bias).view(length, count, d)

    q = plain.rms_norm(heads("q_proj", nq), weights[f"{prefix}.q_norm.weight"], cfg.rms_norm_eps).transpose(0, 1)
    k = plain.rms_norm(heads("k_proj", nkv), weights[f"{prefix}.k_norm.weight"], cfg.rms_norm_eps).transpose(0, 1)
    cosine, sine = plain.rotary_tables(torch.arange(length), d, cfg.rope_theta, x.dtype)
    q, k = plain.apply_rotary(q, cosine, sine), rounded(plain.apply_rotary(k, cosine, sine))
    v = rounded(heads("v_proj", nkv)).transpose(0, 1)
    k, v = (t.repeat_interleave(nq // nkv, dim=0) for t in (k, v))
    scores = q @ k.transpose(1, 2) * d ** -0.5 + plain.causal_mask(length, x.dtype, window, x.device)
    out = (torch.softmax(scores, -1) @ v).transpose(0, 1).reshape(length, nq * d)
    return plain.linear(out, weights[f"{prefix}.o_proj.weight"], weights[f"{prefix}.o_proj.bias"] if cfg.attention_bias else None)


def test_steps_in_portions_equal_one_portion_and_replay(folder) -> None:
    """A sequence in one portion, in several, and token by token gives logits within rounding of one another; graphs replay
    what eager steps compute."""
    from forge_engine_b200.engine import StepEntry

    path, cfg, _ = folder
    ids = random_ids(cfg.vocab_size, 40, 3)
    outs = []
    for cuts, graphs in (((40,), False), ((17, 1, 1, 20, 1), False), ((17, 1, 1, 20, 1), True), ((1,) * 40, True)):
        runner = runner_of(path, use_graphs=graphs)
        runner.begin("a")
        at, rows = 0, []
        for n in cuts:
            logits = runner.step([StepEntry("a", ids[at : at + n], [n - 1])])
            rows.append((at + n - 1, logits[0].float().cpu()))
            at += n
        runner.check_status()
        outs.append(dict(rows))
        k, v = runner.cache.read("a", 0)
        assert k.shape == v.shape == (40, cfg.num_key_value_heads, cfg.head_dim) and k.dtype == torch.bfloat16
        outs[-1]["k"] = k.float().cpu()
        runner.end("a")
        runner.cache.check_consistency()
    scale = outs[0][39].abs().max()
    for other in outs[1:]:
        # bfloat16 products and 8-bit keys that may round the other way where sums differ in their last bits
        assert float((other[39] - outs[0][39]).abs().max()) <= 6e-2 * float(scale)
    shared = [p for p in outs[1] if p in outs[2] and p != "k"]
    assert shared and all(torch.equal(outs[1][p], outs[2][p]) or float((outs[1][p] - outs[2][p]).abs().max()) <= 2e-2 * float(scale) for p in shared)
    # the first layer's keys depend on the embeddings alone: the same codes however the sequence was cut, but for ties
    for other in outs[1:]:
        assert float((other["k"] != outs[0]["k"]).float().mean()) < 0.02


def test_logits_against_plain_implementation(folder, monkeypatch) -> None:
    from forge_engine_b200.engine import StepEntry

    path, cfg, weights = folder
    ids = random_ids(cfg.vocab_size, 37, 11)
    monkeypatch.setattr(plain, "attention", attention_of_rounded)
    want = plain.forward_logits(ids, weights, cfg).float().cpu()
    runner = runner_of(path)
    runner.begin("a")
    got = runner.step([StepEntry("a", ids[:20], list(range(20)))]).float().cpu()
    rest = [runner.step([StepEntry("a", [t], [0])]).float().cpu() for t in ids[20:]]
    runner.check_status()
    got = torch.cat([got, *rest])
    assert float((got - want).abs().max()) <= 6e-2 * float(want.abs().max())
    tv = 0.5 * (torch.softmax(got, -1) - torch.softmax(want, -1)).abs().sum(-1)
    assert float(tv.max()) <= 0.04


def test_mixed_steps_filler_entries_and_generation(folder) -> None:
    from forge_engine_b200.config import EngineConfig, SchedulerConfig
    from forge_engine_b200.engine import Engine

    path, cfg, _ = folder
    prompts = [random_ids(cfg.vocab_size, n, 70 + n) for n in (3, 19, 34)]

    def generate():
        engine = Engine.from_pretrained(path, engine_config=EngineConfig(max_new_tokens=7, cache_dtype="float8"),
                                        scheduler_config=SchedulerConfig(block_size=16, block_capacity=32, token_budget=24, chunk_size=8))
        outputs = engine.generate(prompts)
        assert engine.runner.cache.bytes_per_token() == cfg.num_hidden_layers * cfg.num_key_value_heads * 2 * (cfg.head_dim + 1)
        return outputs

    first = generate()
    assert [len(o) for o in first] == [7, 7, 7] and generate() == first


def test_trace_run_takes_the_option(folder, tmp_path) -> None:
    path, cfg, _ = folder
    steps = [{"step": 0, "entries": [{"id": "a", "tokens": random_ids(cfg.vocab_size, 9, 1), "want": [8]}]},
             {"step": 1, "entries": [{"id": "a", "tokens": [5], "want": [0]}], "end": ["a"]}]
    got = run_trace(path, tmp_path / "out", "bfloat16", 64, steps, ("--cache-dtype", "float8"))
    assert set(got) == {0, 1} and all(torch.isfinite(torch.from_numpy(v)).all() for v in got.values())


def test_a_cache_is_read_back(folder) -> None:
    """``CacheManager.read`` of both kinds of cache; positions a request does not hold are refused."""
    from forge_engine_b200.engine import ModelRunner, StepEntry

    path, cfg, _ = folder
    ids = random_ids(cfg.vocab_size, 21, 2)
    both = []
    for cache_dtype in (None, "float8"):
        runner = ModelRunner.from_folder(path, dtype="bfloat16", page_size=4, num_pages=64, max_requests=2, cache_dtype=cache_dtype)
        runner.begin("a")
        runner.step([StepEntry("a", ids, [20])])
        k, v = runner.cache.read("a", 0, first=3, count=11, dtype=torch.float32)
        assert k.shape == (11, cfg.num_key_value_heads, cfg.head_dim) and k.dtype == torch.float32
        both.append((k.cpu(), v.cpu()))
        for first, count in ((-1, 2), (20, 2), (22, None)):
            with pytest.raises(ValueError):
                runner.cache.read("a", 0, first=first, count=count)
        with pytest.raises(KeyError):
            runner.cache.read("b", 0)
    for exact, eight in zip(*both):
        want = rounded(exact.double())
        # the bfloat16 cache rounded once more on its way (2^-8): at a border that makes another code, one step off, which
        # is at most 2^-3 of the number (just above a power of two); a number is off by half a step, 2^-4, and those 2^-8
        off = float(((eight - want).abs() / exact.abs().clamp(min=1e-9)).masked_fill(exact.abs() < 2.0 ** -6 * exact.abs().max(), 0).max())
        assert off <= 2.0 ** -3 * (1 + 2.0 ** -4)
        assert float((eight - exact).abs().max() / exact.abs().max()) <= 2.0 ** -4 + 2.0 ** -8
        assert float((eight.double() - want).abs().gt(1e-6).double().mean()) < 0.2


def test_layers_without_an_8_bit_form_are_refused(folder) -> None:
    from forge_engine_b200.engine import ModelRunner
    from forge_engine_b200.errors import ConfigError
    import plain_tekilorn as pt

    path, _, _ = folder
    with pytest.raises(ConfigError):
        ModelRunner.from_folder(path, dtype="float32", page_size=16, num_pages=8, max_requests=2, cache_dtype="float8")
    with pytest.raises(ValueError):
        ModelRunner.from_folder(path, dtype="bfloat16", page_size=16, num_pages=8, max_requests=2, cache_dtype="int8")
    raw = pt.config([pt.window_layer()])
    with pytest.raises(ConfigError):
        ModelRunner.from_random(raw, 0, dtype="bfloat16", page_size=16, num_pages=8, max_requests=2, cache_dtype="float8")
