"""The engine over an 8-bit cache where its kernels cut: contexts of thousands of tokens, heads of 64 and 128, captured steps
with fillers, and layers that are rotated in part, not normalised or read another layer's cache.  Bounds:
``test_gpu_kv8_engine.py``."""

from __future__ import annotations

import pytest
import torch

import plain_qwen3 as plain
from helpers import make_model_folder, random_ids
from test_gpu_kv8_engine import attention_of_rounded, rounded

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E128 = dict(plain.TINY_E, num_attention_heads=8, head_dim=128, use_sliding_window=False, sliding_window=None)
CONFIGS = {"heads of 64, a window": plain.TINY_E, "heads of 128": E128, "heads of 96": dict(E128, head_dim=96)}
CONTEXT = 2300


@pytest.fixture(scope="module", params=sorted(CONFIGS))
def folder(request, tmp_path_factory):
    raw = dict(CONFIGS[request.param], eos_token_id=None)
    path = tmp_path_factory.mktemp("kv8long") / "model"
    cfg, weights = make_model_folder(path, raw, 9)
    ids = random_ids(cfg.vocab_size, CONTEXT, 3)
    kept, plain.attention = plain.attention, attention_of_rounded
    try:
        want = plain.forward_logits(ids, weights, cfg).float().cpu()
    finally:
        plain.attention = kept
    return path, cfg, ids, want


@pytest.fixture
def plans(monkeypatch):
    """The plans that the steps of a test make."""
    from forge_engine_b200.ops import native

    made, real = [], native.kv8_plan

    def plan(*args):
        made.append(real(*args))
        return made[-1]

    monkeypatch.setattr(native, "kv8_plan", plan)
    return made


def runner_of(path, graphs: bool, capture_after: int = 0):
    from forge_engine_b200.engine import ModelRunner

    runner = ModelRunner.from_folder(path, dtype="bfloat16", page_size=16, num_pages=400, max_requests=4, cache_dtype="float8", use_graphs=graphs)
    runner.graphs.capture_after = capture_after
    return runner


def assert_near(got: torch.Tensor, want: torch.Tensor) -> None:
    assert float((got - want).abs().max()) <= 6e-2 * float(want.abs().max())
    tv = 0.5 * (torch.softmax(got, -1) - torch.softmax(want, -1)).abs().sum(-1)
    assert float(tv.max()) <= 0.04


def test_long_contexts_cut_and_replayed(folder, plans) -> None:
    """A prompt in two large portions, a small one, then single tokens: eager steps and replayed ones against the plain
    model, with cut entries, the workspace in the graph, and one captured step for many lengths."""
    from forge_engine_b200.engine import StepEntry

    path, cfg, ids, want = folder
    cuts = (1500, 700, 60) + (1,) * (CONTEXT - 2260)
    both = []
    for graphs in (False, True):
        runner = runner_of(path, graphs)
        plans.clear()
        runner.begin("a")
        at, rows = 0, {}
        for n in cuts:
            logits = runner.step([StepEntry("a", ids[at : at + n], [n - 1])])
            at += n
            rows[at - 1] = logits[0].float().cpu()
        runner.check_status()
        assert any(p[1] > 1 for p in plans) and any(p[5] > 1 for p in plans)          # cut single tokens, cut portions
        if graphs:
            assert 2 <= len(runner.graphs.captured) <= 4                # the small portion, single tokens under a plan or two
        both.append(torch.stack([rows[p] for p in sorted(rows)]))
        places = sorted(rows)
        runner.end("a")
        runner.cache.check_consistency()
    for got in both:
        assert_near(got, want[places])
    assert float((both[0] - both[1]).abs().max()) <= 2e-2 * float(both[0].abs().max())


def test_captured_steps_with_fillers(folder, plans) -> None:
    """Mixed steps replayed with a filler entry: of a kind the plan has, of one it has not, and with more row tiles than the plan
    counted; the same logits as eager steps, and nothing is told."""
    from forge_engine_b200.engine import StepEntry

    path, cfg, ids, want = folder
    # (tokens of a, of b, of c) per step; b and c follow their own parts of a's sequence from the start
    steps = [(1, 70, 0), (1, 0, 0), (1, 70, 2), (1, 2, 0), (2, 3, 1), (1, 100, 100), (1, 1, 1), (1, 9, 0)]
    both = []
    for graphs in (False, True):
        runner = runner_of(path, graphs)
        at = {"a": 1900, "b": 0, "c": 0}
        for key in at:
            runner.begin(key)
        runner.step([StepEntry("a", ids[:1900])])
        rows = []
        for counts in steps:
            entries = []
            for key, n in zip("abc", counts):
                if n:
                    entries.append(StepEntry(key, ids[at[key] : at[key] + n], [n - 1]))
                    at[key] += n
            logits = runner.step(entries).float().cpu()
            rows.extend((at[e.key] - 1, logits[i]) for i, e in enumerate(entries))
            runner.check_status()
        if graphs:
            assert len(runner.graphs.captured) >= 6
        both.append(torch.stack([row for _, row in rows]))
        places = [p for p, _ in rows]
        for key in at:
            runner.end(key)
        runner.cache.check_consistency()
    for got in both:
        assert_near(got, want[places])
    assert float((both[0] - both[1]).abs().max()) <= 2e-2 * float(both[0].abs().max())


HIDDEN, HEADS, NKV, DIM, ROT, VOCAB, EPS, THETA, SCALE = 96, 8, 2, 64, 24, 131, 1e-5, 1e4, 0.11


def mixed_model(seed: int) -> tuple:
    """(spec, weights): a layer rotated in its first 24 elements without a norm, one normalised and not rotated in a window, the
    first again over the first's cache, and the second again over a cache of its own."""
    from forge_engine_b200.config import AttentionSpec, GatedMLPSpec, LayerSpec, ModelSpec, NormSpec, RotarySpec, RunSpec
    from forge_engine_b200.config.specs import NoPositionSpec
    from forge_engine_b200.models import expected_tensors
    from forge_engine_b200.weights import random_tensors

    norm, ffn = NormSpec(HIDDEN, EPS), GatedMLPSpec(HIDDEN, 104)
    mixers = (AttentionSpec(HIDDEN, HEADS, NKV, DIM, False, EPS, False, SCALE, RotarySpec(DIM, THETA, ROT), None),
              AttentionSpec(HIDDEN, HEADS, NKV, DIM, True, EPS, True, SCALE, NoPositionSpec(), 200))

    def names(i):
        return {"input_norm": f"l{i}.n1", "mixer": f"l{i}.mix", "post_norm": f"l{i}.n2", "ffn": f"l{i}.ffn"}

    layers = tuple(LayerSpec(norm, mixer, norm, ffn, names(i)) for i, mixer in enumerate(mixers))
    schedule = (RunSpec(0), RunSpec(1), RunSpec(0, cache_of=0), RunSpec(1))
    spec = ModelSpec(VOCAB, HIDDEN, layers, schedule, norm, True, 4096, (), "emb.weight", "fnorm", "head.weight")
    return spec, {name: t.to(torch.bfloat16) for name, t in random_tensors(expected_tensors(spec), seed=seed, std=0.1).items()}


def mixed_plain(ids, w) -> torch.Tensor:
    n = len(ids)
    h = w["emb.weight"][torch.tensor(ids)]
    angle = torch.arange(n).float()[:, None] * (1.0 / THETA ** (torch.arange(0, ROT, 2).float() / ROT))
    cosine, sine = angle.cos()[:, None], angle.sin()[:, None]

    def rotated(x):
        a, b = x[..., : ROT // 2], x[..., ROT // 2 : ROT]
        return torch.cat((a * cosine - b * sine, b * cosine + a * sine, x[..., ROT:]), -1)

    def heads(x, p, name, count):
        y = x @ w[f"{p}.{name}.weight"].t()
        return (y + w[f"{p}.{name}.bias"] if f"{p}.{name}.bias" in w else y).view(n, count, DIM)

    def attention(x, layer, source):
        p = f"l{layer}.mix"
        q, k, v = heads(x, p, "q_proj", HEADS), heads(source, p, "k_proj", NKV), heads(source, p, "v_proj", NKV)
        if layer == 0:
            q, k = rotated(q), rotated(k)
        else:
            q, k = plain.rms_norm(q, w[p + ".q_norm.weight"], EPS), plain.rms_norm(k, w[p + ".k_norm.weight"], EPS)
        k, v = (rounded(t).repeat_interleave(HEADS // NKV, 1) for t in (k, v))
        s = torch.einsum("thd,shd->hts", q, k) * SCALE + plain.causal_mask(n, torch.float32, None if layer == 0 else 200)
        o = torch.einsum("hts,shd->thd", torch.softmax(s, -1), v).reshape(n, HEADS * DIM)
        y = o @ w[p + ".o_proj.weight"].t()
        return y + w[p + ".o_proj.bias"] if p + ".o_proj.bias" in w else y

    first = None
    for run, layer in enumerate((0, 1, 0, 1)):
        x = plain.rms_norm(h, w[f"l{layer}.n1.weight"], EPS)
        first = x if run == 0 else first
        h = h + attention(x, layer, first if run == 2 else x)
        h = h + plain.feed_forward(plain.rms_norm(h, w[f"l{layer}.n2.weight"], EPS), w, f"l{layer}.ffn")
    return plain.rms_norm(h, w["fnorm.weight"], EPS) @ w["emb.weight"].t()


@pytest.mark.parametrize("graphs", [False, True])
def test_shared_caches_partial_rotation_and_layers_without_a_norm(graphs) -> None:
    from forge_engine_b200.engine import ModelRunner, StepEntry

    spec, weights = mixed_model(4)
    runner = ModelRunner.from_tensors(spec, {k: v.to(DEV) for k, v in weights.items()}, dtype="bfloat16", device=DEV, page_size=16, num_pages=100,
                                      max_requests=2, cache_dtype="float8", use_graphs=graphs)
    runner.graphs.capture_after = 0
    assert [g.units for g in runner.cache.groups] == [[0], [1, 3]]
    assert runner.cache.view(2).scales[0].data_ptr() == runner.cache.view(0).scales[0].data_ptr() and not runner.cache.view(2).owns
    ids = random_ids(VOCAB, 700, 6)
    want = mixed_plain(ids, {k: v.float() for k, v in weights.items()})
    for key in "ab":
        runner.begin(key)
    at, rows, places = 0, [], []
    for n in (600, 50, 20, 3) + (1,) * 27:
        entries = [StepEntry("a", ids[at : at + n], [n - 1])]
        if n < 600 and at + n - 650 < 60 and at >= 650:
            entries.append(StepEntry("b", ids[at - 650 : at + n - 650], [n - 1]))
        logits = runner.step(entries).float().cpu()
        rows.append(logits)
        places.append(at + n - 1)
        if len(entries) > 1:
            places.append(at + n - 651)
        at += n
    runner.check_status()
    assert at == 700 and (not graphs or runner.graphs.captured)
    assert_near(torch.cat(rows), want[places])
    for run in (0, 2):
        k, v = runner.cache.read("a", run)
        assert k.shape == v.shape == (700, NKV, DIM)
    runner.end("a"), runner.end("b")
    runner.cache.check_consistency()
