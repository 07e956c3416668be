"""The 8-bit key/value cache: what it is measured by.

Keys and values lie in pages as e4m3 numbers with one power-of-two scale (e8m0) per token, kv head
and matrix.  Four operators, by ``"kind"``:

* ``write``  - the finished projection of a step's tokens: norm per head and rotation of q and k,
               k and v quantised into their pages, q rounded to bfloat16; without heads of q and
               without a norm it is the plain writing of given keys and values.
* ``read``   - cached positions back as bfloat16 or 32-bit rows.
* ``single`` - attention of requests that bring one token (or a few) each.
* ``portion``- attention of requests that bring a portion of a prompt each, from anywhere on.

Both attentions see every earlier key, or a window and a few first tokens that stay visible.

The caches are full of other requests' tokens and a request's pages lie scattered over them.
Keys have the spread that a norm per head and its weights leave, some channels larger than others;
values differ in size from token to token.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
LARGEST = 448.0            # e4m3's largest number
LEAST, MOST = -64, 64      # bounds of a scale's exponent


def listed() -> list:
    base = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 16}
    return [
        # one user's next token: the latency of the launch that every layer has
        {"name": "write-1", "kind": "write", **base, "tokens": 1, "context": 2048, "norm": True, "dtype": "f32"},
        # a busy server's decode step: 64 requests, 32-bit sums of the projection
        {"name": "write-64", "kind": "write", **base, "tokens": 64, "context": 3001, "norm": True, "dtype": "f32"},
        # a whole prompt of a step's token budget
        {"name": "write-4096", "kind": "write", **base, "tokens": 4096, "context": 0, "norm": True, "dtype": "bf16"},
        # a short request's context copied out
        {"name": "read-700", "kind": "read", **base, "entries": 1, "context": 700, "dtype": "bf16"},
        # contexts of several requests handed to 32-bit code, heads of 64
        {"name": "read-ragged", "kind": "read", "heads": 32, "kv_heads": 4, "dim": 64, "page": 16, "entries": 9,
         "context": 8192, "dtype": "f32"},
        # one user, one long document
        {"name": "single-1x32768", "kind": "single", **base, "entries": 1, "new": 1, "context": 32768, "window": 0, "keep": 0},
        # the everyday decode step
        {"name": "single-8x2048", "kind": "single", **base, "entries": 8, "new": 1, "context": 2048, "window": 0, "keep": 0},
        # a busy server: contexts of every length, three checked tokens each, windows with kept first tokens
        {"name": "single-48-window", "kind": "single", "heads": 40, "kv_heads": 8, "dim": 128, "page": 16, "entries": 48,
         "new": 3, "context": 9001, "window": 4096, "keep": 4},
        # the last few tokens of two prompts: hardly more rows than a single token's kernel takes
        {"name": "portion-short", "kind": "portion", **base, "entries": 2, "new": 9, "context": 1500, "window": 0, "keep": 0},
        # a portion of the default token budget behind a medium context, heads of 64, a window
        {"name": "portion-window", "kind": "portion", "heads": 24, "kv_heads": 8, "dim": 64, "page": 16, "entries": 3,
         "new": 255, "context": 5000, "window": 1024, "keep": 4},
        # a whole prompt
        {"name": "portion-2048", "kind": "portion", **base, "entries": 1, "new": 2048, "context": 0, "window": 0, "keep": 0},
        # a later portion of a long document
        {"name": "portion-long", "kind": "portion", **base, "entries": 1, "new": 509, "context": 32259, "window": 0, "keep": 0},
    ]


def _log(rng, low, high) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("write", "read", "single", "portion")}
    while True:
        kind = rng.choice(("write", "read", "single", "single", "portion", "portion"))
        kv_heads = rng.choice((1, 2, 4, 8, 8, 8))
        groups = rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 16))
        case = {"kind": kind, "heads": kv_heads * groups, "kv_heads": kv_heads, "dim": rng.choice((32, 64, 64, 96, 128, 128, 128, 256)),
                "page": rng.choice((4, 8, 16, 16, 16, 32, 64))}
        if kind == "write":
            case.update(tokens=_log(rng, 1, 4096), context=rng.choice((0, _log(rng, 1, 9000))), norm=rng.random() < 0.7,
                        dtype=rng.choice(("bf16", "f32")))
            if not case["norm"]:
                case["heads"] = 0
        elif kind == "read":
            case.update(entries=_log(rng, 1, 16), context=_log(rng, 1, 16000), dtype=rng.choice(("bf16", "f32")))
        else:
            window = rng.choice((0, 0, _log(rng, 16, 8192)))
            case.update(entries=_log(rng, 1, 64) if kind == "single" else _log(rng, 1, 5),
                        new=rng.randint(1, max(1, 16 // groups)) if kind == "single" else 16 // groups + _log(rng, 1, 2000),
                        context=_log(rng, 1, 33000), window=window, keep=rng.choice((0, 1, 4, 20)) if window else 0)
        if _cost(case) <= most[kind] and _padded(case) <= 1.5e9:
            return case


# -- sizes of a case, the same for everybody ----------------------------------------------------


def _spread(case, i) -> tuple:
    """(cached, new) tokens of request ``i``: around the case's figures, each its own."""
    n, context, new = case["entries"], case["context"], case.get("new", 0)
    if n == 1:
        return context, new
    cached = max(0, context * (2 * i + 1) // (2 * n) + (i * 5) % 7 - 3) if case["kind"] != "single" or n > 8 else max(0, context - 3 * i)
    return cached, new if case["kind"] == "single" else max(16 * case["kv_heads"] // case["heads"] + 1, new - 11 * i)


def _requests(case) -> list:
    """(cached, new) per request."""
    if case["kind"] == "write":
        if case["context"] == 0:
            return [(0, case["tokens"])]                          # one prompt from its start
        return [(case["context"] + 13 * i, 1) for i in range(case["tokens"])]
    if case["kind"] == "read":
        return [(0, max(1, _spread(case, i)[0])) for i in range(case["entries"])]
    return [_spread(case, i) for i in range(case["entries"])]


def _seen(case) -> float:
    """Pairs of a query and a key it sees, over all requests."""
    total, window, keep = 0, case.get("window", 0), case.get("keep", 0)
    for cached, new in _requests(case):
        for i in range(new):
            keys = cached + i + 1
            total += keys if not window else min(keys, window) + min(keep, max(0, keys - window))
    return total


def _keys(case) -> float:
    """Cached positions that some query of the call sees."""
    total, window, keep = 0, case.get("window", 0), case.get("keep", 0)
    for cached, new in _requests(case):
        if not window or not new:
            total += cached + new
        else:
            first = max(0, cached - window + 1)
            total += cached + new - first + min(keep, first)
    return total


def work(case) -> dict:
    requests = _requests(case)
    tokens = sum(new for _, new in requests)
    cell = case["kv_heads"] * (case["dim"] + 1) * 2              # codes and scales of one position
    item = 2 if case.get("dtype") == "bf16" else 4
    q, kv = case["heads"] * case["dim"], 2 * case["kv_heads"] * case["dim"]
    if case["kind"] == "write":
        return {"bytes": tokens * ((q + kv) * item + 2 * q + cell + (4 * case["dim"] if case["norm"] else 0) + 8), "flops": 8 * tokens * (q + kv)}
    if case["kind"] == "read":
        return {"bytes": tokens * (cell + kv * item + 8), "flops": tokens * kv}
    return {"bytes": _keys(case) * cell + tokens * 2 * q * 2, "flops": 4 * _seen(case) * q}


def _cost(case) -> float:
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _padded(case) -> float:
    """Scores of the plain form, whose requests are padded to the longest."""
    if case["kind"] in ("write", "read"):
        return 0
    requests = _requests(case)
    return len(requests) * max(n for _, n in requests) * max(c + n for c, n in requests) * case["heads"]


# -- inputs ---------------------------------------------------------------------------------------


def _scales_of(x):
    """Exponent of the scale of every row of ``x`` (last axis): the least e with max |x| <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    e = exponent - 9 + (mantissa > 0.875).int()
    return torch.where(mantissa == 0, LEAST, e.clamp(LEAST, MOST))


def _quantised(x) -> tuple:
    """(codes as bytes, scales as bytes) of 32-bit rows."""
    e = _scales_of(x)
    codes = torch.ldexp(x, -e.unsqueeze(-1)).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    requests = _requests(case)
    nkv, dim, page = case["kv_heads"], case["dim"], case["page"]
    host = random.Random(seed)
    counts = [-(-(cached + new) // page) for cached, new in requests]
    pages = sum(counts) + 5
    ids = list(range(pages))
    host.shuffle(ids)
    width = max(max(counts), 1)
    rows, at = [], 0
    for count in counts:
        rows.append(ids[at : at + count] + [-1] * (width - count))
        at += count
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    draw_ = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    channel = torch.exp(0.4 * draw_(nkv, 1, dim))                 # some channels of a head are larger
    codes, scales = [], []
    for spread in (channel, torch.exp(0.5 * draw_(pages, nkv, page, 1))):
        c, s = _quantised(draw_(pages, nkv, page, dim) * spread)
        codes.append(c.view(torch.float8_e4m3fn))
        scales.append(s.view(torch.float8_e8m0fnu))
    state = {"case": dict(case), "k_cache": codes[0], "v_cache": codes[1], "k_scale": scales[0], "v_scale": scales[1],
             "block_table": ints(rows), "status": torch.zeros(1, dtype=torch.int32, device=DEVICE), "requests": requests}
    tokens = sum(n for _, n in requests)
    state["token_entry"] = ints([e for e, (_, n) in enumerate(requests) for _ in range(n)])
    state["positions"] = ints([c + i for c, n in requests for i in range(n)])
    if case["kind"] == "read":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        state["k_out"], state["v_out"] = (torch.empty((tokens, nkv, dim), dtype=dtype, device=DEVICE) for _ in range(2))
        return state
    q = case["heads"] * dim
    if case["kind"] == "write":
        rows_ = draw_(tokens, q + 2 * nkv * dim) * torch.exp(0.3 * draw_(tokens, 1)) * 2.0
        state["qkv"] = rows_.to(torch.bfloat16) if case["dtype"] == "bf16" else rows_
        state["q_out"] = torch.empty((tokens, q), dtype=torch.bfloat16, device=DEVICE)
        if case["norm"]:
            state["q_norm"], state["k_norm"] = (torch.exp(0.3 * draw_(dim)) for _ in range(2))
            inv_freq = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
            angle = state["positions"].double()[:, None] * inv_freq
            state["table"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        return state
    state["q"] = (draw_(tokens, q) * 1.5).to(torch.bfloat16)
    state["out"] = torch.zeros((tokens, q), dtype=torch.bfloat16, device=DEVICE)
    state["starts"] = ints([c for c, _ in requests])
    ends = [0]
    for _, n in requests:
        ends.append(ends[-1] + n)
    state["cu_tokens"] = ints(ends)
    state["offset"] = ints([i for _, n in requests for i in range(n)])
    state["max_new"] = max(n for _, n in requests)
    return state


# -- one pass ---------------------------------------------------------------------------------------


def run(state):
    return {"write": _write, "read": _read, "single": _attend, "portion": _attend}[state["case"]["kind"]](state)


def _caches(s) -> tuple:
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _write(s):
    c = s["case"]
    q_width, kv_width = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
    q, k, v = s["qkv"].split((q_width, kv_width, kv_width), dim=1)
    if own:
        from forge_engine_b200.ops import native

        native.kv8_write(k, v, s["positions"], s["token_entry"], *_caches(s), s["block_table"], s["status"],
                         q=q if q_width else None, q_out=s["q_out"] if q_width else None, q_norm=s.get("q_norm"),
                         k_norm=s.get("k_norm"), eps=EPS, table=s.get("table"))
        return [s["q_out"], *_caches(s)]
    rows = lambda x: x.float().unflatten(1, (-1, c["dim"]))  # noqa: E731
    q, k, v = rows(q) if q_width else None, rows(k), rows(v)
    if c["norm"]:
        cos, sin = s["table"][:, None, :, 0], s["table"][:, None, :, 1]

        def finished(x, weight):
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
            a, b = x.chunk(2, dim=-1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        q, k = finished(q, s["q_norm"]), finished(k, s["k_norm"])
    if q_width:
        s["q_out"].copy_(q.flatten(1))
    at = s["positions"].long()
    page, slot = s["block_table"][s["token_entry"].long(), at // c["page"]].long(), at % c["page"]
    for x, cache, scale in ((k, s["k_cache"], s["k_scale"]), (v, s["v_cache"], s["v_scale"])):
        codes, exponents = _quantised(x)
        cache.view(torch.uint8)[page, :, slot] = codes
        scale.view(torch.uint8)[page, :, slot] = exponents
    return [s["q_out"], *_caches(s)]


def _read(s):
    c = s["case"]
    if own:
        from forge_engine_b200.ops import native

        native.kv8_read(*_caches(s), s["block_table"], s["positions"], s["token_entry"], s["k_out"], s["v_out"], s["status"])
        return [s["k_out"], s["v_out"]]
    at = s["positions"].long()
    page, slot = s["block_table"][s["token_entry"].long(), at // c["page"]].long(), at % c["page"]
    for cache, scale, out in ((s["k_cache"], s["k_scale"], s["k_out"]), (s["v_cache"], s["v_scale"], s["v_out"])):
        codes, exponents = cache.view(torch.uint8)[page, :, slot], scale.view(torch.uint8)[page, :, slot]
        out.copy_(codes.view(torch.float8_e4m3fn).float() * exponents.view(torch.float8_e8m0fnu).float().unsqueeze(-1))
    return [s["k_out"], s["v_out"]]


def _attend(s):
    c = s["case"]
    if own:
        from forge_engine_b200.ops import native

        plan = native.kv8_plan(s["requests"], c["heads"], c["kv_heads"], c["dim"], c["window"], c["keep"])
        native.attention_kv8(s["q"], *_caches(s), s["block_table"], s["cu_tokens"], s["starts"], len(s["requests"]), s["max_new"],
                             c["heads"], c["window"], c["keep"], c["dim"] ** -0.5, s["out"], s["status"], plan)
        return s["out"]
    entries, new, nkv, dim = len(s["requests"]), s["max_new"], c["kv_heads"], c["dim"]
    groups = c["heads"] // nkv
    entry, offset = s["token_entry"].long(), s["offset"].long()
    table = s["block_table"].long().clamp(min=0)

    def keys(cache, scale):
        x = cache.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
        x = x * scale.view(torch.uint8)[table].view(torch.float8_e8m0fnu).float().unsqueeze(-1)
        return x.transpose(1, 2).flatten(2, 3)                       # [entries, kv heads, positions, dim]

    q = torch.zeros((entries, new, nkv, groups, dim), device=DEVICE)
    q[entry, offset] = s["q"].float().view(-1, nkv, groups, dim)
    scores = q.permute(0, 2, 3, 1, 4).flatten(2, 3) @ keys(s["k_cache"], s["k_scale"]).transpose(2, 3)
    scores = scores.unflatten(2, (groups, new)) * dim ** -0.5
    pos = s["starts"].long()[:, None] + torch.arange(new, device=DEVICE)
    key = torch.arange(scores.shape[-1], device=DEVICE)
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= (pos[..., None] - key < c["window"]) | (key < c["keep"])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    weights /= weights.sum(-1, keepdim=True)
    out = weights.flatten(2, 3) @ keys(s["v_cache"], s["v_scale"])
    out = out.unflatten(2, (groups, new)).permute(0, 3, 1, 2, 4)[entry, offset]
    s["out"].copy_(out.flatten(1))
    return s["out"]


# -- the same in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["kind"] == "write":
        return _exact_write(case, s)

    def values(cache, scale, row, length):
        ids = s["block_table"][row, : -(-length // page)].long()
        x = cache.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        x = x * torch.exp2(scale.view(torch.uint8)[ids].double() - 127.0)[..., None]
        return x.permute(0, 2, 1, 3).reshape(-1, case["kv_heads"], case["dim"])[:length]      # [positions, kv heads, dim]

    if case["kind"] == "read":
        return [torch.cat([values(s[a], s[b], row, n) for row, (_, n) in enumerate(s["requests"])])
                for a, b in (("k_cache", "k_scale"), ("v_cache", "v_scale"))]
    groups = case["heads"] // case["kv_heads"]
    outs, at = [], 0
    for row, (cached, new) in enumerate(s["requests"]):
        length = cached + new
        k, v = (values(s[a], s[b], row, length) for a, b in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
        q = s["q"][at : at + new].double().view(new, case["heads"], case["dim"])
        at += new
        distance = torch.arange(cached, length, device=DEVICE)[:, None] - torch.arange(length, device=DEVICE)[None, :]
        hidden = distance < 0
        if case["window"]:
            kept = torch.arange(length, device=DEVICE)[None, :] < case["keep"]
            hidden = hidden | ((distance >= case["window"]) & ~kept)
        heads = []
        for h in range(case["heads"]):
            t = torch.einsum("nd,ld->nl", q[:, h], k[:, h // groups]) / math.sqrt(case["dim"])
            t = t.masked_fill(hidden, -math.inf)
            heads.append(torch.softmax(t, dim=1) @ v[:, h // groups])
        outs.append(torch.stack(heads, 1).reshape(new, -1))
    return torch.cat(outs)


def _exact_write(case, s):
    """Codes and scales as the numbers they are; what the call does not write keeps its place."""
    dim, nkv, nq, page = case["dim"], case["kv_heads"], case["heads"], case["page"]
    x = s["qkv"].double().view(-1, nq + 2 * nkv, dim)
    q, k, v = x[:, :nq], x[:, nq : nq + nkv], x[:, nq + nkv :]
    if case["norm"]:
        c, n = s["table"][..., 0].double()[:, None], s["table"][..., 1].double()[:, None]
        turned = []
        for y, weight in ((q, s["q_norm"]), (k, s["k_norm"])):
            y = y / (y.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.double()
            first, second = y[..., : dim // 2], y[..., dim // 2 :]
            turned.append(torch.cat((first * c - second * n, second * c + first * n), -1))
        q, k = turned
    where = s["block_table"][s["token_entry"].long(), torch.div(s["positions"], page, rounding_mode="floor").long()].long()
    slot = s["positions"].long() % page
    result = [q.flatten(1)]
    codes_scales = []
    for y, cache, scale in ((k, "k_cache", "k_scale"), (v, "v_cache", "v_scale")):
        top = y.abs().amax(-1)
        e = torch.where(top > 0, torch.ceil(torch.log2(top / LARGEST)), torch.full_like(top, LEAST))
        e = torch.where(top > LARGEST * torch.exp2(e), e + 1, e)
        e = torch.where((top > 0) & (top <= LARGEST * torch.exp2(e - 1)), e - 1, e).clamp(LEAST, MOST)
        z = y / torch.exp2(e)[..., None]
        # e4m3: four significant bits, steps of 2^-9 below 2^-6, ties to even
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        z = (torch.round(z / step) * step).clamp(-LARGEST, LARGEST)
        all_codes = s[cache].view(torch.uint8).view(torch.float8_e4m3fn).double()
        all_scales = torch.exp2(s[scale].view(torch.uint8).double() - 127.0)
        all_codes[where, :, slot] = z
        all_scales[where, :, slot] = torch.exp2(e)
        codes_scales.append((all_codes, all_scales))
    (kc, ks), (vc, vs) = codes_scales
    return result + [kc, vc, ks, vs]
