"""Operator cases: what a long decode loop does with its paged cache besides the attention itself.

"axes" is the append of new tokens whose rotary positions are given, one for each axis (time, height and width of an image's
patches), "weights" the attention of one new token a sequence that adds each cached token's attention weight to a running
sum, and "evict" the eviction of the tokens of smallest sums from sequences that have outgrown their budget.  Where
``own`` is false they are computed in elementary torch operations in 32 bits, else by the framework's kernels.
Activations are random with a few outlier channels, pages lie in the pool in random order, and the pages' unused slots hold
stale values.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

THETA = 1e6
E4M3_MAX = 448.0
SMALLEST = 2.0 ** -126
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
# query heads, key / value heads, head dimension, rotated part of it
HEADS = {"mixtral": (32, 8, 128, 128), "olmoe": (16, 16, 128, 128), "a3b": (16, 2, 256, 64), "a3b_4kv": (32, 4, 128, 128),
         "small": (14, 2, 64, 64), "one_kv": (20, 1, 128, 128)}
# the pairs of each axis, by their number
SECTIONS = {(64, 3): (24, 20, 20), (64, 2): (32, 32), (64, 1): (64,), (32, 3): (11, 11, 10), (32, 2): (20, 12), (32, 1): (32,)}
IMAGE = 24  # patches in an image's row


def _axes(name, heads, batch, new, context, dtype, cache, page, axes, interleaved):
    return {"name": name, "kind": "axes", "heads": heads, "batch": batch, "new": new, "context": context, "dtype": dtype,
            "cache": cache, "page": page, "axes": axes, "interleaved": interleaved}


def _weights(name, heads, batch, shortest, longest, dtype, cache, page, window=0, idle=0):
    return {"name": name, "kind": "weights", "heads": heads, "batch": batch, "shortest": shortest, "longest": longest,
            "dtype": dtype, "cache": cache, "page": page, "window": window, "idle": idle}


def _evict(name, heads, batch, shortest, longest, cache, page, budget, limit, sink, recent):
    return {"name": name, "kind": "evict", "heads": heads, "batch": batch, "shortest": shortest, "longest": longest,
            "cache": cache, "page": page, "budget": budget, "limit": limit, "sink": sink, "recent": recent}


def listed():
    return [
        # a serving batch's decode step behind prompts with images: one token a sequence
        _axes("axes_decode_b16", "mixtral", 16, 1, 2000, "fp16", "fp16", 16, 3, True),
        # prompts with images of different lengths in one batch, onto an empty cache
        _axes("axes_prompts_t8192", "mixtral", 8, 1024, 0, "bf16", "bf16", 64, 3, False),
        # a prompt's next chunk into an 8-bit cache, heads of which a quarter is rotated
        _axes("axes_chunk_e4m3", "a3b", 3, 683, 1500, "fp16", "e4m3", 32, 3, True),
        # one user's chat: a cache of a thousand tokens
        _weights("weights_b1_1k", "mixtral", 1, 1000, 1000, "bf16", "bf16", 16),
        # a serving batch whose sequences' lengths differ by a factor of hundreds, two of its places idle
        _weights("weights_b16_ragged", "mixtral", 16, 20, 8000, "fp16", "fp16", 16, idle=2),
        # one long document, before its first eviction
        _weights("weights_b1_128k", "a3b_4kv", 1, 131072, 131072, "bf16", "bf16", 64),
        # a full serving batch on an 8-bit cache
        _weights("weights_b64_8k_e4m3", "mixtral", 64, 4000, 8192, "bf16", "e4m3", 32),
        # wide heads, pages that no tile divides
        _weights("weights_b8_wide", "a3b", 8, 1000, 16000, "bf16", "bf16", 20),
        # one user's chat, a step in which nothing is due
        _evict("evict_b1_none", "mixtral", 1, 2100, 2100, "bf16", 16, 2048, 2176, 4, 256),
        # a serving batch at its limit: a stretch of the oldest unused tokens leaves each sequence
        _evict("evict_b16_slack", "mixtral", 16, 4225, 4225, "fp16", 16, 4096, 4224, 4, 512),
        # one long document after its prompt
        _evict("evict_b1_128k", "a3b_4kv", 1, 131072, 131072, "bf16", 64, 16384, 16384, 64, 1000),
        # a full batch of prompts of different lengths on an 8-bit cache, some of them still short enough
        _evict("evict_b32_e4m3", "mixtral", 32, 1500, 8192, "e4m3", 32, 2048, 2048, 16, 500),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    kind = rng.choice(("axes", "axes", "weights", "weights", "weights", "evict", "evict", "evict"))
    dtype = rng.choice(("fp16", "bf16"))
    heads = rng.choice(sorted(HEADS))
    cache = rng.choice((dtype, dtype, "e4m3"))
    page = rng.choice((16, 16, 32, 64, 128, 256, rng.randint(1, 100)))
    q_heads, kv_heads, dim, _ = HEADS[heads]
    batch = spread(1, 64)
    size = DTYPES[cache].itemsize
    if kind == "axes":
        most = 8192 * 48 * 128 // ((q_heads + 2 * kv_heads) * dim * batch)
        new = 1 if rng.random() < 0.4 else min(spread(1, 4096), most)
        case = _axes("", heads, batch, new, rng.choice((0, spread(1, 4000))), dtype, cache, page, rng.choice((1, 2, 3, 3)),
                     rng.random() < 0.5)
    elif kind == "weights":
        most = min(64 * 8192 * 8 * 128 // max(q_heads // 4, kv_heads), 380_000_000 // (kv_heads * size)) // (dim * batch)
        longest = min(spread(1, 131072), most)
        shortest = spread(1, longest)
        window = spread(16, longest) if longest > 64 and rng.random() < 0.25 else 0
        idle = rng.randint(1, batch - 1) // 4 if batch > 1 else 0
        case = _weights("", heads, batch, shortest, longest, dtype, cache, page, window, idle)
    else:
        most = 260_000_000 // (kv_heads * size * dim * batch)
        longest = min(spread(1, 131072), most)
        budget = min(spread(1, longest), 16384, 60_000_000 // (kv_heads * size * dim * batch))
        limit = budget + rng.choice((0, 0, spread(1, 256)))
        sink = min(rng.choice((0, 4, 64)), budget // 2)
        recent = rng.randint(0, budget - sink) if rng.random() < 0.8 else 0
        case = _evict("", heads, batch, spread(1, longest), longest, cache, page, budget, limit, sink, recent)
    del case["name"]
    return case


# -------------------------------------------------------------------------------------------------- inputs


def _lengths(case):
    """Each sequence's length: from the shortest to the longest, spread evenly over their logarithm, and the idle ones."""
    idle = case.get("idle", 0)
    lo, hi, count = case["shortest"], case["longest"], case["batch"] - idle
    if count == 1:
        return [hi] + [0] * idle
    return [int(round(lo * (hi / lo) ** (i / (count - 1)))) for i in range(count)] + [0] * idle


def _new_tokens(case):
    """Each sequence's new tokens: case["new"] on average, one for a decode step."""
    mean, count = case["new"], case["batch"]
    return [mean if mean == 1 else max(1, mean - mean // 2 + (i * (mean // 2 * 2)) // max(1, count - 1) if count > 1 else mean)
            for i in range(count)]


def _channels(gen, dim, outliers=4, scale=6.0):
    """A factor for each channel: near one, a few large ones."""
    f = torch.exp(0.3 * torch.randn(dim, generator=gen, device="cuda"))
    f[torch.randperm(dim, generator=gen, device="cuda")[:outliers]] *= scale
    return f


def _tables(dim, positions):
    """cos and sin of position * theta^(-2i/dim), in 64 bits before they are rounded."""
    freq = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq[None]
    return angle.cos().float(), angle.sin().float()


def _pool(gen, pages, heads, page, dim, dtype, keys):
    """A cache's values: (the pool, its scales or None)."""
    factor = _channels(gen, dim, scale=2.0) if keys else torch.ones(dim, device="cuda")
    out = torch.empty((pages, heads, page, dim), dtype=dtype, device="cuda")
    scales = torch.empty((pages, heads, page), device="cuda") if dtype == torch.float8_e4m3fn else None
    step = max(1, (64 << 20) // (heads * page * dim))
    for i in range(0, pages, step):
        x = torch.randn((min(step, pages - i), heads, page, dim), generator=gen, device="cuda") * factor
        if scales is not None:
            s = x.abs().amax(-1) / E4M3_MAX
            scales[i: i + step] = s
            x = x / s[..., None]
        out[i: i + step] = x.to(dtype)
    return out, scales


def _image_positions(case, gen, new, before, starts, tokens):
    """The new tokens' positions on each axis, [axes, tokens]: of a prompt the first two thirds are an image, whose patches
    share their time and have rows and columns, and the rest is text, one position a token on every axis.  A decode
    step's token continues past its cache's places."""
    first = before + torch.randint(0, 100, before.shape, generator=gen, device="cuda")
    if starts is None:
        return first.expand(case["axes"], -1).to(torch.int32).contiguous()
    t = torch.arange(tokens, device="cuda")
    seq = (t[:, None] >= starts[None, 1:]).sum(1)
    i, image = t - starts[seq], new[seq] * 2 // 3
    text = torch.maximum(image // IMAGE, torch.full_like(image, IMAGE)) + i - image
    rows = [torch.where(i < image, x, text) + first[seq] for x in (torch.zeros_like(i), i // IMAGE, i % IMAGE)]
    return torch.stack(rows[: case["axes"]]).to(torch.int32)


def _sums(gen, case, lengths, heads, positions):
    """Attention weights summed over some steps: a few tokens have most, many very little, some none at all; zeros past the
    sequence."""
    shape = (len(lengths), heads, positions)
    w = 0.002 * torch.exp(2.0 * torch.randn(shape, generator=gen, device="cuda"))
    w.masked_fill_(torch.rand(shape, generator=gen, device="cuda") < 0.05, 0.0)
    return w.masked_fill_(torch.arange(positions, device="cuda") >= lengths[:, None, None], 0.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    q_heads, kv_heads, dim, rot = HEADS[case["heads"]]
    cache, page, batch = DTYPES[case["cache"]], case["page"], case["batch"]
    if case["kind"] == "axes":
        new = torch.tensor(_new_tokens(case), device="cuda")
        new = new[torch.randperm(batch, generator=gen, device="cuda")]
        before = torch.randint(case["context"] // 2, case["context"] + 1, (batch,), generator=gen, device="cuda")
        lengths, most = before + new, case["context"] + max(_new_tokens(case))
    else:
        lengths = torch.tensor(_lengths(case), device="cuda")
        lengths, most = lengths[torch.randperm(batch, generator=gen, device="cuda")], case["longest"]
    if case["kind"] == "evict":
        most = max(most, case["budget"])
    per = -(-most // page)
    pages = batch * per + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[: batch * per].reshape(batch, per).to(torch.int32)
    state = {"kind": case["kind"], "table": table, "lengths": lengths.to(torch.int32), "page": page}
    state["k_cache"], state["k_scale"] = _pool(gen, pages, kv_heads, page, dim, cache, True)
    state["v_cache"], state["v_scale"] = _pool(gen, pages, kv_heads, page, dim, cache, False)
    if case["kind"] != "axes":
        state["sums"] = _sums(gen, case, lengths, kv_heads, per * page)
    if case["kind"] == "evict":
        state["sums_now"] = torch.empty_like(state["sums"])
        return state | {name: case[name] for name in ("budget", "limit", "sink", "recent")}
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "weights":
        state["q"] = (randn(batch, q_heads, dim) * _channels(gen, dim, scale=2.0)).to(dtype)
        state["window"] = case["window"]
        return state
    tokens = sum(_new_tokens(case))
    state["q"] = (randn(tokens, q_heads, dim) * _channels(gen, dim)).to(dtype)
    state["k"] = (randn(tokens, kv_heads, dim) * _channels(gen, dim)).to(dtype)
    state["v"] = randn(tokens, kv_heads, dim).to(dtype)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    state["starts"] = starts.to(torch.int32) if case["new"] > 1 else None
    state["positions"] = _image_positions(case, gen, new, before, starts if case["new"] > 1 else None, tokens)
    state["cos"], state["sin"] = _tables(rot, most + 200)
    state["sections"], state["interleaved"] = SECTIONS[rot // 2, case["axes"]], case["interleaved"]
    return state


# -------------------------------------------------------------------------------------------------- passes


def _places(s, tokens):
    """Each token's page and slot."""
    t = torch.arange(tokens, device="cuda")
    lengths = s["lengths"].long()
    if s["starts"] is None:
        seq, pos = t, lengths - 1
    else:
        starts = s["starts"].long()
        seq = (t[:, None] >= starts[None, 1:]).sum(1)
        pos = lengths[seq] - (starts[seq + 1] - t)
    return s["table"][seq, pos // s["page"]].long(), pos % s["page"]


def _pair_axes(sections, interleaved, half):
    """Each pair's axis: its section's, or in turn while an axis has pairs left, then the first."""
    i, axes = torch.arange(half, device="cuda"), len(sections)
    most = torch.tensor(sections, device="cuda")
    if interleaved:
        return torch.where(i < axes * most[i % axes], i % axes, torch.zeros_like(i))
    return (i[:, None] >= most.cumsum(0)[None]).sum(1)


def _rotated(x, cos, sin):
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = x[..., :half], x[..., half: 2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _plain_axes(s):
    page, slot = _places(s, s["q"].shape[0])
    half = s["cos"].shape[1]
    at = s["positions"].long()[_pair_axes(s["sections"], s["interleaved"], half)].T  # [tokens, pairs]
    pair = torch.arange(half, device="cuda")
    cos, sin = s["cos"][at, pair], s["sin"][at, pair]
    q = _rotated(s["q"].float(), cos, sin).to(s["q"].dtype)
    for x, cache, scale in ((_rotated(s["k"].float(), cos, sin), s["k_cache"], s["k_scale"]),
                            (s["v"].float(), s["v_cache"], s["v_scale"])):
        if scale is not None:
            f = (x.abs().amax(-1) / E4M3_MAX).clamp_min(SMALLEST)
            scale[page, :, slot] = f
            x = x / f[..., None]
        cache[page, :, slot] = x.to(cache.dtype)
    return {"q": q} | _cache(s)


def _cache(s):
    return {name: s[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale") if s[name] is not None}


def _gathered(cache, scale, table, mask):
    """A cache's values of every sequence, [batch, heads, length, dim] in 32 bits, zeros where the mask is false."""
    x = cache[table].float()
    if scale is not None:
        x = x * scale[table][..., None]
    batch, pages, heads, page, dim = x.shape
    x = x.permute(0, 2, 1, 3, 4).reshape(batch, heads, pages * page, dim)
    return x.masked_fill_(~mask[:, None, :, None], 0.0)


def _plain_weights(s):
    q, table, lengths = s["q"].float(), s["table"].long(), s["lengths"].long()
    batch, q_heads, dim = q.shape
    kv_heads = s["k_cache"].shape[1]
    j = torch.arange(table.shape[1] * s["page"], device="cuda")[None]
    mask = j < lengths[:, None]
    if s["window"]:
        mask &= j >= lengths[:, None] - s["window"]
    q = q.reshape(batch, kv_heads, q_heads // kv_heads, dim) * dim ** -0.5
    k = _gathered(s["k_cache"], s["k_scale"], table, mask)
    score = torch.matmul(q, k.transpose(2, 3)).masked_fill_(~mask[:, None, None], -math.inf)
    del k
    p = torch.exp(score - score.amax(-1, keepdim=True)).masked_fill_(~mask[:, None, None], 0.0)
    p /= p.sum(-1, keepdim=True).masked_fill_((lengths == 0)[:, None, None, None], 1.0)  # an idle place attends to nothing
    s["sums"] += p.sum(2)
    v = _gathered(s["v_cache"], s["v_scale"], table, mask)
    return torch.matmul(p, v).reshape(batch, q_heads, dim).to(s["q"].dtype), s["sums"]


def _plain_evict(s):
    sums, lengths, budget, page = s["sums_now"], s["lengths"].long(), s["budget"], s["page"]
    sums.copy_(s["sums"])
    batch, heads, positions = sums.shape
    j = torch.arange(positions, device="cuda")
    n = lengths[:, None, None]
    due = n > s["limit"]
    held = (j < s["sink"]) | (j >= n - s["recent"])
    order = sums.masked_fill(held, math.inf).masked_fill_(j >= n, -math.inf).sort(stable=True, dim=-1, descending=True).indices
    place = j[:budget]
    kept = torch.where(due, order[..., :budget].sort(-1).values, place)
    b, h = torch.arange(batch, device="cuda")[:, None, None], torch.arange(heads, device="cuda")[:, None]
    table = s["table"].long()
    src, dst = table[b, kept // page], table[b, place // page]
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if s[name] is not None:
            rows = s[name][src, h, kept % page]
            s[name][dst, h, place % page] = rows
    moved = torch.cat([sums.gather(2, kept), sums.new_zeros((batch, heads, positions - budget))], 2)
    sums.copy_(torch.where(due, moved, sums))
    left = torch.where(due[:, 0, 0], budget, lengths).to(torch.int32)
    return {"lengths": left, "kept": torch.where(due, kept, -1).to(torch.int32), "sums": sums} | _cache(s)


@functools.lru_cache(None)
def _framework():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neurips26-tris-moe_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from tris_moe_amd import ext

    return ext


def _own(s):
    ext = _framework()
    if s["kind"] == "axes":
        q = ext.rotary_append_paged(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["table"],
                                    s["lengths"], query_start=s["starts"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                    positions=s["positions"], sections=s["sections"], interleaved=s["interleaved"])
        return {"q": q} | _cache(s)
    if s["kind"] == "weights":
        y = ext.paged_attention_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], window=s["window"],
                                       k_scale=s["k_scale"], v_scale=s["v_scale"], weight_sum=s["sums"])
        return y, s["sums"]
    s["sums_now"].copy_(s["sums"])
    left, kept = ext.paged_cache_evict(s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["sums_now"], s["budget"],
                                       limit=s["limit"], sink=s["sink"], recent=s["recent"], k_scale=s["k_scale"],
                                       v_scale=s["v_scale"])
    return {"lengths": left, "kept": kept, "sums": s["sums_now"]} | _cache(s)


PLAIN = {"axes": _plain_axes, "weights": _plain_weights, "evict": _plain_evict}


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


def work(case):
    q_heads, kv_heads, dim, rot = HEADS[case["heads"]]
    row = dim * DTYPES[case["cache"]].itemsize + (4 if case["cache"] == "e4m3" else 0)
    if case["kind"] == "axes":
        tokens = sum(_new_tokens(case))
        each = (2 * q_heads + 2 * kv_heads) * dim * 2 + 2 * kv_heads * row + 4 * rot + 4 * case["axes"]
        return {"bytes": float(tokens * each), "flops": 3.0 * tokens * (q_heads + kv_heads) * rot}
    if case["kind"] == "weights":
        keys = sum(min(n, case["window"] or n) for n in _lengths(case))
        return {"bytes": float(keys * kv_heads * (2 * row + 8) + 4 * case["batch"] * q_heads * dim),
                "flops": 4.0 * keys * q_heads * dim + 4.0 * keys * q_heads}
    budget, due = case["budget"], [n for n in _lengths(case) if n > case["limit"]]
    moved = len(due) * (budget - case["sink"])
    # the sums before and after, the kept places, and the rows that change their place
    return {"bytes": float(kv_heads * (8 * sum(due) + 4 * budget * case["batch"] + 4 * row * moved) + 8 * case["batch"]),
            "flops": float(kv_heads * sum(due))}


# ------------------------------------------------------------------------------------------------- 64 bits


def _exact_axes(s):
    starts = range(s["q"].shape[0] + 1) if s["starts"] is None else s["starts"].tolist()
    half, page, sections = s["cos"].shape[1], s["page"], s["sections"]
    if s["interleaved"]:
        axis = [i % len(sections) if i // len(sections) < sections[i % len(sections)] else 0 for i in range(half)]
    else:
        axis = [a for a, count in enumerate(sections) for _ in range(count)]
    where = [s["positions"][a].long() for a in axis]
    angle = torch.stack([torch.complex(s["cos"][p, i].double(), s["sin"][p, i].double()) for i, p in enumerate(where)], 1)
    out = {"q": s["q"].double()} | {name: x.double() for name, x in _cache(s).items()}
    k = s["k"].double()
    for x in (out["q"], k):
        turned = torch.complex(x[..., :half].clone(), x[..., half: 2 * half].clone()) * angle[:, None]
        x[..., :half], x[..., half: 2 * half] = turned.real, turned.imag
    for b, n in enumerate(s["lengths"].tolist()):
        lo, hi = starts[b], starts[b + 1]
        at = torch.arange(n - (hi - lo), n, device="cuda")
        at = (s["table"][b].long()[torch.div(at, page, rounding_mode="floor")], slice(None), at % page)
        for name, x in (("k", k[lo:hi]), ("v", s["v"][lo:hi].double())):
            if s["k_scale"] is not None:
                top = x.abs().max(-1).values / E4M3_MAX
                out[name + "_scale"][at] = top
                x = x / top[..., None]
            out[name + "_cache"][at] = x
    return out


def _exact_weights(s):
    batch, q_heads, dim = s["q"].shape
    kv_heads = s["k_cache"].shape[1]
    out = torch.zeros((batch, q_heads, dim), dtype=torch.float64, device="cuda")
    sums = s["sums"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - s["window"]) if s["window"] else 0
        at = torch.arange(first, n, device="cuda")
        pages, slots = s["table"][b].long()[torch.div(at, s["page"], rounding_mode="floor")], at % s["page"]
        for g in range(kv_heads):
            mine = slice(g * (q_heads // kv_heads), (g + 1) * (q_heads // kv_heads))
            k, v = s["k_cache"][pages, g, slots].double(), s["v_cache"][pages, g, slots].double()
            if s["k_scale"] is not None:
                k = k * s["k_scale"][pages, g, slots].double()[:, None]
                v = v * s["v_scale"][pages, g, slots].double()[:, None]
            weight = torch.softmax(s["q"][b, mine].double() @ k.T / math.sqrt(dim), 1)
            out[b, mine] = weight @ v
            sums[b, g, first:n] += weight.sum(0)
    return out, sums


def _exact_evict(s):
    budget, page = s["budget"], s["page"]
    batch, heads, _ = s["sums"].shape
    sums = s["sums"].double()
    before = {name: x.double() for name, x in _cache(s).items()}
    after = {name: x.clone() for name, x in before.items()}
    left, kept = s["lengths"].clone(), torch.full((batch, heads, budget), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        if n <= s["limit"]:
            continue
        left[b] = budget
        lo, hi, want = s["sink"], n - s["recent"], budget - s["sink"] - s["recent"]
        table = s["table"][b].long()
        for h in range(heads):
            middle = sums[b, h, lo:hi]
            keep = torch.ones(n, dtype=torch.bool, device="cuda")
            keep[lo:hi] = False
            if want:
                bar = torch.kthvalue(middle, hi - lo - want + 1).values  # the want-th largest
                keep[lo:hi] = middle > bar
                level = torch.nonzero(middle == bar)[:, 0]
                keep[lo + level[: want - int((middle > bar).sum())]] = True
            at = torch.nonzero(keep)[:, 0]
            kept[b, h] = at
            old, to = sums[b, h, at].clone(), torch.arange(budget, device="cuda")
            sums[b, h] = 0
            sums[b, h, :budget] = old
            for name, x in before.items():
                after[name][table[to // page], h, to % page] = x[table[at // page], h, at % page]
    return {"lengths": left, "kept": kept, "sums": sums} | after


def exact(case, seed):
    s = prepare(case, seed)
    return {"axes": _exact_axes, "weights": _exact_weights, "evict": _exact_evict}[s["kind"]](s)
