"""Queries on an installed prefix, as cases that can be timed and compared.

After a handoff has published a request's history in the target's paged pool,
the target model answers on it. A case is one pass through an operator of that
path, at the geometry of one layer (all layers for the eviction):

- ``install``: new tokens' queries and keys are rotated to their positions and
               their K/V rows stored into the requests' pages;
- ``attend``:  attention of the new tokens over the paged cache;
- ``weights``: the attention each cached token got, summed over new tokens and
               heads and added to what it had;
- ``evict``:   the kept tokens of each request (the first, the last and the
               heaviest between them) are copied, in order, to other pages.

A request's new tokens are the last of its cached ones. With ``ragged`` its
cached length is drawn around ``tokens`` (lognormal, sigma 0.5) and its new
tokens between 1 and ``new``. Keys and values are N(0, 1) times a lognormal
scale per channel, pages are drawn from a shuffled free list.
"""

from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(op, tokens, new, *, requests=1, ragged=False, heads=(16, 2), head_dim=128, dtype="bf16", **more):
    return dict(op=op, tokens=tokens, new=new, requests=requests, ragged=ragged, query_heads=heads[0],
                kv_heads=heads[1], head_dim=head_dim, dtype=dtype, **more)


def _install(tokens, new, *, rotary_dim=None, interleaved=False, scaling="none", theta=1e6, **more):
    c = _case("install", tokens, new, **more)
    return dict(c, rotary_dim=rotary_dim or c["head_dim"], interleaved=interleaved, scaling=scaling, theta=theta)


def _attend(tokens, new, *, window=0, cap=0.0, bias=False, prefix=0, lse=False, spread=1.0, **more):
    return dict(_case("attend", tokens, new, **more), window=window, cap=cap, bias=bias, prefix=prefix, lse=lse,
                spread=spread)


def _weights(tokens, new, *, window=0, cap=0.0, **more):
    return dict(_case("weights", tokens, new, **more), window=window, cap=cap, bias=False, prefix=0, spread=1.0)


def _evict(tokens, budget, *, layers=64, first=4, last=32, **more):
    return dict(_case("evict", tokens, 1, **more), budget=budget, layers=layers, first=first, last=last)


def listed():
    named = [
        # One decoding step of 64 requests, every head of the target on one
        # GPU: the smallest call, its time is the launch.
        ("install step 64", _install(2048, 1, requests=64, ragged=True, heads=(64, 8))),
        # A prompt chunk behind a handed-off prefix, one tensor-parallel
        # rank's heads, frequencies scaled for a long context.
        ("install chunk 2048", _install(32768, 2048, scaling="yarn")),
        # The decoding step of an admitted cohort of 64 ragged requests (one
        # tensor-parallel rank's share).
        ("step 64", _attend(2048, 1, requests=64, ragged=True)),
        # The decoding step of one request with a long history, all heads.
        ("step 1 of 32768", _attend(32768, 1, heads=(64, 8))),
        # The question asked right after a 4096-token handoff.
        ("query 37 over 4096", _attend(4133, 37, lse=True)),
        # A long document's next chunk behind its installed prefix.
        ("chunk 2048 over 32768", _attend(32768, 2048)),
        # A whole prompt through a sliding-window layer of head size 256, in
        # half precision, scores capped.
        ("windows 8192 dim256", _attend(8192, 8192, window=1024, cap=30.0, spread=3.0, heads=(16, 8), head_dim=256,
                                        dtype="fp16")),
        # The small fp32 model's shape: a prompt with a prefix that sees
        # itself whole, scores biased by distance.
        ("prefix fp32 250", _attend(250, 250, prefix=100, bias=True, lse=True, heads=(4, 2), head_dim=64, dtype="fp32")),
        # What the last 32 tokens of a long history attend to, which decides
        # what is kept of it.
        ("weights 32 of 32768", _weights(32768, 32)),
        # The running sums of a cohort's decoding step.
        ("weights step 64", _weights(2048, 1, requests=64, ragged=True)),
        # A long history of one tensor-parallel rank shrunk to a quarter.
        ("evict 16384 to 4096", _evict(16384, 4096)),
        # A ragged cohort shrunk to a common budget.
        ("evict 16 to 700", _evict(2048, 700, requests=16, ragged=True, heads=(16, 2), layers=62)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["install", "install", "step", "step", "query", "chunk", "chunk", "model", "small", "weights",
                         "weights", "evict"])
    heads = rng.choice([(16, 2), (16, 2), (8, 8), (10, 2), (16, 4)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if family == "install":
        head_dim = rng.choice([64, 96, 128, 128, 256])
        new = _log_uniform(rng, 1, 2048)
        return _install(_log_uniform(rng, new, 32768), new, requests=1 if new > 64 else rng.randint(1, 64),
                        ragged=rng.random() < 0.5, heads=heads, head_dim=head_dim,
                        dtype=rng.choice(["bf16", "fp16", "fp32"]),
                        rotary_dim=head_dim if rng.random() < 0.6 else head_dim // 2, interleaved=rng.random() < 0.4,
                        scaling=rng.choice(["none", "yarn", "linear"]), theta=rng.choice([1e4, 1e6]))
    if family == "step":
        requests = rng.randint(1, 64)
        return _attend(_log_uniform(rng, 16, 32768 if requests < 9 else 4096), 1, requests=requests,
                       ragged=rng.random() < 0.7, heads=rng.choice([heads, (64, 8)]),
                       head_dim=rng.choice([64, 128, 128, 256]), dtype=dtype, window=rng.choice([0, 0, 0, 1024]))
    if family == "query":
        new = rng.randint(2, 100)
        return _attend(_log_uniform(rng, new, 16384), new, requests=rng.randint(1, 8), ragged=True, heads=heads,
                       head_dim=rng.choice([64, 128, 128, 256]), dtype=dtype, lse=rng.random() < 0.5)
    if family == "chunk":
        new = _log_uniform(rng, 100, 2048)
        return _attend(_log_uniform(rng, new, 32768), new, heads=heads, head_dim=rng.choice([64, 128, 128]), dtype=dtype)
    if family == "model":
        new = _log_uniform(rng, 64, 8192)
        return _attend(new, new, heads=rng.choice([(16, 8), (8, 4)]), head_dim=rng.choice([128, 256]), dtype=dtype,
                       window=rng.choice([0, 512, 1024]), cap=rng.choice([0.0, 30.0]), spread=2.0)
    if family == "small":
        new = _log_uniform(rng, 1, 1000)
        return _attend(_log_uniform(rng, new, 2000), new, heads=rng.choice([(4, 2), (6, 6)]),
                       head_dim=rng.choice([64, 80, 128]), dtype=rng.choice(["fp32", "fp32", "bf16"]),
                       prefix=rng.choice([0, 0, 60]), bias=rng.random() < 0.5, lse=rng.random() < 0.5)
    if family == "weights":
        new = rng.choice([1, 1, rng.randint(2, 128)])
        return _weights(_log_uniform(rng, max(new, 100), 32768 if new > 1 else 4096), new,
                        requests=1 if new > 1 else rng.randint(1, 64), ragged=new == 1, heads=heads,
                        head_dim=rng.choice([64, 128, 128, 256]), dtype=dtype, window=rng.choice([0, 0, 1024]))
    tokens = _log_uniform(rng, 200, 8192)
    return _evict(tokens, max(40, int(tokens * rng.uniform(0.1, 0.6))), layers=rng.choice([16, 62, 64]),
                  requests=1 if tokens > 2000 else rng.randint(1, 8), ragged=rng.random() < 0.5, dtype=dtype)


# ---------------------------------------------------------------------------
# Geometry of a case
# ---------------------------------------------------------------------------


def _requests(case):
    """Cached length and new tokens of each request."""
    n, tokens, new = case["requests"], case["tokens"], case["new"]
    if not case["ragged"]:
        return [tokens] * n, [new] * n
    rng = random.Random(1000 * tokens + new)
    lengths = [min(max(round(tokens * math.exp(rng.gauss(0.0, 0.5))), new, 16), 8 * tokens) for _ in range(n)]
    return lengths, [rng.randint(1, new) for _ in range(n)]


def _visible(case, length, new):
    """(query, key) pairs of one request that see each other, and its cached tokens that any query sees."""
    window, prefix = case["window"], min(case["prefix"], length)
    pairs = seen = 0
    for p in range(length - new, length):
        first = max(0, p - window + 1) if window else 0
        pairs += p + 1 - first + max(0, prefix - p - 1) + max(0, min(first, prefix))
    first = max(0, length - new - window + 1) if window else 0
    seen = length - first + min(first, prefix)
    return pairs, seen


def work(case):
    lengths, new = _requests(case)
    e = DTYPES[case["dtype"]].itemsize
    hq, hk, d = case["query_heads"], case["kv_heads"], case["head_dim"]
    n = sum(new)
    if case["op"] == "install":
        moved = 2 * n * (hq + 2 * hk) * d * e
        return {"bytes": moved + 8 * n, "flops": 3 * n * (hq + hk) * case["rotary_dim"]}
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in lengths)
        return {"bytes": 4 * case["layers"] * kept * hk * d * e + 4 * sum(lengths) + 8 * kept, "flops": 0}
    pairs, seen = (sum(x) for x in zip(*(_visible(case, l, m) for l, m in zip(lengths, new))))
    if case["op"] == "attend":
        return {"bytes": 2 * n * hq * d * e + 2 * seen * hk * d * e + (4 * n * hq if case["lse"] else 0),
                "flops": 4 * d * hq * pairs}
    return {"bytes": n * hq * (d * e + 4) + seen * hk * d * e + 8 * seen, "flops": 2 * d * hq * pairs}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _frequencies(case):
    """Rotations per token of each rotated pair, in radians, and the tables' magnitude."""
    dim, theta = case["rotary_dim"], case["theta"]
    inv = theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if case["scaling"] == "linear":
        return inv / 4.0, 1.0
    if case["scaling"] == "none":
        return inv, 1.0
    # YaRN from an 8192-token window to four times that.
    turns = [dim * math.log(8192 / (r * 2 * math.pi)) / (2 * math.log(theta)) for r in (32.0, 1.0)]
    low, high = max(math.floor(turns[0]), 0), min(math.ceil(turns[1]), dim - 1)
    keep = 1 - ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return inv / 4.0 * (1 - keep) + inv * keep, 0.1 * math.log(4.0) + 1.0


def prepare(case, seed):
    dev, dtype = "cuda", DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    lengths, new = _requests(case)
    hq, hk, d, n, op = case["query_heads"], case["kv_heads"], case["head_dim"], sum(new), case["op"]
    scale = torch.exp(0.5 * torch.randn(d, generator=g, device=dev))

    def values(*shape):
        return (torch.randn(*shape, d, generator=g, device=dev) * scale).to(dtype)

    pages = [-(-x // PAGE) for x in lengths]
    kept = [min(x, case["budget"]) for x in lengths] if op == "evict" else []
    kept_pages = [-(-x // PAGE) for x in kept]
    width = max(pages)
    # Storing new tokens touches the last pages only: the pool holds those.
    held = [x // PAGE - (x - m) // PAGE + 1 for x, m in zip(lengths, new)] if op == "install" else pages
    total = sum(held) + sum(kept_pages)
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = order[torch.randint(0, total, (len(lengths), width), generator=g, device=dev)]
    at = 0
    for b, (p, h) in enumerate(zip(pages, held)):
        h = min(h, p)
        table[b, p - h:p] = order[at:at + h]
        at += h
    s = {
        "case": dict(case),
        "table": table,
        "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
        "query_start": torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32),
        "max_query": max(new), "max_length": max(lengths), "softmax_scale": d ** -0.5,
    }
    if op == "evict":
        target = torch.full((len(lengths), max(kept_pages)), 0, dtype=torch.int32, device=dev)
        for b, p in enumerate(kept_pages):
            target[b, :p] = order[at:at + p]
            at += p
        s["target"] = target
        s["k"] = values(case["layers"], total * PAGE, hk)
        s["v"] = values(case["layers"], total * PAGE, hk)
        # What decoding adds up: a few heavy tokens, most near nothing, many alike.
        w = torch.randn(len(lengths), max(lengths), generator=g, device=dev).mul(2).exp()
        s["weights"] = torch.where(w < 0.2, torch.zeros_like(w), w)
        return s
    if op == "install":
        fused = values(n, hq + 2 * hk)
        s["q"], s["new_k"], s["new_v"] = fused.split([hq, hk, hk], dim=1)
        s["k"] = torch.zeros(1, total * PAGE, hk, d, dtype=dtype, device=dev)
        s["v"] = torch.zeros_like(s["k"])
        inv, s["magnitude"] = _frequencies(case)
        s["inv_freq"] = inv.to(dev)
        return s
    s["q"] = (torch.randn(n, hq, d, generator=g, device=dev) * case["spread"]).to(dtype)
    s["k"], s["v"] = values(1, total * PAGE, hk), values(1, total * PAGE, hk)
    if case["bias"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev, dtype=torch.float32) / hq)
    if case["prefix"]:
        s["prefix"] = torch.tensor([min(case["prefix"], x) for x in lengths], dtype=torch.int32, device=dev)
    if op == "weights":
        s["lse"] = _lse(s)
        s["weights"] = torch.rand(len(lengths), max(lengths), generator=g, device=dev)
    return s


def _lse(s):
    """The new tokens' softmax normalisers, which their attention has left."""
    score, row, _ = _scores(s)
    return torch.logsumexp(score, -1).permute(0, 2, 1)[row]


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"install": _plain_install, "attend": _plain_attend, "weights": _plain_weights,
            "evict": _plain_evict}[op](state)


def _own(s, op):
    from cachebridge_amd.online.queries import (QueryBatch, Rotary, add_key_weights, evict_tokens, install_tokens,
                                                paged_attention)
    from cachebridge_amd.plan import rows_from_stacked

    c = s["case"]

    def batch(table):
        rows = rows_from_stacked(s["k"], s["v"], block_table=table.view(-1), page_size=PAGE)
        return QueryBatch(rows, s["query_start"], s["lengths"], request_stride=table.shape[1] * PAGE,
                          max_query=s["max_query"], max_length=s["max_length"])

    requests = batch(s["table"])
    if op == "install":
        rotary = Rotary(s["inv_freq"], magnitude=s["magnitude"], interleaved=c["interleaved"])
        q = install_tokens(requests, 0, s["q"], s["new_k"], s["new_v"], rotary)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "evict":
        kept = evict_tokens(requests, s["weights"], batch(s["target"]), budget=c["budget"], first=c["first"],
                            last=c["last"])
        return {"tokens": kept.tokens, "lengths": kept.lengths, "weights": kept.weights, "k": s["k"], "v": s["v"]}
    scores = dict(scale=s["softmax_scale"], window=c["window"], cap=c["cap"], slopes=s.get("slopes"),
                  prefix_lengths=s.get("prefix"))
    if op == "weights":
        weights = s["weights"].clone()  # the sums before this step stay for the next pass
        add_key_weights(requests, 0, s["q"], s["lse"], weights, **scores)
        return {"weights": weights}
    out = paged_attention(requests, 0, s["q"], return_lse=c["lse"], **scores)
    return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}


def _slots(table, tokens):
    """Pool rows of ``tokens`` [B, n] of each request."""
    return table.gather(1, tokens // PAGE).long() * PAGE + tokens % PAGE


def _padded(s):
    """Index of each new token in [B, max_query], the flat positions of that layout and their validity."""
    start, m = s["query_start"].long(), s["max_query"]
    count = start.diff()
    i = torch.arange(m, device=start.device)
    valid = i < count[:, None]
    token = (s["lengths"].long() - count)[:, None] + i
    return (start[:-1, None] + i).clamp(max=int(s["q"].shape[0]) - 1), token, valid


def _scores(s):
    """Masked scores [B, heads, new, cached] in fp32, the valid new tokens and each pair's visibility."""
    c = s["case"]
    flat, token, valid = _padded(s)
    b, hk, d = flat.shape[0], c["kv_heads"], c["head_dim"]
    j = torch.arange(s["max_length"], device=flat.device)
    inside = j < s["lengths"][:, None]
    rows = _slots(s["table"], torch.where(inside, j, 0))
    k = s["k"][0][rows].float().permute(0, 2, 3, 1).contiguous()                 # [B, kv, D, T]
    q = s["q"][flat].float().permute(0, 2, 1, 3)                                 # [B, heads, n, D]
    q = q.reshape(b, hk, -1, d).contiguous()
    score = (q @ k).view(b, c["query_heads"], flat.shape[1], -1) * s["softmax_scale"]
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    away = j - token[..., None]                                                  # [B, n, T]
    if "slopes" in s:
        score = score - s["slopes"][:, None, None] * away[:, None].abs().float()
    see = away <= 0
    if c["window"]:
        see = see & (away > -c["window"])
    if "prefix" in s:
        see = see | (j < s["prefix"][:, None])[:, None]
    see = see & inside[:, None] & valid[..., None]
    return score.masked_fill(~see[:, None], -math.inf), valid, rows


def _plain_attend(s):
    c = s["case"]
    score, valid, rows = _scores(s)
    b, hk, d = score.shape[0], c["kv_heads"], c["head_dim"]
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = s["v"][0][rows].float().permute(0, 2, 1, 3).contiguous()                 # [B, kv, T, D]
    out = (p.view(b, hk, -1, p.shape[-1]) @ v).view(b, c["query_heads"], -1, d) / total.clamp(min=1e-30)
    out = out.permute(0, 2, 1, 3)[valid].to(s["q"].dtype)
    if not c["lse"]:
        return {"out": out}
    return {"out": out, "lse": (torch.log(total) + top)[..., 0].permute(0, 2, 1)[valid]}


def _plain_weights(s):
    score, valid, _ = _scores(s)
    lse = torch.zeros(*valid.shape, score.shape[1], device=score.device)
    lse[valid] = s["lse"]
    got = torch.exp(score - lse.permute(0, 2, 1)[..., None]).sum((1, 2))
    return {"weights": s["weights"] + got}


def _rotated(x, cos, sin, rotary_dim, interleaved):
    y = x.float()
    turn, rest = y[..., :rotary_dim], y[..., rotary_dim:]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turn.chunk(2, -1)
        turn = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turn, rest), -1).to(x.dtype)


def _plain_install(s):
    c = s["case"]
    _, token, valid = _padded(s)
    # Far positions turn by thousands of radians: the angle is kept in 64 bits.
    angle = token[valid].double()[:, None, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    rows = _slots(s["table"], torch.where(valid, token, 0))[valid]
    s["k"][0][rows] = _rotated(s["new_k"], cos, sin, c["rotary_dim"], c["interleaved"])
    s["v"][0][rows] = s["new_v"]
    return {"q": _rotated(s["q"], cos, sin, c["rotary_dim"], c["interleaved"]), "k": s["k"], "v": s["v"]}


def _plain_evict(s):
    c, lengths = s["case"], s["lengths"].long()[:, None]
    j = torch.arange(s["max_length"], device=lengths.device)
    inside = j < lengths
    rank = s["weights"].masked_fill((j < c["first"]) | (j >= lengths - c["last"]), math.inf).masked_fill(~inside, -1.0)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    count = lengths.clamp(max=c["budget"])
    n = torch.arange(c["budget"], device=j.device)
    taken = order[:, :c["budget"]]
    n, valid = n[:taken.shape[1]], n[:taken.shape[1]] < count
    tokens = torch.where(valid, taken, s["max_length"]).sort(-1).values
    src = _slots(s["table"], torch.where(valid, tokens, 0))[valid]
    dst = _slots(s["target"], torch.where(valid, n, 0))[valid]
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    shape = (lengths.shape[0], c["budget"])
    kept = torch.full(shape, -1, dtype=torch.int32, device=j.device)
    weights = torch.zeros(shape, device=j.device)
    kept[:, :n.numel()] = torch.where(valid, tokens, -1).int()
    weights[:, :n.numel()] = torch.where(valid, s["weights"].gather(1, torch.where(valid, tokens, 0)), 0.0)
    return {"tokens": kept, "lengths": count[:, 0].int(), "weights": weights, "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------------------
# The definition, in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op, lengths, new = case["op"], *_requests(case)
    rows = [[int(x) for x in r] for r in s["table"].tolist()]

    def slots(pages, first, stop):
        at = torch.arange(first, stop)
        return (torch.tensor(pages)[at // PAGE] * PAGE + at % PAGE).cuda()

    if op == "install":
        return _exact_install(case, s, lengths, new, rows, slots)
    if op == "evict":
        return None  # copies and choices: there is nothing to round
    group = case["query_heads"] // case["kv_heads"]
    out, lses, heavy, at = [], [], s["weights"].double() if op == "weights" else None, 0
    for b, (length, m) in enumerate(zip(lengths, new)):
        where = slots(rows[b], 0, length)
        pos = torch.arange(length - m, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        mask = key <= pos
        if case["window"]:
            mask &= pos - key < case["window"]
        if case["prefix"]:
            mask |= key < case["prefix"]
        per_head = []
        for h in range(case["query_heads"]):
            q = s["q"][at:at + m, h].double()
            x = q.mm(s["k"][0, where, h // group].double().t().contiguous()) / math.sqrt(case["head_dim"])
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            if case["bias"]:
                x = x - 2.0 ** (-8.0 * (h + 1) / case["query_heads"]) * (pos - key).abs()
            x[~mask] = -math.inf
            if op == "weights":
                heavy[b, :length] += (x - s["lse"][at:at + m, h].double()[:, None]).exp().sum(0)
                continue
            norm = torch.logsumexp(x, 1, keepdim=True)
            per_head.append(((x - norm).exp().mm(s["v"][0, where, h // group].double()), norm[:, 0]))
        if op == "attend":
            out.append(torch.stack([o for o, _ in per_head], 1))
            lses.append(torch.stack([z for _, z in per_head], 1))
        at += m
    if op == "weights":
        return {"weights": heavy}
    return {"out": torch.cat(out), "lse": torch.cat(lses)} if case["lse"] else {"out": torch.cat(out)}


def _exact_install(case, s, lengths, new, rows, slots):
    dim, half = case["rotary_dim"], case["rotary_dim"] // 2
    pos = torch.cat([torch.arange(x - m, x, dtype=torch.float64) for x, m in zip(lengths, new)])
    turn = torch.polar(torch.full((len(pos), half), s["magnitude"], dtype=torch.float64),
                       pos[:, None] * s["inv_freq"].cpu()[None, :]).cuda()[:, None]

    def spin(x):
        x = x.double()
        pairs = x[..., :dim].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        if not case["interleaved"]:
            z = z.transpose(-1, -2)
        return torch.cat((z.flatten(-2), x[..., dim:]), -1)

    k, v = s["k"].double(), s["v"].double()
    where = torch.cat([slots(r, x - m, x) for r, x, m in zip(rows, lengths, new)])
    k[0, where], v[0, where] = spin(s["new_k"]), s["new_v"].double()
    return {"q": spin(s["q"]), "k": k, "v": v}
