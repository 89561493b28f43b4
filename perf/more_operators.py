"""Queries on an 8-bit cache, as cases that can be timed and compared.

A pool holds K and V rows in 8-bit floating point (e4m3) with one power of two
as scale for each page of tokens and KV head. A case is one pass through an
operator of that path, at the geometry of one layer (all layers for
``quantize``):

- ``quantize``: an installed prefix moves from a 16- or 32-bit pool into an
                8-bit one, all layers: every page of a head gets the scale that
                its largest element needs;
- ``append``:   new tokens' queries and keys are rotated to their positions and
                their K/V rows stored into the requests' 8-bit pages. A page
                that holds cached tokens keeps its scale unless the new rows
                need a larger one; its rows are then rounded again;
- ``axes``:     the same rotation and store with a position of several axes
                (time, height, width) per token, each pair of elements turning
                by one of them, into an 8-bit or a 16-bit pool;
- ``attend``:   attention of the new tokens over the 8-bit cache.

A request's new tokens are the last of its cached ones. With ``ragged`` its
cached length is drawn around ``tokens`` (lognormal, sigma 0.5) and its new
tokens between 1 and ``new``. Keys and values are N(0, 1) times a lognormal
scale per channel, pages are drawn from a shuffled free list.

The scale of a page and head is 2^e with the smallest e for which the largest
finite element is at most 448 * 2^e, 2^-126 if all are zero; rows that come in
fp16 have e at most 7 (the values stay in that type's range), larger elements
are stored as the largest.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
SOURCE_PAGE = 16  # tokens a page of the pools that hold 16- and 32-bit rows


def _case(op, tokens, new, *, requests=1, ragged=False, heads=(16, 2), head_dim=128, dtype="bf16", page=16, **more):
    return dict(op=op, tokens=tokens, new=new, requests=requests, ragged=ragged, query_heads=heads[0],
                kv_heads=heads[1], head_dim=head_dim, dtype=dtype, page=page, **more)


def _quantize(tokens, *, layers=64, **more):
    return dict(_case("quantize", tokens, 1, **more), layers=layers)


def _append(tokens, new, *, rotary_dim=None, interleaved=False, theta=1e6, **more):
    c = _case("append", tokens, new, **more)
    return dict(c, rotary_dim=rotary_dim or c["head_dim"], interleaved=interleaved, theta=theta, sections="",
                cyclic=False, quantized=True)


def _axes(tokens, new, sections, *, cyclic=False, quantized=True, **more):
    c = _append(tokens, new, rotary_dim=2 * sum(sections), **more)
    return dict(c, op="axes", sections=",".join(map(str, sections)), cyclic=cyclic, quantized=quantized)


def _attend(tokens, new, *, window=0, cap=0.0, bias=False, prefix=0, lse=False, spread=1.0, **more):
    return dict(_case("attend", tokens, new, **more), window=window, cap=cap, bias=bias, prefix=prefix, lse=lse,
                spread=spread)


def listed():
    named = [
        # A handed-off history of one tensor-parallel rank goes into the 8-bit
        # pool that its requests are answered from, every layer at once.
        ("quantize 4096", _quantize(4096)),
        # The same for an admitted ragged cohort of half-precision requests,
        # pages of 32 tokens.
        ("quantize cohort 16", _quantize(1024, requests=16, ragged=True, layers=62, dtype="fp16", page=32)),
        # One decoding step of 64 requests, every head of the target on one
        # GPU: the smallest call, its time is the launch.
        ("append step 64", _append(2048, 1, requests=64, ragged=True, heads=(64, 8))),
        # A prompt chunk behind a handed-off prefix, one rank's heads.
        ("append chunk 2048", _append(32768, 2048, page=64)),
        # A prompt of text and image patches into a 16-bit pool: three axes,
        # a quarter of each head of 256 turns, axes in turn from pair to pair.
        ("axes prompt 2048 16-bit", _axes(2048, 2048, (11, 11, 10), cyclic=True, quantized=False, heads=(16, 2),
                                          head_dim=256)),
        # The decoding steps behind such prompts on the 8-bit pool, axes in
        # blocks of pairs.
        ("axes step 32", _axes(4096, 1, (16, 24, 24), requests=32, ragged=True, heads=(28, 4))),
        # The decoding step of an admitted cohort of 64 ragged requests (one
        # tensor-parallel rank's share).
        ("step 64", _attend(2048, 1, requests=64, ragged=True)),
        # The decoding step of one request with a long history, all heads.
        ("step 1 of 32768", _attend(32768, 1, heads=(64, 8))),
        # A decoding step of many long requests: the largest cache.
        ("step 64 of 8192", _attend(8192, 1, requests=64, page=64)),
        # The question asked right after a 4096-token handoff.
        ("query 37 over 4096", _attend(4133, 37, lse=True)),
        # A long document's next chunk behind its installed prefix.
        ("chunk 2048 over 32768", _attend(32768, 2048, page=64)),
        # A whole prompt through a sliding-window layer of head size 256, in
        # half precision, scores capped.
        ("windows 8192 dim256", _attend(8192, 8192, window=1024, cap=30.0, spread=3.0, heads=(16, 8), head_dim=256,
                                        dtype="fp16", page=32)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["quantize", "quantize", "append", "append", "axes", "axes", "step", "step", "step", "query",
                         "chunk", "model", "small"])
    heads = rng.choice([(16, 2), (16, 2), (8, 8), (10, 2), (16, 4)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([1, 16, 16, 24, 32, 64, 128])
    if family == "quantize":
        tokens = _log_uniform(rng, 50, 4096)
        return _quantize(tokens, layers=rng.choice([16, 62, 64]), requests=1 if tokens > 1000 else rng.randint(1, 8),
                         ragged=rng.random() < 0.5, heads=rng.choice([(16, 2), (8, 4)]),
                         head_dim=rng.choice([64, 96, 128]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                         page=max(page, 16))
    if family in ("append", "axes"):
        head_dim = rng.choice([64, 96, 128, 128, 256])
        new = _log_uniform(rng, 1, 2048)
        more = dict(requests=1 if new > 64 else rng.randint(1, 64), ragged=rng.random() < 0.5, heads=heads,
                    head_dim=head_dim, dtype=rng.choice(["bf16", "fp16", "fp32"]), page=page,
                    interleaved=rng.random() < 0.4, theta=rng.choice([1e4, 1e6]))
        tokens = _log_uniform(rng, new, 32768)
        if family == "append":
            return _append(tokens, new, rotary_dim=head_dim if rng.random() < 0.6 else head_dim // 2, **more)
        pairs = rng.choice([head_dim // 2, head_dim // 4])
        third = pairs // 3
        return _axes(tokens, new, (pairs - 2 * third, third, third), cyclic=rng.random() < 0.5,
                     quantized=rng.random() < 0.5, **more)
    if family == "step":
        requests = rng.randint(1, 64)
        return _attend(_log_uniform(rng, 16, 32768 if requests < 9 else 4096), 1, requests=requests,
                       ragged=rng.random() < 0.7, heads=rng.choice([heads, (64, 8)]),
                       head_dim=rng.choice([64, 128, 128, 256]), dtype=dtype, window=rng.choice([0, 0, 0, 1024]),
                       page=page)
    if family == "query":
        new = rng.randint(2, 100)
        return _attend(_log_uniform(rng, new, 16384), new, requests=rng.randint(1, 8), ragged=True, heads=heads,
                       head_dim=rng.choice([64, 128, 128, 256]), dtype=dtype, lse=rng.random() < 0.5, page=page)
    if family == "chunk":
        new = _log_uniform(rng, 100, 2048)
        return _attend(_log_uniform(rng, new, 32768), new, heads=heads, head_dim=rng.choice([64, 128, 128]),
                       dtype=dtype, page=page)
    if family == "model":
        new = _log_uniform(rng, 64, 8192)
        return _attend(new, new, heads=rng.choice([(16, 8), (8, 4)]), head_dim=rng.choice([128, 256]), dtype=dtype,
                       window=rng.choice([0, 512, 1024]), cap=rng.choice([0.0, 30.0]), spread=2.0, page=page)
    new = _log_uniform(rng, 1, 1000)
    return _attend(_log_uniform(rng, new, 2000), new, heads=rng.choice([(4, 2), (6, 6)]),
                   head_dim=rng.choice([64, 80, 128]), dtype=rng.choice(["fp32", "fp16", "bf16"]),
                   prefix=rng.choice([0, 0, 60]), bias=rng.random() < 0.5, lse=rng.random() < 0.5, page=page)


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


def _sections(case):
    return [int(x) for x in case["sections"].split(",")] if case["sections"] else []


def work(case):
    lengths, new = _requests(case)
    e, page = DTYPES[case["dtype"]].itemsize, case["page"]
    hq, hk, d = case["query_heads"], case["kv_heads"], case["head_dim"]
    n = sum(new)
    if case["op"] == "quantize":
        scales = 2 * hk * sum(-(-x // page) for x in lengths)
        return {"bytes": case["layers"] * (2 * sum(lengths) * hk * d * (e + 1) + scales), "flops": 0}
    if case["op"] in ("append", "axes"):
        stored = 1 if case["quantized"] else e
        moved = n * (2 * hq * d * e + 2 * hk * d * (e + stored))
        return {"bytes": moved + 8 * n * max(1, len(_sections(case))), "flops": 3 * n * (hq + hk) * case["rotary_dim"]}
    pairs, seen = (sum(x) for x in zip(*(_visible(case, l, m) for l, m in zip(lengths, new))))
    return {"bytes": 2 * n * hq * d * e + 2 * seen * hk * d + 2 * hk * (seen // page) + (4 * n * hq if case["lse"] else 0),
            "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------------------
# 8-bit rows with a scale for each page and head
# ---------------------------------------------------------------------------


def _exponent(top, dtype):
    """e of the scale 2^e for finite elements up to ``top`` (448 is 0.875 * 2^9)."""
    m, k = torch.frexp(top)
    return (k - 9 + (m > 0.875)).masked_fill(top == 0, -126).clamp(-126, 7 if dtype == torch.float16 else 127)


def _byte(e):
    return (e + 127).to(torch.uint8)


def _codes(x, e):
    """fp32 ``x`` over 2^e, rounded to e4m3."""
    return torch.ldexp(x, -e).clamp(-448, 448).to(E4M3)


def _quantized(x, dtype):
    """``x`` [..., page, heads, dim] as e4m3 and the exponents [..., heads]."""
    x = x.float()
    e = _exponent(x.abs().amax((-3, -1)), dtype)
    return _codes(x, e[..., None, :, None]), e


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _tables(total, pages, held, g, dev):
    """[requests, width] page tables whose last ``held`` entries of each request are pages of its own."""
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = order[torch.randint(0, total, (len(pages), max(pages)), generator=g, device=dev)]
    at = 0
    for b, (p, h) in enumerate(zip(pages, held)):
        table[b, p - h:p] = order[at:at + h]
        at += h
    return table


def prepare(case, seed):
    dev, dtype, page = "cuda", DTYPES[case["dtype"]], case["page"]
    g = torch.Generator(device=dev).manual_seed(seed)
    lengths, new = _requests(case)
    hq, hk, d, n, op = case["query_heads"], case["kv_heads"], case["head_dim"], sum(new), case["op"]
    scale = torch.exp(0.5 * torch.randn(d, generator=g, device=dev))

    def values(*shape):
        return (torch.randn(*shape, d, generator=g, device=dev) * scale).to(dtype)

    pages = [-(-x // page) for x in lengths]
    # Storing new tokens touches the last pages only: the pool holds those.
    storing = op in ("append", "axes")
    held = [p - (x - m) // page for p, x, m in zip(pages, lengths, new)] if storing else pages
    total = sum(held)
    s = {
        "case": dict(case), "page": page,
        "table": _tables(total, pages, held, g, dev),
        "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
        "query_start": torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32),
        "max_query": max(new), "max_length": max(lengths), "softmax_scale": d ** -0.5,
    }
    if op == "quantize":
        source = [-(-x // SOURCE_PAGE) for x in lengths]
        s["source_table"] = _tables(sum(source), source, source, g, dev)
        s["source_k"] = values(case["layers"], sum(source) * SOURCE_PAGE, hk)
        s["source_v"] = values(case["layers"], sum(source) * SOURCE_PAGE, hk)
        shape = (case["layers"], total * page, hk, d)
        for name in ("k", "v"):
            s[name] = torch.zeros(shape, dtype=torch.uint8, device=dev).view(E4M3)
            s[name + "_scale"] = torch.ones(case["layers"], total, hk, dtype=torch.uint8, device=dev).view(E8M0)
        return s
    for name in ("k", "v"):
        x = values(1, total, page, hk)
        if storing and not case["quantized"]:
            s[name] = x.flatten(1, 2)
            continue
        codes, e = _quantized(x, dtype)
        s[name], s[name + "_scale"] = codes.flatten(1, 2), _byte(e).view(E8M0)
    if storing:
        fused = values(n, hq + 2 * hk)
        s["q"], s["new_k"], s["new_v"] = fused.split([hq, hk, hk], dim=1)
        dim = case["rotary_dim"]
        s["inv_freq"] = (case["theta"] ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).to(dev)
        if op == "axes":
            s["positions"] = _positions(case, lengths, new, dev)
        return s
    s["q"] = (torch.randn(n, hq, d, generator=g, device=dev) * case["spread"]).to(dtype)
    if case["bias"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev, dtype=torch.float32) / hq)
    if case["prefix"]:
        s["prefix"] = torch.tensor([min(case["prefix"], x) for x in lengths], dtype=torch.int32, device=dev)
    return s


def _positions(case, lengths, new, dev):
    """[axes, tokens] positions: text counts on along all axes, patches of an image (grids of 16 columns, at places
    512 to 1023 of every 1024) share a time and have a row and a column."""
    place = torch.cat([torch.arange(x - m, x) for x, m in zip(lengths, new)])
    inside = place % 1024
    base = place - inside + 512
    patch = inside >= 512
    rows = torch.stack((base, base + (inside - 512) // 16, base + (inside - 512) % 16))
    return torch.where(patch, rows, place).to(torch.int32).to(dev)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"quantize": _plain_quantize, "append": _plain_store, "axes": _plain_store, "attend": _plain_attend}[op](state)


def _stored(s):
    names = ("k", "v", "k_scale", "v_scale")
    return {name: s[name] for name in names if name in s}


def _batch(s):
    """The requests and their 8-bit (or 16-bit) pages: built once for all layers of a step, as a program does."""
    from cachebridge_amd.online.queries import QueryBatch
    from cachebridge_amd.plan import BlockScales, rows_from_stacked

    c = s["case"]

    def batch(k, v, table, page, scales=None):
        rows = rows_from_stacked(k, v, block_table=table.view(-1), page_size=page, scales=scales)
        return QueryBatch(rows, s["query_start"], s["lengths"], request_stride=table.shape[1] * page,
                          max_query=s["max_query"], max_length=s["max_length"])

    scales = BlockScales(s["k_scale"], s["v_scale"], s["page"], DTYPES[c["dtype"]]) if "k_scale" in s else None
    s["batch"] = batch(s["k"], s["v"], s["table"], s["page"], scales)
    if c["op"] == "quantize":
        s["source"] = batch(s["source_k"], s["source_v"], s["source_table"], SOURCE_PAGE)
    return s["batch"]


def _own(s, op):
    from cachebridge_amd.online.queries import Rotary, install_tokens, paged_attention, quantize_tokens

    c = s["case"]
    batch = s["batch"] if "batch" in s else _batch(s)
    if op == "quantize":
        return {"lengths": quantize_tokens(s["source"], batch), **_stored(s)}
    if op in ("append", "axes"):
        if "rotary" not in s:  # one for all layers and steps
            s["rotary"] = Rotary(s["inv_freq"], interleaved=c["interleaved"],
                                 axes=Rotary.axis_of_pairs(_sections(c), cyclic=c["cyclic"]) if op == "axes" else None)
        q = install_tokens(batch, 0, s["q"], s["new_k"], s["new_v"], s["rotary"], positions=s.get("positions"))
        return {"q": q, **_stored(s)}
    out = paged_attention(batch, 0, s["q"], scale=s["softmax_scale"], window=c["window"], cap=c["cap"],
                          slopes=s.get("slopes"), prefix_lengths=s.get("prefix"), return_lse=c["lse"])
    return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}


def _slots(table, tokens, page):
    """Pool rows of ``tokens`` [B, n] of each request."""
    return table.gather(1, tokens // page).long() * page + tokens % page


def _plain_quantize(s):
    c, page, dtype = s["case"], s["page"], DTYPES[s["case"]["dtype"]]
    lengths = s["lengths"].long()[:, None]
    width = s["table"].shape[1]
    j = torch.arange(width * page, device=lengths.device)
    inside = j < lengths                                                         # [B, T]
    rows = _slots(s["source_table"], torch.where(inside, j, 0), SOURCE_PAGE)
    live = (torch.arange(width, device=j.device) * page < lengths)               # [B, pages]
    at = s["table"][live].long()
    mask = inside.view(-1, width, page)[live]                                    # [P, page]
    where = rows.view(-1, width, page)[live]
    for name in ("k", "v"):
        x = s["source_" + name][:, where]                                        # [L, P, page, heads, D]
        codes, e = _quantized(x.masked_fill(~mask[..., None, None], 0), dtype)
        held = s[name].view(torch.uint8).view(c["layers"], -1, page, *x.shape[3:])
        held[:, at] = torch.where(mask[..., None, None], codes.view(torch.uint8), held[:, at])
        s[name + "_scale"].view(torch.uint8)[:, at] = _byte(e)
    return {"lengths": s["lengths"].clone(), **_stored(s)}


def _rotated(x, cos, sin, rotary_dim, interleaved):
    """Rotated in 32 bits, not yet rounded to the type of ``x``."""
    y = x.float()
    turn, rest = y[..., :rotary_dim], y[..., rotary_dim:]
    if interleaved:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turn.chunk(2, -1)
        turn = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turn, rest), -1)


def _pair_axes(case):
    """The axis that each pair turns by."""
    sections = _sections(case)
    pairs, n = case["rotary_dim"] // 2, max(1, len(sections))
    if case["cyclic"]:
        return [i % n if i // n < sections[i % n] else 0 for i in range(pairs)]
    return [a for a, m in enumerate(sections) for _ in range(m)] or [0] * pairs


def _plain_store(s):
    c, page, dtype = s["case"], s["page"], DTYPES[s["case"]["dtype"]]
    count = s["query_start"].long().diff()
    lengths = s["lengths"].long()
    request = torch.repeat_interleave(torch.arange(count.numel(), device=count.device), count,
                                      output_size=s["q"].shape[0])
    place = (lengths - count)[request] + torch.arange(s["q"].shape[0], device=count.device) - s["query_start"][request]
    if c["op"] == "axes":
        position = s["positions"][torch.tensor(_pair_axes(c), device=count.device)].t()  # [tokens, pairs]
    else:
        position = place[:, None]
    # Far positions turn by thousands of radians: the angle is kept in 64 bits.
    angle = (position.double() * s["inv_freq"])[:, None]
    cos, sin = (angle.cos(), angle.sin()) if dtype == torch.float32 else (angle.cos().float(), angle.sin().float())
    q = _rotated(s["q"], cos, sin, c["rotary_dim"], c["interleaved"]).to(dtype)
    k = _rotated(s["new_k"], cos, sin, c["rotary_dim"], c["interleaved"]).float()
    pages = s["table"][request, place // page].long()
    if not c["quantized"]:
        rows = pages * page + place % page
        s["k"][0][rows], s["v"][0][rows] = k.to(dtype), s["new_v"]
        return {"q": q, **_stored(s)}
    # Every page that gets a row: which of its rows are cached already (its first `old` ones), which are new.
    p, at = pages.unique(return_inverse=True)
    fresh = torch.full((p.numel(),), page, device=p.device).scatter_reduce(0, at, place % page, "amin")
    slot = torch.arange(page, device=p.device)
    old = (slot < fresh[:, None])[..., None, None]
    new = torch.zeros(p.numel(), page, dtype=torch.bool, device=p.device).index_put((at, place % page), torch.tensor(True, device=p.device))
    for name, x in (("k", k), ("v", s["new_v"].float())):
        held = s[name][0].view(torch.uint8).view(-1, page, *x.shape[1:])
        scale = s[name + "_scale"][0].view(torch.uint8)
        rows = torch.zeros(p.numel(), page, *x.shape[1:], device=p.device).index_put((at, place % page), x)
        had = torch.where((fresh > 0)[:, None], scale[p].int() - 127, -126)
        e = torch.maximum(had, _exponent(rows.abs().amax((1, 3)), dtype).int())  # [pages, heads]
        again = _codes(held[p].view(E4M3).float(), (e - had)[:, None, :, None])
        codes = _codes(rows, e[:, None, :, None])
        held[p] = torch.where(new[..., None, None], codes.view(torch.uint8),
                              torch.where(old, again.view(torch.uint8), held[p]))
        scale[p] = _byte(e)
    return {"q": q, **_stored(s)}


def _padded(s):
    """Index of each new token in [B, max_query], the flat positions of that layout and their validity."""
    start, m = s["query_start"].long(), s["max_query"]
    count = start.diff()
    i = torch.arange(m, device=start.device)
    valid = i < count[:, None]
    token = (s["lengths"].long() - count)[:, None] + i
    return (start[:-1, None] + i).clamp(max=int(s["q"].shape[0]) - 1), token, valid


def _plain_attend(s):
    c, page = s["case"], s["page"]
    flat, token, valid = _padded(s)
    b, hk, d = flat.shape[0], c["kv_heads"], c["head_dim"]
    j = torch.arange(s["max_length"], device=flat.device)
    inside = j < s["lengths"][:, None]
    rows = _slots(s["table"], torch.where(inside, j, 0), page)
    k, v = (s[name][0].view(torch.uint8)[rows].view(E4M3).float() *
            s[name + "_scale"][0].view(torch.uint8)[rows // page].view(E8M0).float()[..., None] for name in ("k", "v"))
    q = s["q"][flat].float().permute(0, 2, 1, 3)                                 # [B, heads, n, D]
    q = q.reshape(b, hk, -1, d).contiguous()
    k = k.permute(0, 2, 3, 1).contiguous()                                       # [B, kv, D, T]
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
    score = score.masked_fill(~see[:, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    w = torch.exp(score - top)
    total = w.sum(-1, keepdim=True)
    v = v.permute(0, 2, 1, 3).contiguous()                                       # [B, kv, T, D]
    out = (w.view(b, hk, -1, w.shape[-1]) @ v).view(b, c["query_heads"], -1, d) / total.clamp(min=1e-30)
    out = out.permute(0, 2, 1, 3)[valid].to(s["q"].dtype)
    if not c["lse"]:
        return {"out": out}
    return {"out": out, "lse": (torch.log(total) + top)[..., 0].permute(0, 2, 1)[valid]}


# ---------------------------------------------------------------------------
# The definition, in 64 bits: stored rows are elements over their scale before they are rounded
# ---------------------------------------------------------------------------


def _least_scale(top, case):
    """log2 of a page's scale, from the definition: the smallest power of two with 448 of it at least ``top``."""
    e = torch.ceil(torch.log2(top.double().clamp(min=1e-300) / 448.0) - 1e-12)
    e = torch.where(448.0 * 2.0 ** (e - 1) >= top, e - 1, e)
    e = torch.where(448.0 * 2.0 ** e < top, e + 1, e)
    return torch.where(top == 0, -126.0, e).clamp(-126, 7 if case["dtype"] == "fp16" else 127)


def exact(case, seed):
    s = prepare(case, seed)
    op, lengths, new, page = case["op"], *_requests(case), case["page"]
    tables = [[int(x) for x in r] for r in s["table"].tolist()]

    def slots(pages, first, stop, size=page):
        at = torch.arange(first, stop)
        return (torch.tensor(pages, dtype=torch.int64)[at // size] * size + at % size).cuda()

    if op == "quantize":
        return _exact_quantize(case, s, lengths, tables, slots)
    if op in ("append", "axes"):
        return _exact_store(case, s, lengths, new, tables, slots)
    group = case["query_heads"] // case["kv_heads"]
    out, lses, at = [], [], 0
    for b, (length, m) in enumerate(zip(lengths, new)):
        where = slots(tables[b], 0, length)
        pos = torch.arange(length - m, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        mask = key <= pos
        if case["window"]:
            mask &= pos - key < case["window"]
        if case["prefix"]:
            mask |= key < case["prefix"]
        per_head = []
        for h in range(case["query_heads"]):
            k, v = (s[n].double()[0, where, h // group] * s[n + "_scale"].double()[0, where // page, h // group, None]
                    for n in ("k", "v"))
            q = s["q"][at:at + m, h].double()
            x = q.mm(k.t().contiguous()) / math.sqrt(case["head_dim"])
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            if case["bias"]:
                x = x - 2.0 ** (-8.0 * (h + 1) / case["query_heads"]) * (pos - key).abs()
            x[~mask] = -math.inf
            norm = torch.logsumexp(x, 1, keepdim=True)
            per_head.append(((x - norm).exp().mm(v), norm[:, 0]))
        out.append(torch.stack([o for o, _ in per_head], 1))
        lses.append(torch.stack([z for _, z in per_head], 1))
        at += m
    return {"out": torch.cat(out), "lse": torch.cat(lses)} if case["lse"] else {"out": torch.cat(out)}


def _exact_quantize(case, s, lengths, tables, slots):
    got = {"lengths": None}
    source = [[int(x) for x in r] for r in s["source_table"].tolist()]
    page = case["page"]
    for name in ("k", "v"):
        codes, scales = s[name].double(), s[name + "_scale"].double()
        for b, length in enumerate(lengths):
            x = s["source_" + name][:, slots(source[b], 0, length, SOURCE_PAGE)].double()
            tops = torch.nn.functional.pad(x.abs().amax(-1), (0, 0, 0, -length % page))
            e = _least_scale(tops.unflatten(1, (-1, page)).amax(2), case)         # [L, pages, heads]
            at = torch.arange(length, device="cuda") // page
            codes[:, slots(tables[b], 0, length)] = x / (2.0 ** e)[:, at][..., None]
            scales[:, torch.tensor(tables[b][:e.shape[1]], device="cuda")] = 2.0 ** e
        got[name], got[name + "_scale"] = codes, scales
    return got


def _exact_store(case, s, lengths, new, tables, slots):
    dim, half, page = case["rotary_dim"], case["rotary_dim"] // 2, case["page"]
    pos = torch.cat([torch.arange(x - m, x, dtype=torch.float64) for x, m in zip(lengths, new)])[:, None].expand(-1, half)
    if case["op"] == "axes":
        sections = _sections(case)
        per = torch.zeros(half, dtype=torch.int64)
        for a in (1, 2):
            first = sum(sections[:a])
            per[slice(a, a + 3 * sections[a], 3) if case["cyclic"] else slice(first, first + sections[a])] = a
        pos = torch.stack([s["positions"].cpu().double()[int(a)] for a in per], 1)
    turn = torch.polar(torch.ones(1, dtype=torch.float64), pos * s["inv_freq"].cpu()[None, :]).cuda()[:, None]

    def spin(x):
        x = x.double()
        pairs = x[..., :dim].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        if not case["interleaved"]:
            z = z.transpose(-1, -2)
        return torch.cat((z.flatten(-2), x[..., dim:]), -1)

    got = {"q": spin(s["q"])}
    for name, rows in (("k", spin(s["new_k"])), ("v", s["new_v"].double())):
        held, at = s[name].double(), 0
        scales = s[name + "_scale"].double() if case["quantized"] else None
        for b, (x, m) in enumerate(zip(lengths, new)):
            mine, at = rows[at:at + m], at + m
            if not case["quantized"]:
                held[0, slots(tables[b], x - m, x)] = mine
                continue
            first, stop = (x - m) // page, -(-x // page)
            lead = (x - m) - first * page
            tops = torch.nn.functional.pad(mine.abs().amax(-1), (0, 0, lead, stop * page - x))
            e = _least_scale(tops.unflatten(0, (-1, page)).amax(1), case)         # [pages, heads]
            where = torch.tensor(tables[b][first:stop], device="cuda")
            if lead:
                had = scales[0, where[0]].clone()
                e[0] = torch.maximum(e[0], torch.log2(had))
                before = slots(tables[b], first * page, first * page + lead)
                held[0, before] = held[0, before] * (had / 2.0 ** e[0])[None, :, None]
            scales[0, where] = 2.0 ** e
            page_of = (torch.arange(x - m, x, device="cuda") // page) - first
            held[0, slots(tables[b], x - m, x)] = mine / (2.0 ** e)[page_of][..., None]
        got[name] = held
        if case["quantized"]:
            got[name + "_scale"] = scales
    return got
