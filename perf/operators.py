"""Attention over the blocks that a router chooses, as cases that can be timed: rotary positions applied to queries and
keys on their way into the cache (``append``), the choice of blocks by their statistics (``route``) and the attention of
each query over its chosen blocks and its local window (``attend``), each for one decode position, for rows with a
sequence and a position of their own, and for whole sequences.

``run`` with ``own`` false is the plain form in elementary tensor operations, with ``own`` true the calls that a user of
this library makes.  ``exact`` is the same in 64 bits, written apart from the plain form.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ROUTER_HEADS, ROUTER_WIDTH, BUCKETS = 4, 16, 12


# ---------------------------------------------------------------------------- the cases
#
# form: "decode" (every sequence at the same position), "rows" (each row its own sequence and position) or "prefill"
# (all positions of every sequence).


def _append(name, form, dtype, batch, rows, context, heads, kv_heads, width, rotary, interleaved):
    return {"name": name, "op": "append", "form": form, "dtype": dtype, "batch": batch, "rows": rows, "context": context,
            "heads": heads, "kv_heads": kv_heads, "width": width, "rotary": rotary, "interleaved": interleaved}


def _route(name, form, dtype, batch, rows, context, block, window, top, strict):
    return {"name": name, "op": "route", "form": form, "dtype": dtype, "batch": batch, "rows": rows, "context": context,
            "block": block, "window": window, "top": top, "strict": strict}


def _attend(name, form, dtype, batch, rows, context, heads, kv_heads, width, block, window, top, shared):
    return {"name": name, "op": "attend", "form": form, "dtype": dtype, "batch": batch, "rows": rows, "context": context,
            "heads": heads, "kv_heads": kv_heads, "width": width, "block": block, "window": window, "top": top,
            "shared": shared}


def listed():
    return [
        # one position of a handful of sequences: the launch is what counts
        _append("append, decode, 8 sequences", "decode", "bf16", 8, 8, 512, 8, 2, 64, 64, False),
        # whole sequences on their way into the cache, half of each head rotated
        _append("append, prefill, 8 x 4096", "prefill", "fp16", 8, 32768, 4096, 16, 4, 128, 64, True),
        # pieces of text of several sequences, far into a long cache, in single precision
        _append("append, rows, 1237 of 3", "rows", "fp32", 3, 1237, 65536, 12, 12, 64, 64, False),
        # one position of one sequence at the sizes of the decode benchmark
        _route("route, decode, 1 sequence", "decode", "bf16", 1, 1, 512, 32, 64, 2, True),
        # a decode batch of long sequences, each with a length of its own
        _route("route, rows, 256 long sequences", "rows", "fp16", 256, 256, 65536, 64, 512, 16, True),
        # every position of a batch of sequences
        _route("route, prefill, 8 x 4096", "prefill", "bf16", 8, 32768, 4096, 64, 64, 4, False),
        # one position of one sequence: latency
        _attend("attend, decode, 1 sequence", "decode", "bf16", 1, 1, 512, 8, 2, 64, 32, 64, 2, True),
        # a decode batch of long sequences, a choice for each key head
        _attend("attend, rows, 64 long sequences", "rows", "bf16", 64, 64, 32768, 32, 8, 128, 64, 512, 16, False),
        # rows of a few sequences in single precision, one key head for each query head
        _attend("attend, rows, 77 in fp32", "rows", "fp32", 5, 77, 1984, 12, 12, 64, 32, 100, 4, True),
        # whole sequences, grouped heads
        _attend("attend, prefill, 8 x 4096", "prefill", "bf16", 8, 32768, 4096, 8, 2, 64, 64, 64, 4, True),
        # whole sequences of an odd length, one key head under sixteen query heads
        _attend("attend, prefill, 3 x 1999", "prefill", "fp16", 3, 5997, 2048, 16, 1, 128, 64, 128, 8, False),
    ]


def _span(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "route", "attend"))
    form = rng.choice(("decode", "rows", "prefill"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    block = rng.choice((16, 32, 64))
    if form == "prefill":
        length = _span(rng, 40, 4096)
        batch = _span(rng, 1, max(1, min(8, 32768 // length)))
        context, rows = -(-length // block) * block, batch * length
    else:
        context = block * _span(rng, 3, 65536 // block)
        batch = _span(rng, 1, 256 if form == "decode" else 64)
        rows = batch if form == "decode" else min(_span(rng, 1, 1024), batch * (context // 2))
    name = f"{op}, {form}, {dtype}"
    window = _span(rng, 1, 512)
    top = _span(rng, 1, 16)
    if op == "route":
        return {**_route(name, form, dtype, batch, rows, context, block, window, top, rng.random() < 0.5)}
    width = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 8) if kv_heads < 8 else (1, 2, 4))
    if form != "prefill":                                # what a state holds: two caches
        batch = max(1, min(batch, (1 << 28) // (context * kv_heads * width)))
        rows = batch if form == "decode" else min(rows, batch * (context // 2))
    if op == "append":
        rotary = rng.choice((width, width // 2, width // 4))
        return _append(name, form, dtype, batch, rows, context, heads, kv_heads, width, rotary, rng.random() < 0.5)
    if form == "prefill":                                # no more work than the largest listed pass
        top = min(top, 8)
        window = min(window, 256)
        keys = top * block + window
        limit = max(1, 28_000_000 // (keys * kv_heads * width // 64))
        length = min(rows // batch, max(40, limit))
        batch = max(1, min(batch, limit // length))
        context, rows = -(-length // block) * block, batch * length
        if dtype == "fp32":
            heads = kv_heads * min(4, heads // kv_heads)
    else:
        rows = max(1, min(rows, 900_000 // ((top * block + window) * kv_heads)))
        if form == "decode":
            batch = rows
    return _attend(name, form, dtype, batch, rows, context, heads, kv_heads, width, block, window, top, rng.random() < 0.5)


# ---------------------------------------------------------------------------- what a program holds


def _positions(case):
    """(sequence, position) of every row, by the case alone."""
    batch, rows, context = case["batch"], case["rows"], case["context"]
    if case["form"] == "prefill":
        length = rows // batch
        return [(i // length, i % length) for i in range(rows)]
    if case["form"] == "decode":
        return [(i, context - 1 - context // 13) for i in range(rows)]
    # rows: distinct positions, spread over the last three quarters of each sequence
    per = -(-rows // batch)
    return [(i % batch, context - 1 - (i // batch) * max(1, (3 * context // 4) // per) % context) for i in range(rows)]


def _rows(case):
    batch, position = zip(*_positions(case))
    return (torch.tensor(batch, dtype=torch.int32, device="cuda"), torch.tensor(position, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, kind=dtype):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(kind)

    batch, rows, context = case["batch"], case["rows"], case["context"]
    state = {"case": case}
    state["row_batch"], state["row_position"] = _rows(case)
    if case["form"] == "decode":
        state["position"] = state["row_position"][:1].to(torch.int64).reshape(())
    if case["op"] == "route":
        blocks = context // case["block"]
        state["query"] = normal(rows, ROUTER_HEADS * ROUTER_WIDTH)
        state["mean"] = normal(batch, blocks, ROUTER_HEADS, ROUTER_WIDTH, scale=0.5)
        state["std"] = normal(batch, blocks, ROUTER_HEADS, ROUTER_WIDTH, scale=0.5).abs_()
        state["gamma"] = normal(ROUTER_HEADS, kind=torch.float32)
        state["bias"] = normal(ROUTER_HEADS, BUCKETS, kind=torch.float32)
        return state
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    state["query"] = normal(rows, heads, width)
    state["key_cache"] = normal(batch, context, kv_heads, width)
    state["value_cache"] = normal(batch, context, kv_heads, width)
    if case["op"] == "append":
        state["key"], state["value"] = normal(rows, kv_heads, width), normal(rows, kv_heads, width)
        # positions stretched by four, as for a context of four times the trained one
        steps = torch.arange(case["rotary"] // 2, dtype=torch.float64, device="cuda")
        state["frequencies"] = 0.25 * 10000.0 ** (-2.0 * steps / case["rotary"])
        return state
    # blocks as a router hands them out: distinct, whole and before the window, the better ones first, -1 where none is left;
    # neighbouring positions mostly agree
    block, top = case["block"], case["top"]
    blocks = context // block
    choices = 1 if case["shared"] else kv_heads
    group = (state["row_batch"].long() * 4096 + state["row_position"].long() // 16) % 8191
    score = torch.rand(8191, choices, blocks, generator=g, device="cuda")[group]
    score += 0.5 * torch.rand(rows, choices, blocks, generator=g, device="cuda")
    start = (state["row_position"].long() - case["window"] + 1).clamp_(min=0)
    whole = torch.arange(1, blocks + 1, device="cuda") * block <= start[:, None]
    score.masked_fill_(~whole[:, None], -1.0)
    found = score.topk(min(top, blocks), dim=-1)
    index = torch.full((rows, choices, top), -1, dtype=torch.int32, device="cuda")
    index[..., :found.indices.size(-1)] = torch.where(found.values >= 0, found.indices, -1).to(torch.int32)
    state["index"] = index.expand(rows, kv_heads, top)
    state["scale"] = 1.0 / math.sqrt(width)
    return state


# ---------------------------------------------------------------------------- one pass


def run(state):
    return {"append": _append_pass, "route": _route_pass, "attend": _attend_pass}[state["case"]["op"]](state)


def _library():
    package = os.path.join(os.getcwd(), "relation-lm_b200")
    if package not in sys.path:
        sys.path.insert(1, package)
    from relation_lm.kernels import block_attention

    return block_attention


def _where(state):
    """The arguments that say where the rows are, in the case's form."""
    case = state["case"]
    if case["form"] == "decode":
        return (state["position"],)
    if case["form"] == "rows":
        return (state["row_batch"], state["row_position"])
    return (case["rows"] // case["batch"],)


_SUFFIX = {"decode": "", "rows": "_rows", "prefill": "_prefill"}


def _append_pass(state):
    case = state["case"]
    q, k, v, k_cache, v_cache = (state[n] for n in ("query", "key", "value", "key_cache", "value_cache"))
    if own:
        call = getattr(_library(), "rotary_append" + _SUFFIX[case["form"]])
        out = call(q, k, v, k_cache, v_cache, state["frequencies"], *_where(state), case["interleaved"], 1.0)
        return out, k_cache, v_cache
    angle = state["row_position"].double()[:, None] * state["frequencies"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rotate(x):
        turned, rest = x[..., :case["rotary"]].float(), x[..., case["rotary"]:]
        if case["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = turned.chunk(2, -1)
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned.to(x.dtype), rest), -1)

    where = (state["row_batch"].long(), state["row_position"].long())
    k_cache[where] = rotate(k)
    v_cache[where] = v
    return rotate(q), k_cache, v_cache


def _route_pass(state):
    case = state["case"]
    block, window, top = case["block"], case["window"], case["top"]
    if own:
        call = getattr(_library(), "route_blocks" + _SUFFIX[case["form"]])
        return call(state["query"], state["mean"], state["std"], state["gamma"], state["bias"], *_where(state), block,
                    window, top, case["strict"])
    # in 64 bits: two blocks' scores may be near one another, and which is the larger decides
    batch, blocks = case["batch"], state["mean"].size(1)
    q = state["query"].double().view(-1, ROUTER_HEADS, ROUTER_WIDTH)
    mean, std = (state[n].double().permute(0, 2, 3, 1) for n in ("mean", "std"))           # [B, heads, width, blocks]
    if case["form"] == "rows":
        near, spread = (torch.matmul(x.unsqueeze(2), y[state["row_batch"].long()]).squeeze(2)
                        for x, y in ((q, mean), (q.abs(), std)))
    else:
        q = q.view(batch, -1, ROUTER_HEADS, ROUTER_WIDTH).transpose(1, 2)                   # [B, heads, positions, width]
        near, spread = (torch.matmul(x, y).transpose(1, 2).reshape(-1, ROUTER_HEADS, blocks)
                        for x, y in ((q, mean), (q.abs(), std)))
    soft = torch.log1p(state["gamma"].double().exp())
    t = state["row_position"].long()[:, None]
    last = torch.arange(1, blocks + 1, device="cuda") * block - 1
    bucket = torch.frexp((t - last).clamp(min=0).add(1).double())[1].sub(1).long().clamp(max=BUCKETS - 1)
    head = (near + soft[:, None] * spread) * 0.25 + state["bias"].double()[:, bucket].transpose(0, 1)
    score = head.exp().sum(1).log()
    able = last <= t
    if case["strict"]:
        able = able & (last < (t - window + 1).clamp(min=0))
    score = torch.where(able, score, -math.inf)
    value, index = score.sort(dim=-1, descending=True, stable=True)
    value, index = value[:, :top], index[:, :top]
    if top > blocks:
        value = torch.nn.functional.pad(value, (0, top - blocks), value=-math.inf)
        index = torch.nn.functional.pad(index, (0, top - blocks))
    return torch.where(value > -math.inf, index, -1).to(torch.int32), value.float()


def _attend_pass(state):
    case = state["case"]
    block, window, kv_heads = case["block"], case["window"], case["kv_heads"]
    q, k_cache, v_cache, index = (state[n] for n in ("query", "key_cache", "value_cache", "index"))
    if own:
        call = getattr(_library(), "block_attention" + _SUFFIX[case["form"]])
        return call(q, k_cache, v_cache, index, *_where(state), block, window, state["scale"])
    rows = q.size(0)
    t = state["row_position"].long()
    start = (t - window + 1).clamp(min=0)
    near = start[:, None] + torch.arange(window, device="cuda")
    far = index.long()[..., None] * block + torch.arange(block, device="cuda")              # [rows, kv, top, block]
    place = torch.cat((far.flatten(2), near[:, None].expand(-1, kv_heads, -1)), -1)
    live = torch.cat(((far >= 0).logical_and_(far < start[:, None, None, None]).flatten(2),
                      (near <= t[:, None])[:, None].expand(-1, kv_heads, -1)), -1)
    where = (state["row_batch"].long()[:, None, None], place.clamp_(0, k_cache.size(1) - 1),
             torch.arange(kv_heads, device="cuda")[:, None])
    k = k_cache[where].float()                                                              # [rows, kv, keys, width]
    grouped = q.float().view(rows, kv_heads, -1, q.size(2))
    score = torch.matmul(grouped, k.transpose(2, 3)).mul_(state["scale"])
    del k
    score.masked_fill_(~live[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v_cache[where].float()).div_(total)
    return out.view_as(q).to(q.dtype), (total.log() + top).view(rows, -1)


# ---------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    rows, batch, context = case["rows"], case["batch"], case["context"]
    if case["op"] == "append":
        q, kv = rows * case["heads"] * case["width"], rows * case["kv_heads"] * case["width"]
        turned = rows * (case["heads"] + case["kv_heads"]) * case["rotary"]
        return {"bytes": e * (2 * q + 4 * kv), "flops": 3 * turned}
    block, window, top = case["block"], case["window"], case["top"]
    places = _positions(case)
    if case["op"] == "route":
        able = [min(context, t + 1) // block for _, t in places]
        if case["form"] == "prefill":
            read = batch * (max(able) if able else 0)
        else:
            most = {}
            for (b, _), n in zip(places, able):
                most[b] = max(most.get(b, 0), n)
            read = sum(most.values())
        return {"bytes": e * 64 * (rows + 2 * read) + 8 * rows * top, "flops": sum(able) * (4 * 64 + 4 * 8)}
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    keys = [min(window, t + 1) + block * min(top, max(0, t + 1 - window) // block) for _, t in places]
    total = sum(keys)
    cached = batch * min(context, max(t for _, t in places) + 1)       # no more than what the caches hold
    choices = 1 if case["shared"] else kv_heads
    return {"bytes": 2 * e * kv_heads * width * min(total, cached) + 2 * e * rows * heads * width + 4 * rows * heads
                     + 4 * rows * choices * top,
            "flops": 4 * width * heads * total}


# ---------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _append_exact, "route": _route_exact, "attend": _attend_exact}[case["op"]](case, state)


def _append_exact(case, state):
    """Pairs of components as complex numbers, turned by exp(i angle)."""
    half = case["rotary"] // 2
    angle = state["row_position"].double().view(-1, 1, 1) * state["frequencies"].view(1, 1, half)
    turn = torch.polar(torch.ones_like(angle), angle)

    def rotated(x):
        x = x.double()
        y = x.clone()
        one = slice(0, case["rotary"], 2) if case["interleaved"] else slice(0, half)
        two = slice(1, case["rotary"], 2) if case["interleaved"] else slice(half, case["rotary"])
        z = torch.complex(x[..., one], x[..., two]) * turn
        y[..., one], y[..., two] = z.real, z.imag
        return y

    keys, values = state["key_cache"].double(), state["value_cache"].double()
    flat = state["row_batch"].long() * case["context"] + state["row_position"].long()
    keys.flatten(0, 1).index_copy_(0, flat, rotated(state["key"]))
    values.flatten(0, 1).index_copy_(0, flat, state["value"].double())
    return rotated(state["query"]), keys, values


def _route_exact(case, state):
    """A sequence at a time: the scores as one product of queries and (mean, spread), the choice by counting better blocks."""
    top, block = case["top"], case["block"]
    blocks = state["mean"].size(1)
    soft = torch.nn.functional.softplus(state["gamma"].double()).view(1, -1, 1)
    end = (torch.arange(blocks, device="cuda") + 1) * block - 1
    index = torch.full((case["rows"], top), -1, dtype=torch.int32, device="cuda")
    value = torch.full((case["rows"], top), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        mine = (state["row_batch"] == b).nonzero()[:, 0]
        if not mine.numel():
            continue
        q = state["query"][mine].double().view(-1, ROUTER_HEADS, ROUTER_WIDTH)
        both = torch.cat((state["mean"][b].double(), soft.view(1, -1, 1) * state["std"][b].double()), -1)
        raw = torch.einsum("rhw,nhw->rhn", torch.cat((q, q.abs()), -1), both) / 4
        t = state["row_position"][mine].long().view(-1, 1)
        away = (t - end).clamp(min=0) + 1
        bucket = sum((away >= 1 << i).long() for i in range(1, BUCKETS))
        raw = raw + state["bias"].double().t()[bucket].permute(0, 2, 1)
        score = torch.logsumexp(raw, 1)
        limit = (t - case["window"]).clamp(min=-1) if case["strict"] else t
        score = torch.where(end <= limit, score, -math.inf)
        best, at = score.topk(min(top, blocks), dim=-1)
        index[mine, :best.size(1)] = torch.where(best > -math.inf, at, -1).to(torch.int32)
        value[mine, :best.size(1)] = best
    return index, value


def _attend_exact(case, state):
    """Every position of the cache against every row, a mask for those that a row may see; a key head of a sequence at a time."""
    if case["rows"] * case["heads"] * case["context"] > 3e9:
        return None
    block, window, kv_heads = case["block"], case["window"], case["kv_heads"]
    group = case["heads"] // kv_heads
    where = torch.arange(case["context"], device="cuda")
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(state["query"].shape[:2], dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        mine = (state["row_batch"] == b).nonzero()[:, 0]
        for piece in mine.split(1024):
            t = state["row_position"][piece].long()[:, None]
            near = (where <= t) & (where > t - window)
            before = where <= t - window
            for h in range(kv_heads):
                picked = state["index"][piece, h].long()
                chosen = torch.zeros(len(piece), case["context"] // block + 1, dtype=torch.bool, device="cuda")
                chosen.scatter_(1, torch.where(picked >= 0, picked, chosen.size(1) - 1), True)
                seen = near | (before & chosen[:, where // block] & (where // block < chosen.size(1) - 1))
                key, value = state["key_cache"][b, :, h].double(), state["value_cache"][b, :, h].double()
                for j in range(h * group, (h + 1) * group):
                    s = state["query"][piece, j].double() @ key.t() * state["scale"]
                    s = torch.where(seen, s, -math.inf)
                    lse[piece, j] = torch.logsumexp(s, -1)
                    out[piece, j] = torch.softmax(s, -1) @ value
    return out, lse
