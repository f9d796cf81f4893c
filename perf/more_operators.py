"""Drafted tokens' trees over the paged key and value cache, and the eviction
of positions from it by the attention they have gathered, as cases to time and
to check: what each reads, writes and computes, its plain form in elementary
torch operations, and its definition in 64 bits.

- `tree` (`HipOps.attentionTree`): attention of drafted tokens over the cache.
  A row sees the positions before its sequence's drafted tokens, and of those
  the ones whose bits its mask has (its ancestors and itself);
- `mass` (`HipOps.attentionMass`): what each cached position gathers of the
  rows' attention, summed over the rows and the heads that share a key head,
  added to what it had;
- `heaviest` (`HipOps.heaviest`): a sequence's positions to keep, for each key
  head: its first, its last, and the heaviest of those between;
- `keep` (`HipOps.cacheKeep`): the kept positions' keys and values moved
  together, in place or into other pages: a verified path of drafted tokens,
  or what an eviction leaves.

A case's `tokens` counts the new rows of the whole call. `context` is the
positions before them: the most that any sequence has, the others' shorter.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# (heads, key heads, values a head)
HEADS = ((32, 8, 128), (28, 4, 128), (16, 2, 256), (16, 4, 64), (24, 24, 128), (12, 3, 80), (9, 3, 72), (8, 1, 96))


def _case(name, op, dtype, cache, sequences, tokens, context, heads, page, window=0, sinks=0, keep=0, into=False):
    return {"name": name, "op": op, "type": dtype, "cache": cache, "sequences": sequences, "tokens": tokens,
            "context": context, "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "page": page,
            "window": window, "sinks": sinks, "keep": keep, "into": into}


def listed():
    return [
        # one conversation's drafted tokens early on: the smallest call, where latency counts
        _case("tree one", "tree", "bf16", "f16", 1, 8, 517, (32, 8, 128), 16),
        # a server's step that checks a small tree for each of 32 conversations
        _case("tree batch", "tree", "bf16", "f16", 32, 601, 8000, (32, 8, 128), 16),
        # wide trees, groups of 7 heads, over the 8-bit cache
        _case("tree wide i8", "tree", "bf16", "i8", 16, 811, 4000, (28, 4, 128), 64),
        # a windowed layer's trees in the runner's own activations (F32), 2 key heads of 256
        _case("tree window f32", "tree", "f32", "f16", 5, 63, 12345, (16, 2, 256), 32, 1024, 4),
        # a decode step's attention added to what 64 conversations' positions have gathered
        _case("mass step", "mass", "bf16", "f16", 64, 64, 8000, (32, 8, 128), 16),
        # a long prompt's positions weighed by its last 64 tokens
        _case("mass last rows", "mass", "bf16", "f16", 1, 64, 32000, (32, 8, 128), 64),
        # a long prompt's positions weighed by all of it: the largest
        _case("mass prompt", "mass", "bf16", "f16", 1, 8192, 0, (32, 8, 128), 16),
        # chunks and single tokens in one call over the 8-bit cache, in F32
        _case("mass mixed i8", "mass", "f32", "i8", 24, 1811, 3000, (16, 4, 64), 16),
        # a conversation cut to 512 positions: a small call again
        _case("heaviest one", "heaviest", "f32", "f16", 1, 0, 1900, (32, 8, 128), 16, keep=512),
        # 48 conversations cut to 2,048 positions each
        _case("heaviest batch", "heaviest", "f32", "f16", 48, 0, 16000, (32, 8, 128), 16, keep=2048),
        # the accepted path of each of 32 conversations' trees
        _case("keep accepted", "keep", "f32", "f16", 32, 64, 8000, (32, 8, 128), 16, keep=7),
        # 32 conversations' caches cut in place, with the masses of what is kept
        _case("keep evicted i8", "keep", "f32", "i8", 32, 0, 8000, (32, 8, 128), 16, keep=2048),
    ]


# What a drawn case may cost, as the largest listed one: visible pairs times
# heads times values a head; and, for the plain form's memory, its scores.
MOST_PAIR_VALUES = 8192 * 8193 // 2 * 32 * 128
MOST_SCORES = 8192 * 8192 * 32
MOST_CACHE = 1 << 28  # values of the keys


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    while True:
        op = rng.choice(("tree", "tree", "mass", "mass", "heaviest", "keep"))
        heads, page = rng.choice(HEADS), rng.choice((16, 16, 32, 48, 64, 128))
        cache, dtype = rng.choice(("f16", "i8")), rng.choice(("f32", "bf16"))
        sequences, context = rng.choice((1, log_int(2, 64))), log_int(1, 32000)
        window = sinks = keep = tokens = 0
        into = False
        if op == "tree":
            tokens = max(sequences, int(sequences * log_int(1, 160) * rng.uniform(0.5, 1.0)))
            window = log_int(16, 8192) if rng.random() < 0.3 else 0
            sinks = rng.choice((0, 1, 4, 37)) if window else 0
        elif op == "mass":
            tokens = sequences if rng.random() < 0.5 else max(sequences, log_int(1, 8192))
        elif op == "heaviest":
            context, dtype, cache = log_int(16, 131072), "f32", "f16"
            keep = log_int(8, max(context // 2, 9))
        else:
            context, dtype, into = max(context, 64), "f32", rng.random() < 0.4
            if rng.random() < 0.4:
                tokens, keep = 64, rng.randint(1, 9)  # the accepted path of a tree of 64
            else:
                keep = log_int(8, context * 3 // 10)
        c = _case("", op, dtype, cache, sequences, tokens, context, heads, page, window, sinks, keep, into)
        del c["name"]
        most, count = int(_new_tokens(c).max()) if tokens else 0, sequences
        positions = count * (context + most + 2 * page + (keep + page if into else 0))
        if positions * heads[1] * (1 if op == "heaviest" else heads[2]) > MOST_CACHE:
            continue
        if op in ("tree", "mass"):
            scores = count * most * (context + most) * heads[0]
            if scores > MOST_SCORES or _pairs(c) * heads[0] * heads[2] > MOST_PAIR_VALUES:
                continue
        return c


# ------------------------------------------------------------------ a case's layout

def _new_tokens(case):
    """New tokens of each sequence."""
    count, tokens = case["sequences"], case["tokens"]
    if case["op"] == "keep":  # a tree of so many each, one path of which is kept
        return np.full(count, tokens, np.int64)
    each = np.ones(count, np.int64)
    if count == 1:
        each[0] = tokens
    elif tokens > count:
        # a tree's sizes uneven; of a mass, every fourth sequence brings a chunk
        more = np.arange(0, count, 1 if case["op"] == "tree" else 4)
        share = 1.0 + np.random.RandomState(count).random_sample(len(more))
        extra = np.floor(share / share.sum() * (tokens - count)).astype(np.int64)
        extra[0] += tokens - count - extra.sum()
        each[more] += extra
    return each


def _starts(case):
    """Positions each sequence holds before its new tokens."""
    count, context = case["sequences"], case["context"]
    low = 0.05 if case["op"] in ("tree", "mass") else 0.62
    share = np.random.RandomState(1000 + count).random_sample(count)
    starts = np.floor(context * (low + (1 - low) * share)).astype(np.int64)
    starts[-1] = context
    return starts


def _trees(case):
    """What each drafted token sees of its sequence's, as rows of bits [tokens, 64-bit words]: itself and its
    ancestors."""
    each = _new_tokens(case)
    words = -(-int(each.max()) // 64)
    rows = np.zeros((int(each.sum()), words), np.uint64)
    rng = np.random.RandomState(7 + int(each.sum()))
    first = 0
    for n in each:
        for i in range(int(n)):
            if i > 0:  # a child of one of the last eight, or of any before
                low = max(0, i - 8) if rng.random_sample() < 0.7 else 0
                rows[first + i] = rows[first + rng.randint(low, i)]
            rows[first + i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
        first += int(n)
    return rows


def _seen_of(rows):
    return np.unpackbits(rows.view(np.uint8), axis=1).sum(1).astype(np.int64)


def _pairs(case):
    """Visible (token, position) pairs."""
    starts, each = _starts(case), _new_tokens(case)
    start = np.repeat(starts, each)
    if case["op"] == "mass":
        at = start + np.arange(each.sum()) - np.repeat(np.cumsum(each) - each, each)
        return int((at + 1).sum())
    own_seen = _seen_of(_trees(case))
    seen = start
    if case["window"]:
        low = np.clip(start + own_seen - case["window"], 0, start)
        seen = start - low + np.minimum(case["sinks"], low)
    return int((seen + own_seen).sum())


def _lengths(case):
    return _starts(case) + (_new_tokens(case) if case["tokens"] else 0)


def _kept(case):
    """Rows that a `keep` leaves each sequence."""
    count, keep = case["sequences"], case["keep"]
    if case["tokens"]:  # accepted paths of 1 to `keep` tokens
        return np.random.RandomState(3 + count).randint(1, keep + 1, count).astype(np.int64)
    return np.full(count, keep, np.int64)


def work(case):
    kv, dim, count = case["kv_heads"], case["dim"], case["sequences"]
    row = dim * 2 if case["cache"] == "f16" else dim + 4  # a position's key, or value, of a head as cached
    lengths = _lengths(case)
    tables = 4 * int(np.ceil(lengths / case["page"]).sum())
    if case["op"] == "heaviest":
        return {"bytes": int(lengths.sum()) * kv * 4 + tables + 4 * count * (kv * case["keep"] + 2), "flops": 0}
    if case["op"] == "keep":
        moved = int(_kept(case).sum()) * kv
        listed_rows = count * case["keep"] * (1 if case["tokens"] else kv)
        mass = 0 if case["tokens"] else 8 * moved
        return {"bytes": 2 * moved * 2 * row + mass + 4 * listed_rows, "flops": 0}
    wide = 4 if case["type"] == "f32" else 2
    query = case["tokens"] * case["heads"] * dim * wide
    if case["op"] == "mass":
        cached = int(lengths.sum()) * kv
        return {"bytes": query + cached * (row + 4) + int(_starts(case).sum()) * kv * 4 + tables,
                "flops": 2 * _pairs(case) * case["heads"] * dim}
    positions = lengths
    if case["window"]:
        low = np.maximum(_starts(case) + 1 - case["window"], 0)
        positions = lengths - low + np.minimum(case["sinks"], low)
    return {"bytes": 2 * query + int(positions.sum()) * kv * 2 * row + tables + _trees(case).nbytes,
            "flops": 4 * _pairs(case) * case["heads"] * dim}


# ------------------------------------------------------------------ inputs

def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)

    def ints(x):
        return torch.from_numpy(np.ascontiguousarray(x)).to(DEV, torch.int32)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=DEV, dtype=torch.float32)

    op, kv, dim, page = case["op"], case["kv_heads"], case["dim"], case["page"]
    starts, lengths, count = _starts(case), _lengths(case), case["sequences"]
    used = -(-lengths // page)
    room = -(-(starts * bool(case["tokens"]) + case["keep"]) // page) * case["into"]  # of the pages moved into
    columns, pages = int(used.max()), int(used.sum() + room.sum()) + 3
    # each sequence's pages among the cache's, in no order; entries past its last page name no page
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)

    def tables_of(used, pages_of):
        tables = torch.full((count, max(int(used.max()), 1)), -1, dtype=torch.int32, device=DEV)
        filled = torch.arange(tables.shape[1], device=DEV)[None, :] < torch.from_numpy(used).to(DEV)[:, None]
        tables[filled] = pages_of
        return tables

    s = {"case": case, "tables": tables_of(used, order[:int(used.sum())]), "starts": ints(starts),
         "lengths": ints(lengths)}
    if op == "heaviest":
        # a few positions gather most of a head's attention
        s["mass"] = torch.exp(2.5 * normal(pages, kv, page))
        s["kept"] = torch.zeros(count, kv, case["keep"], dtype=torch.int32, device=DEV)
        s["counts"] = torch.zeros(count, dtype=torch.int32, device=DEV)
        return s
    # keys after their norm and rotation have values about 1, with some strong channels; one draw serves all pages
    # in turns of a prime length, so that making a large cache stays quick
    channels = 1.0 + 2.0 * (uniform(kv, dim) < 0.05)
    turns = torch.arange(pages, device=DEV) % min(pages, 509)
    if case["cache"] == "f16":
        s["keys"] = (normal(min(pages, 509), page, kv, dim) * channels).half()[turns]
        s["values"] = normal(min(pages, 509), kv, dim, page).half()[turns]
    else:
        def codes(*shape):
            return torch.randint(-127, 128, (min(pages, 509),) + shape, generator=gen, device=DEV,
                                 dtype=torch.int8)[turns]

        s["keys"], s["values"] = codes(page, kv, dim), codes(kv, dim, page)
        s["key_scales"] = (0.5 + uniform(pages, kv, page)) * 2.0 / 127
        s["value_scales"] = (0.5 + uniform(pages, kv, page)) * 2.5 / 127
    if op == "keep":
        keep = case["keep"]
        s["counts"] = ints(_kept(case))
        if case["tokens"]:
            # an accepted path's places among the drafted tokens: the first, then such as lie past the path's own
            # length, so that moving them a second time leaves them as they are
            path = torch.rand(count, case["tokens"] - keep, generator=gen, device=DEV).argsort(1)[:, :keep - 1]
            path = torch.cat([torch.zeros(count, 1, device=DEV, dtype=torch.int64), path.sort(1).values + keep], 1)
            s["kept"] = (s["starts"].long()[:, None] + path).to(torch.int32)
            s["to"] = s["starts"]
        else:
            # the first four, then such as lie past the kept ones' number, for the same reason
            draws = uniform(count, kv, int(lengths.max()))
            draws.masked_fill_(torch.arange(draws.shape[2], device=DEV) >= s["lengths"][:, None, None], -1.0)
            draws[:, :, :keep] = -1.0
            far = draws.topk(keep - 4, dim=2).indices.sort(2).values
            near = torch.arange(4, device=DEV).expand(count, kv, 4)
            s["kept"] = torch.cat([near, far], 2).to(torch.int32)
            s["to"] = torch.zeros_like(s["starts"])
            s["mass"] = torch.exp(2.5 * normal(pages, kv, page))
        s["into"] = tables_of(room, order[int(used.sum()):int(used.sum() + room.sum())]) if case["into"] else s["tables"]
        return s
    each = _new_tokens(case)
    s["offsets"] = ints(np.concatenate([[0], np.cumsum(each)]))
    # queries sharp enough that a few positions carry most of a row
    s["queries"] = normal(case["tokens"], case["heads"], dim, dtype=TYPES[case["type"]], scale=2.0)
    s["scale"] = 1.0 / math.sqrt(dim)
    if op == "tree":
        s["sees"] = torch.from_numpy(_trees(case).view(np.int32)).to(DEV)
        s["out"] = torch.zeros_like(s["queries"])
    else:
        s["before"] = 0.01 * torch.exp(2.5 * normal(pages, kv, page))
        s["mass"] = torch.zeros(pages, kv, page, device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from drift_amd import ops as d

        s["hip"] = d.HipOps()
        if case["op"] != "heaviest":
            if case["cache"] == "f16":
                s["cache"] = d.KvCache(s["keys"], s["values"], case["page"])
            else:
                s["cache"] = d.QuantizedKvCache(s["keys"], s["values"], s["key_scales"], s["value_scales"],
                                                case["page"])
        s["window"] = d.AttentionWindow(case["window"], case["sinks"]) if case["window"] else None
        if case["op"] in ("tree", "mass"):
            step = case["tokens"] == case["sequences"]
            s["batch"] = d.Sequences(s["tables"], s["starts"], None if step else s["offsets"])
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    op = s["case"]["op"]
    if own:
        hip = s["hip"]
        if op == "tree":
            hip.attentionTree(s["queries"], s["cache"], s["batch"], s["sees"], s["scale"], s["out"], s["window"])
        elif op == "mass":
            hip.attentionMass(s["queries"], s["cache"], s["batch"], s["scale"], s["mass"], s["before"])
        elif op == "heaviest":
            hip.heaviest(s["mass"], s["tables"], s["lengths"], min(4, s["case"]["keep"] // 4), s["case"]["keep"] // 4,
                         s["kept"], s["counts"])
        else:
            hip.cacheKeep(s["cache"], s["tables"], s["kept"], s["counts"], s["to"],
                          s["into"] if s["case"]["into"] else None, s.get("mass"))
    else:
        {"tree": _plain_tree, "mass": _plain_mass, "heaviest": _plain_heaviest, "keep": _plain_keep}[op](s)
    return {what: s[what] for what in {"tree": ("out",), "mass": ("mass",), "heaviest": ("kept", "counts"),
                                       "keep": ("keys", "values", "key_scales", "value_scales", "mass")}[op]
            if what in s}


def _columns(s):
    """Every sequence's rows side by side, as many columns as the most rows that one has: the token row of each
    (clamped where it has none), and which there are."""
    offsets, most = s["offsets"].long(), int(_new_tokens(s["case"]).max())
    column = torch.arange(most, device=DEV)
    rows = (offsets[:-1, None] + column).clamp(max=s["case"]["tokens"] - 1)
    return rows, column < (offsets[1:] - offsets[:-1])[:, None]


def _plain_scores(s, seen):
    """Scores of every sequence's rows [sequences, kv, rows, group, length], -infinity where not `seen`
    [sequences, rows, length]."""
    c, tables = s["case"], s["tables"].clamp(min=0).long()
    kv, dim, group, count = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"], tables.shape[0]
    keys = s["keys"][tables].float()
    if c["cache"] == "i8":  # scales [sequences, pages, kv, page]
        keys = keys * s["key_scales"][tables].permute(0, 1, 3, 2)[..., None]
    length = tables.shape[1] * c["page"]
    k = keys.reshape(count, length, kv, dim).permute(0, 2, 3, 1).contiguous().view(count * kv, dim, length)
    rows, _ = _columns(s)
    most = rows.shape[1]
    q = s["queries"].float()[rows]  # [sequences, most, heads, dim]
    q = q.view(count, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(count * kv, most * group, dim)
    scores = torch.bmm(q, k).mul_(s["scale"]).view(count, kv, most, group, length)
    return scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)


def _plain_weights(scores):
    """In place: the exponentials of scores less their rows' largest; and their sums."""
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    return scores.sum(-1, keepdim=True)


def _plain_tree(s):
    c, tables = s["case"], s["tables"].clamp(min=0).long()
    kv, dim, group, count = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"], tables.shape[0]
    length = tables.shape[1] * c["page"]
    rows, there = _columns(s)
    start = s["starts"].long()[:, None, None]
    j = torch.arange(length, device=DEV)
    bits = s["sees"][rows]  # [sequences, most, words]
    mine = (bits[..., None] >> torch.arange(32, device=DEV) & 1).flatten(2).bool()
    mine &= torch.arange(mine.shape[2], device=DEV) < there.sum(1)[:, None, None]
    nth = (j - start).clamp(min=0, max=mine.shape[2] - 1).expand(count, rows.shape[1], length)
    seen = (j >= start) & (j < start + mine.shape[2]) & mine.gather(2, nth)
    cached = j < start
    if c["window"]:
        at = start + mine.sum(2, keepdim=True) - 1
        cached = cached & ((j > at - c["window"]) | (j < c["sinks"]))
    scores = _plain_scores(s, seen | cached)
    total = _plain_weights(scores)
    values = s["values"][tables].float()
    if c["cache"] == "i8":
        values = values * s["value_scales"][tables][..., None, :]
    v = values.permute(0, 2, 1, 4, 3).contiguous().view(count * kv, length, dim)
    most = rows.shape[1]
    out = torch.bmm(scores.view(count * kv, most * group, length), v).view(count, kv, most, group, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 2, 1, 3, 4).reshape(count, most, c["heads"], dim)
    s["out"][rows[there]] = out[there].to(s["out"].dtype)


def _plain_mass(s):
    c, tables = s["case"], s["tables"].long()
    length = tables.shape[1] * c["page"]
    rows, there = _columns(s)
    start = s["starts"].long()[:, None]
    j = torch.arange(length, device=DEV)
    at = start + torch.arange(rows.shape[1], device=DEV)
    scores = _plain_scores(s, (j <= at[..., None]) & there[..., None])
    total = _plain_weights(scores)
    gathered = scores.div_(torch.where(total > 0, total, torch.ones_like(total))).sum((2, 3))  # [sequences, kv, length]
    held = s["before"][tables.clamp(min=0)].permute(0, 2, 1, 3).flatten(2)
    gathered = torch.where((j < start)[:, None], held + gathered, gathered)
    mine = j < start + there.sum(1)[:, None]
    which, where = mine.nonzero(as_tuple=True)
    s["mass"][tables[which, where // c["page"]], :, where % c["page"]] = gathered.transpose(1, 2)[which, where]


def _plain_heaviest(s):
    c, keep = s["case"], s["case"]["keep"]
    sinks, recent = min(4, keep // 4), keep // 4
    mass = s["mass"][s["tables"].clamp(min=0).long()].permute(0, 2, 1, 3).flatten(2)  # [sequences, kv, length]
    j = torch.arange(mass.shape[2], device=DEV)
    length = s["lengths"].long()[:, None, None]
    mass = torch.where((j < sinks) | (j >= length - recent), math.inf, mass)
    mass = torch.where(j < length, mass, -math.inf)
    order = mass.sort(dim=2, descending=True, stable=True).indices
    count = length.clamp(max=keep)
    order = order[:, :, :keep]
    if order.shape[2] < keep:
        order = torch.cat([order, order.new_zeros(*order.shape[:2], keep - order.shape[2])], 2)
    nth = torch.arange(keep, device=DEV)
    order = torch.where(nth < count, order, mass.shape[2]).sort(2).values
    s["kept"].copy_(torch.where(nth < count, order, -1))
    s["counts"].copy_(count[:, 0, 0])


def _plain_keep(s):
    c, page = s["case"], s["case"]["page"]
    kv, kept = c["kv_heads"], s["kept"].long()
    if kept.dim() == 2:
        kept = kept[:, None].expand(-1, kv, -1)
    nth = torch.arange(kept.shape[2], device=DEV)
    which, head, row = (nth < s["counts"][:, None, None]).expand_as(kept).nonzero(as_tuple=True)
    source, to = kept[which, head, row], s["to"].long()[which] + row
    source_page, to_page = s["tables"].long()[which, source // page], s["into"].long()[which, to // page]
    source, to = source % page, to % page
    s["keys"][to_page, to, head] = s["keys"][source_page, source, head]
    s["values"][to_page, head, :, to] = s["values"][source_page, head, :, source]
    for what in ("key_scales", "value_scales", "mass"):
        if what in s:
            s[what][to_page, head, to] = s[what][source_page, head, source]


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    if case["op"] == "heaviest":
        return None  # whole numbers alone
    s = _inputs(case, seed)
    starts, lengths = _starts(case), _lengths(case)
    page, kv, group = case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]

    if case["op"] == "keep":
        # sequence by sequence, every head's rows taken out of a copy of the cache as it was
        kept, counts = s["kept"].cpu().numpy(), _kept(case)
        table, into, to = s["tables"].cpu().numpy(), s["into"].cpu().numpy(), s["to"].cpu().numpy()
        names = [w for w in ("keys", "values", "key_scales", "value_scales", "mass") if w in s]
        old = {w: s[w].clone() for w in names}
        for n in range(case["sequences"]):
            there = to[n] + np.arange(counts[n])
            for h in range(kv):
                at = (kept[n] if kept.ndim == 2 else kept[n, h])[:counts[n]]
                a, b = (torch.from_numpy(x.astype(np.int64)).to(DEV) for x in (table[n, at // page], at % page))
                p, q = (torch.from_numpy(x.astype(np.int64)).to(DEV) for x in (into[n, there // page], there % page))
                s["keys"][p, q, h] = old["keys"][a, b, h]
                for w in names[1:]:
                    if w == "values":
                        s[w][p, h, :, q] = old[w][a, h, :, b]
                    else:
                        s[w][p, h, q] = old[w][a, h, b]
        return {w: s[w].double() if s[w].dtype != torch.int8 else None for w in names}

    def dense(n, length, what):
        """Sequence n's cached keys or values, [kv, length, dim] in 64 bits."""
        table = s["tables"][n, :-(-length // page)].long()
        x = s[what][table].double()
        if what == "keys":
            x = x.permute(2, 0, 1, 3).reshape(kv, -1, case["dim"])
        else:
            x = x.permute(1, 0, 3, 2).reshape(kv, -1, case["dim"])
        if case["cache"] == "i8":
            scales = s["key_scales" if what == "keys" else "value_scales"][table].double()
            x = x * scales.permute(1, 0, 2).reshape(kv, -1, 1)
        return x[:, :length]

    each = _new_tokens(case)
    first = np.cumsum(each) - each
    tree = np.unpackbits(_trees(case).view(np.uint8), axis=1, bitorder="little") if case["op"] == "tree" else None
    out = torch.zeros(s["queries"].shape, dtype=torch.float64, device=DEV)
    mass = torch.zeros(s["keys"].shape[0], kv, page, dtype=torch.float64, device=DEV)
    for n in range(len(starts)):
        start, length = int(starts[n]), int(lengths[n])
        k = dense(n, length, "keys")
        v = dense(n, length, "values") if case["op"] == "tree" else None
        j = torch.arange(length, device=DEV)
        gathered = torch.zeros(kv, length, dtype=torch.float64, device=DEV)
        for a in range(0, int(each[n]), 1024):
            b = min(a + 1024, int(each[n]))
            rows = slice(int(first[n]) + a, int(first[n]) + b)
            if tree is None:
                hidden = j > torch.arange(start + a, start + b, device=DEV)[:, None]
            else:
                bits = torch.from_numpy(tree[rows, :int(each[n])].astype(bool)).to(DEV)
                hidden = torch.zeros(b - a, length, dtype=torch.bool, device=DEV)
                hidden[:, start:] = ~bits
                if case["window"]:
                    last = start - 1 + bits.sum(1, keepdim=True)
                    hidden |= (j < start) & (j <= last - case["window"]) & (j >= case["sinks"])
            for h in range(case["heads"]):
                logits = s["queries"][rows, h].double() @ k[h // group].T.contiguous() * s["scale"]
                logits[hidden] = -math.inf
                p = torch.softmax(logits, -1)
                if tree is None:
                    gathered[h // group] += p.sum(0)
                else:
                    out[rows, h] = p @ v[h // group]
        if tree is None:
            table = s["tables"][n].long()[j // page]
            held = s["before"][table, :, j % page].double().T
            held[:, start:] = 0.0
            mass[table, :, j % page] = (held + gathered).T
    return {"out": out} if tree is not None else {"mass": mass}
