"""The attention over the paged key and value cache, and the cache in 8 bits,
as cases to time and to check: what each reads, writes and computes, its
plain form in elementary torch operations, and its definition in 64 bits.

- attention of new tokens over the paged cache, for one sequence
  (`HipOps.attention`) and for several (`HipOps.attentionSequences`), over the
  F16 cache and the 8-bit one;
- the same with a sliding window and first positions that stay visible;
- keys and values quantised into the 8-bit cache as they are written
  (`cacheWrite`, `cacheWriteSequences`) and read back (`cacheRead`,
  `cacheReadSequences`).

A case's `sequences` is 0 for one sequence given by itself (its page table and
its start on the host), else the number of sequences of a batch (page tables,
starts and offsets on the device). `tokens` counts the new tokens of the whole
call: a batch with as many tokens as sequences has one each (a decode step), one
with more is a mix of single tokens and chunks. `context` is the positions
before them: a sequence's own, and the most that any has in a batch.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# (heads, key heads, values a head)
HEADS = ((32, 8, 128), (28, 4, 128), (16, 2, 256), (16, 4, 64), (24, 24, 128), (12, 3, 80), (9, 3, 72), (8, 1, 96))


def _case(name, op, dtype, cache, sequences, tokens, context, heads, page, window=0, sinks=0, read=0):
    return {"name": name, "op": op, "type": dtype, "cache": cache, "sequences": sequences, "tokens": tokens,
            "context": context, "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "page": page,
            "window": window, "sinks": sinks, "read": read}


def listed():
    return [
        # a chat's next token early on: the smallest call, where latency counts
        _case("decode one", "attention", "bf16", "f16", 0, 1, 517, (32, 8, 128), 16),
        # a server's decode step: 64 conversations of ragged lengths
        _case("decode batch", "attention", "bf16", "f16", 64, 64, 8000, (32, 8, 128), 16),
        # the next chunk of a prompt in the runner's own activations (F32), 2 key heads of 256
        _case("chunk f32", "attention", "f32", "f16", 0, 509, 3591, (16, 2, 256), 16),
        # a long prompt from its start
        _case("prefill", "attention", "bf16", "f16", 0, 8192, 0, (32, 8, 128), 16),
        # continuous batching: decode tokens and prompts' chunks in one call, groups of 7 heads
        _case("mixed batch", "attention", "bf16", "f16", 24, 1811, 6000, (28, 4, 128), 64),
        # long conversations whose layers see a window and the first four positions
        _case("window decode", "attention", "bf16", "f16", 32, 32, 32000, (32, 8, 128), 64, 4096, 4),
        # a prompt's chunk in a windowed layer with narrow heads
        _case("window chunk", "attention", "bf16", "f16", 0, 4096, 12345, (16, 4, 64), 32, 1024, 4),
        # a decode step's keys and values into the 8-bit cache, its newest positions taken out again
        _case("i8 write step", "write_read", "bf16", "i8", 64, 64, 4000, (32, 8, 128), 16, read=33),
        # a prompt's keys and values quantised, the whole sequence read back (to move it elsewhere)
        _case("i8 write prompt", "write_read", "f32", "i8", 0, 8192, 1000, (32, 8, 128), 16, read=9192),
        # the decode step over the 8-bit cache
        _case("i8 decode batch", "attention", "bf16", "i8", 64, 64, 8000, (32, 8, 128), 16),
        # the next token in F32 over the 8-bit cache, 2 key heads of 256
        _case("i8 decode one", "attention", "f32", "i8", 0, 1, 1900, (16, 2, 256), 16),
        # a prompt's chunk over the 8-bit cache
        _case("i8 chunk", "attention", "bf16", "i8", 0, 1021, 2500, (32, 8, 128), 16),
    ]


# What a drawn case may cost, as the largest listed one: visible pairs times
# heads times values a head; and, for the plain form's memory, its scores.
MOST_PAIR_VALUES = 8192 * 8193 // 2 * 32 * 128
MOST_SCORES = 8192 * 8192 * 32
MOST_CACHE = 1 << 31  # values of the keys


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    while True:
        heads = rng.choice(HEADS)
        cache = rng.choice(("f16", "i8"))
        op = "write_read" if cache == "i8" and rng.random() < 0.35 else "attention"
        sequences = rng.choice((0, 0, log_int(2, 100)))
        step = sequences > 0 and rng.random() < 0.5
        tokens = sequences if step else max(sequences, log_int(1, 8192))
        context = log_int(1, 32000)
        window = log_int(16, 8192) if op == "attention" and rng.random() < 0.4 else 0
        sinks = rng.choice((0, 1, 4, 37)) if window else 0
        read = rng.randint(1, context) if op == "write_read" else 0
        c = _case("", op, rng.choice(("f32", "bf16")), cache, sequences, tokens, context, heads,
                  rng.choice((16, 16, 32, 48, 64, 128)), window, sinks, read)
        del c["name"]
        most, count = int(_new_tokens(c).max()), max(sequences, 1)
        positions = count * (context + most + c["page"])
        scores = count * most * (context + most) * heads[0]
        if positions * heads[1] * heads[2] > MOST_CACHE:
            continue
        if op == "write_read":
            if read * count * heads[1] * heads[2] <= MOST_CACHE // 8:
                return c
        elif scores <= MOST_SCORES and _pairs(c) * heads[0] * heads[2] <= MOST_PAIR_VALUES:
            return c


# ------------------------------------------------------------------ a case's layout

def _new_tokens(case):
    """New tokens of each sequence."""
    count, tokens = max(case["sequences"], 1), case["tokens"]
    each = np.ones(count, np.int64)
    if count == 1:
        each[0] = tokens
    elif tokens > count:  # every fourth sequence brings a chunk, the sizes uneven
        chunks = np.arange(0, count, 4)
        share = 1.0 + np.random.RandomState(count).random_sample(len(chunks))
        more = np.floor(share / share.sum() * (tokens - count)).astype(np.int64)
        more[0] += tokens - count - more.sum()
        each[chunks] += more
    return each


def _starts(case):
    """Positions each sequence holds before its new tokens."""
    count, context = max(case["sequences"], 1), case["context"]
    if count == 1:
        return np.array([context], np.int64)
    share = np.random.RandomState(1000 + count).random_sample(count)
    starts = np.floor(context * (0.05 + 0.95 * share)).astype(np.int64)
    starts[-1] = context
    return starts


def _visible_positions(case):
    """Positions that some new token of each sequence sees."""
    starts, each = _starts(case), _new_tokens(case)
    ends = starts + each
    if not case["window"]:
        return ends
    low = np.maximum(starts - case["window"] + 1, 0)
    return ends - low + np.minimum(case["sinks"], low)


def _pairs(case):
    """Visible (token, position) pairs."""
    starts, each = _starts(case), _new_tokens(case)
    at = np.repeat(starts, each) + np.arange(each.sum()) - np.repeat(np.cumsum(each) - each, each)
    if not case["window"]:
        return int((at + 1).sum())
    seen = np.minimum(at + 1, case["window"])
    return int((seen + np.minimum(case["sinks"], at + 1 - seen)).sum())


def work(case):
    wide = 4 if case["type"] == "f32" else 2
    kv, dim, tokens = case["kv_heads"], case["dim"], case["tokens"]
    row = 2 * (dim * 2 if case["cache"] == "f16" else dim + 4)  # a position's key and value of a head, as cached
    tables = 4 * int(np.ceil((_starts(case) + _new_tokens(case)) / case["page"]).sum())
    if case["op"] == "write_read":
        read = case["read"] * max(case["sequences"], 1)
        return {"bytes": (tokens + read) * kv * (2 * dim * wide + row) + tables, "flops": 0}
    return {"bytes": 2 * tokens * case["heads"] * dim * wide + int(_visible_positions(case).sum()) * kv * row + tables,
            "flops": 4 * _pairs(case) * case["heads"] * dim}


# ------------------------------------------------------------------ inputs

def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)

    starts, each = _starts(case), _new_tokens(case)
    kv, dim, page, dtype = case["kv_heads"], case["dim"], case["page"], TYPES[case["type"]]
    used = -(-(starts + each) // page)
    columns, pages = int(used.max()), int(used.sum()) + 3
    # each sequence's pages among the cache's, in no order; entries past its last page name no page
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((len(starts), columns), -1, dtype=torch.int32, device=DEV)
    filled = torch.arange(columns, device=DEV)[None, :] < torch.from_numpy(used).to(DEV)[:, None]
    tables[filled] = order[:int(used.sum())]
    s = {"case": case, "tables": tables,
         "starts": torch.from_numpy(starts).to(DEV, torch.int32),
         "offsets": torch.from_numpy(np.concatenate([[0], np.cumsum(each)])).to(DEV, torch.int32)}
    # keys after their norm and rotation have values about 1, with some strong channels; one draw serves all pages
    # in turns of a prime length, so that making a large cache stays quick
    channels = 1.0 + 2.0 * (torch.rand(kv, dim, generator=gen, device=DEV) < 0.05)
    if case["cache"] == "f16":
        base = normal(min(pages, 509), page, kv, dim) * channels
        s["keys"] = base.half()[torch.arange(pages, device=DEV) % base.shape[0]]
        base = normal(min(pages, 509), kv, dim, page)
        s["values"] = base.half()[torch.arange(pages, device=DEV) % base.shape[0]]
    else:
        def codes(*shape):
            return torch.randint(-127, 128, (min(pages, 509),) + shape, generator=gen, device=DEV,
                                 dtype=torch.int8)[torch.arange(pages, device=DEV) % min(pages, 509)]

        def scales(most):
            return (0.5 + torch.rand(pages, kv, page, generator=gen, device=DEV)) * most / 127

        s["keys"], s["key_scales"] = codes(page, kv, dim), scales(2.0)
        s["values"], s["value_scales"] = codes(kv, dim, page), scales(2.5)
    tokens = case["tokens"]
    if case["op"] == "attention":
        # queries sharp enough that a few positions carry most of a row
        s["queries"] = normal(tokens, case["heads"], dim, dtype=dtype, scale=2.0)
        s["out"] = torch.zeros(tokens, case["heads"], dim, dtype=dtype, device=DEV)
        s["scale"] = 1.0 / math.sqrt(dim)
    else:
        s["k"] = (normal(tokens, kv, dim) * channels).to(dtype)
        s["v"] = normal(tokens, kv, dim, dtype=dtype)
        # read back: the newest `read` positions of each sequence (fewer where it holds fewer)
        count = np.minimum(case["read"], starts + each)
        s["read_starts"] = torch.from_numpy(starts + each - count).to(DEV, torch.int32)
        s["read_offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(count)])).to(DEV, torch.int32)
        s["k_out"] = torch.zeros(int(count.sum()), kv, dim, dtype=dtype, device=DEV)
        s["v_out"] = torch.zeros_like(s["k_out"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from drift_amd import ops as d

        s["hip"] = d.HipOps()
        if case["cache"] == "f16":
            s["cache"] = d.KvCache(s["keys"], s["values"], case["page"])
        else:
            s["cache"] = d.QuantizedKvCache(s["keys"], s["values"], s["key_scales"], s["value_scales"], case["page"])
        s["window"] = d.AttentionWindow(case["window"], case["sinks"]) if case["window"] else None
        if case["sequences"]:
            step = case["tokens"] == case["sequences"]
            s["batch"] = d.Sequences(s["tables"], s["starts"], None if step else s["offsets"])
            if case["op"] == "write_read":
                s["read_batch"] = d.Sequences(s["tables"], s["read_starts"], s["read_offsets"])
        else:
            s["table"], s["start"] = s["tables"][0], case["context"]
            if case["op"] == "write_read":
                s["read_start"] = int(s["read_starts"][0])
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    attention = s["case"]["op"] == "attention"
    if own:
        hip, cache = s["hip"], s["cache"]
        if attention:
            if s["case"]["sequences"]:
                hip.attentionSequences(s["queries"], cache, s["batch"], s["scale"], s["out"], s["window"])
            else:
                hip.attention(s["queries"], cache, s["table"], s["start"], s["scale"], s["out"], s["window"])
            return s["out"]
        if s["case"]["sequences"]:
            hip.cacheWriteSequences(s["k"], s["v"], cache, s["batch"])
            hip.cacheReadSequences(cache, s["read_batch"], s["k_out"], s["v_out"])
        else:
            hip.cacheWrite(s["k"], s["v"], cache, s["table"], s["start"])
            hip.cacheRead(cache, s["table"], s["read_start"], s["k_out"], s["v_out"])
        return {"keys": s["k_out"], "values": s["v_out"]}
    return _plain_attention(s) if attention else _plain_write_read(s)


def _places(offsets, count):
    """Of `count` token rows, packed by `offsets`: each one's sequence, and its place among that sequence's."""
    row = torch.arange(count, device=DEV)
    sequence = torch.searchsorted(offsets[1:], row, right=True)
    return sequence, row - offsets[sequence]


def _plain_attention(s):
    c, tables = s["case"], s["tables"].clamp(min=0).long()
    kv, dim, group, count = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"], tables.shape[0]
    keys, values = s["keys"][tables].float(), s["values"][tables].float()
    if c["cache"] == "i8":  # scales [sequences, pages, kv, page]
        keys = keys * s["key_scales"][tables].permute(0, 1, 3, 2)[..., None]
        values = values * s["value_scales"][tables][..., None, :]
    length = tables.shape[1] * c["page"]
    k = keys.reshape(count, length, kv, dim).permute(0, 2, 3, 1).contiguous().view(count * kv, dim, length)
    v = values.permute(0, 2, 1, 4, 3).contiguous().view(count * kv, length, dim)
    # every sequence's rows side by side, as many columns as the longest chunk has
    most, offsets = int(_new_tokens(c).max()), s["offsets"].long()
    column = torch.arange(most, device=DEV)
    rows = (offsets[:-1, None] + column).clamp(max=c["tokens"] - 1)
    at = s["starts"].long()[:, None] + column
    q = s["queries"].float()[rows]  # [sequences, most, heads, dim]
    q = q.view(count, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(count * kv, most * group, dim)
    j = torch.arange(length, device=DEV)
    seen = j <= at[..., None]
    if c["window"]:
        seen &= (j > at[..., None] - c["window"]) | (j < c["sinks"])
    scores = torch.bmm(q, k).mul_(s["scale"]).view(count, kv, most, group, length)
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.bmm(scores.view(count * kv, most * group, length), v).view(count, kv, most, group, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 2, 1, 3, 4).reshape(count, most, c["heads"], dim)
    s["out"].copy_(out[_places(offsets, c["tokens"])])
    return s["out"]


def _plain_quantise(x):
    x = x.double()
    scale = (x.abs().amax(-1) / 127).float()
    step = scale.double()[..., None]
    codes = torch.floor(x.abs() / torch.where(step > 0, step, torch.ones_like(step)) + 0.5).clamp(max=127)
    return (codes * x.sign()).to(torch.int8), scale


def _plain_write_read(s):
    c = s["case"]
    tables, page = s["tables"].long(), c["page"]

    def places(starts, offsets, rows):
        sequence, nth = _places(offsets.long(), rows)
        at = starts.long()[sequence] + nth
        return tables[sequence, at // page], at % page

    to, slot = places(s["starts"], s["offsets"], c["tokens"])
    codes, scale = _plain_quantise(s["k"])
    s["keys"][to, slot] = codes
    s["key_scales"][to, :, slot] = scale
    codes, scale = _plain_quantise(s["v"])
    s["values"][to, :, :, slot] = codes
    s["value_scales"][to, :, slot] = scale
    at, slot = places(s["read_starts"], s["read_offsets"], s["k_out"].shape[0])
    s["k_out"].copy_(s["keys"][at, slot].float() * s["key_scales"][at, :, slot][..., None])
    s["v_out"].copy_(s["values"][at, :, :, slot].float() * s["value_scales"][at, :, slot][..., None])
    return {"keys": s["k_out"], "values": s["v_out"]}


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    starts, each = _starts(case), _new_tokens(case)
    first = np.cumsum(each) - each
    page, kv, group = case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]

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

    if case["op"] == "attention":
        out = torch.zeros(case["tokens"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
        for n in range(len(starts)):
            length = int(starts[n] + each[n])
            k, v = dense(n, length, "keys"), dense(n, length, "values")
            j = torch.arange(length, device=DEV)
            for a in range(0, int(each[n]), 1024):
                b = min(a + 1024, int(each[n]))
                p = torch.arange(int(starts[n]) + a, int(starts[n]) + b, device=DEV)[:, None]
                hidden = j > p
                if case["window"]:
                    hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
                rows = slice(int(first[n]) + a, int(first[n]) + b)
                for h in range(case["heads"]):
                    logits = s["queries"][rows, h].double() @ k[h // group].T.contiguous() * s["scale"]
                    logits[hidden] = -math.inf
                    out[rows, h] = torch.softmax(logits, -1) @ v[h // group]
        return out
    # the codes of a row: its values over the row's F32 scale, to the nearest whole number, halves away from 0
    new = {}
    for what in ("k", "v"):
        x = s[what].double()
        d = (x.abs().amax(-1, keepdim=True) / 127).float().double()
        d1 = torch.where(d > 0, d, torch.ones_like(d))
        new[what] = torch.sign(x) * torch.clamp(torch.trunc(torch.abs(x) / d1 + 0.5), max=127.0) * d
    got = {"keys": [], "values": []}
    for n in range(len(starts)):
        length = int(starts[n] + each[n])
        for what, fresh in (("keys", "k"), ("values", "v")):
            x = dense(n, length, what)
            x[:, int(starts[n]):] = new[fresh][int(first[n]):int(first[n] + each[n])].transpose(0, 1)
            got[what].append(x[:, length - min(case["read"], length):].transpose(0, 1))
    return {what: torch.cat(x) for what, x in got.items()}
