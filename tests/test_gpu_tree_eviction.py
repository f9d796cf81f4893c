"""Attention over trees of drafted tokens, the attention that cached positions
gather, the choice of the heaviest and the move of kept rows on the GPU, against
plain implementations in 64 bits.

Bars, derived from the roundings on the way:
- trees: those of attention over the paged cache (test_gpu_paged_attention.py
  has them with their derivation), which they are but for what a row sees;
- masses: a row's weight for a position is relatively off by its score's error
  and by that of the row's sum: with S' = scale sum |q||k| up to the row's
  largest, D values and n visible positions, d = 2 (4 2^-24 (sqrt(D) + 4) S' +
  2^-20) + 2^-24 (sqrt(n) + 8), the exponential, the sum's own weights' errors
  and the divisions in it. The sum of r weights in F32 adds at most 2^-24 (r + 2)
  of their sum and of what was there before (a sum of r terms in order, or in
  parts). Weights below 2^-126 may count as 0: r 2^-126. Held to
  (max d + 2^-24 (r + 2)) (sum + before) + r 2^-126;
- what is chosen and what is moved: exact.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

from drift_amd import _lib
from drift_amd import ops as d
from tests.helpers import DEV, dev_i32, step
from tests.test_gpu_paged_attention import CACHES, DTYPES, TYPES, Case, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return d.HipOps()


# ------------------------------------------------------------------ trees

def trees(rows, seed=0, shape="random"):
    """What each row sees of its sequence's: bool [rows of it, rows of it], a sequence after another."""
    rng = np.random.default_rng(seed)
    found = []
    for n in rows:
        sees = np.zeros((n, n), bool)
        for i in range(n):
            if i > 0 and shape != "roots":
                parent = i - 1 if shape == "chain" else int(rng.integers(max(0, i - 9), i))
                sees[i] = sees[parent]
            sees[i, i] = True
        if shape == "any":  # no tree at all: rows that see anything, or nothing
            sees = rng.random((n, n)) < 0.5
            sees[::5] = False
        found.append(sees)
    return found


def packed(sees, words, total=None, seed=3):
    """As I32 words; bits of rows that the sequence does not have are set at random."""
    rng = np.random.default_rng(seed)
    rows = sum(len(s) for s in sees) if total is None else total
    bits = rng.random((rows, words * 32)) < 0.5
    at = 0
    for s in sees:
        n = len(s)
        bits[at:at + n, :n] = s[:, :words * 32]
        at += n
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()).to(DEV)


def tree_rows(case, queries, scale, sees, window=None, hidden=()):
    """The rows in 64 bits, and their bars."""
    tokens, heads, dim = queries.shape
    q, f32 = queries.cpu().double(), queries.dtype == torch.float32
    out, bar = torch.zeros(tokens, heads, dim).double(), torch.zeros(tokens, heads, dim).double()
    for s, (k, v) in enumerate(case.dense):
        start, n = int(case.starts[s]), int(case.rows[s])
        if n == 0:
            continue
        rows = slice(int(case.offsets[s]), int(case.offsets[s + 1]))
        seen = torch.zeros(n, start + n, dtype=torch.bool)
        mine = torch.from_numpy(sees[s])
        seen[:, start:] = mine
        j = torch.arange(start)
        seen[:, :start] = True
        if window is not None:
            at = start - 1 + mine.sum(1, keepdim=True)
            seen[:, :start] = (j > at - window.positions) | (j < window.sinks)
        for sequence, position in hidden:
            if sequence == s:
                seen[:, position] = False
        for h in range(heads):
            kh, vh = k[:, h // (heads // case.kv)], v[:, h // (heads // case.kv)]
            hide = ~seen
            logits = (scale * (q[rows, h] @ kh.nan_to_num(0).T)).masked_fill(hide, -math.inf)
            some = seen.any(1, keepdim=True)
            p = torch.where(some, torch.softmax(torch.where(some, logits, 0.0), -1), 0.0)
            size = (scale * (q[rows, h].abs() @ kh.nan_to_num(0).abs().T)).masked_fill(hide, 0.0).amax(1, keepdim=True)
            count = seen.sum(1, keepdim=True).double()
            value = vh.nan_to_num(0)
            mass = p @ value.abs()
            out[rows, h] = p @ value
            lost = p.amax(1, keepdim=True) * (seen.double() @ value.abs() if case.kind == "f16" else
                                              2 * case.scales[s][:, h // (heads // case.kv)].max() * 127 * count)
            bar[rows, h] = 4 * (2.0 ** -24 * (math.sqrt(dim) + 4) * size + 2.0 ** -20 + 2.0 ** -24 * count.sqrt()) * \
                mass + (2.0 ** -39 if f32 else 2.0 ** -32) * lost
            if not f32:
                bar[rows, h] += 2.0 ** -11 * mass
    if not f32:
        bar += 2.0 ** -8 * out.abs()
    return out, bar + 1e-30


def assert_tree(case, queries, scale, sees, got, window=None, hidden=(), what=""):
    out, bar = tree_rows(case, queries, scale, sees, window, hidden)
    off = (got.cpu().double() - out).abs()
    worst = float((off / bar).max())
    print(f"[gpu]   worst {worst:.3f} of the bar", flush=True)
    assert bool((off <= bar).all()), f"{what}: worst {worst:.2f} times the bar, first {(off > bar).nonzero()[0].tolist()}"


def attend(hip, case, queries, sees, scale, window=None, offsets=True, longest=0, bad=None):
    out = torch.full(queries.shape, 7.0, dtype=queries.dtype, device=DEV)
    hip.attentionTree(queries, case.cache, case.sequences(offsets, longest), sees, scale, out, window, bad)
    return out


TREES = [
    # (starts, rows, heads, kv heads, dim, page, shape): single nodes, trees that start and end inside pages, tiles and
    # words, one whose rows see anything; groups of 1 to 16 heads; sizes whole, padded and odd
    ([0], [1], 2, 1, 64, 16, "random"), ([517], [8], 32, 8, 128, 16, "random"), ([3], [33], 8, 2, 128, 16, "random"),
    ([0, 700, 63], [7, 64, 13], 8, 2, 128, 32, "random"), ([31, 1000], [70, 129], 9, 3, 72, 16, "random"),
    ([250], [100], 28, 4, 128, 64, "any"), ([100, 0, 48], [12, 25, 0], 16, 2, 256, 48, "any"),
    ([64], [64], 16, 16, 64, 16, "roots"), ([2500], [20], 16, 1, 128, 128, "random"), ([40], [9], 4, 2, 20, 16, "any"),
    ([33, 5], [3, 40], 2, 1, 512, 16, "random"), ([90], [6], 3, 3, 7, 16, "any"), ([1200], [300], 4, 1, 96, 16, "any"),
]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,rows,heads,kv,dim,page,shape", TREES)
def test_trees(hip, kind, dtype, starts, rows, heads, kv, dim, page, shape):
    step(f"trees {kind} {dtype} {rows} rows at {starts}, {heads}/{kv} heads of {dim}, pages of {page}, {shape}")
    case = Case(kind, starts, rows, kv, dim, page, seed=sum(starts) + sum(rows))
    q = normal(5, (case.tokens, heads, dim), TYPES[dtype], 2.0).to(DEV)
    sees, scale = trees(rows, len(rows), shape), 1 / math.sqrt(dim)
    words = -(-max(rows) // 32)
    got = attend(hip, case, q, packed(sees, words), scale)
    assert_tree(case, q, scale, sees, got, what="tree")
    # the words may be more than the rows need
    assert torch.equal(attend(hip, case, q, packed(sees, words + 2, seed=4), scale), got)


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("positions,sinks", [(1, 0), (5, 1), (40, 3), (700, 4), (4096, 50)])
@pytest.mark.parametrize("starts,rows,heads,kv,dim", [([900, 3, 0], [12, 40, 70], 8, 2, 128), ([130], [9], 3, 3, 20)])
def test_trees_in_windows(hip, kind, dtype, positions, sinks, starts, rows, heads, kv, dim):
    step(f"trees in a window of {positions} + {sinks} {kind} {dtype} {rows} rows at {starts}, heads of {dim}")
    case = Case(kind, starts, rows, kv, dim, 16, seed=21)
    q = normal(6, (case.tokens, heads, dim), TYPES[dtype], 2.0).to(DEV)
    window, scale = d.AttentionWindow(positions, sinks), 1 / math.sqrt(dim)
    for shape in ("random", "any"):
        sees = trees(rows, 2, shape)
        got = attend(hip, case, q, packed(sees, 3), scale, window)
        assert_tree(case, q, scale, sees, got, window, what=shape)


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [None, d.AttentionWindow(50, 3)])
@pytest.mark.parametrize("rows", [[1, 5, 17, 1, 30], [200, 1, 90, 1, 64]])
def test_a_chain_is_attention_of_the_sequences(hip, kind, dtype, window, rows):
    step(f"chains {kind} {dtype} {window} {rows}")
    case = Case(kind, [0, 700, 30, 1500, 9], rows, 2, 128, 16, seed=11)
    q = normal(8, (case.tokens, 8, 128), TYPES[dtype], 2.0).to(DEV)
    want = torch.empty_like(q)
    hip.attentionSequences(q, case.cache, case.sequences(), 0.1, want, window)
    sees = trees(rows, 0, "chain")
    if window is not None:  # what the window hides of the new tokens is the caller's to leave out
        for s, start in zip(sees, case.starts):
            i = np.arange(len(s))
            s &= (i > i[:, None] - window.positions) | (start + i < window.sinks)
    got = attend(hip, case, q, packed(sees, -(-max(rows) // 32)), 0.1, window)
    assert_tree(case, q, 0.1, sees, got, window, what="chain")
    assert_tree(case, q, 0.1, sees, want, window, what="attention")


def test_tokens_past_the_words_are_not_seen(hip):
    step("tokens past the words")
    case = Case("f16", [20], [90], 2, 64, 16, seed=12)
    q = normal(9, (90, 4, 64), torch.float32, 2.0).to(DEV)
    sees = trees([90], 5)
    words = packed(sees, 1)
    sees[0][:, 32:] = False
    assert_tree(case, q, 0.125, sees, attend(hip, case, q, words, 0.125), what="one word")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dim", [64, 128, 20])
def test_a_step_without_offsets(hip, kind, dim):
    step(f"trees of one node without offsets {kind} {dim}")
    starts = [0, 15, 900, 64]
    case = Case(kind, starts, [1] * 4, 2, dim, 16, seed=13)
    q = normal(10, (4, 8, dim), torch.bfloat16, 2.0).to(DEV)
    sees = [np.ones((1, 1), bool), np.zeros((1, 1), bool), np.ones((1, 1), bool), np.zeros((1, 1), bool)]
    assert_tree(case, q, 0.1, sees, attend(hip, case, q, packed(sees, 1), 0.1, offsets=False), what="without")
    assert_tree(case, q, 0.1, sees, attend(hip, case, q, packed(sees, 1), 0.1, longest=1), what="by offsets")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[6, 3], [90, 50]])
def test_what_a_trees_rows_do_not_see_has_no_part(hip, kind, dtype, rows):
    step(f"a tree's masked places {kind} {dtype} {rows}")
    case = Case(kind, [100, 40], rows, 2, 128, 16, seed=14)
    q = normal(11, (case.tokens, 8, 128), TYPES[dtype], 2.0).to(DEV)
    sees = trees(rows, 6)
    for s in sees:  # no row but its own sees row 2, which holds no numbers
        s[:, 2] = False
        s[2, 2] = True
    words = packed(sees, -(-max(rows) // 32))
    position = int(case.starts[0]) + 2
    page, off = int(case.tables[0, position // 16]), position % 16
    if kind == "f16":
        case.cache.keys[page, off] = float("inf")
        case.cache.values[page, :, :, off] = float("nan")
    else:
        case.cache.keyScales[page, :, off] = float("nan")
        case.cache.valueScales[page, :, off] = float("inf")
    got = attend(hip, case, q, words, 0.1)
    assert not bool(torch.isfinite(got[2]).any())
    others = torch.arange(case.tokens, device=DEV) != 2
    case.dense[0][0][position] = 0
    case.dense[0][1][position] = 0
    out, bar = tree_rows(case, q, 0.1, sees)
    off = ((got.cpu().double() - out).abs() / bar)[others.cpu()]
    assert float(off.max()) <= 1, float(off.max())


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("rows", [[5], [150]])
def test_a_trees_pages_outside_the_cache(hip, kind, rows):
    step(f"a tree's pages outside the cache {kind} {rows}")
    case = Case(kind, [200], rows, 2, 128, 16, seed=15)
    hidden = []
    for column, entry in ((2, -1), (5, case.cache.pages), (12, 1 << 30)):
        case.tables[0, column] = entry
        hidden += [(0, column * 16 + i) for i in range(16) if column * 16 + i < 200 + rows[0]]
    q = normal(12, (case.tokens, 8, 128), torch.float32, 2.0).to(DEV)
    sees = trees(rows, 7)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = attend(hip, case, q, packed(sees, 5), 0.1, bad=bad)
    assert int(bad.item()) == 1
    assert_tree(case, q, 0.1, sees, got, hidden=hidden, what="pages")


@pytest.mark.parametrize("rows_each", [[1, 1], [5, 40]])
def test_a_trees_rows_outside_every_sequence_stay(hip, rows_each):
    step(f"a tree's rows outside every sequence {rows_each}")
    case = Case("f16", [30, 700], rows_each, 2, 128, 16, seed=16)
    first, tokens = 3, case.tokens + 8
    q = normal(9, (tokens, 4, 128), torch.bfloat16).to(DEV)
    sees = trees(rows_each, 8)
    words = torch.full((tokens, 2), -1, dtype=torch.int32, device=DEV)
    words[first:first + case.tokens] = packed(sees, 2)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    batch = d.Sequences(dev_i32(case.tables), dev_i32(case.starts), dev_i32(case.offsets + first))
    hip.attentionTree(q, case.cache, batch, words, 0.1, out)
    inside = slice(first, first + case.tokens)
    assert bool((out[:first] == 7).all()) and bool((out[first + case.tokens:] == 7).all())
    assert_tree(case, q[inside], 0.1, sees, out[inside], what="inside")
    # a sequence with an end past its page table gets nothing done
    out.fill_(7)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    batch = d.Sequences(dev_i32(case.tables), dev_i32([30, 1 << 30]), dev_i32(case.offsets + first))
    hip.attentionTree(q, case.cache, batch, words, 0.1, out, badPage=bad)
    assert int(bad.item()) == 1 and bool((out[first + rows_each[0]:] == 7).all())


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("rows", [[9] * 6, [80, 3, 160]])
def test_trees_give_the_same_bits_on_another_stream_and_off_16_bytes(hip, kind, rows):
    step(f"trees twice {kind} {rows}")
    case = Case(kind, [800 + 13 * i for i in range(len(rows))], rows, 2, 128, 16, seed=17)
    q = normal(13, (case.tokens, 16, 128), torch.bfloat16, 2.0).to(DEV)
    sees = trees(rows, 9)
    words = packed(sees, 5)
    want = attend(hip, case, q, words, 0.1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    other = d.HipOps(stream)
    torch.cuda.synchronize()
    out = torch.empty_like(q)
    other.attentionTree(q, case.cache, case.sequences(), words, 0.1, out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    flat = torch.empty(q.numel() + 4, dtype=q.dtype, device=DEV)[4:].view(q.shape)
    flat.copy_(q)
    assert_tree(case, q, 0.1, sees, attend(hip, case, flat, words, 0.1), what="queries off 16 bytes")


# ------------------------------------------------------------------ masses

def wanted_mass(case, queries, scale, before, hidden=()):
    """Per sequence: masses and bars [kv, length] in 64 bits. `before`: the same, or None."""
    tokens, heads, dim = queries.shape
    q, group, found = queries.cpu().double(), heads // case.kv, []
    for s, (k, _) in enumerate(case.dense):
        start, n = int(case.starts[s]), int(case.rows[s])
        rows = slice(int(case.offsets[s]), int(case.offsets[s + 1]))
        j = torch.arange(start + n)
        seen = j <= (start + torch.arange(n))[:, None]
        for sequence, position in hidden:
            if sequence == s:
                seen[:, position] = False
        mass, bar = torch.zeros(case.kv, start + n).double(), torch.zeros(case.kv, start + n).double()
        for h in range(heads):
            kh = k[:, h // group]
            logits = scale * (q[rows, h] @ kh.T)
            logits = torch.where(seen, logits, -math.inf)
            p = torch.where(seen, torch.softmax(logits, -1), 0.0)
            size = torch.where(seen, abs(scale) * (q[rows, h].abs() @ kh.abs().T), 0.0).amax(1, keepdim=True)
            delta = 2 * (4 * 2.0 ** -24 * (math.sqrt(dim) + 4) * size + 2.0 ** -20) + \
                2.0 ** -24 * (seen.sum(1, keepdim=True).double().sqrt() + 8)
            mass[h // group] += p.sum(0)
            bar[h // group] += (p * delta.nan_to_num(0)).sum(0)
        if before is not None:
            mass[:, :start] += before[s][:, :start].double()
        found.append((mass, bar + 2.0 ** -24 * (n * group + 2) * mass.abs() + n * group * 2.0 ** -126))
    return found


def gathered(case, mass):
    """Per sequence, [kv, length]."""
    found = []
    for s in range(len(case.starts)):
        j = torch.arange(int(case.starts[s] + case.rows[s]))
        page = torch.from_numpy(case.tables[s].astype(np.int64))[j // case.page]
        found.append(mass.cpu()[page.clamp(0, mass.shape[0] - 1), :, j % case.page].T)
    return found


def assert_mass(case, queries, scale, mass, before=None, hidden=(), what=""):
    held = None if before is None else gathered(case, before)
    for s, ((want, bar), got) in enumerate(zip(wanted_mass(case, queries, scale, held, hidden), gathered(case, mass))):
        keep = torch.ones(want.shape[1], dtype=torch.bool)
        for sequence, position in hidden:
            if sequence == s:
                keep[position] = False
        if case.rows[s] == 0:
            continue
        want, bar, got = want[:, keep], bar[:, keep], got.double()[:, keep]
        nan = torch.isnan(want)
        assert bool((torch.isnan(got) == nan).all()), f"{what}: NaN in other places of sequence {s}"
        off = ((got - want).abs() / bar)[~nan]
        worst = float(off.max()) if off.numel() else 0.0
        print(f"[gpu]   worst {worst:.3f} of the bar", flush=True)
        assert worst <= 1, f"{what}: sequence {s}, {worst:.2f} times the bar"


def masses(case, seed, scale=0.01):
    gen = torch.Generator().manual_seed(seed)
    return (torch.exp(2 * torch.randn(case.cache.pages, case.kv, case.page, generator=gen)) * scale).to(DEV)


MASSES = [
    # (starts, rows, heads, kv heads, dim, page)
    ([0], [1], 1, 1, 64, 16), ([0], [1], 8, 2, 128, 16), ([15], [1], 28, 4, 128, 64), ([517], [1], 32, 8, 128, 16),
    ([3000], [1], 16, 2, 256, 16), ([0, 15, 900, 333, 64, 31], [1] * 6, 8, 2, 128, 16), ([9000], [3], 16, 1, 128, 128),
    ([0], [130], 8, 2, 128, 16), ([5], [37], 9, 3, 72, 16), ([700, 3], [64, 33], 12, 3, 80, 48),
    ([100, 0, 64, 7], [65, 1, 0, 200], 16, 4, 64, 32), ([250], [129], 4, 2, 256, 16), ([1], [300], 8, 8, 96, 16),
    ([40], [20], 4, 2, 20, 16), ([9], [5], 3, 3, 7, 16), ([33], [3], 2, 1, 512, 16), ([64], [40], 4, 4, 264, 32),
    ([1200], [17], 16, 1, 64, 16), ([2000], [16], 4, 1, 128, 16), ([10 * i for i in range(70)], [1 + i % 3 for i in range(70)], 4, 2, 64, 16),
]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,rows,heads,kv,dim,page", MASSES)
def test_masses(hip, kind, dtype, starts, rows, heads, kv, dim, page):
    step(f"masses {kind} {dtype} {rows} rows at {starts}, {heads}/{kv} heads of {dim}, pages of {page}")
    case = Case(kind, starts, rows, kv, dim, page, seed=sum(starts) + 1)
    q = normal(5, (case.tokens, heads, dim), TYPES[dtype], 2.0).to(DEV)
    scale, before = 1 / math.sqrt(dim), masses(case, 3)
    mass = torch.full_like(before, 7.0)
    hip.attentionMass(q, case.cache, case.sequences(), scale, mass, before)
    assert_mass(case, q, scale, mass, before, what="added")
    # what no sequence holds is left as it is
    held = torch.zeros(mass.shape, dtype=torch.bool)
    for s in range(len(starts)):
        j = torch.arange(int(case.starts[s] + case.rows[s]) if rows[s] else 0)
        held[torch.from_numpy(case.tables[s].astype(np.int64))[j // page], :, j % page] = True
    assert bool((mass.cpu()[~held] == 7).all())
    # in place, and anew
    same = before.clone()
    hip.attentionMass(q, case.cache, case.sequences(longest=1), scale, same, same)
    assert_mass(case, q, scale, same, before, what="in place")
    assert bool((same.cpu()[~held] == before.cpu()[~held]).all())
    hip.attentionMass(q, case.cache, case.sequences(), scale, mass)
    assert_mass(case, q, scale, mass, what="anew")
    if rows == [1] * len(rows):
        hip.attentionMass(q, case.cache, case.sequences(offsets=False), scale, mass, before)
        assert_mass(case, q, scale, mass, before, what="without offsets")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_a_rows_masses_add_up_to_its_heads(hip, kind, dtype, tokens):
    step(f"masses' sums {kind} {dtype} {tokens}")
    case = Case(kind, [1000], [tokens], 2, 128, 16, seed=31)
    q = normal(5, (tokens, 12, 128), TYPES[dtype], 3.0).to(DEV)
    mass = torch.zeros(case.cache.pages, 2, 16, device=DEV)
    hip.attentionMass(q, case.cache, case.sequences(), 0.1, mass)
    assert torch.allclose(mass.double().sum((0, 2)), torch.full((2,), 6.0 * tokens, device=DEV).double(), rtol=1e-5)


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim", [(1, 128), (9, 64), (100, 128), (2, 20)])
def test_masses_of_what_is_no_number(hip, kind, dtype, tokens, dim):
    step(f"masses of what is no number {kind} {dtype} {tokens} {dim}")
    case = Case(kind, [150], [tokens], 2, dim, 16, seed=32)
    q = normal(5, (tokens, 4, dim), TYPES[dtype], 2.0)
    q[..., 0] = q[..., 0].abs() + 1.0
    last = 150 + tokens - 1
    if kind == "f16":
        # a key of minus infinity where every query is above 0: weight 0, in one head; of a NaN in the other, seen by
        # the last row alone
        page, off = int(case.tables[0, 70 // 16]), 70 % 16
        case.cache.keys[page, off, 0, 0] = -math.inf
        case.dense[0][0][70, 0, 0] = -math.inf
        page, off = int(case.tables[0, last // 16]), last % 16
        case.cache.keys[page, off, 1, 3] = math.nan
        case.dense[0][0][last, 1, 3] = math.nan
    else:
        page, off = int(case.tables[0, last // 16]), last % 16
        case.cache.keyScales[page, 1, off] = math.nan
        case.dense[0][0][last, 1] = math.nan
    mass = torch.zeros(case.cache.pages, 2, 16, device=DEV)
    hip.attentionMass(q.to(DEV), case.cache, case.sequences(), 0.1, mass)
    held = gathered(case, mass)[0]
    assert bool(torch.isnan(held[1]).all()), "the last row's NaN reaches every position it sees"
    if kind == "f16":
        assert bool((held[0, 70] == 0))
        case.dense[0][0][70, 0, 0] = -1e300
    # (scores up to 50: 2 (4 2^-24 (sqrt(128) + 4) 50) is 4e-4 relative at most)
    (want, _), = wanted_mass(case, q, 0.1, None)
    assert bool(((held[0].double() - want[0]).abs() <= 4e-4 * want[0].abs() + 1e-30).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 50])
@pytest.mark.parametrize("what", ["nan", "inf", "huge", "tiny"])
def test_masses_of_unlike_queries(hip, dtype, tokens, what):
    step(f"masses of queries {what} {dtype} {tokens}")
    case = Case("f16", [100], [tokens], 2, 64, 16, seed=33)
    q = normal(5, (tokens, 4, 64), TYPES[dtype], 2.0)
    mass = torch.zeros(case.cache.pages, 2, 16, device=DEV)
    if what in ("nan", "inf"):
        q[-1, 1, 5] = float(what)
        hip.attentionMass(q.to(DEV), case.cache, case.sequences(), 0.1, mass)
        held = gathered(case, mass)[0]
        assert bool(torch.isnan(held[0]).all()) and bool(torch.isfinite(held[1]).all())
        return
    q[-1] *= 2.0 ** 90 if what == "huge" else 2.0 ** -100
    scale = 0.1 * 2.0 ** -85 if what == "huge" else 0.1
    hip.attentionMass(q.to(DEV), case.cache, case.sequences(), scale, mass)
    assert_mass(case, q, scale, mass, what=what)


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("tokens", [1, 150])
def test_masses_on_pages_outside_the_cache(hip, kind, tokens):
    step(f"masses on pages outside the cache {kind} {tokens}")
    case = Case(kind, [200], [tokens], 2, 128, 16, seed=34)
    hidden = []
    for column, entry in ((0, -1), (2, -1), (5, case.cache.pages), (9, 1 << 30)):
        case.tables[0, column] = entry
        hidden += [(0, column * 16 + i) for i in range(16)]
    q = normal(12, (tokens, 8, 128), torch.float32, 2.0).to(DEV)
    mass, bad = torch.zeros(case.cache.pages, 2, 16, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    hip.attentionMass(q, case.cache, case.sequences(), 0.1, mass, badPage=bad)
    assert int(bad.item()) == 1
    assert_mass(case, q, 0.1, mass, hidden=hidden, what="pages")


def test_masses_of_wrongly_described_sequences(hip):
    step("masses of wrongly described sequences")
    case = Case("f16", [30] * 4, [20] * 4, 2, 64, 16, seed=35)
    q = normal(12, (80, 4, 64), torch.float32, 2.0).to(DEV)
    for offsets, starts, good in (([0, 20, 40, 60, 81], [30] * 4, [0, 1, 2]), ([0, 20, 40, 60, 80], [30, -1, 1 << 30, 30], [0, 3]),
                                  ([0, 20, 40, 60, 20], [30] * 4, [0, 1, 2])):
        mass, bad = torch.full((case.cache.pages, 2, 16), 7.0, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        hip.attentionMass(q, case.cache, d.Sequences(dev_i32(case.tables), dev_i32(starts), dev_i32(offsets)), 0.1,
                          mass, badPage=bad)
        assert int(bad.item()) == 1
        for s, ((want, bar), got) in enumerate(zip(wanted_mass(case, q, 0.1, None), gathered(case, mass))):
            if s in good:
                assert bool(((got.double() - want).abs() <= bar).all()), s
            else:
                assert bool((got == 7).all()), s


def test_masses_of_no_rows(hip):
    step("masses of no rows")
    case = Case("f16", [5], [0], 2, 64, 16)
    mass = torch.full((case.cache.pages, 2, 16), 7.0, device=DEV)
    hip.attentionMass(torch.empty(0, 4, 64, device=DEV), case.cache, case.sequences(), 0.1, mass)
    empty = d.Sequences(dev_i32(np.zeros((0, 3))), dev_i32([]), dev_i32([0]))
    hip.attentionMass(torch.zeros(3, 4, 64, device=DEV), case.cache, empty, 0.1, mass)
    assert bool((mass == 7).all())


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("rows", [[1, 1, 1], [200, 1, 9]])
def test_masses_the_same_bits_every_time(hip, kind, rows):
    step(f"masses twice {kind} {rows}")
    case = Case(kind, [3000, 100, 999], rows, 2, 128, 16, seed=36)
    q = normal(13, (case.tokens, 16, 128), torch.bfloat16, 2.0).to(DEV)
    first, second, third = (torch.zeros(case.cache.pages, 2, 16, device=DEV) for _ in range(3))
    hip.attentionMass(q, case.cache, case.sequences(), 0.1, first)
    hip.attentionMass(q, case.cache, case.sequences(), 0.1, second)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    d.HipOps(stream).attentionMass(q, case.cache, case.sequences(), 0.1, third)
    torch.cuda.synchronize()
    assert torch.equal(first, second) and torch.equal(first, third)
    flat = torch.empty(q.numel() + 4, dtype=q.dtype, device=DEV)[4:].view(q.shape)
    flat.copy_(q)
    hip.attentionMass(flat, case.cache, case.sequences(), 0.1, third)
    assert_mass(case, q, 0.1, third, what="queries off 16 bytes")


# ------------------------------------------------------------------ the heaviest

def pick(mass, tables, lengths, sinks, recent, keep):
    """kept and counts as the definition has them."""
    pages, kv, page = mass.shape
    kept, counts = np.full((len(lengths), kv, keep), -1, np.int32), np.zeros(len(lengths), np.int32)
    for s, n in enumerate(lengths):
        counts[s] = min(n, keep)
        for h in range(kv):
            if n <= keep:
                kept[s, h, :n] = np.arange(n)
                continue
            j = np.arange(sinks, n - recent)
            at = tables[s, j // page].astype(np.int64)
            there = (at >= 0) & (at < pages)
            m = mass[np.where(there, at, 0), h, j % page].astype(np.float64)
            m = np.where(np.isnan(m), np.inf, m)
            nan = np.isnan(mass[np.where(there, at, 0), h, j % page])
            order = np.lexsort((j, -np.where(there, m, -np.inf), ~(nan & there), ~there))
            chosen = np.sort(j[order[:keep - sinks - recent]])
            kept[s, h] = np.concatenate([np.arange(sinks), chosen, np.arange(n - recent, n)])
    return kept, counts


def choose(hip, mass, tables, lengths, sinks, recent, keep, bad=None):
    kept = torch.full((len(lengths), mass.shape[1], keep), 99, dtype=torch.int32, device=DEV)
    counts = torch.full((len(lengths),), 99, dtype=torch.int32, device=DEV)
    hip.heaviest(torch.from_numpy(mass).to(DEV), dev_i32(tables), dev_i32(lengths), sinks, recent, kept, counts, bad)
    return kept.cpu().numpy(), counts.cpu().numpy()


def tables_for(lengths, page, seed, spare=2):
    rng = np.random.default_rng(seed)
    used = [-(-int(n) // page) for n in lengths]
    pages = sum(used) + spare
    order, at = rng.permutation(pages), 0
    tables = np.full((len(used), max(used) + 1), -9, np.int32)
    for s, n in enumerate(used):
        tables[s, :n] = order[at:at + n]
        at += n
    return tables, pages


KEEPS = [
    # (lengths, kv, page, sinks, recent, keep)
    ([1], 1, 16, 0, 0, 1), ([5, 0, 8, 9], 2, 16, 1, 2, 8), ([1900], 8, 16, 4, 128, 512), ([700, 64, 65, 4000], 2, 48, 4, 16, 64),
    ([300], 3, 16, 0, 0, 299), ([300], 3, 16, 10, 20, 30), ([300, 20], 3, 16, 0, 0, 0), ([1025, 1088, 1024], 2, 64, 0, 0, 1000),
    ([40000], 2, 128, 4, 64, 1000), ([131073], 1, 16, 3, 7, 5000), ([66000, 12], 1, 256, 0, 1, 3), ([17000, 9], 5, 16, 1, 0, 16000),
]


@pytest.mark.parametrize("kind", ["spread", "equal", "few", "zeros", "signs", "nan"])
@pytest.mark.parametrize("lengths,kv,page,sinks,recent,keep", KEEPS)
def test_the_heaviest(hip, kind, lengths, kv, page, sinks, recent, keep):
    step(f"heaviest {keep} of {lengths}, {kv} heads, pages of {page}, {kind}")
    rng = np.random.default_rng(len(lengths) + keep)
    tables, pages = tables_for(lengths, page, 5)
    mass = np.exp(2.5 * rng.standard_normal((pages, kv, page))).astype(np.float32)
    if kind == "equal":
        mass[:] = 0.37
    elif kind == "few":  # ties everywhere
        mass = rng.integers(0, 4, mass.shape).astype(np.float32)
    elif kind == "zeros":
        mass = np.where(rng.random(mass.shape) < 0.97, np.where(rng.random(mass.shape) < 0.5, 0.0, -0.0), mass).astype(np.float32)
    elif kind == "signs":
        mass = (rng.standard_normal(mass.shape) * 1e-42 * 10.0 ** rng.integers(0, 70, mass.shape)).astype(np.float32)
        mass = np.where(rng.random(mass.shape) < 0.02, np.where(rng.random(mass.shape) < 0.5, np.inf, -np.inf), mass).astype(np.float32)
    elif kind == "nan":
        mass = np.where(rng.random(mass.shape) < 0.2, np.where(rng.random(mass.shape) < 0.5, np.nan, np.inf), mass).astype(np.float32)
    want, counts = pick(mass, tables, lengths, sinks, recent, keep)
    got, told = choose(hip, mass, tables, lengths, sinks, recent, keep)
    assert np.array_equal(told, counts)
    assert np.array_equal(got, want), (got[got != want][:5], want[got != want][:5])


def test_the_heaviest_of_wrong_lengths_and_pages(hip):
    step("heaviest of wrong lengths and pages")
    tables, pages = tables_for([200, 200, 200], 16, 6)
    mass = np.abs(np.random.default_rng(3).standard_normal((pages, 2, 16))).astype(np.float32)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    good = choose(hip, mass, tables, [200, 100, 3], 2, 3, 50, bad)
    assert int(bad.item()) == 0
    got, counts = choose(hip, mass, tables, [200, -1, 5000], 2, 3, 50, bad)
    assert int(bad.item()) == 1 and counts.tolist() == [50, 0, 0]
    assert np.array_equal(got[0], good[0][0]) and bool((got[1:] == -1).all())
    bad.zero_()
    tables[0, 3], tables[0, 5] = -1, pages
    got, counts = choose(hip, mass, tables, [200, 100, 3], 2, 3, 190, bad)
    assert int(bad.item()) == 1
    want, _ = pick(mass, tables, [200, 100, 3], 2, 3, 190)
    assert np.array_equal(got, want)


# ------------------------------------------------------------------ moves

def cache_of(kind, pages, page, kv, dim, seed):
    """A cache of any bits, and masses."""
    gen = torch.Generator().manual_seed(seed)
    if kind == "f16":
        def bits(*shape):
            return torch.randint(-2 ** 15, 2 ** 15, shape, generator=gen, dtype=torch.int16).view(torch.float16).to(DEV)
        cache = d.KvCache(bits(pages, page, kv, dim), bits(pages, kv, dim, page), page)
    else:
        def codes(*shape):
            return torch.randint(-128, 128, shape, generator=gen, dtype=torch.int8).to(DEV)
        cache = d.QuantizedKvCache(codes(pages, page, kv, dim), codes(pages, kv, dim, page),
                                   torch.randn(pages, kv, page, generator=gen).to(DEV),
                                   torch.randn(pages, kv, page, generator=gen).to(DEV), page)
    return cache, torch.randn(pages, kv, page, generator=gen).to(DEV)


def parts(cache, mass=None):
    """Its tensors' bits on the host, by name."""
    found = {"keys": cache.keys, "values": cache.values}
    if isinstance(cache, d.QuantizedKvCache):
        found.update(key_scales=cache.keyScales, value_scales=cache.valueScales)
    if mass is not None:
        found["mass"] = mass
    return {w: t.cpu().view(torch.int16 if t.dtype == torch.float16 else t.dtype).numpy().copy() for w, t in found.items()}


def moved(old, tables, kept, counts, starts, into, page):
    """What the parts hold after the move."""
    new = {w: t.copy() for w, t in old.items()}
    pages, kv = old["values"].shape[:2]
    for s in range(len(tables)):
        if not (0 <= counts[s] <= kept.shape[-1] and starts[s] >= 0):
            continue
        for h in range(kv):
            for i in range(counts[s]):
                a = int(kept[s, h, i] if kept.ndim == 3 else kept[s, i])
                b = int(starts[s]) + i
                if not (0 <= a < tables.shape[1] * page and b < into.shape[1] * page):
                    continue
                p, q = int(tables[s, a // page]), int(into[s, b // page])
                if not (0 <= p < pages and 0 <= q < pages):
                    continue
                a, b = a % page, b % page
                new["keys"][q, b, h] = old["keys"][p, a, h]
                new["values"][q, h, :, b] = old["values"][p, h, :, a]
                for w in ("key_scales", "value_scales", "mass"):
                    if w in old:
                        new[w][q, h, b] = old[w][p, h, a]
    return new


def assert_parts(cache, mass, want):
    got = parts(cache, mass)
    for w in want:
        assert np.array_equal(got[w].view(np.uint8), want[w].view(np.uint8)), w


MOVES = [
    # (lengths, kv, dim, page, most, start of what is moved to, apart for each head)
    ([40], 2, 128, 16, 1, 37, False), ([200, 33, 90], 8, 128, 16, 7, 20, False), ([500, 130], 2, 64, 32, 64, 0, True),
    ([700], 4, 96, 48, 65, 5, True), ([300, 1, 64], 1, 256, 16, 130, 0, True), ([2000], 3, 72, 64, 900, 0, True),
    ([90, 90], 2, 20, 16, 33, 3, True), ([64], 2, 7, 16, 20, 1, False), ([400], 1, 512, 16, 100, 16, True),
    ([3000, 2500], 2, 128, 128, 1024, 0, True), ([250], 2, 1, 16, 100, 0, True),
]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("order", ["ascending", "any"])
@pytest.mark.parametrize("lengths,kv,dim,page,most,start,heads", MOVES)
def test_moves(hip, kind, order, lengths, kv, dim, page, most, start, heads):
    step(f"moves {kind} {order} {most} of {lengths}, {kv} heads of {dim}, pages of {page}, to {start}")
    rng = np.random.default_rng(most + dim)
    count = len(lengths)
    tables, pages = tables_for([max(n, start + most) for n in lengths], page, 8, spare=4)
    counts = [min(most, n) for n in lengths]
    shape = (count, kv, most) if heads else (count, most)
    kept = np.zeros(shape, np.int32)
    for s, n in enumerate(lengths):
        for h in range(kv if heads else 1):
            row = rng.choice(n, counts[s], replace=order == "any")
            kept[(s, h) if heads else s][:counts[s]] = np.sort(row) if order == "ascending" else row
            kept[(s, h) if heads else s][counts[s]:] = rng.integers(-3, 10 ** 9)
    starts = [start] * count
    for mass_too in (False, True):
        cache, mass = cache_of(kind, pages, page, kv, dim, 7)
        old = parts(cache, mass)
        want = moved(old, tables, kept, counts, starts, tables, page)
        if not mass_too:
            want["mass"] = old["mass"]
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept), dev_i32(counts), dev_i32(starts), None,
                      mass if mass_too else None, bad)
        assert_parts(cache, mass, want)
        assert int(bad.item()) == 0
    # into pages of their own
    rooms, more = tables_for([start + most] * count, page, 9, spare=0)
    into = np.where(rooms >= 0, rooms + pages, rooms)
    cache, mass = cache_of(kind, pages + more, page, kv, dim, 10)
    old = parts(cache, mass)
    hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept), dev_i32(counts), dev_i32(starts), dev_i32(into), mass)
    assert_parts(cache, mass, moved(old, tables, kept, counts, starts, into, page))


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("most", [5, 200])
@pytest.mark.parametrize("apart", [False, True])
def test_moves_of_entries_that_are_none(hip, kind, most, apart):
    step(f"moves of entries that are none {kind} {most} {apart}")
    page, kv, dim = 16, 2, 64
    tables, pages = tables_for([300] * 4, page, 11, spare=40)
    tables[0, 3], tables[1, 0] = -1, pages  # sources, and a place that rows go to
    into = tables if not apart else tables_for([300] * 4, page, 12)[0] + pages
    if apart:
        into[2, 0] = 1 << 30
    rng = np.random.default_rng(5)
    kept = rng.integers(0, 300, (4, kv, most)).astype(np.int32)
    kept[2, 0, 1], kept[2, 1, 2], kept[3, 0, 0] = -1, 1 << 30, -2 ** 31
    cache, mass = cache_of(kind, pages + (200 if apart else 0), page, kv, dim, 13)
    for counts, starts in (([most] * 4, [0] * 4), ([most, -1, most + 1, most], [0, 0, 0, -5]), ([1, 0, most, 2], [299, 5, 2 ** 31 - 1, 30])):
        old = parts(cache, mass)
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept), dev_i32(counts), dev_i32(starts),
                      dev_i32(into) if apart else None, mass, bad)
        want = moved(old, tables, kept, counts, starts, into, page)
        assert_parts(cache, mass, want)
        assert int(bad.item()) == 1


@pytest.mark.parametrize("kind", CACHES)
def test_moves_without_counts_and_starts_and_of_nothing(hip, kind):
    step(f"moves without counts and starts {kind}")
    tables, pages = tables_for([100, 80], 16, 14)
    kept = np.stack([np.arange(99, 59, -1), np.arange(40)]).astype(np.int32)
    cache, mass = cache_of(kind, pages, 16, 3, 48, 15)
    old = parts(cache, mass)
    hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept))
    assert_parts(cache, None, moved({w: t for w, t in old.items() if w != "mass"}, tables, kept, [40, 40], [0, 0], tables, 16))
    now = parts(cache, mass)
    hip.cacheKeep(cache, dev_i32(tables), dev_i32(np.zeros((2, 0))))
    hip.cacheKeep(cache, dev_i32(np.zeros((0, 3))), dev_i32(np.zeros((0, 4))))
    hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept), dev_i32([0, 0]))
    assert_parts(cache, mass, now)
    # page tables given a second time are in place
    hip.cacheKeep(cache, t := dev_i32(tables), dev_i32(kept), None, None, t)
    assert_parts(cache, None, moved({w: x for w, x in now.items() if w != "mass"}, tables, kept, [40, 40], [0, 0], tables, 16))


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_drafted_tree_checked_and_its_path_kept(hip, kind, dtype):
    """A server's step, captured once and replayed: the drafted tokens' keys
    and values go into the cache, their tree attends, the accepted path's rows
    are moved together, and the next token attends to them: it is what it is in
    a cache that only ever held the path."""
    step(f"a drafted tree, checked {kind} {dtype}")
    heads, kv, dim, page, t = 8, 2, 128, 16, TYPES[dtype]
    prompts, nodes = [70, 23, 250], 12
    make = d.KvCache.allocate if kind == "f16" else d.QuantizedKvCache.allocate
    tables, pages = tables_for([n + nodes + 8 for n in prompts], page, 21)
    tree_cache, path_cache = make(pages, page, kv, dim), make(pages, page, kv, dim)
    device_tables, starts = dev_i32(tables), dev_i32(prompts)
    chunk = d.Sequences(device_tables, dev_i32([0] * 3), dev_i32(np.concatenate([[0], np.cumsum(prompts)])))
    k, v = normal(30, (sum(prompts), kv, dim), t).to(DEV), normal(31, (sum(prompts), kv, dim), t).to(DEV)
    for cache in (tree_cache, path_cache):
        hip.cacheWriteSequences(k, v, cache, chunk)
    sees = trees([nodes] * 3, 22)
    words = packed(sees, 1)
    # an accepted path: the ancestors of a leaf, and it
    paths = [np.flatnonzero(s[leaf]) for s, leaf in zip(sees, (11, 9, 7))]
    most = max(len(p) for p in paths)
    kept = np.zeros((3, most), np.int32)
    for s, p in enumerate(paths):
        kept[s, :len(p)] = prompts[s] + p
    accepted, device_kept = dev_i32([len(p) for p in paths]), dev_i32(kept)
    drafted = d.Sequences(device_tables, starts, dev_i32(np.arange(4) * nodes))
    after = d.Sequences(device_tables, dev_i32([n + len(p) for n, p in zip(prompts, paths)]))
    dk, dv, dq = (torch.empty(3 * nodes, h, dim, dtype=t, device=DEV) for h in (kv, kv, heads))
    nk, nv, nq = (torch.empty(3, h, dim, dtype=t, device=DEV) for h in (kv, kv, heads))
    tree_out, next_out = torch.empty_like(dq), torch.empty_like(nq)

    def calls():
        hip.cacheWriteSequences(dk, dv, tree_cache, drafted)
        hip.attentionTree(dq, tree_cache, drafted, words, 0.1, tree_out)
        hip.cacheKeep(tree_cache, device_tables, device_kept, accepted, starts)
        hip.cacheWriteSequences(nk, nv, tree_cache, after)
        hip.attentionSequences(nq, tree_cache, after, 0.1, next_out)

    for x in (dk, dv, dq, nk, nv, nq):
        x.normal_()
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    want_next, want_path = torch.empty_like(nq), torch.empty(sum(len(p) for p in paths), heads, dim, dtype=t, device=DEV)
    for i in range(3):
        for n, x in enumerate((dk, dv, dq, nk, nv, nq)):
            x.copy_(normal(100 * i + n, x.shape, t, 2.0 if x.shape[1] == heads else 1.0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        rows = torch.cat([torch.from_numpy(p + s * nodes) for s, p in enumerate(paths)]).to(DEV)
        path = d.Sequences(device_tables, starts, dev_i32(np.concatenate([[0], np.cumsum([len(p) for p in paths])])))
        hip.cacheWriteSequences(dk[rows].contiguous(), dv[rows].contiguous(), path_cache, path)
        hip.attentionSequences(dq[rows].contiguous(), path_cache, path, 0.1, want_path)
        hip.cacheWriteSequences(nk, nv, path_cache, after)
        hip.attentionSequences(nq, path_cache, after, 0.1, want_next)
        torch.cuda.synchronize()
        assert torch.equal(next_out, want_next), f"replay {i}"
        # the path's rows of the tree are the chain's, but for where their positions lie
        off = float((tree_out[rows].double() - want_path.double()).abs().max() / want_path.double().abs().max())
        assert off <= (2.0 ** -7 if dtype == "bf16" else 1e-5), f"replay {i}: {off}"


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_cache_cut_to_its_heaviest(hip, kind, dtype):
    """A prompt's masses, a step's added to them, the heaviest kept, the cache
    cut to them in place and decoding gone on with: each head's next row is
    the attention over the positions that it kept. Captured and replayed, too."""
    step(f"a cache cut to its heaviest {kind} {dtype}")
    heads, kv, dim, page, t, keep = 8, 2, 64, 16, TYPES[dtype], 40
    case = Case(kind, [0, 0, 0], [130, 60, 33], kv, dim, page, seed=41)
    lengths = [130, 60, 33]
    device_tables = dev_i32(case.tables)
    q = normal(42, (case.tokens, heads, dim), t, 2.0).to(DEV)
    last = torch.tensor(case.offsets[1:] - 1, device=DEV)
    mass, saved = torch.zeros(case.cache.pages, kv, page, device=DEV), parts(case.cache)
    first = torch.empty_like(mass)
    kept = torch.zeros(3, kv, keep, dtype=torch.int32, device=DEV)
    counts, device_lengths = torch.zeros(3, dtype=torch.int32, device=DEV), dev_i32(lengths)
    prompt, step_rows = case.sequences(), d.Sequences(device_tables, dev_i32([n - 1 for n in lengths]))
    q1, out = q[last].contiguous(), torch.empty(3, heads, dim, dtype=t, device=DEV)

    def calls():
        hip.attentionMass(q, case.cache, prompt, 0.125, mass)
        first.copy_(mass)
        hip.attentionMass(q1, case.cache, step_rows, 0.125, mass, mass)
        hip.heaviest(mass, device_tables, device_lengths, 2, 8, kept, counts)
        hip.cacheKeep(case.cache, device_tables, kept, counts, mass=mass)
        hip.attentionSequences(q1, case.cache, d.Sequences(device_tables, counts - 1), 0.125, out)

    def restore():
        for w, x in (("keys", case.cache.keys), ("values", case.cache.values)):
            x.copy_(torch.from_numpy(saved[w]).view(x.dtype))
        if kind == "i8":
            case.cache.keyScales.copy_(torch.from_numpy(saved["key_scales"]))
            case.cache.valueScales.copy_(torch.from_numpy(saved["value_scales"]))

    calls()
    torch.cuda.synchronize()
    eager = out.clone(), kept.clone(), mass.clone()
    # the step's own position is anew in its masses: its row alone has seen it
    assert_mass(case, q, 0.125, first, what="the prompt's")
    tables = case.tables
    chosen = kept.cpu().numpy()
    assert counts.tolist() == [40, 40, 33]
    for s, n in enumerate(lengths):
        k, v = case.dense[s]
        for h in range(heads):
            at = chosen[s, h // (heads // kv)][:min(n, keep)]
            assert (np.diff(at) > 0).all() and at[:2].tolist() == [0, 1] and at[-8:].tolist() == list(range(n - 8, n))
            logits = 0.125 * (k[at, h // (heads // kv)] @ q1[s, h].cpu().double())
            want = torch.softmax(logits, 0) @ v[at, h // (heads // kv)]
            off = float((out[s, h].cpu().double() - want).abs().max() / want.abs().max())
            assert off <= (2.0 ** -7 if dtype == "bf16" else 1e-5)
    restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for _ in range(3):
        restore()
        mass.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager[:2], (out, kept)))
        held = [torch.equal(gathered(case, eager[2])[s], gathered(case, mass)[s]) for s in range(3)]
        assert all(held), held


# ------------------------------------------------------------------ calls beside each other, and far ones

@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("order", ["ascending", "any"])
@pytest.mark.parametrize("count,kv,dim,page,most,start", [(24, 4, 128, 16, 300, 5), (40, 8, 64, 32, 257, 64)])
def test_moves_of_many_lists(hip, kind, order, count, kv, dim, page, most, start):
    """As many as keep a block each for all their chunks: in order, and (rows that come from places already
    written) by way of the workspace."""
    step(f"moves of many lists {kind} {order} {count} of {most}")
    rng = np.random.default_rng(most)
    lengths = [start + most + int(n) for n in rng.integers(1, 200, count)]
    tables, pages = tables_for(lengths, page, 51)
    counts = rng.integers(most - 140, most + 1, count)
    counts[0], counts[1], counts[2] = most, 0, 128
    kept = np.zeros((count, kv, most), np.int32)
    for s, n in enumerate(lengths):
        for h in range(kv):
            row = rng.choice(n, most, replace=order == "any")  # (with the same position more than once)
            kept[s, h] = np.sort(row) if order == "ascending" else row
    if order == "ascending":  # from `start` on, no row comes from before its place
        kept = np.maximum(kept, start + np.arange(most, dtype=np.int32))
    cache, mass = cache_of(kind, pages, page, kv, dim, 52)
    old = parts(cache, mass)
    hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept), dev_i32(counts), dev_i32([start] * count), mass=mass)
    assert_parts(cache, mass, moved(old, tables, kept, counts, [start] * count, tables, page))


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,rows,group,dim", [([700, 3, 64], [7, 8, 1], 4, 128), ([0, 2000], [3, 2], 7, 64), ([95], [17], 1, 256),
                                                  ([40, 0, 5], [32, 30, 33], 1, 80)])
def test_masses_of_rows_past_a_unit_of_16(hip, kind, dtype, starts, rows, group, dim):
    step(f"masses of rows past a unit {kind} {dtype} {rows} of {group} heads of {dim}")
    case = Case(kind, starts, rows, 2, dim, 32, seed=67)
    q = normal(68, (case.tokens, 2 * group, dim), TYPES[dtype], 2.0).to(DEV)
    before = masses(case, 69)
    mass = torch.zeros_like(before)
    hip.attentionMass(q, case.cache, case.sequences(), 1 / math.sqrt(dim), mass, before)
    assert_mass(case, q, 1 / math.sqrt(dim), mass, before, what="rows past a unit")


@pytest.mark.parametrize("kind", CACHES)
def test_masses_of_steps_with_more_scores_than_are_kept(hip, kind):
    """Page tables with room for so many positions that a step's scores are taken twice."""
    step(f"masses of steps over wide page tables {kind}")
    case = Case(kind, [700, 90, 0], [1, 1, 1], 2, 128, 16, seed=53)
    case.tables = np.concatenate([case.tables, np.full((3, 400_000), -7, np.int32)], 1)
    q = normal(54, (3, 8, 128), torch.bfloat16, 2.0).to(DEV)
    before = masses(case, 55)
    mass = torch.zeros_like(before)
    hip.attentionMass(q, case.cache, case.sequences(offsets=False, longest=701), 0.1, mass, before)
    assert_mass(case, q, 0.1, mass, before, what="wide page tables")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 70])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_masses_of_scales_that_are_not_above_zero(hip, dtype, tokens, scale):
    step(f"masses of a scale of {scale} {dtype} {tokens}")
    case = Case("f16", [333], [tokens], 2, 64, 16, seed=56)
    q = normal(57, (tokens, 4, 64), TYPES[dtype], 2.0).to(DEV)
    mass = torch.zeros(case.cache.pages, 2, 16, device=DEV)
    hip.attentionMass(q, case.cache, case.sequences(), scale, mass)
    assert_mass(case, q, scale, mass, what=f"scale {scale}")


@pytest.mark.parametrize("kind", CACHES)
def test_a_cache_of_more_values_than_32_bits_count(hip, kind):
    """The same sequences in a small cache and on the first and last pages of a
    large one: the same bits."""
    step(f"a large cache {kind}")
    kv, dim, page, heads = 8, 128, 64, 16
    pages = (1 << 32) // (page * kv * dim) + 100
    case = Case(kind, [600, 500], [20, 1], kv, dim, page, seed=58)
    small = case.cache
    make = d.KvCache.allocate if kind == "f16" else d.QuantizedKvCache.allocate
    large = make(pages, page, kv, dim)
    place = torch.arange(small.pages)
    place[1::2] += pages - small.pages  # every other page at the far end
    far = np.where(case.tables >= 0, place.numpy()[np.clip(case.tables, 0, None)], case.tables).astype(np.int32)
    names = ("keys", "values") + (("keyScales", "valueScales") if kind == "i8" else ())

    def fill():
        for w in names:
            getattr(large, w)[place.to(DEV)] = getattr(small, w)

    fill()
    near_rows = case.sequences()
    far_rows = d.Sequences(dev_i32(far), near_rows.starts, near_rows.offsets)
    q = normal(59, (21, heads, dim), torch.bfloat16, 2.0).to(DEV)
    sees = trees([20, 1], 60)
    words = packed(sees, 1)
    outs = []
    for cache, rows in ((small, near_rows), (large, far_rows)):
        out, mass = torch.empty_like(q), torch.zeros(cache.pages, kv, page, device=DEV)
        hip.attentionTree(q, cache, rows, words, 0.1, out)
        hip.attentionMass(q, cache, rows, 0.1, mass)
        one = torch.zeros_like(mass)
        hip.attentionMass(q[19:].contiguous(), cache, d.Sequences(rows.pageTables, dev_i32([619, 500])), 0.1, one, mass)
        kept = torch.zeros(2, kv, 200, dtype=torch.int32, device=DEV)
        counts = torch.zeros(2, dtype=torch.int32, device=DEV)
        hip.heaviest(one, rows.pageTables, dev_i32([620, 501]), 4, 30, kept, counts)
        hip.cacheKeep(cache, rows.pageTables, kept, counts, mass=one)
        at = torch.arange(small.pages) if cache is small else place
        outs.append([out.cpu(), kept.cpu(), counts.cpu()] + [x[at.to(DEV)].cpu() for x in (mass, one)] +
                    [getattr(cache, w)[at.to(DEV)].cpu() for w in names])
    for near, far_one in zip(*outs):
        assert torch.equal(near.view(torch.uint8), far_one.view(torch.uint8))


def test_graphs_beside_each_other(hip):
    """Each captured call's workspace is its own: two graphs of all the calls, replayed at once on two streams with
    eager calls on a third, give what each gives alone."""
    step("graphs beside each other")
    heads, kv, dim, page, runs = 8, 2, 128, 16, []
    for n, rows in enumerate(([9, 40, 3], [70, 1, 130])):
        case = Case("f16", [700, 350, 1200], rows, kv, dim, page, seed=61 + n)
        q = normal(63 + n, (case.tokens, heads, dim), torch.bfloat16, 2.0).to(DEV)
        words = packed(trees(rows, n), 5)
        mass = torch.zeros(case.cache.pages, kv, page, device=DEV)
        kept, counts = torch.zeros(3, kv, 150, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
        out, rest, tables = torch.empty_like(q), case.sequences(), dev_i32(case.tables)
        lengths = dev_i32(case.starts + case.rows)
        saved = case.cache.keys.clone(), case.cache.values.clone()
        stream = torch.cuda.Stream()
        ops = d.HipOps(stream)

        def calls(ops=ops, case=case, q=q, words=words, mass=mass, kept=kept, counts=counts, out=out, rest=rest,
                  tables=tables, lengths=lengths, saved=saved):
            case.cache.keys.copy_(saved[0])
            case.cache.values.copy_(saved[1])
            ops.attentionTree(q, case.cache, rest, words, 0.1, out)
            ops.attentionMass(q, case.cache, rest, 0.1, mass)
            ops.heaviest(mass, tables, lengths, 2, 16, kept, counts)
            ops.cacheKeep(case.cache, tables, kept, counts, mass=mass)

        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            calls()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls()
        held = [out, mass, kept, counts, case.cache.keys, case.cache.values]
        want = [x.clone() for x in held]
        runs.append((graph, stream, held, want, calls))  # (the calls hold what a graph reads)
    case = Case("i8", [900], [30], kv, dim, page, seed=65)
    q = normal(66, (30, heads, dim), torch.bfloat16, 2.0).to(DEV)
    alone, now = (torch.zeros(case.cache.pages, kv, page, device=DEV) for _ in range(2))
    sequence = case.sequences()
    hip.attentionMass(q, case.cache, sequence, 0.1, alone)
    for turn in range(4):
        for _, _, held, _, _ in runs:
            for x in held[:4]:
                x.zero_()
        torch.cuda.synchronize()
        for graph, stream, _, _, _ in runs * 3:
            with torch.cuda.stream(stream):
                graph.replay()
        hip.attentionMass(q, case.cache, sequence, 0.1, now)
        torch.cuda.synchronize()
        assert torch.equal(now, alone), turn
        for _, _, held, want, _ in runs:
            for x, y in zip(held, want):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), turn


# ------------------------------------------------------------------ weights' bits

def cancelling_codes(weights, dim, rng):
    """Whole numbers [positions, dim] within 127 that almost cancel: sum_j weights[j] codes[j] is next to nothing
    beside sum_j weights[j] |codes[j]|."""
    codes = rng.integers(-127, 128, (len(weights), dim)).astype(np.float64)
    rest = weights @ codes
    for j in np.argsort(-weights):
        to = np.clip(codes[j] - np.round(rest / weights[j]), -127, 127)
        rest += weights[j] * (to - codes[j])
        codes[j] = to
    return codes


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,rows,dim", [(300, 3, 128), (300, 12, 64), (900, 70, 128), (2900, 150, 64), (500, 40, 256),
                                            (1500, 200, 80)])
def test_trees_weights_have_22_bits(hip, kind, dtype, start, rows, dim):
    """Values whose weighted sum almost cancels: what is left of a row's
    result are its weights' roundings. Rows of the same queries, +-1, that see
    what lies before the tree; keys are whole numbers, so that scores are
    exact but for the factor's, the scale's and the difference's roundings, 3
    2^-24 of their size. So a row is off by 4 (3 2^-24 max|s| + 2^-20 + 2^-24
    sqrt(n)) of its sum of p |v| and 2^-39 max p sum |v| as above, and BF16
    results by half a step."""
    step(f"trees' weights {kind} {dtype} {rows} rows after {start}, heads of {dim}")
    kv, heads = 2, 4
    case = Case(kind, [start], [rows], kv, dim, 16, seed=71)
    rng = np.random.default_rng(start + dim)
    j = np.arange(start)
    page, off = torch.from_numpy(case.tables[0, j // 16].astype(np.int64)).to(DEV), torch.from_numpy(j % 16).to(DEV)
    q = rng.choice([-1.0, 1.0], (kv, dim))
    out, mass, lost, most = (np.zeros((kv, dim)), np.zeros((kv, dim)), np.zeros((kv, dim)), 0.0)
    for h in range(kv):
        keys = rng.integers(-4, 5, (start, dim)).astype(np.float64)
        scores = keys @ q[h] / 16
        most = max(most, float(np.abs(scores).max()))
        p = np.exp(scores - scores.max())
        p /= p.sum()
        scales = np.ones(start) if kind == "f16" else (0.5 + rng.random(start, np.float32)).astype(np.float32).astype(np.float64)
        codes = cancelling_codes(p * scales, dim, rng)
        values = codes * scales[:, None]
        out[h], mass[h], lost[h] = p @ values, p @ np.abs(values), p.max() * np.abs(values).sum(0)
        if kind == "i8":
            lost[h] = p.max() * 2 * scales.max() * 127 * start
            case.cache.keyScales[page, h, off] = 1.0
            case.cache.valueScales[page, h, off] = torch.from_numpy(scales.astype(np.float32)).to(DEV)
        case.cache.keys[page, off, h] = torch.from_numpy(keys).to(DEV, case.cache.keys.dtype)
        case.cache.values[page, h, :, off] = torch.from_numpy(codes).to(DEV, case.cache.values.dtype)
    queries = torch.from_numpy(np.repeat(q, heads // kv, 0)).to(DEV, TYPES[dtype]).expand(rows, heads, dim).contiguous()
    got = attend(hip, case, queries, packed([np.zeros((rows, rows), bool)], -(-rows // 32)), 1 / 16).cpu().double().numpy()
    bar = 4 * (3 * 2.0 ** -24 * most + 2.0 ** -20 + 2.0 ** -24 * math.sqrt(start)) * mass + 2.0 ** -39 * lost
    if dtype == "bf16":
        bar += 2.0 ** -8 * np.abs(out)
    worst = np.abs(got - np.repeat(out, heads // kv, 0)) / np.repeat(bar, heads // kv, 0)
    print(f"[gpu]   worst {worst.max():.3f} of the bar, {2.0 ** -12 * (mass / bar).max():.1f} bars are 2^-12 of the sizes", flush=True)
    assert worst.max() <= 1, worst.max()


# ------------------------------------------------------------------ moves' page tables

@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("most", [60, 300])
def test_moves_into_a_sequences_first_pages(hip, kind, most):
    """One sequence's first pages, as `into` the same memory as its page tables: in place, and rows past those pages
    move nothing."""
    step(f"moves into the first pages {kind} {most}")
    tables, pages = tables_for([500], 16, 73)
    device_tables = dev_i32(tables)
    kept = np.random.default_rng(74).permutation(500)[:most].astype(np.int32)[None]
    into = device_tables[:, :14]
    assert into.data_ptr() == device_tables.data_ptr()
    cache, mass = cache_of(kind, pages, 16, 3, 64, 75)
    old = parts(cache, mass)
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    hip.cacheKeep(cache, device_tables, dev_i32(kept), None, None, into, mass, bad)
    assert_parts(cache, mass, moved(old, tables, kept, [most], [0], tables[:, :14], 16))
    assert int(bad.item()) == (most > 14 * 16)


# ------------------------------------------------------------------ kernels' other forms

@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("order", ["ascending", "any"])
@pytest.mark.parametrize("dim", [8, 24, 40, 72, 200, 264])
@pytest.mark.parametrize("most,start", [(129, 0), (300, 7)])
def test_moves_of_heads_in_pieces_of_8_bytes(hip, kind, order, dim, most, start):
    """Heads of other than multiples of 16 values over 8 bits, with few and many pieces a thread."""
    step(f"moves in pieces {kind} {order} {dim} {most}")
    rng = np.random.default_rng(dim + most)
    lengths, kv, page = [start + most + 150, start + most + 3], 3, 16
    tables, pages = tables_for(lengths, page, 76)
    counts = [most, most - 2]
    kept = np.zeros((2, kv, most), np.int32)
    for s, n in enumerate(lengths):
        for h in range(kv):
            row = rng.choice(n, most, replace=order == "any")
            kept[s, h] = np.sort(row) if order == "ascending" else row
    cache, mass = cache_of(kind, pages, page, kv, dim, 77)
    old = parts(cache, mass)
    hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept), dev_i32(counts), dev_i32([start] * 2), mass=mass)
    assert_parts(cache, mass, moved(old, tables, kept, counts, [start] * 2, tables, page))
    rooms, more = tables_for([start + most] * 2, page, 78, spare=0)
    into = np.where(rooms >= 0, rooms + pages, rooms)
    cache, mass = cache_of(kind, pages + more, page, kv, dim, 79)
    old = parts(cache, mass)
    hip.cacheKeep(cache, dev_i32(tables), dev_i32(kept), dev_i32(counts), dev_i32([start] * 2), dev_i32(into), mass)
    assert_parts(cache, mass, moved(old, tables, kept, counts, [start] * 2, into, page))


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,chunk,group,dim,at", [(64, 401, 4, 64, 333), (40, 143, 7, 128, 1501), (70, 517, 2, 80, 2)])
def test_masses_of_one_long_chunk_among_single_tokens(hip, kind, dtype, count, chunk, group, dim, at):
    """So many single tokens that the call's rows are few on average: a chunk of more rows than are added up at a
    time keeps its scores too."""
    step(f"masses of a chunk of {chunk} among {count} tokens {kind} {dtype} {group} heads of {dim}")
    rows, starts = [1] * count, [(37 * i) % 90 for i in range(count)]
    rows[count // 2], starts[count // 2] = chunk, at
    assert sum(rows) * group <= count * 32 and chunk * group > 256
    case = Case(kind, starts, rows, 1, dim, 16, seed=81)
    q = normal(82, (case.tokens, group, dim), TYPES[dtype], 2.0).to(DEV)
    before = masses(case, 83)
    for longest in (0, 1):
        mass = torch.zeros_like(before)
        hip.attentionMass(q, case.cache, case.sequences(longest=longest), 1 / math.sqrt(dim), mass, before)
        assert_mass(case, q, 1 / math.sqrt(dim), mass, before, what=f"longest {longest}")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [None, d.AttentionWindow(200, 3)])
@pytest.mark.parametrize("starts,rows,dim", [([900, 31, 0, 64, 1200, 5], [9, 16, 3, 10, 1, 12], 128),
                                             ([400 + 7 * i for i in range(10)], [5, 4, 8, 1, 40, 6, 5, 3, 9, 0], 64),
                                             ([2500, 100, 900], [10, 9, 8], 256)])
def test_small_trees_together(hip, kind, dtype, window, starts, rows, dim):
    """Trees of 17 to 64 rows a key head with few on average, one of more among them."""
    step(f"small trees together {kind} {dtype} {window} {rows} rows, heads of {dim}")
    case = Case(kind, starts, rows, 2, dim, 16, seed=84)
    q = normal(85, (case.tokens, 8, dim), TYPES[dtype], 2.0).to(DEV)
    for shape in ("random", "any"):
        sees = trees(rows, 3, shape)
        got = attend(hip, case, q, packed(sees, 2), 0.1, window)
        assert_tree(case, q, 0.1, sees, got, window, what=shape)


# ------------------------------------------------------------------ one sequence by the entry points' arguments

@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,rows,dim", [(0, 1, 64), (517, 7, 128), (700, 90, 128), (33, 300, 64), (90, 9, 20)])
def test_one_sequence_without_starts_and_offsets(hip, kind, dtype, start, rows, dim):
    """The C entry points take one sequence of all rows at `start` without device arrays of either."""
    step(f"one sequence by arguments {kind} {dtype} {rows} rows at {start}, heads of {dim}")
    case = Case(kind, [start], [rows], 2, dim, 16, seed=86)
    q, heads, scale = normal(87, (rows, 8, dim), TYPES[dtype], 2.0).to(DEV), 8, 0.1
    tables, c, stream = dev_i32(case.tables), case.cache, torch.cuda.current_stream().cuda_stream
    p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())  # noqa: E731
    scales = (c.keyScales, c.valueScales) if kind == "i8" else (None, None)
    room = case.tables.shape[1] * 16

    def scratch(entry, *numbers):
        told = ctypes.c_int64()
        _lib.call(entry, *numbers, ctypes.byref(told))
        return torch.empty(max(told.value, 16), dtype=torch.uint8, device=DEV)

    sees = trees([rows], 88)
    words = packed(sees, -(-rows // 32))
    out, space = torch.full_like(q, 7.0), scratch("drift_tree_attention_workspace", 1, rows, heads, 2, dim, 0, 0, room)
    _lib.call(f"drift_tree_attention_{dtype}", p(q), p(c.keys), p(c.values), p(scales[0]), p(scales[1]), p(tables),
              case.tables.shape[1], c.pages, None, None, 1, start, rows, heads, 2, dim, 16, scale, 0, 0, room, p(words),
              words.shape[1], p(out), p(space), space.numel(), None, stream)
    assert_tree(case, q, scale, sees, out, what="tree")
    before = masses(case, 89)
    mass, space = torch.zeros_like(before), scratch("drift_attention_mass_workspace", 1, rows, heads, 2, dim, room, room)
    _lib.call(f"drift_attention_mass_{dtype}", p(q), p(c.keys), p(scales[0]), p(tables), case.tables.shape[1], c.pages, None,
              None, 1, start, rows, heads, 2, dim, 16, scale, room, p(before), p(mass), p(space), space.numel(), None, stream)
    assert_mass(case, q, scale, mass, before, what="mass")
