"""Attention over the paged cache and the 8-bit cache's rows on the GPU,
against plain implementations in 64 bits.

Bars, derived from the roundings on the way:
- the 8-bit cache's codes and scales, and what is read back of either cache:
  exact (the scale is one correctly rounded F32 quotient, a code the nearest
  whole number of the exact quotient, a value read back one F32 product rounded
  to the output's type);
- attention, F32: the row's result is off by the products' and sums' F32
  roundings. With n visible positions, D values a head and a score's size up to
  S, a score is off by at most (D + 4) 2^-24 S', S' = scale sum |q||k|; a weight
  relatively by that and 2^-20 (exponential, running rescales); weighted sums by
  a further (n + 8) 2^-24 in the worst case, sqrt(n) in earnest. Held to
  4 (2^-24 (sqrt(D) + 4) S' + 2^-20 + 2^-24 sqrt(n)) times the row's sum of p |v|.
- and for both types, what a weight that is small next to its row's largest
  loses: weights are F16 terms lifted so that the largest is 2^14 (its
  first term exact), and F16's last step is 2^-24, half of it 2^-25, so the
  last term of a weight is off by at most 2^-39 of the largest weight however
  small the weight is. With the values that is 2^-39 max p sum |v| over the
  visible positions; in 8 bits, where a weight is p times the value's scale w over
  a power of two above every scale so far (less than twice the largest), and the
  values are codes up to 127, 2^-39 max p 2 max w 127 n. BF16's one term is lifted
  by 2^7 at least, which makes it 2^-32. (It shows where a row's one strong
  position has a value of 0.)
"""

import math

import numpy as np
import pytest
import torch

from drift_amd import ops as d
from tests.helpers import DEV, dev_i32, step

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def hip():
    return d.HipOps()


def normal(seed, shape, dtype=torch.float32, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


# ------------------------------------------------------------------ a cache and its sequences

class Case:
    """A cache of random values with several sequences' shuffled pages in it.
    What no sequence holds is filled with NaN (F16) or scales of NaN (I8)."""

    def __init__(self, kind, starts, rows, kv, dim, page, seed=0, spare=2, value_scale=1.0):
        rng = np.random.default_rng(seed)
        self.kind, self.kv, self.dim, self.page = kind, kv, dim, page
        self.starts, self.rows = np.asarray(starts), np.asarray(rows)
        lengths = self.starts + self.rows
        used = -(-lengths // page)
        pages = int(used.sum()) + spare
        order = rng.permutation(pages)
        self.tables = np.full((len(used), int(used.max(initial=0)) + 1), -7, np.int32)
        at = 0
        for s, n in enumerate(used):
            self.tables[s, :n] = order[at:at + n]
            at += n
        self.tokens = int(self.rows.sum())
        self.offsets = np.concatenate([[0], np.cumsum(self.rows)])
        # dense keys and values of each sequence, and the cache that holds them
        self.dense, self.scales = [], []
        if kind == "f16":
            keys = torch.full((pages, page, kv, dim), float("nan"), dtype=torch.float16)
            values = torch.full((pages, kv, dim, page), float("nan"), dtype=torch.float16)
        else:
            keys = torch.full((pages, page, kv, dim), 99, dtype=torch.int8)
            values = torch.full((pages, kv, dim, page), -99, dtype=torch.int8)
            key_scales = torch.full((pages, kv, page), float("nan"))
            value_scales = torch.full((pages, kv, page), float("nan"))
        for s, n in enumerate(lengths):
            n = int(n)
            position = torch.arange(n)
            p = torch.from_numpy(self.tables[s].astype(np.int64))[position // page]
            o = position % page
            if kind == "f16":
                k = normal(1000 * seed + 2 * s, (n, kv, dim), torch.float16)
                v = normal(1000 * seed + 2 * s + 1, (n, kv, dim), torch.float16, value_scale)
                keys[p, o], values[p, :, :, o] = k, v
                self.dense.append((k.double(), v.double()))
            else:
                gen = torch.Generator().manual_seed(1000 * seed + s)
                k = torch.randint(-127, 128, (n, kv, dim), generator=gen, dtype=torch.int8)
                v = torch.randint(-127, 128, (n, kv, dim), generator=gen, dtype=torch.int8)
                ks = (0.5 + torch.rand((n, kv), generator=gen)) * 2.5 / 127
                vs = (0.5 + torch.rand((n, kv), generator=gen)) * 2.5 / 127 * value_scale
                keys[p, o], values[p, :, :, o] = k, v
                key_scales[p, :, o], value_scales[p, :, o] = ks, vs
                self.scales.append(vs.double())
                self.dense.append((k.double() * ks.double()[..., None], v.double() * vs.double()[..., None]))
        if kind == "f16":
            self.cache = d.KvCache(keys.to(DEV), values.to(DEV), page)
        else:
            self.cache = d.QuantizedKvCache(keys.to(DEV), values.to(DEV), key_scales.to(DEV), value_scales.to(DEV), page)

    def sequences(self, offsets=True, longest=0):
        return d.Sequences(dev_i32(self.tables), dev_i32(self.starts), dev_i32(self.offsets) if offsets else None,
                           longest)


def wanted(case, queries, scale, window=None, hidden=()):
    """The rows in 64 bits, and each value's bar's parts: the sum of p |v|, and
    the largest S' of the row's scores. `hidden`: (sequence, position) masked."""
    tokens, heads, dim = queries.shape
    q = queries.double()
    out, mass = torch.zeros(tokens, heads, dim, dtype=torch.float64), torch.zeros(tokens, heads, dim, dtype=torch.float64)
    size, count = torch.zeros(tokens, heads, 1, dtype=torch.float64), torch.zeros(tokens, heads, 1, dtype=torch.float64)
    small_weights = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    group = heads // case.kv
    for s, (k, v) in enumerate(case.dense):
        rows = slice(int(case.offsets[s]), int(case.offsets[s + 1]))
        at = torch.arange(int(case.rows[s]))[:, None] + int(case.starts[s])
        j = torch.arange(k.shape[0])[None, :]
        seen = j <= at
        if window is not None:
            seen &= (j > at - window.positions) | (j < window.sinks)
        for sequence, position in hidden:
            if sequence == s:
                seen[:, position] = False
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            logits = scale * (q[rows, h] @ kh.T)
            logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
            top = logits.amax(-1, keepdim=True) if logits.shape[1] else logits
            p = torch.exp(logits - torch.where(top == -math.inf, torch.zeros_like(top), top))
            p = torch.where(seen, p, torch.zeros_like(p))
            total = p.sum(-1, keepdim=True)
            p = torch.where(seen.any(-1, keepdim=True), p / total, torch.zeros_like(p))
            # what is not seen has no part, whatever it holds
            def weigh(x):
                return torch.where(seen[..., None], p[..., None] * x[None], torch.zeros(())).sum(1) if x.shape[0] \
                    else torch.zeros(p.shape[0], dim, dtype=torch.float64)
            small = not bool(torch.isfinite(vh).all())
            out[rows, h] = weigh(vh) if small else p @ vh
            mass[rows, h] = weigh(vh.abs()) if small else p @ vh.abs()
            if k.shape[0]:
                sizes = torch.where(seen, abs(scale) * (q[rows, h].abs() @ kh.abs().T), torch.zeros(()).double())
                size[rows, h] = sizes.amax(-1, keepdim=True)
            count[rows, h] = seen.sum(-1, keepdim=True).double()
            if k.shape[0]:
                if case.kind == "f16":
                    lost = p.amax(-1, keepdim=True) * (seen.double() @ vh.abs().nan_to_num(0, 0, 0))
                else:
                    lost = p.amax(-1, keepdim=True) * 2 * case.scales[s][:, h // group].max() * 127 * count[rows, h]
                small_weights[rows, h] = (2.0 ** -39 if queries.dtype == torch.float32 else 2.0 ** -32) * \
                    lost.nan_to_num(0)
    return out, mass, size, count, small_weights


def assert_rows(case, queries, scale, got, window=None, hidden=(), what=""):
    out, mass, size, count, small_weights = wanted(case, queries.cpu(), scale, window, hidden)
    got = got.cpu().double()
    same_nan = torch.isnan(out) == torch.isnan(got)
    assert bool(same_nan.all()), f"{what}: NaN in other places, {int((~same_nan).sum())}"
    inf = torch.isinf(out)
    assert bool((got[inf] == out[inf]).all()), f"{what}: infinities differ"
    fine = torch.isfinite(out)
    bar = 4 * (2.0 ** -24 * (math.sqrt(case.dim) + 4) * size + 2.0 ** -20 + 2.0 ** -24 * count.sqrt()) * mass
    if queries.dtype == torch.bfloat16:
        bar = bar + 2.0 ** -11 * mass + 2.0 ** -8 * out.abs()
    bar = bar + small_weights + 1e-30
    off = (got - out).abs()
    bad = fine & ~(off <= bar)
    worst = float((off / bar)[fine].max()) if bool(fine.any()) else 0.0
    print(f"[gpu]   worst {worst:.3f} of the bar", flush=True)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} values beyond the bar, worst {worst:.2f} times it, " \
        f"first at {bad.nonzero()[0].tolist()}"


def run(hip, case, queries, scale, window=None, single=False, offsets=True, longest=0, bad=None):
    out = torch.full(queries.shape, 7.0, dtype=queries.dtype, device=DEV)
    if single:
        hip.attention(queries, case.cache, dev_i32(case.tables[0]), int(case.starts[0]), scale, out, window, bad)
    else:
        hip.attentionSequences(queries, case.cache, case.sequences(offsets, longest), scale, out, window, bad)
    return out


CACHES = ["f16", "i8"]
DTYPES = ["f32", "bf16"]


# one sequence: a first token, one token after few and many, chunks that start and end inside pages and tiles; heads that
# share keys 1, 3, 4, 7 and 16 ways; sizes whole, padded and odd
SINGLE = [
    # (start, tokens, heads, kv heads, dim, page)
    (0, 1, 1, 1, 64, 16), (0, 1, 8, 2, 128, 16), (15, 1, 8, 2, 128, 16), (16, 1, 28, 4, 128, 64),
    (517, 1, 32, 8, 128, 16), (3000, 1, 16, 2, 256, 16), (700, 1, 6, 6, 128, 48), (9000, 1, 16, 1, 128, 128),
    (0, 7, 8, 2, 128, 16), (5, 37, 9, 3, 72, 16), (31, 33, 12, 3, 80, 48), (100, 65, 16, 4, 64, 32),
    (0, 130, 4, 2, 256, 16), (250, 129, 28, 4, 128, 64), (1, 300, 8, 8, 96, 16), (640, 257, 7, 1, 128, 16),
    (40, 20, 4, 2, 20, 16), (9, 5, 3, 3, 7, 16), (33, 3, 2, 1, 512, 16), (64, 40, 4, 4, 264, 32), (12, 70, 4, 1, 16, 16),
]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,tokens,heads,kv,dim,page", SINGLE)
def test_one_sequence(hip, kind, dtype, start, tokens, heads, kv, dim, page):
    step(f"attention {kind} {dtype} {tokens} tokens at {start}, {heads}/{kv} heads of {dim}, pages of {page}")
    case = Case(kind, [start], [tokens], kv, dim, page, seed=start + tokens)
    q = normal(5, (tokens, heads, dim), TYPES[dtype], 2.0).to(DEV)
    scale = 1 / math.sqrt(dim)
    assert_rows(case, q, scale, run(hip, case, q, scale, single=True), what="one sequence")


WINDOWS = [
    # (start, tokens, heads, kv, dim, page, window, sinks)
    (0, 1, 8, 2, 128, 16, 1, 0), (500, 1, 8, 2, 128, 16, 1, 1), (2000, 1, 32, 8, 128, 16, 333, 4),
    (100, 60, 8, 2, 64, 16, 40, 3), (0, 200, 8, 2, 128, 16, 17, 0), (300, 150, 16, 4, 64, 32, 128, 37),
    (777, 70, 4, 1, 256, 48, 100, 200), (50, 40, 4, 2, 128, 16, 4096, 4), (5000, 90, 7, 1, 128, 64, 64, 1),
    (30, 20, 3, 3, 20, 16, 9, 2), (1000, 33, 2, 2, 80, 16, 31, 1000),
]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,tokens,heads,kv,dim,page,positions,sinks", WINDOWS)
def test_windows_and_sinks(hip, kind, dtype, start, tokens, heads, kv, dim, page, positions, sinks):
    step(f"window {positions} + {sinks} {kind} {dtype} {tokens} tokens at {start}, {heads}/{kv} heads of {dim}")
    case = Case(kind, [start], [tokens], kv, dim, page, seed=start + 1)
    q = normal(6, (tokens, heads, dim), TYPES[dtype], 2.0).to(DEV)
    scale = 1 / math.sqrt(dim)
    window = d.AttentionWindow(positions, sinks)
    assert_rows(case, q, scale, run(hip, case, q, scale, window, single=True), window, what="window")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("longest", [0, 40, 100000])
def test_a_decode_step_of_several_sequences(hip, kind, dtype, longest):
    step(f"decode step {kind} {dtype} longest {longest}")
    starts = [0, 15, 16, 1, 900, 333, 64, 31, 2500]
    case = Case(kind, starts, [1] * len(starts), 2, 128, 16, seed=3)
    q = normal(7, (len(starts), 8, 128), TYPES[dtype], 2.0).to(DEV)
    scale = 1 / math.sqrt(128)
    assert_rows(case, q, scale, run(hip, case, q, scale, offsets=False, longest=longest), what="decode")
    assert_rows(case, q, scale, run(hip, case, q, scale, offsets=True, longest=longest), what="decode by offsets")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [None, d.AttentionWindow(50, 3)])
def test_a_mixed_batch(hip, kind, dtype, window):
    step(f"mixed batch {kind} {dtype} {window}")
    # sequences without rows among them, chunks of all sizes, and more than 64 sequences
    starts = [0, 700, 3, 50, 0, 1200, 17, 64, 5] + [10 * i for i in range(70)]
    rows = [130, 1, 0, 17, 1, 70, 200, 0, 33] + [1] * 70
    case = Case(kind, starts, rows, 2, 64, 32, seed=4)
    q = normal(8, (case.tokens, 14, 64), TYPES[dtype], 2.0).to(DEV)
    assert_rows(case, q, 0.125, run(hip, case, q, 0.125, window), window, what="mixed")


def test_no_rows_and_no_sequences(hip):
    step("attention of nothing")
    case = Case("f16", [5], [0], 2, 64, 16)
    q = torch.empty(0, 4, 64, device=DEV)
    hip.attention(q, case.cache, dev_i32(case.tables[0]), 5, 0.125, torch.empty_like(q))
    empty = d.Sequences(dev_i32(np.zeros((0, 3))), dev_i32([]), dev_i32([0]))
    kept = torch.full((3, 4, 64), 7.0, device=DEV)
    hip.attentionSequences(torch.zeros(3, 4, 64, device=DEV), case.cache, empty, 0.125, kept)
    assert bool((kept == 7).all())


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("rows_each", [[1, 1, 1], [5, 40, 1]])
def test_rows_outside_every_sequence_stay(hip, kind, rows_each):
    step(f"rows outside every sequence {kind} {rows_each}")
    case = Case(kind, [30, 100, 700], rows_each, 2, 128, 16, seed=5)
    first, tokens = 3, case.tokens + 8
    q = normal(9, (tokens, 4, 128), torch.bfloat16).to(DEV)
    batch = d.Sequences(dev_i32(case.tables), dev_i32(case.starts), dev_i32(case.offsets + first))
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    hip.attentionSequences(q, case.cache, batch, 0.1, out)
    inside = slice(first, first + case.tokens)
    assert bool((out[:first] == 7).all()) and bool((out[first + case.tokens:] == 7).all())
    assert_rows(case, q[inside], 0.1, out[inside], what="inside")
    k = torch.full((tokens, 2, 128), 7.0, device=DEV)
    v = k.clone()
    hip.cacheReadSequences(case.cache, batch, k, v)
    assert bool((k[:first] == 7).all()) and bool((v[first + case.tokens:] == 7).all())


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("tokens", [1, 20, 150])
def test_wrongly_described_sequences_get_nothing_done(hip, kind, tokens):
    step(f"wrongly described sequences {kind} {tokens}")
    # rows past the tensors, before them, backwards; a negative start; an end past the page table
    case = Case(kind, [30, 30, 30, 30, 30], [tokens] * 5, 2, 128, 16, seed=6)
    n = tokens
    for offsets, starts, good in (
            ([0, n, 2 * n, 3 * n, 4 * n, 5 * n + 1], [30] * 5, [0, 1, 2, 3]),
            ([-1, n, 2 * n, 3 * n, 4 * n, 5 * n], [30] * 5, [1, 2, 3, 4]),
            ([0, n, 2 * n, 3 * n, 4 * n, 5 * n], [30, -1, 30, 1 << 30, 30], [0, 2, 4]),
            ([0, n, 2 * n, 3 * n, 2 * n, 2 * n], [30] * 5, [0, 1, 2])):
        q = normal(10, (5 * n, 4, 128), torch.bfloat16).to(DEV)
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        hip.attentionSequences(q, case.cache, d.Sequences(dev_i32(case.tables), dev_i32(starts), dev_i32(offsets)),
                               0.1, out, badPage=bad)
        assert int(bad.item()) == 1
        want, *_ = wanted(case, q.cpu(), 0.1)
        for s in good:
            if starts[s] == 30 and offsets[s + 1] - offsets[s] == n:
                rows = slice(offsets[s], offsets[s + 1])
                assert float((out[rows].cpu().double() - want[rows]).abs().max()) < 0.05
        if offsets[1] == n and starts[1] == -1:
            assert bool((out[n:2 * n] == 7).all()) and bool((out[3 * n:4 * n] == 7).all())


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 9, 100])
def test_pages_outside_the_cache_are_not_seen(hip, kind, dtype, tokens):
    step(f"pages outside the cache {kind} {dtype} {tokens}")
    page = 16
    case = Case(kind, [200], [tokens], 2, 128, page, seed=7)
    for column, entry in ((2, -1), (5, case.cache.pages), (9, 1 << 30)):
        case.tables[0, column] = entry
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = normal(11, (tokens, 6, 128), TYPES[dtype], 2.0).to(DEV)
    hidden = [(0, p) for column in (2, 5, 9) for p in range(column * page, (column + 1) * page)]
    assert_rows(case, q, 0.09, run(hip, case, q, 0.09, single=True, bad=bad), hidden=hidden, what="bad pages")
    assert int(bad.item()) == 1
    # no page at all: nothing seen, zeros
    case.tables[:] = -1
    bad.zero_()
    assert bool((run(hip, case, q, 0.09, single=True, bad=bad) == 0).all())
    assert int(bad.item()) == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,tokens", [(300, 1), (90, 12), (200, 140)])
def test_what_is_masked_has_no_part(hip, dtype, start, tokens):
    step(f"infinities and NaN in masked places {dtype} {tokens} at {start}")
    window = d.AttentionWindow(60, 5)
    case = Case("f16", [start], [tokens], 2, 128, 16, seed=8)
    values, keys = case.cache.values, case.cache.keys
    table = case.tables[0]
    dense_k, dense_v = case.dense[0]

    def put(position, k=None, v=None):
        page, off = int(table[position // 16]), position % 16
        if k is not None:
            keys[page, off] = k
            dense_k[position] = k
        if v is not None:
            values[page, :, :, off] = v
            dense_v[position] = v

    # between the sinks and the window of every row, of some rows, and ahead of some rows
    last = start + tokens - 1
    put(6, k=float("nan"), v=float("nan"))
    put(start - 60 if start >= 66 else 7, k=float("inf"), v=float("-inf"))
    put(last, v=float("inf"))          # the last row's own: +inf for it alone
    if tokens > 3:
        put(last - 2, k=float("nan"))  # NaN for the rows that see it
        put(start + 1, v=float("-inf"))
    q = normal(12, (tokens, 4, 128), TYPES[dtype], 1.0).to(DEV)
    assert_rows(case, q, 0.05, run(hip, case, q, 0.05, window, single=True), window, what="masked")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("tokens", [1, 90])
def test_queries_large_small_and_not_numbers(hip, dtype, kind, tokens):
    step(f"extreme queries {dtype} {kind} {tokens}")
    case = Case(kind, [150], [tokens], 2, 64, 16, seed=9)
    q = normal(13, (tokens, 8, 64), torch.float32, 1.0)
    q[:, 0] *= 1e30
    q[:, 1] *= 1e-30
    q[:, 2] = 0
    q[0, 3, 5] = float("nan")
    q[0, 4, 6] = float("inf")
    q[:, 5, 1:] *= 1e-6   # one strong value among weak ones
    q = q.to(TYPES[dtype]).to(DEV)
    # head 0: scaled to scores of ordinary size; the others: weights near even
    for scale, heads in ((1e-30, [0]), (0.125, [1, 2, 3, 4, 5, 6, 7])):
        out = run(hip, case, q, scale, single=True)
        want, mass, size, count, small_weights = wanted(case, q.cpu(), scale)
        got = out.cpu().double()
        for h in heads:
            if h in (3, 4):
                assert bool(torch.isnan(got[0, h]).all())
                got[0, h], want[0, h] = 0, 0
            bar = (4 * (2.0 ** -24 * 12 * size + 2.0 ** -20 + 2.0 ** -24 * count.sqrt())) * mass + small_weights
            if dtype == "bf16":
                bar = bar + 2.0 ** -11 * mass + 2.0 ** -8 * want.abs()
            assert bool(((got - want).abs()[:, h] <= bar[:, h].nan_to_num(0) + 1e-30).all()), f"head {h}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("tokens", [1, 80])
def test_value_rows_of_unlike_sizes(hip, dtype, kind, tokens):
    step(f"value rows of unlike sizes {dtype} {kind} {tokens}")
    # rows whose own values are small next to others' that they hardly weigh
    case = Case(kind, [100], [tokens], 1, 64, 16, seed=10)
    page = case.page
    for position in range(0, 100 + tokens, 3):
        p, off = int(case.tables[0, position // page]), position % page
        factor = 2.0 ** -8 if position % 2 else 2.0 ** 6
        if kind == "f16":
            case.cache.values[p, :, :, off] *= factor
            case.dense[0][1][position] = case.cache.values[p, :, :, off].cpu().double()
        else:
            case.cache.valueScales[p, :, off] *= factor
            case.dense[0][1][position] *= factor
            case.scales[0][position] *= factor
    q = normal(14, (tokens, 4, 64), TYPES[dtype], 8.0).to(DEV)
    assert_rows(case, q, 0.125, run(hip, case, q, 0.125, single=True), what="unlike sizes")


@pytest.mark.parametrize("kind", CACHES)
def test_scores_far_apart(hip, kind):
    step(f"scores far apart {kind}")
    # the maximum rises by hundreds from tile to tile, so the sums so far vanish
    case = Case(kind, [400], [70], 1, 128, 16, seed=11)
    q = normal(15, (70, 2, 128), torch.float32, 30.0).to(DEV)
    assert_rows(case, q, 1.0, run(hip, case, q, 1.0, single=True), what="far apart")


@pytest.mark.parametrize("tokens", [1, 40, 200])
def test_unaligned_tensors(hip, tokens):
    step(f"queries off 16 bytes {tokens}")
    case = Case("f16", [90], [tokens], 2, 128, 16, seed=12)
    for dtype in (torch.float32, torch.bfloat16):
        flat = torch.empty(tokens * 4 * 128 + 1, dtype=dtype, device=DEV)
        q = flat[1:].view(tokens, 4, 128)
        q.copy_(normal(16, (tokens, 4, 128), dtype))
        out = torch.empty(tokens * 4 * 128 + 1, dtype=dtype, device=DEV)[1:].view(tokens, 4, 128)
        hip.attention(q, case.cache, dev_i32(case.tables[0]), 90, 0.1, out)
        assert_rows(case, q, 0.1, out, what="unaligned")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("tokens", [1, 24, 600])
def test_the_same_bits_every_time_and_on_another_stream(hip, kind, tokens):
    step(f"the same bits every time {kind} {tokens}")
    case = Case(kind, [3000], [tokens], 2, 128, 16, seed=13)
    q = normal(17, (tokens, 8, 128), torch.bfloat16, 2.0).to(DEV)
    first = run(hip, case, q, 0.09, single=True)
    stream = torch.cuda.Stream()
    other = d.HipOps(stream)
    torch.cuda.synchronize()
    for _ in range(3):
        assert torch.equal(run(hip, case, q, 0.09, single=True), first)
        out = torch.empty_like(first)
        table = dev_i32(case.tables[0])
        torch.cuda.synchronize()
        other.attention(q, case.cache, table, 3000, 0.09, out)
        again = run(hip, case, q, 0.09, single=True)  # at the same time, on this stream
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(again, first)


# ------------------------------------------------------------------ rows into and out of the caches

def quantised(x):
    """Codes and scales by the definition: d = fl32(max|x| / 127); codes to the nearest, halves away from 0."""
    x = x.double()
    top = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    scale = torch.where(fine, (top / 127).float(), torch.tensor(float("nan")))
    step_ = scale.double()[..., None]
    codes = torch.floor(x.abs() / step_ + 0.5).clamp(max=127) * x.sign()
    codes = torch.where((fine & (scale > 0))[..., None], codes, torch.zeros_like(codes))
    return codes.nan_to_num(0).to(torch.int8), scale


ROWS = [
    # (starts, rows, kv, dim, page)
    ([14], [1], 8, 128, 16), ([0], [1], 1, 8, 16), ([5], [37], 2, 128, 16), ([30], [5], 3, 72, 16),
    ([7], [431], 3, 136, 48), ([3], [50], 2, 512, 16), ([9], [20], 2, 7, 16), ([0], [33], 1, 600, 32),
    ([0, 15, 16, 200], [1, 1, 1, 1], 8, 128, 16), ([0, 31, 5, 64, 9], [40, 0, 1, 17, 200], 2, 64, 32),
    ([3 * i for i in range(90)], [1 + i % 3 for i in range(90)], 2, 256, 64),
]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,rows,kv,dim,page", ROWS)
def test_written_and_read_back(hip, kind, dtype, starts, rows, kv, dim, page):
    step(f"write and read {kind} {dtype} {len(starts)} sequences, {kv} heads of {dim}, pages of {page}")
    case = Case(kind, starts, rows, kv, dim, page, seed=20)
    cache, n = case.cache, case.tokens
    k, v = normal(21, (n, kv, dim), TYPES[dtype], 3.0), normal(22, (n, kv, dim), TYPES[dtype], 0.2)
    k[0, 0] = 0  # a row of zeros
    before = [t.cpu().clone() for t in (cache.keys, cache.values)]
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    single = len(starts) == 1
    if single and kind == "i8":
        hip.cacheWrite(k.to(DEV), v.to(DEV), cache, dev_i32(case.tables[0]), starts[0], bad)
    else:
        hip.cacheWriteSequences(k.to(DEV), v.to(DEV), cache, case.sequences(), bad)
    want_k, want_v = before
    if kind == "i8":
        kc, ks = quantised(k)
        vc, vs = quantised(v)
        read_k = (kc.float() * ks[..., None]).to(TYPES[dtype])
        read_v = (vc.float() * vs[..., None]).to(TYPES[dtype])
    else:
        kc, vc = k.half(), v.half()
        read_k, read_v = kc.to(TYPES[dtype]), vc.to(TYPES[dtype])
    for s in range(len(starts)):
        for t in range(rows[s]):
            position, row = starts[s] + t, int(case.offsets[s]) + t
            p, off = int(case.tables[s, position // page]), position % page
            want_k[p, off], want_v[p, :, :, off] = kc[row], vc[row]
            if kind == "i8":
                assert torch.equal(cache.keyScales[p, :, off].cpu(), ks[row])
                assert torch.equal(cache.valueScales[p, :, off].cpu(), vs[row])
    same = (lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))) if kind == "f16" else torch.equal
    assert same(cache.keys.cpu(), want_k) and same(cache.values.cpu(), want_v)
    got_k = torch.full(k.shape, 5.0, dtype=k.dtype, device=DEV)
    got_v = torch.full_like(got_k, 5.0)
    if single:
        hip.cacheRead(cache, dev_i32(case.tables[0]), starts[0], got_k, got_v, bad)
    else:
        hip.cacheReadSequences(cache, case.sequences(), got_k, got_v, bad)
    assert torch.equal(got_k.cpu(), read_k) and torch.equal(got_v.cpu(), read_v)
    assert int(bad.item()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 13])
def test_rows_that_are_not_numbers_and_ties(hip, dtype, dim):
    step(f"quantised rows that are not numbers, ties {dtype} {dim}")
    case = Case("i8", [0], [8], 1, dim, 16, seed=23)
    x = normal(24, (8, 1, dim), TYPES[dtype])
    x[0, 0, 3], x[1, 0, 2], x[2, 0, 1] = float("nan"), float("inf"), float("-inf")
    x[3] = 0
    x[4] = 1e-45 if dtype == "f32" else 1e-38
    # multiples of 1/2 with 127 among them: scale 1, every half a tie that goes away from 0
    x[5, 0] = (torch.arange(dim) - dim // 2).to(x.dtype) / 2
    x[5, 0, 0] = 127
    x[6] = 3e38
    hip.cacheWrite(x.to(DEV), x.to(DEV), case.cache, dev_i32(case.tables[0]), 0)
    codes, scales = quantised(x)
    page = int(case.tables[0, 0])
    assert torch.equal(case.cache.keys[page, :8].cpu(), codes)
    assert torch.equal(case.cache.values[page, :, :, :8].permute(2, 0, 1).cpu(), codes)
    for got in (case.cache.keyScales, case.cache.valueScales):
        assert torch.equal(got[page, :, :8].T.cpu().isnan(), scales.isnan())
        assert torch.equal(got[page, :, :8].T.cpu().nan_to_num(0), scales.nan_to_num(0))


def test_codes_at_the_halves(hip):
    step("codes next to halves")
    # x one F32 step either side of d (n + 1/2), for scales with full mantissas: where a quotient in F32 errs
    rng = np.random.default_rng(25)
    rows = 64
    x = np.zeros((rows, 1, 256), np.float32)
    for r in range(rows):
        top = np.float32(rng.uniform(0.5, 2.0))
        step_ = np.float32(np.float64(top) / 127)
        n = np.arange(84)
        near = (np.float64(step_) * (n + 0.5)).astype(np.float32)
        x[r, 0, 0] = top
        x[r, 0, 1:85], x[r, 0, 85:169] = near, np.nextafter(near, np.float32(9))
        x[r, 0, 169:253] = -np.nextafter(near, np.float32(0))
    case = Case("i8", [0], [rows], 1, 256, 16, seed=26)
    t = torch.from_numpy(x)
    hip.cacheWrite(t.to(DEV), t.to(DEV), case.cache, dev_i32(case.tables[0]), 0)
    codes, _ = quantised(t)
    for r in range(rows):
        page, off = int(case.tables[0, r // 16]), r % 16
        assert torch.equal(case.cache.keys[page, off].cpu(), codes[r])


@pytest.mark.parametrize("kind", CACHES)
def test_rows_on_pages_outside_the_cache(hip, kind):
    step(f"rows on pages outside the cache {kind}")
    case = Case(kind, [10], [30], 2, 64, 16, seed=27)
    case.tables[0, 1] = case.cache.pages  # positions 16 to 31
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    k = normal(28, (30, 2, 64)).to(DEV)
    hip.cacheWriteSequences(k, k, case.cache, case.sequences(), bad)
    assert int(bad.item()) == 1
    bad.zero_()
    got = torch.full((30, 2, 64), 5.0, device=DEV)
    got_v = got.clone()
    hip.cacheReadSequences(case.cache, case.sequences(), got, got_v, bad)
    assert int(bad.item()) == 1
    assert bool((got[6:22] == 5).all()) and bool((got_v[6:22] == 5).all())
    assert float((got[:6] - k[:6]).abs().max()) < 0.05 and float((got_v[22:] - k[22:]).abs().max()) < 0.05


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", CACHES)
def test_a_prompt_then_steps_in_a_graph(hip, dtype, kind):
    """A server's run: two prompts' keys and values go into the cache and
    their chunks attend; then decode steps, captured once and replayed as the
    sequences grow (their starts move on the device), each against the same
    calls made eagerly in another cache."""
    step(f"prompt and captured steps {dtype} {kind}")
    heads, kv, dim, page, t = 8, 2, 128, 16, TYPES[dtype]
    prompts, steps = [70, 23], 6
    make = d.KvCache.allocate if kind == "f16" else d.QuantizedKvCache.allocate
    caches = [make(14, page, kv, dim) for _ in range(2)]
    tables = dev_i32([[3, 1, 9, 12, 0, 7], [2, 5, 13, 4, 6, 8]])
    offsets = dev_i32(np.concatenate([[0], np.cumsum(prompts)]))
    chunk = d.Sequences(tables, dev_i32([0, 0]), offsets)
    n = sum(prompts)
    k, v = normal(30, (n, kv, dim), t).to(DEV), normal(31, (n, kv, dim), t).to(DEV)
    q = normal(32, (n, heads, dim), t, 2.0).to(DEV)
    outs = []
    for cache in caches:
        hip.cacheWriteSequences(k, v, cache, chunk)
        out = torch.empty_like(q)
        hip.attentionSequences(q, cache, chunk, 0.1, out)
        outs.append(out)
    assert torch.equal(*outs)
    starts = dev_i32(prompts)
    batch = d.Sequences(tables, starts)
    k1, v1 = torch.empty(2, kv, dim, dtype=t, device=DEV), torch.empty(2, kv, dim, dtype=t, device=DEV)
    q1, graph_out = torch.empty(2, heads, dim, dtype=t, device=DEV), torch.empty(2, heads, dim, dtype=t, device=DEV)
    graph_windowed, windowed = torch.empty_like(graph_out), torch.empty_like(graph_out)
    window = d.AttentionWindow(33, 2)

    def calls(cache, whole, part):
        hip.cacheWriteSequences(k1, v1, cache, batch)
        hip.attentionSequences(q1, cache, batch, 0.1, whole)
        hip.attentionSequences(q1, cache, batch, 0.1, part, window)

    for x in (k1, v1, q1):
        x.normal_()
    calls(caches[0], graph_out, graph_windowed)  # warm; the same places are written again below
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(caches[0], graph_out, graph_windowed)
    eager_out = torch.empty_like(graph_out)
    for i in range(steps):
        starts.copy_(dev_i32([p + i for p in prompts]))
        k1.copy_(normal(40 + i, (2, kv, dim), t))
        v1.copy_(normal(50 + i, (2, kv, dim), t))
        q1.copy_(normal(60 + i, (2, heads, dim), t, 2.0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        calls(caches[1], eager_out, windowed)
        torch.cuda.synchronize()
        assert torch.equal(graph_out, eager_out) and torch.equal(graph_windowed, windowed), f"step {i}"
    # what the caches hold now, read back, carries the last step's result
    longest = prompts[0] + steps
    back_k, back_v = (torch.empty(longest, kv, dim, dtype=torch.float32, device=DEV) for _ in range(2))
    hip.cacheRead(caches[0], tables[0].contiguous(), 0, back_k, back_v)
    logits = torch.einsum("hd,jhd->hj", q1[0].double().cpu(),
                          back_k.double().cpu().repeat_interleave(heads // kv, 1)) * 0.1
    want = torch.einsum("hj,jhd->hd", torch.softmax(logits, -1), back_v.double().cpu().repeat_interleave(heads // kv, 1))
    bar = 2.0 ** -7 if dtype == "bf16" else 1e-5
    assert float((graph_out[0].double().cpu() - want).abs().max()) < bar * float(want.abs().max())


def test_two_captured_graphs_at_the_same_time(hip):
    """Their scratch is their own: replayed together on two streams they give
    what they give alone."""
    step("two captured graphs at the same time")
    case = Case("f16", [6000], [1], 2, 128, 16, seed=33)
    table = dev_i32(case.tables[0])
    made = []
    for i in range(2):
        q = normal(70 + i, (1, 16, 128), torch.bfloat16, 2.0).to(DEV)
        out = torch.empty_like(q)
        hip.attention(q, case.cache, table, 6000, 0.09, out)
        torch.cuda.synchronize()
        alone = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                hip.attention(q, case.cache, table, 6000, 0.09, out)
        made.append((graph, out, alone, q))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for (graph, *_), stream in zip(made, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, alone, _ in made:
            assert torch.equal(out, alone)
            out.zero_()
        torch.cuda.synchronize()


# ------------------------------------------------------------------ more of what a program may do

@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [None, d.AttentionWindow(2700, 4)])
def test_unlike_sequences_in_splits(hip, kind, dtype, dim, window):
    step(f"unlike sequences in splits {kind} {dtype} heads of {dim} {window}")
    # long chunks split in several, short ones written at once; chunks of few rows among the chunks of many
    case = Case(kind, [5000, 100, 2900, 2600, 0, 640], [40, 1, 30, 5, 3, 1], 2, dim, 16, seed=30)
    q = normal(31, (case.tokens, 16, dim), TYPES[dtype], 2.0).to(DEV)
    scale = 1 / math.sqrt(dim)
    out = run(hip, case, q, scale, window)
    assert_rows(case, q, scale, out, window, what="unlike sequences")
    assert torch.equal(out, run(hip, case, q, scale, window))


ROW_BY_ROW = [
    # (start, tokens, heads, kv, dim, page, window, sinks): heads past 256 values, and off eights
    (1500, 3, 4, 2, 320, 16, 100, 7), (1500, 3, 4, 2, 36, 48, 100, 70), (900, 70, 2, 1, 512, 64, 64, 0),
    (257, 2, 6, 2, 264, 16, 1, 1), (255, 2, 3, 3, 13, 16, 200, 0), (300, 5, 2, 2, 300, 16, 63, 129),
]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,tokens,heads,kv,dim,page,positions,sinks", ROW_BY_ROW)
def test_windows_of_rows_by_themselves(hip, kind, dtype, start, tokens, heads, kv, dim, page, positions, sinks):
    step(f"row by row, window {positions} + {sinks} {kind} {dtype} {tokens} at {start}, {heads}/{kv} heads of {dim}")
    case = Case(kind, [start], [tokens], kv, dim, page, seed=32)
    q = normal(33, (tokens, heads, dim), TYPES[dtype], 2.0).to(DEV)
    window, scale = d.AttentionWindow(positions, sinks), 1 / math.sqrt(dim)
    assert_rows(case, q, scale, run(hip, case, q, scale, window, single=True), window, what="window")
    assert_rows(case, q, scale, run(hip, case, q, scale, single=True), what="whole")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [320, 36])
def test_masked_places_of_rows_by_themselves(hip, dtype, dim):
    step(f"row by row, NaN and infinities in masked places {dtype} heads of {dim}")
    window = d.AttentionWindow(60, 5)
    case = Case("f16", [300], [3], 2, dim, 16, seed=34)
    dense_k, dense_v = case.dense[0]
    for position, k, v in ((6, float("nan"), float("nan")), (240, float("inf"), float("-inf")), (302, 1.0, float("inf"))):
        page, off = int(case.tables[0, position // 16]), position % 16
        case.cache.keys[page, off], case.cache.values[page, :, :, off] = k, v
        dense_k[position], dense_v[position] = k, v
    q = normal(35, (3, 4, dim), TYPES[dtype]).to(DEV)
    assert_rows(case, q, 0.05, run(hip, case, q, 0.05, window, single=True), window, what="masked")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("tokens,dim", [(1, 128), (20, 128), (150, 128), (2, 320)])
def test_pages_given_back_behind_the_window(hip, kind, tokens, dim):
    step(f"pages given back behind the window {kind} {tokens} tokens, heads of {dim}")
    # no row sees a position of them: nothing is read there and nothing flagged
    case = Case(kind, [400], [tokens], 2, dim, 16, seed=36)
    window = d.AttentionWindow(90, 5)
    case.tables[0, 1:(400 - 90) // 16] = -1
    bad = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = normal(37, (tokens, 4, dim), torch.bfloat16, 2.0).to(DEV)
    assert_rows(case, q, 0.09, run(hip, case, q, 0.09, window, single=True, bad=bad), window, what="pages given back")
    assert int(bad.item()) == 0


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim", [(1, 128), (90, 128), (2, 300)])
def test_scales_of_zero_and_below(hip, kind, dtype, tokens, dim):
    step(f"scales of zero and below {kind} {dtype} {tokens} tokens, heads of {dim}")
    case = Case(kind, [150], [tokens], 2, dim, 16, seed=38)
    q = normal(39, (tokens, 4, dim), TYPES[dtype], 2.0).to(DEV)
    for scale in (-0.1, 0.0):
        assert_rows(case, q, scale, run(hip, case, q, scale, single=True), what=f"scale {scale}")


@pytest.mark.parametrize("kind", CACHES)
def test_sequences_that_share_pages(hip, kind):
    step(f"sequences that share pages {kind}")
    case = Case(kind, [200, 90, 400], [1, 50, 3], 2, 128, 16, seed=40)
    for s, columns in ((1, 4), (2, 9)):  # the first sequence's pages as the others' prefix
        case.tables[s, :columns] = case.tables[0, :columns]
        for mine, first in zip(case.dense[s], case.dense[0]):
            mine[:columns * 16] = first[:columns * 16]
        if kind == "i8":
            case.scales[s][:columns * 16] = case.scales[0][:columns * 16]
    q = normal(41, (case.tokens, 8, 128), torch.bfloat16, 2.0).to(DEV)
    assert_rows(case, q, 0.09, run(hip, case, q, 0.09), what="shared pages")


@pytest.mark.parametrize("tokens", [1, 90])
def test_subnormal_keys_and_values(hip, tokens):
    step(f"subnormal keys and values {tokens}")
    # numbers below F16's normal ones (2^-14) count as they are
    case = Case("f16", [100], [tokens], 1, 64, 16, seed=42)
    case.cache.keys.mul_(2.0 ** -15)
    case.cache.values.mul_(2.0 ** -15)
    k, v = (x.half().mul(2.0 ** -15).double() for x in case.dense[0])
    assert bool((v != 0).float().mean() > 0.9)
    case.dense[0] = (k, v)
    q = normal(43, (tokens, 4, 64), torch.float32, 2.0).to(DEV)
    scale = 2.0 ** 12
    assert_rows(case, q, scale, run(hip, case, q, scale, single=True), what="subnormal")


@pytest.mark.parametrize("kind", CACHES)
def test_a_cache_past_2_31_values(hip, kind):
    step(f"a cache past 2^31 values {kind}")
    # the same rows in the last pages of a large cache and in a small one: the same bits written, read and attended
    page, kv, dim, starts, rows = 16, 8, 128, [300, 40], [1, 100]
    small_pages = 32
    large_pages = (1 << 31) // (page * kv * dim) + small_pages

    def cache(pages):
        if kind == "i8":
            return d.QuantizedKvCache.allocate(pages, page, kv, dim, DEV)
        return d.KvCache(torch.empty((pages, page, kv, dim), dtype=torch.float16, device=DEV),
                         torch.empty((pages, kv, dim, page), dtype=torch.float16, device=DEV), page)

    lengths = [s + r for s, r in zip(starts, rows)]
    offsets, all_offsets = np.cumsum([0] + rows), np.cumsum([0] + lengths)
    tables = np.full((2, 20), -1, np.int32)
    tables[0, :19], tables[1, :9] = np.arange(19), 19 + np.arange(9)
    k, v = (normal(s, (int(all_offsets[-1]), kv, dim)).to(DEV) for s in (44, 45))
    results = []
    for pages, shift in ((small_pages, 0), (large_pages, large_pages - small_pages)):
        c, where = cache(pages), dev_i32(np.where(tables >= 0, tables + shift, -1))
        whole = d.Sequences(where, dev_i32(np.zeros(2)), dev_i32(all_offsets))
        hip.cacheWriteSequences(k, v, c, whole)
        rk, rv = torch.empty_like(k), torch.empty_like(v)
        hip.cacheReadSequences(c, whole, rk, rv)
        made = [rk, rv]
        for dtype in (torch.float32, torch.bfloat16):
            q = normal(46, (sum(rows), 16, dim), dtype, 2.0).to(DEV)
            out = torch.empty_like(q)
            hip.attentionSequences(q, c, d.Sequences(where, dev_i32(starts), dev_i32(offsets)), 0.09, out)
            made.append(out)
        off = torch.empty(1 + sum(rows) * 16 * dim, device=DEV)[1:].view(sum(rows), 16, dim)  # row by row
        off.copy_(normal(46, (sum(rows), 16, dim), torch.float32, 2.0))
        out = torch.empty_like(off)
        hip.attentionSequences(off, c, d.Sequences(where, dev_i32(starts), dev_i32(offsets)), 0.09, out)
        made.append(out)
        results.append([x.cpu() for x in made])
        del c
        torch.cuda.empty_cache()
    for one, other in zip(*results):
        assert bool(torch.isfinite(one).all())
        assert torch.equal(one, other)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 264])
@pytest.mark.parametrize("what", ["keys", "values"])
def test_rows_that_see_a_quantised_nan(hip, dtype, dim, what):
    step(f"rows that see a quantised NaN {dtype} heads of {dim} {what}")
    # a row written with a NaN or an infinity reads as NaN throughout, and so do the rows that see it; no others
    case = Case("i8", [60], [30], 2, dim, 16, seed=47)
    k, v = normal(48, (1, 2, dim)), normal(49, (1, 2, dim))
    (k if what == "keys" else v)[0, 1, 3] = float("inf")
    hip.cacheWrite(k.to(DEV), v.to(DEV), case.cache, dev_i32(case.tables[0]), 70)
    for mine, x in zip(case.dense[0], (k, v)):
        codes, scales = quantised(x)
        mine[70] = (codes.double() * scales.double()[..., None])[0]
    case.scales[0][70] = quantised(v)[1][0].double().nan_to_num(0)
    q = normal(50, (30, 4, dim), TYPES[dtype], 2.0).to(DEV)
    out = run(hip, case, q, 0.09, single=True)
    assert_rows(case, q, 0.09, out, what="a quantised NaN")
    assert bool(torch.isnan(out[10:, 2:]).all()) and bool(torch.isfinite(out[:10]).all())
    assert bool(torch.isfinite(out[:, :2]).all())


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", ["out", "queries"])
@pytest.mark.parametrize("start,tokens,heads", [
    (90, 1, 4),      # few rows
    (3000, 24, 4),   # few rows, in splits that are joined
    (90, 200, 4),    # many rows
    (3000, 90, 16),  # many rows, in splits that are joined
])
def test_queries_or_out_alone_off_16_bytes(hip, kind, dtype, off, start, tokens, heads):
    step(f"{off} alone off 16 bytes {kind} {dtype} {tokens} tokens at {start}")
    case = Case(kind, [start], [tokens], 2, 128, 16, seed=51)
    t = TYPES[dtype]
    q = normal(52, (tokens, heads, 128), t, 2.0).to(DEV)

    def shifted():  # one value past a multiple of 16 bytes, a value to spare at either end
        flat = torch.full((q.numel() + 2,), 7.0, dtype=t, device=DEV)
        return flat, flat[1:-1].view(q.shape)

    flat, moved = shifted()
    queries, out = (q, moved) if off == "out" else (moved.copy_(q), torch.full_like(q, 7.0))
    hip.attention(queries, case.cache, dev_i32(case.tables[0]), start, 0.09, out)
    assert_rows(case, q, 0.09, out, what=f"{off} off 16 bytes")
    assert float(flat[0]) == 7 and float(flat[-1]) == 7


def repeated(case, times):
    """The case's one sequence `times` over, on the same pages."""
    case.starts, case.rows = np.tile(case.starts, times), np.tile(case.rows, times)
    case.tables = np.tile(case.tables, (times, 1))
    case.tokens, case.offsets = case.tokens * times, np.concatenate([[0], np.cumsum(case.rows)])
    case.dense, case.scales = case.dense * times, case.scales * times
    return case


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("sequences,offsets", [(340, False), (340, True), (1100, False)])
def test_more_sequences_than_their_splits_have_blocks(hip, kind, sequences, offsets):
    step(f"{sequences} sequences of 4,001 positions {kind} offsets {offsets}")
    # three splits each, or one, where 4,001 positions alone would take four
    case = repeated(Case(kind, [4000], [1], 16, 16, 16, seed=53), sequences)
    q = normal(54, (sequences, 16, 16), torch.float32, 2.0).to(DEV)
    assert_rows(case, q, 0.25, run(hip, case, q, 0.25, offsets=offsets), what="many sequences")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_and_many_rows_partials_by_place(hip, kind, dtype):
    step(f"a chunk and single tokens in splits, partials by place {kind} {dtype}")
    # the chunk's rows and the single tokens', both in splits, share one range of partials
    case = Case(kind, [3000, 2500, 20, 4000, 1800, 900], [20, 1, 1, 1, 1, 1], 2, 128, 16, seed=55)
    q = normal(56, (case.tokens, 16, 128), TYPES[dtype], 2.0).to(DEV)
    out = run(hip, case, q, 0.09)
    assert_rows(case, q, 0.09, out, what="by place")
    assert torch.equal(out, run(hip, case, q, 0.09))


def scale_rows(case, sequence, position, factor):
    """The 8-bit cache's value row at `position`, its scale times `factor`."""
    p, off = int(case.tables[sequence, position // case.page]), position % case.page
    case.cache.valueScales[p, :, off] *= factor
    case.dense[sequence][1][position] *= factor
    case.scales[sequence][position] *= factor


def assert_rows_of_scales_apart(case, queries, scale, got, window=None, what=""):
    """Value scales w any distance apart: a row's weights are p w in F16 terms
    over a power of two such that the largest is 2^(lift - 17) at least (lift 14
    for F32's two terms, 7 for BF16's one), their last step 2^-24. So with codes
    up to 127 and n positions a row is off by 127 n 2^-25 / 2^(lift - 17) of its
    own largest p w, not of the cache's largest w, beside the other roundings.
    Few rows' weights are 2^(score + log2 w): the logarithm off by a step, its sums
    with the score and the maximum by half of one, 2^-22 |log2 w| ln 2 together."""
    out, mass, size, count, _ = wanted(case, queries.cpu(), scale, window)
    logs = max(float(w.clamp(min=2.0 ** -126).log2().abs().max()) for w in case.scales)
    bar = 4 * (2.0 ** -24 * (math.sqrt(case.dim) + 4) * size + 2.0 ** -20 + 2.0 ** -24 * count.sqrt()) * mass
    bar = bar + math.log(2) * 2.0 ** -22 * logs * mass
    if queries.dtype == torch.bfloat16:
        bar = bar + 2.0 ** -11 * mass + 2.0 ** -8 * out.abs()
    lift, group = 14 if queries.dtype == torch.float32 else 7, queries.shape[1] // case.kv
    for s, (k, _) in enumerate(case.dense):
        rows = slice(int(case.offsets[s]), int(case.offsets[s + 1]))
        at = torch.arange(int(case.rows[s]))[:, None] + int(case.starts[s])
        j = torch.arange(k.shape[0])[None, :]
        seen = (j <= at) if window is None else (j <= at) & ((j > at - window.positions) | (j < window.sinks))
        for h in range(queries.shape[1]):
            logits = scale * (queries[rows, h].double().cpu() @ k[:, h // group].T)
            p = torch.softmax(logits.masked_fill(~seen, -math.inf), -1)
            most = (p * case.scales[s][:, h // group]).amax(-1, keepdim=True)
            bar[rows, h] += 127 * count[rows, h] * 2.0 ** (-25 + 17 - lift) * most
    off = (got.cpu().double() - out).abs()
    print(f"[gpu]   worst {float((off / bar).max()):.3f} of the bar", flush=True)
    assert bool((off <= bar).all()), f"{what}: {int((off > bar).sum())} beyond the bar, {float((off / bar).max()):.2f} of it"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("down", [20, 40, 90])
@pytest.mark.parametrize("where", ["first", "thirds", "tiles", "last", "all but some", "none weighed"])
@pytest.mark.parametrize("start,tokens,heads,dim", [(100, 1, 8, 128), (200, 80, 8, 64), (200, 80, 4, 128),
                                                    (150, 70, 4, 256), (3000, 90, 16, 128)])
def test_value_scales_far_apart(hip, dtype, down, where, start, tokens, heads, dim):
    step(f"value scales 2^{down} apart, {where} {dtype} {tokens} tokens at {start}, heads of {dim}")
    case = Case("i8", [start], [tokens], 2, dim, 16, seed=57, value_scale=4.0)
    length = start + tokens
    small = {"first": [0], "thirds": range(0, length, 3), "tiles": [j for j in range(length) if j // 64 % 2 == 0],
             "last": range(start, length), "all but some": [j for j in range(length) if j % 50 != 49],
             "none weighed": [0, 40]}[where]
    for position in small:
        scale_rows(case, 0, position, 2.0 ** -down)
    q = normal(58, (tokens, heads, dim), torch.float32, 0.5)
    # half of the heads weigh one small row so far above the others that these are e^-20 to e^-30 next to it
    k = case.dense[0][0]
    for h in range(0, heads, 2):
        if where != "none weighed":
            position = list(small)[len(small) // 2 if where != "last" else 0]
            key = k[position, h // (heads // 2)].float()
            q[:, h] += 25 / 0.09 / float(key @ key) * key
    q = q.to(TYPES[dtype]).to(DEV)
    assert_rows_of_scales_apart(case, q, 0.09, run(hip, case, q, 0.09, single=True), what="scales apart")
    window = d.AttentionWindow(70, 3)
    assert_rows_of_scales_apart(case, q, 0.09, run(hip, case, q, 0.09, window, single=True), window, "windowed")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rising", [True, False])
def test_value_scales_far_apart_as_scores_rise(hip, dtype, rising):
    step(f"value scales apart, scores {'rising' if rising else 'falling'} {dtype}")
    # from tile to tile a row's scores go up (or down) by a few nats and its scales the other way, so that every
    # tile's part of the result is of one size
    case = Case("i8", [600], [70], 1, 128, 16, seed=59)
    q = normal(60, (70, 4, 128), torch.float32, 0.25)
    u = torch.sign(normal(61, (128,)))
    case.cache.keyScales.fill_(2.0 / 127)
    for position in range(670):
        tile = position // 64 if rising else 10 - position // 64
        page, off = int(case.tables[0, position // 16]), position % 16
        case.cache.valueScales[page, :, off] *= math.exp(-3.0 * tile)
        codes = (u * 12 * tile).to(torch.int8)  # q.k gains about 3 a tile
        case.cache.keys[page, off, 0] = codes.to(DEV)
        held = case.cache.valueScales[page, :, off].double().cpu()
        case.dense[0][0][position, 0] = codes.double() * float(np.float32(2.0 / 127))
        case.dense[0][1][position] = case.cache.values[page, :, :, off].double().cpu() * held[:, None]
        case.scales[0][position] = held
    q += u * (3.0 / 0.09 / (128 * 12 * 2.0 / 127))
    q = q.to(TYPES[dtype]).to(DEV)
    assert_rows_of_scales_apart(case, q, 0.09, run(hip, case, q, 0.09, single=True), what="scores that rise")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("context", [0, 6000])
def test_a_value_row_next_to_zero_costs_no_more_than_its_tiles(hip, dtype, context):
    step(f"a prompt over a value row next to zero {dtype} after {context}")
    # one value row 2^-30 of the others must not send a prompt's rows to the kernel of single rows, which would take
    # some hundred times as long
    tokens, heads, kv, dim, page = 1024, 16, 4, 128, 16
    pages = (context + tokens) // page
    cache = d.QuantizedKvCache.allocate(pages, page, kv, dim)
    cache.keys.random_(-127, 128)
    cache.values.random_(-127, 128)
    cache.keyScales.fill_(2.0 / 127)
    cache.valueScales.fill_(2.0 / 127)
    table, q = dev_i32(np.arange(pages)), normal(62, (tokens, heads, dim), TYPES[dtype]).to(DEV)
    out = torch.empty_like(q)

    def least():
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            hip.attention(q, cache, table, context, 0.09, out)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    even = least()
    cache.valueScales[0, :, 5] *= 2.0 ** -30
    apart = least()
    print(f"[gpu]   {even * 1e3:.0f} us, {apart * 1e3:.0f} with scales apart", flush=True)
    assert apart < 5 * even


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dim", [128, 36])
@pytest.mark.parametrize("each,before", [(3, 0), (90, 0), (90, 70)])
def test_a_sequence_that_begins_before_an_earlier_ones_end(hip, kind, dim, each, before):
    step(f"offsets that go back {kind} heads of {dim}, {each} rows after {before} sequences")
    # `before` sequences of no rows, then rows 0 to n, back to n / 3, from there to n + n / 3, and n more: the one that
    # begins inside the first's rows gets nothing done (its rows past them are left), the last is done
    n, third = each, each // 3
    case = Case(kind, [40] * 2, [n, n], 2, dim, 16, seed=63)
    tables = np.full((before + 4, case.tables.shape[1]), -1, np.int32)
    tables[before], tables[before + 3] = case.tables
    tables[before + 1], tables[before + 2] = case.tables[0], case.tables[0]
    starts = dev_i32([0] * before + [40, 40, 40, 40])
    ends = [n, third, n + third, 2 * n + third]
    offsets = dev_i32([0] * (before + 1) + ends)
    tokens = ends[-1]
    batch = d.Sequences(dev_i32(tables), starts, offsets)
    q = normal(64, (tokens, 8, dim), torch.float32, 2.0).to(DEV)
    out, bad = torch.full(q.shape, 7.0, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    hip.attentionSequences(q, case.cache, batch, 0.1, out, badPage=bad)
    assert int(bad.item()) == 1
    done = torch.tensor(list(range(n)) + list(range(n + third, tokens)))
    assert_rows(case, q.cpu()[done], 0.1, out.cpu()[done], what="beside offsets that go back")
    assert bool((out[n:n + third] == 7).all())
    # reading: the same rows
    k, v = (torch.full((tokens, 2, dim), 7.0, device=DEV) for _ in range(2))
    bad.zero_()
    hip.cacheReadSequences(case.cache, batch, k, v, bad)
    assert int(bad.item()) == 1
    assert bool((k[n:n + third] == 7).all()) and bool((v[n:n + third] == 7).all())
    want = torch.cat([case.dense[s][0][40:40 + n] for s in (0, 1)])
    assert float((k.cpu().double()[done] - want).abs().max()) < 1e-5
    # an offset past the tokens spoils the two sequences that it bounds, and no other
    offsets = dev_i32([0] * (before + 1) + [n, tokens + 5, n + third, 2 * n + third])
    out.fill_(7.0), bad.zero_()
    hip.attentionSequences(q, case.cache, d.Sequences(dev_i32(tables), starts, offsets), 0.1, out, badPage=bad)
    assert int(bad.item()) == 1
    assert_rows(case, q.cpu()[done], 0.1, out.cpu()[done], what="beside an offset past the tokens")
    assert bool((out[n:n + third] == 7).all())


@pytest.mark.parametrize("kind", CACHES)
def test_a_wrong_sequence_far_behind_the_rows_is_told(hip, kind):
    step(f"a wrong sequence far behind the rows {kind}")
    # one row, the first of 200 sequences'; the 150th ends past the tokens
    case = Case(kind, [5], [1], 2, 64, 16, seed=65)
    offsets = np.ones(201, np.int32)
    offsets[0], offsets[150] = 0, 9
    batch = d.Sequences(dev_i32(np.tile(case.tables, (200, 1))), dev_i32([5] * 200), dev_i32(offsets))
    x, out = normal(66, (1, 2, 64)).to(DEV), torch.empty(1, 2, 64, device=DEV)
    for call in (lambda bad: hip.cacheWriteSequences(x, x, case.cache, batch, bad),
                 lambda bad: hip.cacheReadSequences(case.cache, batch, out, torch.empty_like(out), bad),
                 lambda bad: hip.attentionSequences(x, case.cache, batch, 0.1, out, badPage=bad)):
        bad = torch.zeros(1, dtype=torch.int32, device=DEV)
        call(bad)
        assert int(bad.item()) == 1


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dim", [64, 36])
def test_empty_places_of_a_batch_are_right_whatever_their_start(hip, kind, dim):
    step(f"empty places of a batch {kind} heads of {dim}")
    case = Case(kind, [40, 7], [5, 2], 2, dim, 16, seed=67)
    tables = np.full((5, case.tables.shape[1]), -1, np.int32)
    tables[[1, 3]] = case.tables
    batch = d.Sequences(dev_i32(tables), dev_i32([-1, 40, 2 ** 31 - 1, 7, -(2 ** 31)]), dev_i32([0, 0, 5, 5, 7, 7]))
    q, bad = normal(68, (7, 4, dim), torch.float32, 2.0).to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    out, k, v = torch.empty_like(q), torch.empty(7, 2, dim, device=DEV), torch.empty(7, 2, dim, device=DEV)
    hip.attentionSequences(q, case.cache, batch, 0.1, out, badPage=bad)
    hip.cacheReadSequences(case.cache, batch, k, v, bad)
    hip.cacheWriteSequences(k, v, case.cache, batch, bad)
    assert int(bad.item()) == 0
    assert_rows(case, q, 0.1, out, what="beside empty places")


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start,tokens,heads,dim", [(150, 1, 4, 128), (150, 90, 4, 128), (3000, 90, 16, 64), (150, 2, 4, 300)])
def test_scales_that_are_no_numbers(hip, kind, dtype, start, tokens, heads, dim):
    step(f"scales that are no numbers {kind} {dtype} {tokens} tokens at {start}, heads of {dim}")
    # every score is then a NaN or an infinity, and so is no row of weights a number
    case = Case(kind, [start], [tokens], 2, dim, 16, seed=69)
    q = normal(70, (tokens, heads, dim), TYPES[dtype], 2.0).to(DEV)
    for scale in (math.nan, math.inf, -math.inf):
        assert bool(torch.isnan(run(hip, case, q, scale, single=True)).all()), f"scale {scale}"


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,context", [(64, 130), (128, 400), (256, 3000), (36, 400)])
def test_masked_content_leaves_a_decode_steps_bits_alone(hip, kind, dtype, dim, context):
    step(f"masked content and a decode step's bits {kind} {dtype} heads of {dim}, {context} positions")
    # one token a sequence: all its rows see the same positions, and what they do not see may be anything
    case = Case(kind, [context, context // 3, 17], [1, 1, 1], 2, dim, 16, seed=71)
    window = d.AttentionWindow(60, 5)
    q = normal(72, (3, 8, dim), TYPES[dtype], 2.0).to(DEV)
    first = run(hip, case, q, 0.09, window, offsets=False)
    assert_rows(case, q, 0.09, first, window, what="before")
    cache, held = case.cache, torch.zeros(case.cache.pages, 16, dtype=torch.bool)
    for s, start in enumerate(case.starts):
        for j in range(int(start) + 1):
            if j > start - 60 or j < 5:
                held[int(case.tables[s, j // 16]), j % 16] = True
    page, off = [x.to(DEV) for x in (~held).nonzero(as_tuple=True)]
    assert len(page) > 40
    for junk in (0.0, 65504.0, math.inf, math.nan):
        if kind == "f16":
            cache.keys[page, off], cache.values[page, :, :, off] = junk, -junk
        else:
            cache.keys[page, off], cache.values[page, :, :, off] = -128, 127
            cache.keyScales[page, :, off], cache.valueScales[page, :, off] = junk, junk
        assert torch.equal(run(hip, case, q, 0.09, window, offsets=False), first), f"{junk} in masked places"


@pytest.mark.parametrize("window", [None, d.AttentionWindow(300, 4)])
@pytest.mark.parametrize("start,tokens,heads,kv,dim", [(517, 1, 32, 8, 128), (4000, 1, 32, 8, 128), (2000, 1, 16, 2, 256),
                                                       (900, 3, 16, 4, 64), (700, 12, 8, 2, 128), (33, 5, 6, 2, 20)])
def test_few_rows_results_in_bf16_are_the_f32_ones_rounded(hip, window, start, tokens, heads, kv, dim):
    step(f"BF16 results of few rows {tokens} tokens at {start}, {heads}/{kv} heads of {dim} {window}")
    # a BF16 query is an F32 one whose second F16 term is 0: over the F16 cache nothing else is rounded to fewer bits
    # than for F32 results before the last step
    case = Case("f16", [start], [tokens], kv, dim, 16, seed=73)
    q = normal(74, (tokens, heads, dim), torch.bfloat16, 2.0).to(DEV)
    scale = 1 / math.sqrt(dim)
    one, other = (run(hip, case, x, scale, window, single=True) for x in (q, q.float()))
    assert torch.equal(one, other.bfloat16())
