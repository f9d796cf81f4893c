"""The refusals of attention over trees of drafted tokens, of the masses, of
the choice of the heaviest positions and of the move of kept rows, without a
GPU: HipOps' checks on CPU tensors, and the entry points' own on addresses that
are never followed (each call here fails before a launch)."""

import ctypes

import pytest
import torch

from drift_amd import _lib
from drift_amd import ops as d
from tests.test_paged_checks_cpu import CACHES, I32, P, f16_cache, refusal, zeros


@pytest.fixture(scope="module")
def hip():
    return d.HipOps()


def batch(count=2, pages=4, offsets=True):
    return d.Sequences(zeros(count, pages, dtype=I32), zeros(count, dtype=I32),
                       zeros(count + 1, dtype=I32) if offsets else None)


@pytest.mark.parametrize("make", CACHES)
def test_trees_are_refused(hip, make):
    def tree(queries=zeros(3, 4, 64), sees=zeros(3, 1, dtype=I32), out=None, sequences=batch(), bad=None):
        hip.attentionTree(queries, make(), sequences, sees, 0.1, torch.empty_like(queries) if out is None else out,
                          None, bad)

    with pytest.raises(ValueError, match="device memory"):
        tree()
    with pytest.raises(ValueError, match=r"what the rows see is I32 \[3, words\], not I32 \[2×1\]"):
        tree(sees=zeros(2, 1, dtype=I32))
    for sees in (zeros(3, 0, dtype=I32), zeros(3, dtype=I32), zeros(3, 1), zeros(3, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="what the rows see is I32"):
            tree(sees=sees)
    with pytest.raises(ValueError, match="takes F32 or BF16"):
        tree(zeros(3, 4, 64).half())
    with pytest.raises(ValueError, match="over a cache of 2 heads of 64"):
        tree(zeros(3, 3, 64))
    with pytest.raises(ValueError, match="2 sequences for 3 rows"):
        tree(sequences=batch(offsets=False))
    with pytest.raises(ValueError, match=r"badPage is I32 \[1\]"):
        tree(bad=zeros(1))


@pytest.mark.parametrize("make", CACHES)
def test_masses_are_refused(hip, make):
    def mass(queries=zeros(3, 4, 64), to=zeros(4, 2, 16), before=None, sequences=batch(), bad=None):
        hip.attentionMass(queries, make(), sequences, 0.1, to, before, bad)

    with pytest.raises(ValueError, match="device memory"):
        mass()
    with pytest.raises(ValueError, match="takes F32 or BF16"):
        mass(zeros(3, 4, 64).half())
    with pytest.raises(ValueError, match="over a cache of 2 heads of 64"):
        mass(zeros(3, 4, 32))
    with pytest.raises(ValueError, match=r"masses \[4×16×2\] for a cache"):
        mass(to=zeros(4, 16, 2))
    with pytest.raises(ValueError, match=r"masses are \[pages, kvHeads, pageSize\]"):
        mass(to=zeros(4, 32))
    with pytest.raises(ValueError, match="takes F32, not F16"):
        mass(to=zeros(4, 2, 16).half())
    with pytest.raises(ValueError, match=r"masses \[3×2×16\] for a cache"):
        mass(before=zeros(3, 2, 16))
    with pytest.raises(ValueError, match="2 sequences for 3 rows"):
        mass(sequences=batch(offsets=False))
    with pytest.raises(ValueError, match=r"badPage is I32 \[1\]"):
        mass(bad=zeros(1))


def test_masses_that_overlap_are_refused(hip, monkeypatch):
    monkeypatch.setattr(hip, "_onOneDevice", lambda *_: None)
    flat = zeros(5 * 2 * 16)
    with pytest.raises(ValueError, match="mass overlaps before"):
        hip.attentionMass(zeros(3, 4, 64), f16_cache(), batch(), 0.1, flat[:128].view(4, 2, 16),
                          flat[16:144].view(4, 2, 16))


def test_the_heaviest_are_refused(hip, monkeypatch):
    def pick(mass=zeros(4, 2, 16), tables=zeros(3, 4, dtype=I32), lengths=zeros(3, dtype=I32), sinks=1, recent=2,
             kept=zeros(3, 2, 8, dtype=I32), counts=zeros(3, dtype=I32), bad=None):
        hip.heaviest(mass, tables, lengths, sinks, recent, kept, counts, bad)

    with pytest.raises(ValueError, match="device memory"):
        pick()
    with pytest.raises(ValueError, match="takes F32, not F16"):
        pick(zeros(4, 2, 16).half())
    with pytest.raises(ValueError, match="masses are"):
        pick(zeros(4, 16))
    with pytest.raises(ValueError, match="pages of 24 tokens: not a multiple of 16"):
        pick(zeros(4, 2, 24))
    with pytest.raises(ValueError, match="page tables are I32"):
        pick(tables=zeros(3, 4))
    with pytest.raises(ValueError, match=r"lengths I32 \[2\] for 3 sequences"):
        pick(lengths=zeros(2, dtype=I32))
    with pytest.raises(ValueError, match="counts torch.int64"):
        pick(counts=zeros(3, dtype=torch.int64))
    for kept in (zeros(3, 8, dtype=I32), zeros(3, 3, 8, dtype=I32), zeros(2, 2, 8, dtype=I32), zeros(3, 2, 8)):
        with pytest.raises(ValueError, match="for 3 sequences of 2 heads"):
            pick(kept=kept)
    for sinks, recent in ((-1, 0), (0, -1), (5, 4)):
        with pytest.raises(ValueError, match=f"the first {sinks} and the last {recent} positions of 8 kept"):
            pick(sinks=sinks, recent=recent)
    with pytest.raises(ValueError, match=r"badPage is I32 \[1\]"):
        pick(bad=zeros(1))
    monkeypatch.setattr(hip, "_onOneDevice", lambda *_: None)
    same = zeros(3, dtype=I32)
    with pytest.raises(ValueError, match="counts overlap lengths"):
        pick(lengths=same, counts=same)


@pytest.mark.parametrize("make", CACHES)
def test_moves_are_refused(hip, make):
    def keep(tables=zeros(3, 4, dtype=I32), kept=zeros(3, 2, 8, dtype=I32), counts=None, starts=None, into=None,
             mass=None, bad=None):
        hip.cacheKeep(make(), tables, kept, counts, starts, into, mass, bad)

    with pytest.raises(ValueError, match="device memory"):
        keep()
    with pytest.raises(ValueError, match="page tables are I32"):
        keep(tables=zeros(3, dtype=I32))
    with pytest.raises(ValueError, match=r"counts I32 \[2\] for 3 sequences"):
        keep(counts=zeros(2, dtype=I32))
    with pytest.raises(ValueError, match="starts F32"):
        keep(starts=zeros(3))
    for kept in (zeros(3, 1, 8, dtype=I32), zeros(2, 8, dtype=I32), zeros(3, dtype=I32), zeros(3, 2, 8)):
        with pytest.raises(ValueError, match="for 3 sequences of 2 heads"):
            keep(kept=kept)
    with pytest.raises(ValueError, match=r"into \[2×4\] for 3 sequences"):
        keep(into=zeros(2, 4, dtype=I32))
    with pytest.raises(ValueError, match="page tables are I32"):
        keep(into=zeros(3, 4))
    with pytest.raises(ValueError, match="for a cache"):
        keep(mass=zeros(4, 2, 32))
    with pytest.raises(ValueError, match=r"badPage is I32 \[1\]"):
        keep(bad=zeros(1))


# ------------------------------------------------------------------ the entry points

def attention(queries=16, keys=16, values=16, key_scales=None, value_scales=None, tables=16, table_pages=4,
              cache_pages=4, starts=None, offsets=None, sequences=1, start=0, tokens=3, heads=4, kv_heads=2, dim=64,
              page=16, scale=0.1, window=0, sinks=0, longest=0, sees=16, words=1, out=64, workspace=None, size=0):
    return tuple(P(x) for x in (queries, keys, values, key_scales, value_scales, tables)) + \
        (table_pages, cache_pages, P(starts), P(offsets), sequences, start, tokens, heads, kv_heads, dim, page, scale,
         window, sinks, longest, P(sees), words, P(out), P(workspace), size, None, None)


@pytest.mark.parametrize("entry", ["drift_tree_attention_f32", "drift_tree_attention_bf16"])
def test_tree_entry_points_refuse(entry):
    assert "heads of 520 values (at most 512)" in refusal(entry, *attention(dim=520))
    assert "3 heads over 2 key heads" in refusal(entry, *attention(heads=3))
    assert "a window of 0 positions with 4 sinks" in refusal(entry, *attention(sinks=4))
    assert "pages of 8 tokens" in refusal(entry, *attention(page=8))
    assert "a page table of 4 pages for 65 positions" in refusal(entry, *attention(start=62))
    assert "null tensor" in refusal(entry, *attention(queries=None))
    assert "null tensor" in refusal(entry, *attention(sees=None))
    assert "0 words" in refusal(entry, *attention(words=0))
    assert "not aligned" in refusal(entry, *attention(sees=18))
    assert "out is queries" in refusal(entry, *attention(out=16))
    assert "needs" in refusal(entry, *attention(out=1 << 20, start=5000, table_pages=400, longest=5003))
    assert refusal(entry, *attention(tokens=0)) == "code 0"
    assert refusal(entry, *attention(sequences=0)) == "code 0"


def mass(queries=16, keys=16, key_scales=None, tables=16, table_pages=4, cache_pages=4, starts=None, offsets=None,
         sequences=1, start=0, tokens=3, heads=4, kv_heads=2, dim=64, page=16, scale=0.1, longest=0, before=None,
         to=64, workspace=16, size=1 << 40):
    return tuple(P(x) for x in (queries, keys, key_scales, tables)) + \
        (table_pages, cache_pages, P(starts), P(offsets), sequences, start, tokens, heads, kv_heads, dim, page, scale,
         longest, P(before), P(to), P(workspace), size, None, None)


@pytest.mark.parametrize("entry", ["drift_attention_mass_f32", "drift_attention_mass_bf16"])
def test_mass_entry_points_refuse(entry):
    assert "heads of 520 values (at most 512)" in refusal(entry, *mass(dim=520))
    assert "3 heads over 2 key heads" in refusal(entry, *mass(heads=3))
    assert "pages of 8 tokens" in refusal(entry, *mass(page=8))
    assert "longest" in refusal(entry, *mass(longest=-1))
    assert "a page table of 4 pages for 65 positions" in refusal(entry, *mass(start=62))
    assert "2 sequences of 3 tokens without offsets" in refusal(entry, *mass(sequences=2, starts=16))
    for name in ("queries", "keys", "tables", "to"):
        assert "null tensor" in refusal(entry, *mass(**{name: None}))
    assert "not aligned" in refusal(entry, *mass(queries=17))
    assert "not aligned" in refusal(entry, *mass(keys=17))
    assert "not aligned" in refusal(entry, *mass(key_scales=18))
    assert "not aligned" in refusal(entry, *mass(to=66))
    assert "mass overlaps before" in refusal(entry, *mass(before=1 << 20, to=(1 << 20) + 4 * 2 * 16 * 4 - 4))
    assert "mass overlaps before" in refusal(entry, *mass(before=(1 << 20) + 4, to=1 << 20))
    assert "needs" in refusal(entry, *mass(size=0))
    assert "needs" in refusal(entry, *mass(workspace=None))
    assert "needs" in refusal(entry, *mass(workspace=24))
    assert refusal(entry, *mass(tokens=0)) == "code 0"
    assert refusal(entry, *mass(sequences=0)) == "code 0"


def told(entry, *numbers):
    size = ctypes.c_int64(-1)
    return refusal(entry, *numbers, ctypes.byref(size)), size.value


def test_the_workspaces_are_told():
    assert refusal("drift_tree_attention_workspace", 1, 1, 8, 2, 128, 0, 0, 10, None).endswith("null bytes")
    assert "7 heads over 2" in told("drift_tree_attention_workspace", 1, 1, 7, 2, 128, 0, 0, 10)[0]
    for numbers in ((1, 8, 32, 8, 128, 0, 0, 525), (64, 2000, 32, 8, 256, 4096, 4, 2 ** 31 - 1), (0, 5, 8, 2, 64, 0, 0, 5)):
        code, size = told("drift_tree_attention_workspace", *numbers)
        assert code == "code 0" and 0 <= size < 1 << 40
    assert refusal("drift_attention_mass_workspace", 1, 1, 8, 2, 128, 16, 10, None).endswith("null bytes")
    assert "7 heads over 2" in told("drift_attention_mass_workspace", 1, 1, 7, 2, 128, 16, 10)[0]
    assert "longest" in told("drift_attention_mass_workspace", 1, 1, 8, 2, 128, 16, -1)[0]
    assert "room for -1" in told("drift_attention_mass_workspace", 1, 1, 8, 2, 128, -1, 5)[0]
    for numbers in ((1, 1, 8, 2, 128, 16, 10), (64, 64, 32, 8, 128, 2 ** 31 - 1, 2 ** 31 - 1), (1, 0, 8, 2, 64, 0, 0),
                    (0, 5, 8, 2, 64, 16, 5), (3, 2 ** 20, 64, 8, 256, 2 ** 21, 2 ** 20), (1, 1, 1, 1, 1, 0, 0)):
        code, size = told("drift_attention_mass_workspace", *numbers)
        assert code == "code 0" and 0 <= size < 1 << 40
    assert refusal("drift_cache_keep_workspace", 1, 1, 8, 128, 0, None).endswith("null bytes")
    assert "0 heads" in told("drift_cache_keep_workspace", 1, 1, 0, 128, 0)[0]
    assert "in one call" in told("drift_cache_keep_workspace", 1 << 20, 1 << 20, 8, 128, 0)[0]
    for numbers in ((0, 5, 2, 64, 0), (3, 0, 2, 64, 1), (64, 2048, 8, 128, 0), (1, 100000, 2, 7, 1)):
        code, size = told("drift_cache_keep_workspace", *numbers)
        assert code == "code 0" and 0 <= size < 1 << 40


def heaviest(mass=64, tables=64, table_pages=4, cache_pages=4, lengths=64, sequences=3, kv_heads=2, page=16, sinks=1,
             recent=2, keep=8, kept=64, counts=128, bad=None):
    return (P(mass), P(tables), table_pages, cache_pages, P(lengths), sequences, kv_heads, page, sinks, recent, keep,
            P(kept), P(counts), P(bad), None)


def test_the_heaviests_entry_point_refuses():
    entry = "drift_heaviest"
    assert "-1 sequences" in refusal(entry, *heaviest(sequences=-1))
    assert "0 heads" in refusal(entry, *heaviest(kv_heads=0))
    assert "pages of 8 tokens" in refusal(entry, *heaviest(page=8))
    assert "the first 5 and the last 4 positions of 8 kept" in refusal(entry, *heaviest(sinks=5, recent=4))
    assert "the first 2147483647" in refusal(entry, *heaviest(sinks=2 ** 31 - 1, recent=2 ** 31 - 1))
    assert "-1" in refusal(entry, *heaviest(sinks=0, recent=0, keep=-1))
    for name in ("mass", "tables", "lengths", "kept", "counts"):
        assert "null tensor" in refusal(entry, *heaviest(**{name: None}))
        assert "not aligned" in refusal(entry, *heaviest(**{name: 66}))
    assert "counts overlap lengths" in refusal(entry, *heaviest(counts=72))
    assert "in one call" in refusal(entry, *heaviest(sequences=2 ** 30, kv_heads=2 ** 10, counts=1 << 40))
    assert refusal(entry, *heaviest(sequences=0)) == "code 0"


def move(keys=16, values=16, key_scales=None, value_scales=None, mass=None, tables=16, table_pages=4, into=None,
         into_pages=0, cache_pages=4, kept=16, kept_heads=2, counts=None, starts=None, sequences=3, most=8, kv_heads=2,
         dim=64, page=16, workspace=16, size=1 << 40):
    return tuple(P(x) for x in (keys, values, key_scales, value_scales, mass, tables)) + \
        (table_pages, P(into), into_pages, cache_pages, P(kept), kept_heads, P(counts), P(starts), sequences, most,
         kv_heads, dim, page, P(workspace), size, None, None)


def test_the_moves_entry_point_refuses():
    entry = "drift_cache_keep"
    assert "-1 rows" in refusal(entry, *move(most=-1))
    assert "heads of 0 values" in refusal(entry, *move(dim=0))
    assert "pages of 8 tokens" in refusal(entry, *move(page=8))
    assert "into -1" in refusal(entry, *move(into_pages=-1))
    assert "lists of 3 heads for 2" in refusal(entry, *move(kept_heads=3))
    for name in ("keys", "values", "tables", "kept"):
        assert "null tensor" in refusal(entry, *move(**{name: None}))
    assert "scales of keys or of values alone" in refusal(entry, *move(key_scales=16))
    assert "not aligned" in refusal(entry, *move(keys=17))
    for name in ("mass", "tables", "into", "kept", "counts", "starts"):
        assert "not aligned" in refusal(entry, *move(**{name: 18}))
    assert "needs" in refusal(entry, *move(size=0))
    assert "needs" in refusal(entry, *move(workspace=None))
    assert "needs" in refusal(entry, *move(workspace=24))
    assert "needs" in refusal(entry, *move(into=16, into_pages=4, size=0))  # into is the page tables: in place
    assert "in one call" in refusal(entry, *move(sequences=2 ** 30, most=2 ** 30))
    assert refusal(entry, *move(most=0)) == "code 0"
    assert refusal(entry, *move(sequences=0)) == "code 0"


def test_moves_into_their_own_page_tables_as_others_are_refused(hip):
    """The page tables' memory read as tables of another width would name other sequences' pages as the places that
    rows move to in place."""
    tables = zeros(3, 4, dtype=I32)
    kept = zeros(3, 2, 8, dtype=I32)
    with pytest.raises(ValueError, match=r"into \[3×2\] is the page tables \[3×4\]"):
        hip.cacheKeep(f16_cache(), tables, kept, into=tables.view(-1)[:6].view(3, 2))
    assert "page tables of 4 pages a sequence as ones of 2" in refusal("drift_cache_keep", *move(into=16, into_pages=2))
    # one sequence's first pages, or the same tables, are in place: their own scratch is asked for
    with pytest.raises(ValueError, match="device memory"):
        hip.cacheKeep(f16_cache(), tables[:1], kept[:1], into=tables[:1, :2])
    assert "needs" in refusal("drift_cache_keep", *move(into=16, into_pages=2, sequences=1, size=0))
    assert "needs" in refusal("drift_cache_keep", *move(into=16, into_pages=4, size=0))


@pytest.mark.parametrize("dim,quantized", [(128, 0), (128, 1), (96, 0), (24, 1), (512, 1), (7, 0)])
@pytest.mark.parametrize("most", [1, 7, 128])
def test_short_moves_ask_for_their_rows_bytes_alone(dim, quantized, most):
    """A row's key, value, two scales and mass; a list of up to 128 rows puts no more by."""
    code, size = told("drift_cache_keep_workspace", 32, most, 8, dim, quantized)
    row = -(-dim * 2 * (1 if quantized else 2) // 4) * 4 + 12
    assert code == "code 0" and size == -(-32 * most * 8 * row // 16) * 16
