"""The refusals of the paged cache's rows and of the attention over it,
without a GPU: HipOps' checks on CPU tensors, and the entry points' own on
addresses that are never followed (each call here fails before a launch)."""

import ctypes

import pytest
import torch

from drift_amd import _lib
from drift_amd import ops as d

I32 = torch.int32


@pytest.fixture(scope="module")
def hip():
    return d.HipOps()


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def f16_cache(pages=4, page=16, kv=2, dim=64):
    return d.KvCache.allocate(pages, page, kv, dim, "cpu")


def i8_cache(pages=4, page=16, kv=2, dim=64):
    return d.QuantizedKvCache.allocate(pages, page, kv, dim, "cpu")


CACHES = [f16_cache, i8_cache]


def test_a_quantised_caches_tensors_agree():
    c = i8_cache()
    assert (c.pages, c.kvHeads, c.headDimension) == (4, 2, 64)
    with pytest.raises(ValueError, match="not a multiple of 16"):
        i8_cache(page=24)
    with pytest.raises(ValueError, match="codes are I8"):
        d.QuantizedKvCache(c.keys.half(), c.values, c.keyScales, c.valueScales, 16)
    with pytest.raises(ValueError, match=r"cache values \[4×2×64×16\] for keys \[4×32×2×64\]"):
        d.QuantizedKvCache(zeros(4, 32, 2, 64, dtype=torch.int8), c.values, c.keyScales, c.valueScales, 16)
    with pytest.raises(ValueError, match=r"cache scales \[4×16×2\]"):
        d.QuantizedKvCache(c.keys, c.values, c.keyScales, zeros(4, 16, 2), 16)
    with pytest.raises(ValueError, match="takes F32, not F16"):
        d.QuantizedKvCache(c.keys, c.values, c.keyScales.half(), c.valueScales, 16)


def test_windows():
    assert d.AttentionWindow(5).sinks == 0
    for positions, sinks in ((0, 0), (-1, 0), (4, -1), (1 << 31, 0), (4, 1 << 31)):
        with pytest.raises(ValueError, match="a window of"):
            d.AttentionWindow(positions, sinks)


@pytest.mark.parametrize("make", CACHES)
def test_attention_refuses(hip, make):
    cache, table, q = make(), zeros(4, dtype=I32), zeros(3, 4, 64)

    def attend(queries=q, out=None, pages=table, start=0, over=cache, window=None, bad=None):
        hip.attention(queries, over, pages, start, 0.1, zeros(*queries.shape, dtype=queries.dtype) if out is None
                      else out, window, bad)

    with pytest.raises(ValueError, match="device memory"):
        attend()
    with pytest.raises(ValueError, match="takes F32 or BF16, not F16"):
        attend(q.half())
    with pytest.raises(ValueError, match="one type, not F32 and BF16"):
        attend(out=q.bfloat16())
    with pytest.raises(ValueError, match="equal shapes"):
        attend(out=zeros(3, 4, 32))
    with pytest.raises(ValueError, match=r"takes \[tokens, heads, headDimension\]"):
        attend(zeros(3, 256))
    for heads, dim in ((3, 64), (4, 32), (0, 64)):
        with pytest.raises(ValueError, match="over a cache of 2 heads of 64"):
            attend(zeros(3, heads, dim))
    with pytest.raises(ValueError, match="at most 512"):
        attend(zeros(3, 4, 520), over=make(dim=520))
    with pytest.raises(ValueError, match="a page table of 4 pages for 65 positions"):
        attend(start=62)
    with pytest.raises(ValueError, match="3 tokens from position -1"):
        attend(start=-1)
    with pytest.raises(ValueError, match="page table is I32"):
        attend(pages=zeros(4))
    with pytest.raises(ValueError, match="page table is I32"):
        attend(pages=zeros(1, 4, dtype=I32))
    with pytest.raises(ValueError, match=r"badPage is I32 \[1\]"):
        attend(bad=zeros(1))


def test_a_cache_whose_keys_have_other_pages_is_refused(hip):
    cache = d.KvCache(zeros(4, 32, 2, 64, dtype=torch.float16), zeros(4, 2, 64, 16, dtype=torch.float16), 16)
    with pytest.raises(ValueError, match="pages of 16 tokens in a cache"):
        hip.attention(zeros(1, 4, 64), cache, zeros(4, dtype=I32), 0, 0.1, zeros(1, 4, 64))
    with pytest.raises(ValueError, match="pages of 16 tokens in a cache"):
        hip.cacheRead(cache, zeros(4, dtype=I32), 0, zeros(1, 2, 64), zeros(1, 2, 64))


@pytest.mark.parametrize("make", CACHES)
def test_sequences_are_refused(hip, make):
    cache, q = make(), zeros(5, 4, 64)
    k = zeros(5, 2, 64)

    def calls(sequences, message):
        for call in (lambda: hip.attentionSequences(q, cache, sequences, 0.1, zeros(5, 4, 64)),
                     lambda: hip.cacheWriteSequences(k, k, cache, sequences),
                     lambda: hip.cacheReadSequences(cache, sequences, k, zeros(5, 2, 64))):
            with pytest.raises(ValueError, match=message):
                call()

    tables, starts, offsets = zeros(5, 4, dtype=I32), zeros(5, dtype=I32), zeros(6, dtype=I32)
    calls(d.Sequences(tables, starts), "device memory")
    calls(d.Sequences(tables, starts, offsets), "device memory")
    calls(d.Sequences(tables.float(), starts), "page tables are I32")
    calls(d.Sequences(zeros(5, dtype=I32), starts), "page tables are I32")
    calls(d.Sequences(tables, starts.long()), "starts torch.int64")
    calls(d.Sequences(tables, zeros(4, dtype=I32)), r"starts I32 \[4\] for 5 sequences")
    calls(d.Sequences(tables, starts, zeros(5, dtype=I32)), r"offsets I32 \[5\] for 5 sequences")
    calls(d.Sequences(tables[:3], starts[:3]), "3 sequences for 5 rows")
    calls(d.Sequences(tables, starts, offsets, -1), "longest sequence of -1")


@pytest.mark.parametrize("make", CACHES)
def test_cache_rows_are_refused(hip, make):
    cache, table = make(), zeros(4, dtype=I32)
    for operation in ((lambda k, v, start=0: hip.cacheRead(cache, table, start, k, v)),
                      (lambda k, v, start=0: hip.cacheWrite(k, v, i8_cache(), table, start))):
        with pytest.raises(ValueError, match="device memory"):
            operation(zeros(3, 2, 64), zeros(3, 2, 64))
        with pytest.raises(ValueError, match="for a cache of 2 heads of 64"):
            operation(zeros(3, 2, 32), zeros(3, 2, 32))
        with pytest.raises(ValueError, match="equal shapes"):
            operation(zeros(3, 2, 64), zeros(4, 2, 64))
        with pytest.raises(ValueError, match="takes F32 or BF16"):
            operation(zeros(3, 2, 64).half(), zeros(3, 2, 64).half())
        with pytest.raises(ValueError, match="a page table of 4 pages for 66 positions"):
            operation(zeros(3, 2, 64), zeros(3, 2, 64), 63)


def test_the_fused_inputs_refuse_the_8_bit_cache(hip):
    norms = d.QueryKeyNorms(zeros(64), zeros(64), 1e-6, 0.0, d.Rope(1e4, 64))
    with pytest.raises(ValueError, match="F16 cache"):
        hip.queryKeyNormRopeCache(zeros(3, 4, 64), zeros(3, 2, 64), zeros(3, 2, 64), norms, zeros(3, dtype=I32),
                                  i8_cache(), zeros(4, dtype=I32), 0, zeros(3, 4, 64))


class OnDevice:
    """A tensor's stand-in on another device."""

    def __init__(self, device, contiguous=True):
        self.is_cuda, self.device, self.contiguous = True, device, contiguous

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return self.contiguous


def test_tensors_of_another_device_are_refused(hip, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    hip._onOneDevice("attention", (OnDevice(0), None, OnDevice(0)))
    with pytest.raises(ValueError, match="a tensor on device 1, launched on device 0"):
        hip._onOneDevice("attention", (OnDevice(0), OnDevice(1)))
    with pytest.raises(ValueError, match="dense row-major"):
        hip._onOneDevice("attention", (OnDevice(0, contiguous=False),))


# ------------------------------------------------------------------ the entry points

P = ctypes.c_void_p


def refusal(name, *args):
    lib = _lib.load()
    code = getattr(lib, name)(*args)
    return lib.drift_last_error().decode() if code == 1 else f"code {code}"


def rows(k=16, v=16, keys=16, values=16, key_scales=None, value_scales=None, tables=16, table_pages=4, cache_pages=4,
         starts=None, offsets=None, sequences=1, start=0, tokens=3, kv_heads=2, dim=64, page=16):
    return tuple(P(x) for x in (k, v, keys, values, key_scales, value_scales, tables)) + \
        (table_pages, cache_pages, P(starts), P(offsets), sequences, start, tokens, kv_heads, dim, page, None, None)


@pytest.mark.parametrize("entry", ["drift_paged_write_f32", "drift_paged_write_bf16", "drift_paged_read_f32",
                                   "drift_paged_read_bf16"])
def test_rows_entry_points_refuse(entry):
    assert "pages of 10 tokens: not a multiple of 16" in refusal(entry, *rows(page=10))
    assert "-1 tokens" in refusal(entry, *rows(tokens=-1))
    assert "0 heads" in refusal(entry, *rows(kv_heads=0))
    assert "heads of 0 values" in refusal(entry, *rows(dim=0))
    assert "start -1" in refusal(entry, *rows(start=-1))
    assert "a page table of 4 pages for 65 positions" in refusal(entry, *rows(start=62))
    assert "2147483650 positions" in refusal(entry, *rows(start=2 ** 31 - 1))
    assert "2147483550 positions (at most 2147483520)" in refusal(entry, *rows(start=2147483547, table_pages=2 ** 27))
    assert "2 sequences without starts" in refusal(entry, *rows(sequences=2))
    assert "2 sequences of 3 tokens without offsets" in refusal(entry, *rows(sequences=2, starts=16))
    assert "null tensor" in refusal(entry, *rows(k=None))
    assert "null tensor" in refusal(entry, *rows(keys=None))
    assert "null tensor" in refusal(entry, *rows(tables=None))
    assert "scales of keys or of values alone" in refusal(entry, *rows(key_scales=16))
    assert "not aligned to their elements" in refusal(entry, *rows(keys=17))
    assert "not aligned to their elements" in refusal(entry, *rows(key_scales=18, value_scales=16))
    assert "in one call" in refusal(entry, *rows(tokens=2 ** 31 - 129, table_pages=2 ** 27, kv_heads=64, dim=7))
    assert refusal(entry, *rows(tokens=0)) == "code 0"
    assert refusal(entry, *rows(sequences=0, starts=None)) == "code 0"


def attention(queries=16, keys=16, values=16, key_scales=None, value_scales=None, tables=16, table_pages=4,
              cache_pages=4, starts=None, offsets=None, sequences=1, start=0, tokens=3, heads=4, kv_heads=2, dim=64,
              page=16, scale=0.1, window=0, sinks=0, longest=0, out=64, workspace=None, size=0):
    return tuple(P(x) for x in (queries, keys, values, key_scales, value_scales, tables)) + \
        (table_pages, cache_pages, P(starts), P(offsets), sequences, start, tokens, heads, kv_heads, dim, page, scale,
         window, sinks, longest, P(out), P(workspace), size, None, None)


@pytest.mark.parametrize("entry", ["drift_paged_attention_f32", "drift_paged_attention_bf16"])
def test_attention_entry_points_refuse(entry):
    assert "heads of 520 values (at most 512)" in refusal(entry, *attention(dim=520))
    assert "3 heads over 2 key heads" in refusal(entry, *attention(heads=3))
    assert "0 heads over 2" in refusal(entry, *attention(heads=0))
    assert "a window of -1 positions" in refusal(entry, *attention(window=-1))
    assert "a window of 0 positions with 4 sinks" in refusal(entry, *attention(sinks=4))
    assert "pages of 8 tokens" in refusal(entry, *attention(page=8))
    assert "a page table of 4 pages for 65 positions" in refusal(entry, *attention(start=62))
    assert "null tensor" in refusal(entry, *attention(queries=None))
    assert "null tensor" in refusal(entry, *attention(out=None))
    assert "null tensor" in refusal(entry, *attention(values=None))
    assert "out is queries" in refusal(entry, *attention(out=16))
    assert "not aligned" in refusal(entry, *attention(queries=17))
    assert "longest" in refusal(entry, *attention(longest=-1))
    assert refusal(entry, *attention(tokens=0)) == "code 0"
    assert refusal(entry, *attention(sequences=0)) == "code 0"


def workspace(*numbers):
    told = ctypes.c_int64(-1)
    return refusal("drift_paged_attention_workspace", *numbers, ctypes.byref(told)), told.value


def test_the_workspace_is_told():
    assert refusal("drift_paged_attention_workspace", 1, 1, 8, 2, 128, 0, 0, 10, None).endswith("null bytes")
    assert "7 heads over 2" in workspace(1, 1, 7, 2, 128, 0, 0, 10)[0]
    assert "longest" in workspace(1, 1, 8, 2, 128, 0, 0, -1)[0]
    for numbers in ((1, 1, 8, 2, 128, 0, 0, 10), (64, 64, 32, 8, 128, 4096, 4, 2 ** 31 - 1), (1, 0, 8, 2, 64, 0, 0, 0),
                    (0, 5, 8, 2, 64, 0, 0, 5), (3, 2 ** 20, 64, 8, 256, 0, 0, 2 ** 20)):
        code, size = workspace(*numbers)
        assert code == "code 0" and 0 <= size < 1 << 40


@pytest.mark.parametrize("sequences", [1, 17, 64, 256])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (28, 4, 128), (16, 2, 256), (16, 16, 64)])
def test_a_decode_steps_workspace_is_its_rows_splits(sequences, heads, kv_heads, dim):
    """One token a sequence, by offsets or without: `splits` partial results
    and statistics of each row there is, and no more splits than leave 16,384
    blocks of a sequence, key head and split, however wide the page tables."""
    sizes = []
    for longest in (100, 8016, 32768, 131072, 2 ** 20, 2 ** 31 - 128):
        code, size = workspace(sequences, sequences, heads, kv_heads, dim, 0, 0, longest)
        assert code == "code 0"
        splits = min(1024, max(1, 16384 // (sequences * kv_heads)), -(-longest // 256))
        # (by offsets the rows may be one sequence's, of attend_many: its splits leave up to 512 blocks of 128 rows)
        splits = max(splits, min(-(-longest // 512), -(-512 * 128 // (sequences * heads))))
        assert size <= splits * sequences * heads * (dim + 3) * 4
        sizes.append(size)
    assert sizes == sorted(sizes)


def test_a_mixed_batchs_workspace_has_slots_for_few_rows():
    # 24 sequences, 1,811 tokens of 28 heads over 4: up to 16 rows of each sequence and key head may be split
    code, size = workspace(24, 1811, 28, 4, 128, 0, 0, 131072)
    assert code == "code 0" and 0 < size <= 170 * 24 * 4 * 16 * 131 * 4


@pytest.mark.parametrize("entry,size", [("drift_paged_attention_f32", 4), ("drift_paged_attention_bf16", 2)])
def test_out_that_overlaps_queries_is_refused(entry, size):
    for apart in (16, 3 * 4 * 64 * size - 16):
        assert "out overlaps queries" in refusal(entry, *attention(queries=1 << 20, out=(1 << 20) + apart))
        assert "out overlaps queries" in refusal(entry, *attention(queries=(1 << 20) + apart, out=1 << 20))


def test_out_that_overlaps_queries_is_refused_by_hip_ops(hip, monkeypatch):
    monkeypatch.setattr(hip, "_onOneDevice", lambda *_: None)
    flat, cache, table = zeros(4 * 4 * 64), f16_cache(), zeros(4, dtype=I32)
    queries, over = flat[:768].view(3, 4, 64), flat[256:].view(3, 4, 64)
    for out, what in ((queries, "is"), (over, "overlaps")):
        with pytest.raises(ValueError, match=f"attention: out {what} queries"):
            hip.attention(queries, cache, table, 0, 0.1, out)
    with pytest.raises(ValueError, match="attentionSequences: out overlaps queries"):
        hip.attentionSequences(over, cache, d.Sequences(zeros(3, 4, dtype=I32), zeros(3, dtype=I32)), 0.1, queries)
