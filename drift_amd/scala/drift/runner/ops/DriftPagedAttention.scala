package drift.runner.ops

import drift.runner.tensor.*

import java.lang.foreign.*

/** `KvCache`'s pages in 8 bits: I8 codes `keys` `[pages, pageSize, kvHeads, D]`
  * and `values` `[pages, kvHeads, D, pageSize]`, and F32 scales `[pages,
  * kvHeads, pageSize]`, one a position and head of each: a value is its code
  * times its row's scale, max |x| / 127 of the row.
  */
final case class QuantizedKvCache(keys: Tensor, values: Tensor, keyScales: Tensor, valueScales: Tensor,
                                  pageSize: Int) {
  require(pageSize > 0 && pageSize % 16 == 0, s"pages of $pageSize tokens: not a multiple of 16")
  require(keys.dtype == DType.I8 && values.dtype == DType.I8, "the 8-bit cache's codes are I8")
  require(keys.shape.rank == 4, "the cache's keys and values are 4-dimensional")
  private val Seq(pageCount, size, heads, dimension) = keys.shape.dimensions
  require(size == pageSize && values.shape == Shape.of(pageCount, heads, dimension, size),
    s"cache values ${values.shape} for keys ${keys.shape}")
  Ops.requireF32("the 8-bit cache", keyScales, valueScales)
  Seq(keyScales, valueScales).foreach { scales =>
    require(scales.shape == Shape.of(pageCount, heads, size), s"cache scales ${scales.shape} for keys ${keys.shape}")
  }
  def pages: Int = pageCount.toInt
  def kvHeads: Int = heads.toInt
  def headDimension: Int = dimension.toInt
}

/** What a row at position P sees of the positions j up to P: j > P - positions, or j < sinks. */
final case class AttentionWindow(positions: Int, sinks: Int = 0) {
  require(positions > 0 && sinks >= 0, s"a window of $positions positions with $sinks sinks")
}

/** Several sequences' token rows in one call: sequence s has rows
  * offsets[s] to offsets[s + 1], at positions starts[s] and on, in the pages
  * pageTables[s], all I32 and read on the device; without `offsets` each has one
  * row. `longest` is a guess of the most positions of one, by which attention
  * splits its work (0: what the page tables have room for).
  */
final case class Sequences(pageTables: Tensor, starts: Tensor, offsets: Option[Tensor] = None, longest: Int = 0) {
  require(pageTables.dtype == DType.I32 && pageTables.shape.rank == 2,
    s"page tables are I32 [sequences, pages], not ${pageTables.dtype} ${pageTables.shape}")
  require(starts.dtype == DType.I32 && starts.shape == Shape.of(pageTables.shape.dimensions.head),
    s"starts ${starts.dtype} ${starts.shape} for page tables ${pageTables.shape}")
  offsets.foreach { o =>
    require(o.dtype == DType.I32 && o.shape == Shape.of(pageTables.shape.dimensions.head + 1),
      s"offsets ${o.dtype} ${o.shape} for page tables ${pageTables.shape}")
  }
  require(longest >= 0, s"a longest sequence of $longest positions")
  def count: Int = pageTables.shape.dimensions.head.toInt
}

/** Rows that `cacheKeep` moves: position starts[s] + i (without `starts` i) gets
  * what position kept[s, head, i] holds, for i < counts[s] (without `counts`
  * all); all I32, kept `[sequences, kvHeads, most]`, or `[sequences, most]` for
  * all heads alike. With `into`, page tables `[sequences, pages]`, rows go to
  * those pages, else to the same.
  */
final case class KeptRows(pageTables: Tensor, kept: Tensor, counts: Option[Tensor] = None,
                          starts: Option[Tensor] = None, into: Option[Tensor] = None) {
  require(pageTables.dtype == DType.I32 && pageTables.shape.rank == 2,
    s"page tables are I32 [sequences, pages], not ${pageTables.dtype} ${pageTables.shape}")
  require(kept.dtype == DType.I32 && (kept.shape.rank == 2 || kept.shape.rank == 3) &&
    kept.shape.dimensions.head == pageTables.shape.dimensions.head,
    s"kept ${kept.dtype} ${kept.shape} for page tables ${pageTables.shape}")
  (counts.toSeq ++ starts).foreach { v =>
    require(v.dtype == DType.I32 && v.shape == Shape.of(pageTables.shape.dimensions.head),
      s"counts or starts ${v.dtype} ${v.shape} for page tables ${pageTables.shape}")
  }
  into.foreach { t =>
    require(t.dtype == DType.I32 && t.shape.rank == 2 && t.shape.dimensions.head == pageTables.shape.dimensions.head,
      s"into ${t.dtype} ${t.shape} for page tables ${pageTables.shape}")
  }
}

/** The paged cache of several sequences a call, in F16 and in 8 bits, and
  * attention over it, as libdrift_kernels downcalls; the reference's own
  * attention (ops/HipAttention.scala) has no gfx950 code. The caller owns the
  * attention's scratch: at least `attentionWorkspace` bytes, one for each
  * stream that runs such calls.
  */
private[ops] trait DriftPagedAttention extends DriftAttention {

  /** The most positions of a sequence (csrc/paged.hpp). */
  private val MostPositions: Long = Int.MaxValue - 127L

  /** A cache as the entry points take it: its tensors and sizes. */
  private final case class Paged(keys: Tensor, values: Tensor, keyScales: Option[Tensor], valueScales: Option[Tensor],
                                 pages: Int, kvHeads: Int, headDimension: Int, pageSize: Int)

  private def paged(cache: KvCache): Paged =
    Paged(cache.keys, cache.values, None, None, cache.pages, cache.kvHeads, cache.headDimension, cache.pageSize)

  private def paged(cache: QuantizedKvCache): Paged =
    Paged(cache.keys, cache.values, Some(cache.keyScales), Some(cache.valueScales), cache.pages, cache.kvHeads,
      cache.headDimension, cache.pageSize)

  private def checkRows(operation: String, k: Tensor, v: Tensor, cache: Paged): Int = {
    Ops.checkElementwise(operation, k, v)
    require(k.shape.rank == 3 && k.shape.dimensions.drop(1) == Seq(cache.kvHeads.toLong, cache.headDimension.toLong),
      s"$operation: ${k.shape} for a cache of ${cache.kvHeads} heads of ${cache.headDimension}")
    k.shape.dimensions.head.toInt
  }

  private def checkSequences(operation: String, sequences: Sequences, tokens: Int): Unit =
    require(sequences.offsets.nonEmpty || sequences.count == tokens,
      s"$operation: ${sequences.count} sequences for $tokens rows (several rows a sequence need offsets)")

  /** One sequence's rows quantised into the 8-bit cache at `start`. */
  def cacheWrite(k: Tensor, v: Tensor, cache: QuantizedKvCache, pageTable: Tensor, start: Int): Unit =
    writeRows("cacheWrite", k, v, paged(cache), Left((pageTable, start)))

  /** Several sequences' keys and values into the cache in one launch. */
  def cacheWriteSequences(k: Tensor, v: Tensor, cache: KvCache, sequences: Sequences): Unit =
    writeRows("cacheWriteSequences", k, v, paged(cache), Right(sequences))
  def cacheWriteSequences(k: Tensor, v: Tensor, cache: QuantizedKvCache, sequences: Sequences): Unit =
    writeRows("cacheWriteSequences", k, v, paged(cache), Right(sequences))

  /** Positions start and on of the cache into k and v `[tokens, kvHeads, D]`. */
  def cacheRead(cache: KvCache, pageTable: Tensor, start: Int, k: Tensor, v: Tensor): Unit =
    readRows("cacheRead", paged(cache), Left((pageTable, start)), k, v)
  def cacheRead(cache: QuantizedKvCache, pageTable: Tensor, start: Int, k: Tensor, v: Tensor): Unit =
    readRows("cacheRead", paged(cache), Left((pageTable, start)), k, v)

  def cacheReadSequences(cache: KvCache, sequences: Sequences, k: Tensor, v: Tensor): Unit =
    readRows("cacheReadSequences", paged(cache), Right(sequences), k, v)
  def cacheReadSequences(cache: QuantizedKvCache, sequences: Sequences, k: Tensor, v: Tensor): Unit =
    readRows("cacheReadSequences", paged(cache), Right(sequences), k, v)

  /** A call's page tables, starts (null for one sequence at `start`) and
    * offsets, and the sizes with them.
    */
  private final case class Rows(tables: Tensor, tablePages: Int, starts: Option[Tensor], offsets: Option[Tensor],
                                count: Int, start: Int, longest: Int)

  private def rowsOf(operation: String, cache: Paged, tokens: Int, pages: Either[(Tensor, Int), Sequences]): Rows =
    pages match {
      case Left((table, start)) =>
        require(table.dtype == DType.I32 && table.shape.rank == 1,
          s"a page table is I32 [pages], not ${table.dtype} ${table.shape}")
        val count = table.shape.elementCount
        require(start >= 0 && start.toLong + tokens <= MostPositions, s"$operation: $tokens tokens from position $start")
        require(count * cache.pageSize >= start.toLong + tokens,
          s"a page table of $count pages for ${start.toLong + tokens} positions")
        Rows(table, count.toInt, None, None, 1, start, start + tokens)
      case Right(sequences) =>
        checkSequences(operation, sequences, tokens)
        val tablePages = sequences.pageTables.shape.last.toInt
        val room = (tablePages.toLong * cache.pageSize).min(MostPositions).toInt
        Rows(sequences.pageTables, tablePages, Some(sequences.starts), sequences.offsets, sequences.count, 0,
          if (sequences.longest > 0) sequences.longest.min(room) else room)
    }

  private def writeRows(operation: String, k: Tensor, v: Tensor, cache: Paged,
                        where: Either[(Tensor, Int), Sequences]): Unit = {
    val tokens: Int = checkRows(operation, k, v, cache)
    val rows = rowsOf(operation, cache, tokens, where)
    val (tablePages: Int, pages: Int, count: Int, start: Int) = (rows.tablePages, cache.pages, rows.count, rows.start)
    val (kvHeads: Int, d: Int, pageSize: Int) = (cache.kvHeads, cache.headDimension, cache.pageSize)
    downcall(entry("drift_paged_write", k))(
      (drift.pagedWrite(bf16(k)).invokeExact(pointer(k), pointer(v), pointer(cache.keys), pointer(cache.values),
        optional(cache.keyScales), optional(cache.valueScales), pointer(rows.tables), tablePages, pages,
        optional(rows.starts), optional(rows.offsets), count, start, tokens, kvHeads, d, pageSize, MemorySegment.NULL,
        DefaultStream): Int)
    )
  }

  private def readRows(operation: String, cache: Paged, where: Either[(Tensor, Int), Sequences], k: Tensor,
                       v: Tensor): Unit = {
    val tokens: Int = checkRows(operation, k, v, cache)
    val rows = rowsOf(operation, cache, tokens, where)
    val (tablePages: Int, pages: Int, count: Int, start: Int) = (rows.tablePages, cache.pages, rows.count, rows.start)
    val (kvHeads: Int, d: Int, pageSize: Int) = (cache.kvHeads, cache.headDimension, cache.pageSize)
    downcall(entry("drift_paged_read", k))(
      (drift.pagedRead(bf16(k)).invokeExact(pointer(k), pointer(v), pointer(cache.keys), pointer(cache.values),
        optional(cache.keyScales), optional(cache.valueScales), pointer(rows.tables), tablePages, pages,
        optional(rows.starts), optional(rows.offsets), count, start, tokens, kvHeads, d, pageSize, MemorySegment.NULL,
        DefaultStream): Int)
    )
  }

  /** Attention of one sequence's new tokens over its cache, their own keys
    * and values written to it before: token t at position start + t sees the
    * positions up to its own, or with `window` those of it.
    */
  def attention(queries: Tensor, cache: KvCache, pageTable: Tensor, start: Int, scale: Float, out: Tensor,
                window: Option[AttentionWindow], workspace: Tensor): Unit =
    attend("attention", queries, paged(cache), Left((pageTable, start)), scale, out, window, workspace)
  def attention(queries: Tensor, cache: QuantizedKvCache, pageTable: Tensor, start: Int, scale: Float, out: Tensor,
                window: Option[AttentionWindow], workspace: Tensor): Unit =
    attend("attention", queries, paged(cache), Left((pageTable, start)), scale, out, window, workspace)

  def attentionSequences(queries: Tensor, cache: KvCache, sequences: Sequences, scale: Float, out: Tensor,
                         window: Option[AttentionWindow], workspace: Tensor): Unit =
    attend("attentionSequences", queries, paged(cache), Right(sequences), scale, out, window, workspace)
  def attentionSequences(queries: Tensor, cache: QuantizedKvCache, sequences: Sequences, scale: Float, out: Tensor,
                         window: Option[AttentionWindow], workspace: Tensor): Unit =
    attend("attentionSequences", queries, paged(cache), Right(sequences), scale, out, window, workspace)

  private def attend(operation: String, queries: Tensor, cache: Paged, where: Either[(Tensor, Int), Sequences],
                     scale: Float, out: Tensor, window: Option[AttentionWindow], workspace: Tensor): Unit = {
    Ops.checkElementwise(operation, queries, out)
    require(queries.shape.rank == 3, s"$operation takes [tokens, heads, headDimension], got ${queries.shape}")
    val (tokens, heads) = (queries.shape.dimensions(0).toInt, queries.shape.dimensions(1).toInt)
    require(queries.shape.last == cache.headDimension && cache.kvHeads > 0 && heads > 0 && heads % cache.kvHeads == 0,
      s"$operation: queries ${queries.shape} over a cache of ${cache.kvHeads} heads of ${cache.headDimension}")
    val rows = rowsOf(operation, cache, tokens, where)
    val (tablePages: Int, pages: Int, count: Int, start: Int) = (rows.tablePages, cache.pages, rows.count, rows.start)
    val (kvHeads: Int, d: Int, pageSize: Int) = (cache.kvHeads, cache.headDimension, cache.pageSize)
    val (positions: Int, sinks: Int) = window.fold((0, 0))(w => (w.positions, w.sinks))
    val longest: Int = rows.longest
    val workspaceBytes: Long = workspace.byteSize
    downcall(entry("drift_paged_attention", queries))(
      (drift.pagedAttention(bf16(queries)).invokeExact(pointer(queries), pointer(cache.keys), pointer(cache.values),
        optional(cache.keyScales), optional(cache.valueScales), pointer(rows.tables), tablePages, pages,
        optional(rows.starts), optional(rows.offsets), count, start, tokens, heads, kvHeads, d, pageSize, scale,
        positions, sinks, longest, pointer(out), pointer(workspace), workspaceBytes, MemorySegment.NULL,
        DefaultStream): Int)
    )
  }

  /** Attention of trees of drafted tokens: as `attentionSequences`, but of its
    * sequence's new rows a row sees those that `sees` names (I32 `[tokens,
    * words]`, bit b of word w: row 32 w + b), and every position before them.
    */
  def attentionTree(queries: Tensor, cache: KvCache, sequences: Sequences, sees: Tensor, scale: Float, out: Tensor,
                    window: Option[AttentionWindow], workspace: Tensor): Unit =
    attendTree(queries, paged(cache), sequences, sees, scale, out, window, workspace)
  def attentionTree(queries: Tensor, cache: QuantizedKvCache, sequences: Sequences, sees: Tensor, scale: Float,
                    out: Tensor, window: Option[AttentionWindow], workspace: Tensor): Unit =
    attendTree(queries, paged(cache), sequences, sees, scale, out, window, workspace)

  private def checkQueries(operation: String, queries: Tensor, cache: Paged): (Int, Int) = {
    require(queries.shape.rank == 3, s"$operation takes [tokens, heads, headDimension], got ${queries.shape}")
    val (tokens, heads) = (queries.shape.dimensions(0).toInt, queries.shape.dimensions(1).toInt)
    require(queries.shape.last == cache.headDimension && cache.kvHeads > 0 && heads > 0 && heads % cache.kvHeads == 0,
      s"$operation: queries ${queries.shape} over a cache of ${cache.kvHeads} heads of ${cache.headDimension}")
    (tokens, heads)
  }

  private def attendTree(queries: Tensor, cache: Paged, sequences: Sequences, sees: Tensor, scale: Float, out: Tensor,
                         window: Option[AttentionWindow], workspace: Tensor): Unit = {
    Ops.checkElementwise("attentionTree", queries, out)
    val (tokens: Int, heads: Int) = checkQueries("attentionTree", queries, cache)
    require(sees.dtype == DType.I32 && sees.shape.rank == 2 && sees.shape.dimensions.head == tokens && sees.shape.last > 0,
      s"attentionTree: what the rows see is I32 [$tokens, words], not ${sees.dtype} ${sees.shape}")
    val words: Int = sees.shape.last.toInt
    val rows = rowsOf("attentionTree", cache, tokens, Right(sequences))
    val (tablePages: Int, pages: Int, count: Int, start: Int) = (rows.tablePages, cache.pages, rows.count, rows.start)
    val (kvHeads: Int, d: Int, pageSize: Int) = (cache.kvHeads, cache.headDimension, cache.pageSize)
    val (positions: Int, sinks: Int) = window.fold((0, 0))(w => (w.positions, w.sinks))
    val longest: Int = rows.longest
    val workspaceBytes: Long = workspace.byteSize
    downcall(entry("drift_tree_attention", queries))(
      (drift.treeAttention(bf16(queries)).invokeExact(pointer(queries), pointer(cache.keys), pointer(cache.values),
        optional(cache.keyScales), optional(cache.valueScales), pointer(rows.tables), tablePages, pages,
        optional(rows.starts), optional(rows.offsets), count, start, tokens, heads, kvHeads, d, pageSize, scale,
        positions, sinks, longest, pointer(sees), words, pointer(out), pointer(workspace), workspaceBytes,
        MemorySegment.NULL, DefaultStream): Int)
    )
  }

  private def checkMass(operation: String, mass: Tensor, cache: Paged): Unit = {
    Ops.requireF32(operation, mass)
    require(mass.shape == Shape.of(cache.pages.toLong, cache.kvHeads.toLong, cache.pageSize.toLong),
      s"$operation: masses ${mass.shape} for a cache ${cache.keys.shape}")
  }

  /** What the rows' attention weighs each position of their sequences, into
    * mass F32 `[pages, kvHeads, pageSize]`, added to `before` (which may be
    * mass) where the position precedes the rows.
    */
  def attentionMass(queries: Tensor, cache: KvCache, sequences: Sequences, scale: Float, mass: Tensor,
                    before: Option[Tensor], workspace: Tensor): Unit =
    gatherMass(queries, paged(cache), sequences, scale, mass, before, workspace)
  def attentionMass(queries: Tensor, cache: QuantizedKvCache, sequences: Sequences, scale: Float, mass: Tensor,
                    before: Option[Tensor], workspace: Tensor): Unit =
    gatherMass(queries, paged(cache), sequences, scale, mass, before, workspace)

  private def gatherMass(queries: Tensor, cache: Paged, sequences: Sequences, scale: Float, mass: Tensor,
                         before: Option[Tensor], workspace: Tensor): Unit = {
    Ops.checkElementwise("attentionMass", queries)
    val (tokens: Int, heads: Int) = checkQueries("attentionMass", queries, cache)
    checkMass("attentionMass", mass, cache)
    before.foreach(b => checkMass("attentionMass", b, cache))
    val rows = rowsOf("attentionMass", cache, tokens, Right(sequences))
    val (tablePages: Int, pages: Int, count: Int, start: Int) = (rows.tablePages, cache.pages, rows.count, rows.start)
    val (kvHeads: Int, d: Int, pageSize: Int) = (cache.kvHeads, cache.headDimension, cache.pageSize)
    val longest: Int = rows.longest
    val workspaceBytes: Long = workspace.byteSize
    downcall(entry("drift_attention_mass", queries))(
      (drift.attentionMass(bf16(queries)).invokeExact(pointer(queries), pointer(cache.keys), optional(cache.keyScales),
        pointer(rows.tables), tablePages, pages, optional(rows.starts), optional(rows.offsets), count, start, tokens,
        heads, kvHeads, d, pageSize, scale, longest, optional(before), pointer(mass), pointer(workspace),
        workspaceBytes, MemorySegment.NULL, DefaultStream): Int)
    )
  }

  /** The positions to keep, ascending, into kept I32 `[sequences, kvHeads,
    * keep]`: of a sequence of lengths[s] > keep positions the first `sinks`, the
    * last `recent` and the heaviest between, of a shorter one all; -1 past
    * counts[s].
    */
  def heaviest(mass: Tensor, pageTables: Tensor, lengths: Tensor, sinks: Int, recent: Int, kept: Tensor,
               counts: Tensor): Unit = {
    Ops.requireF32("heaviest", mass)
    require(mass.shape.rank == 3, s"heaviest: masses are [pages, kvHeads, pageSize], got ${mass.shape}")
    require(pageTables.dtype == DType.I32 && pageTables.shape.rank == 2,
      s"heaviest: page tables are I32 [sequences, pages], not ${pageTables.dtype} ${pageTables.shape}")
    val count: Int = pageTables.shape.dimensions.head.toInt
    Seq(lengths, counts).foreach { v =>
      require(v.dtype == DType.I32 && v.shape == Shape.of(count.toLong),
        s"heaviest: lengths or counts ${v.dtype} ${v.shape} for $count sequences")
    }
    val (pages: Int, kvHeads: Int, pageSize: Int) =
      (mass.shape.dimensions(0).toInt, mass.shape.dimensions(1).toInt, mass.shape.last.toInt)
    require(kept.dtype == DType.I32 && kept.shape.rank == 3 &&
      kept.shape.dimensions.take(2) == Seq(count.toLong, kvHeads.toLong),
      s"heaviest: kept ${kept.dtype} ${kept.shape} for $count sequences of $kvHeads heads")
    val (tablePages: Int, keep: Int) = (pageTables.shape.last.toInt, kept.shape.last.toInt)
    require(sinks >= 0 && recent >= 0 && sinks.toLong + recent <= keep,
      s"heaviest: the first $sinks and the last $recent positions of $keep kept")
    downcall("drift_heaviest")(
      (drift.heaviest.invokeExact(pointer(mass), pointer(pageTables), tablePages, pages, pointer(lengths), count,
        kvHeads, pageSize, sinks, recent, keep, pointer(kept), pointer(counts), MemorySegment.NULL,
        DefaultStream): Int)
    )
  }

  /** The kept rows moved together, all read before any is written; `mass` moves
    * with them. `workspace`: `keepWorkspace`'s bytes (none with rows.into).
    */
  def cacheKeep(cache: KvCache, rows: KeptRows, mass: Option[Tensor], workspace: Option[Tensor]): Unit =
    moveRows(paged(cache), rows, mass, workspace)
  def cacheKeep(cache: QuantizedKvCache, rows: KeptRows, mass: Option[Tensor], workspace: Option[Tensor]): Unit =
    moveRows(paged(cache), rows, mass, workspace)

  private def moveRows(cache: Paged, rows: KeptRows, mass: Option[Tensor], workspace: Option[Tensor]): Unit = {
    require(rows.kept.shape.rank == 2 || rows.kept.shape.dimensions(1) == cache.kvHeads.toLong,
      s"cacheKeep: kept ${rows.kept.shape} for ${cache.kvHeads} heads")
    mass.foreach(m => checkMass("cacheKeep", m, cache))
    val count: Int = rows.kept.shape.dimensions.head.toInt
    val most: Int = rows.kept.shape.last.toInt
    val keptHeads: Int = if (rows.kept.shape.rank == 3) cache.kvHeads else 1
    val tablePages: Int = rows.pageTables.shape.last.toInt
    val intoPages: Int = rows.into.fold(0)(_.shape.last.toInt)
    val (pages: Int, kvHeads: Int, d: Int, pageSize: Int) =
      (cache.pages, cache.kvHeads, cache.headDimension, cache.pageSize)
    val workspaceBytes: Long = workspace.fold(0L)(_.byteSize)
    downcall("drift_cache_keep")(
      (drift.cacheKeep.invokeExact(pointer(cache.keys), pointer(cache.values), optional(cache.keyScales),
        optional(cache.valueScales), optional(mass), pointer(rows.pageTables), tablePages, optional(rows.into),
        intoPages, pages, pointer(rows.kept), keptHeads, optional(rows.counts), optional(rows.starts), count, most,
        kvHeads, d, pageSize, optional(workspace), workspaceBytes, MemorySegment.NULL, DefaultStream): Int)
    )
  }
}
