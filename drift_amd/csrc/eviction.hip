// Which positions of a sequence its paged cache keeps, and the move of the
// kept ones (paged.hpp has the cache's layouts): `heaviest` chooses by the
// attention that positions have gathered (attention_mass.hip), `cache_keep`
// moves any chosen rows together, an accepted path of drafted tokens' among
// them.
#include "paged.hpp"

#include <algorithm>
#include <initializer_list>

namespace drift {
namespace {

// ------------------------------------------------------------------ the heaviest

struct HeaviestArgs {
  const float* mass;
  const int32_t *tables, *lengths;
  int32_t sequences, table_pages, cache_pages, page_size, kv_heads, sinks, recent, keep;
  int32_t *kept, *counts, *bad_page;
  UnitColumns columns;
};

// Masses as whole numbers in their order: 0 and -0 are one, a NaN is above every number, and 0 is
// below them all.
__device__ __forceinline__ uint32_t order_of(float mass) {
  const float x = mass + 0.0f;
  const uint32_t bits = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  return bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
}

constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / kWave, kBins = 2048;

// One block a sequence and key head. The `wanted` heaviest of its candidates (the
// positions between the first `sinks` and the last `recent`) are those above a
// threshold, the wanted-th largest order, and as many equal to it as are left, the
// lowest first. Three passes over the orders' digits of 11, 11 and 10 bits find it,
// each by a histogram in LDS of the candidates that share the digits so far; two more
// write the positions in their order, by counts of the waves before and ballots.
// EACH: the candidates a lane keeps in registers, up to 32; 0: more, read again in each pass (us, 16 sequences of 8
// heads, kept / read again: 1,500 positions 9 / 23, 7,000 13 / 31, 14,000 20 / 35, 30,000 42 / 67). The launch takes it
// by what the page tables have room for: 7,000 positions in tables for 32,768 20 us, for more 21 to 32.
//
// The passes over the orders with their additions in LDS bound it, not memory: 48 sequences of up to 16,000 positions, 8
// heads, 31 us for 22 MB in 384 blocks, two a compute unit (vector instructions issue 36% of the time).
template <int EACH>
__global__ void __launch_bounds__(kPickThreads, EACH > 0 && EACH <= 16 ? 8 : 4) pick_heaviest(HeaviestArgs a) {
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t sums[2][kPickWaves];
  __shared__ uint32_t found[3];
  const int thread = threadIdx.x, lane = thread & (kWave - 1), wave = uniform(thread / kWave);
  const int s = blockIdx.x / (unsigned)a.kv_heads, kv = blockIdx.x % (unsigned)a.kv_heads;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.keep;
  int64_t length = a.lengths[s];
  if (length < 0 || length > min((int64_t)a.table_pages * a.page_size, kMostPositions)) {
    if (a.bad_page) *a.bad_page = 1;
    length = 0;
  }
  if (kv == 0 && thread == 0) a.counts[s] = (int32_t)min(length, (int64_t)a.keep);
  if (length <= a.keep) {
    for (int64_t i = thread; i < a.keep; i += kPickThreads) kept[i] = i < length ? (int32_t)i : -1;
    return;
  }
  for (int i = thread; i < a.sinks; i += kPickThreads) kept[i] = i;
  for (int i = thread; i < a.recent; i += kPickThreads) kept[a.keep - a.recent + i] = (int32_t)(length - a.recent + i);
  const uint32_t wanted = a.keep - a.sinks - a.recent;
  if (wanted == 0) return;
  const uint32_t candidates = (uint32_t)(length - a.sinks - a.recent);  // more than are wanted
  const int32_t* table = a.tables + (int64_t)s * a.table_pages;
  auto column_of = [&](uint32_t candidate) { return a.columns.of((candidate + a.sinks) / 16); };
  auto order_at = [&](uint32_t candidate, int32_t page) -> uint32_t {
    if (page < 0 || page >= a.cache_pages) {
      if (a.bad_page) *a.bad_page = 1;
      return 0;
    }
    const uint32_t j = candidate + a.sinks, off = j - column_of(candidate) * a.columns.page_units * 16;
    return order_of(a.mass[((int64_t)page * a.kv_heads + kv) * a.page_size + off]);
  };
  // a wave's candidates lie together, a lane has every 64th of them: their places then follow from the waves' before
  const uint32_t each = (candidates + kPickThreads - 1) / kPickThreads;  // of a lane
  const uint32_t begin = min(wave * each * kWave, candidates), end = min(begin + each * kWave, candidates);
  uint32_t kept_order[EACH > 0 ? EACH : 1];
  if constexpr (EACH > 0) {
    int32_t page[EACH];
#pragma unroll
    for (int n = 0; n < EACH; ++n)
      page[n] = begin + n * kWave + lane < end ? table[column_of(begin + n * kWave + lane)] : 0;
#pragma unroll
    for (int n = 0; n < EACH; ++n)
      kept_order[n] = begin + n * kWave + lane < end ? order_at(begin + n * kWave + lane, page[n]) : 0;
  }
  // `take` with each of the lane's orders, and whether there is one; whole waves
  auto for_each = [&](auto take) {
    if constexpr (EACH > 0) {
#pragma unroll
      for (int n = 0; n < EACH; ++n) {
        const uint32_t i = begin + n * kWave;
        if (i < end) take(i + lane, i + lane < end, kept_order[n]);
      }
    } else {
      constexpr int kAhead = 16;  // on their way together
      for (uint32_t i = begin; i < end; i += kAhead * kWave) {
        int32_t page[kAhead];
        uint32_t order[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) page[n] = table[column_of(min(i + n * kWave + lane, end - 1))];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) order[n] = order_at(min(i + n * kWave + lane, end - 1), page[n]);
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
          if (i + n * kWave < end) take(i + n * kWave + lane, i + n * kWave + lane < end, order[n]);
      }
    }
  };

  uint32_t digits = 0, known = 0, left = wanted;  // the threshold's digits so far, and how many are wanted of those that share them
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 1024 : 2048;
    for (int i = thread; i < kBins; i += kPickThreads) bins[i] = 0;
    __syncthreads();
    for_each([&](uint32_t, bool in, uint32_t order) {
      const bool counts = in && (order & known) == digits;
      const uint32_t bin = order >> shift & (width - 1);
      // (equal masses, as before the first call, are one addition a wave)
      if (__all(counts && bin == uniform(bin))) {
        if (lane == 0) atomicAdd(&bins[bin], (uint32_t)kWave);
      } else if (counts) {
        atomicAdd(&bins[bin], 1u);
      }
    });
    __syncthreads();
    // a thread's two bins, the highest first; those above them
    const int bin = kBins - 2 - 2 * thread;
    const uint32_t high = bins[bin + 1], low = bins[bin];
    uint32_t upto = high + low;
#pragma unroll
    for (int step = 1; step < kWave; step <<= 1) {
      const uint32_t before = __shfl_up(upto, step, kWave);
      if (lane >= step) upto += before;
    }
    if (lane == kWave - 1) sums[0][wave] = upto;
    __syncthreads();
    uint32_t above = upto - high - low;
    for (int w = 0; w < wave; ++w) above += sums[0][w];
    if (above < left && left <= above + high) found[0] = bin + 1, found[1] = above, found[2] = high;
    else if (above + high < left && left <= above + high + low) found[0] = bin, found[1] = above + high, found[2] = low;
    __syncthreads();
    digits |= found[0] << shift;
    known |= (uint32_t)(width - 1) << shift;
    left -= found[1];
    const bool all_taken = found[2] == left;
    __syncthreads();
    if (all_taken) break;  // (every candidate that shares the digits: those with more digits are all taken)
  }

  // above the threshold, or (left of them, the lowest first) sharing its digits
  uint32_t more = 0, equal = 0;
  for_each([&](uint32_t, bool in, uint32_t order) {
    more += __popcll(__ballot(in && (order & known) > digits));
    equal += __popcll(__ballot(in && (order & known) == digits));
  });
  if (lane == 0) sums[0][wave] = more, sums[1][wave] = equal;
  __syncthreads();
  uint32_t more_before = 0, equal_before = 0;
  for (int w = 0; w < wave; ++w) more_before += sums[0][w], equal_before += sums[1][w];
  uint32_t place = a.sinks + more_before + min(equal_before, left);
  const uint64_t below = (1ull << lane) - 1;
  for_each([&](uint32_t i, bool in, uint32_t order) {
    const bool tie = in && (order & known) == digits;
    const uint64_t ties = __ballot(tie);
    const bool taken = (in && (order & known) > digits) || (tie && equal_before + __popcll(ties & below) < left);
    const uint64_t all = __ballot(taken);
    if (taken) kept[place + __popcll(all & below)] = (int32_t)(i + a.sinks);
    place += __popcll(all);
    equal_before += __popcll(ties);
  });
}

// ------------------------------------------------------------------ the kept rows' move

struct KeepArgs {
  void *keys, *values;
  float *key_scales, *value_scales, *mass;
  const int32_t *tables, *into, *kept, *counts, *starts;
  int32_t sequences, table_pages, into_pages, cache_pages, page_size, kept_heads, most, kv_heads, dim;
  char* scratch;
  int32_t* bad_page;
};

// Row i of a sequence's and key head's kept ones: where it lies and where it goes.
struct Move {
  int64_t from_page, from_off, to_page, to_off;
  bool good;
};

__device__ __forceinline__ bool place_of(const KeepArgs& a, const int32_t* table, int32_t columns, int64_t position,
                                         int64_t& page, int64_t& off) {
  if (position < 0 || position >= (int64_t)columns * a.page_size) return false;
  page = table[position / a.page_size];
  off = position % a.page_size;
  return page >= 0 && page < a.cache_pages;
}

__device__ __forceinline__ Move move_of(const KeepArgs& a, int s, int kv, int i) {
  Move m;
  const int32_t count = a.counts ? a.counts[s] : a.most, start = a.starts ? a.starts[s] : 0;
  m.good = count >= 0 && count <= a.most && start >= 0;
  if (!m.good) {
    if (a.bad_page) *a.bad_page = 1;
    return m;
  }
  m.good = i < count;
  if (!m.good) return m;
  const int32_t from = a.kept[((int64_t)s * a.kept_heads + (a.kept_heads == 1 ? 0 : kv)) * a.most + i];
  m.good = place_of(a, a.tables + (int64_t)s * a.table_pages, a.table_pages, from, m.from_page, m.from_off) &&
           place_of(a, a.into + (int64_t)s * a.into_pages, a.into_pages, (int64_t)start + i, m.to_page, m.to_off);
  if (!m.good && a.bad_page) *a.bad_page = 1;
  return m;
}

// What no chunks are made for (heads of 512 in F16, of odd sizes, tensors off 16-byte alignment): a wave a row, 1,024 of
// 4,000 rows of 16 sequences, 4 heads of 512, in place 277 us (537 MB moved twice, 3.9 TB/s), of 20 values 61.
// READ: from the cache, else from the scratch; WRITE: to the cache, else to the
// scratch, which has a row's keys, values, scales and mass one after another.
template <typename E, bool READ, bool WRITE>
__global__ void __launch_bounds__(256) move_rows(KeepArgs a, int64_t rows, int64_t row_bytes) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (row >= rows) return;
  const int i = (int)(row % a.most), kv = (int)(row / a.most % a.kv_heads), s = (int)(row / a.most / a.kv_heads);
  const Move m = move_of(a, s, kv, i);
  if (!m.good) return;
  E* const keys = (E*)a.keys;
  E* const values = (E*)a.values;
  E* const scratch = (E*)(a.scratch + row * row_bytes);
  for (int d = lane; d < a.dim; d += kWave) {
    const E k = READ ? keys[((m.from_page * a.page_size + m.from_off) * a.kv_heads + kv) * a.dim + d] : scratch[d];
    const E v = READ ? values[((m.from_page * a.kv_heads + kv) * a.dim + d) * a.page_size + m.from_off]
                     : scratch[a.dim + d];
    if (WRITE) {
      keys[((m.to_page * a.page_size + m.to_off) * a.kv_heads + kv) * a.dim + d] = k;
      values[((m.to_page * a.kv_heads + kv) * a.dim + d) * a.page_size + m.to_off] = v;
    } else {
      scratch[d] = k;
      scratch[a.dim + d] = v;
    }
  }
  float* const words = (float*)(a.scratch + row * row_bytes + row_bytes - 12);
  float* const of[3] = {a.key_scales, a.value_scales, a.mass};
  if (lane < 3 && of[lane]) {
    const int64_t at = (m.from_page * a.kv_heads + kv) * a.page_size + m.from_off;
    const float x = READ ? of[lane][at] : words[lane];
    if (WRITE) of[lane][(m.to_page * a.kv_heads + kv) * a.page_size + m.to_off] = x;
    else words[lane] = x;
  }
}

// Rows in chunks of 128 by a block: a block has a sequence's and key head's keys with
// their words (scales and masses), or 64 dimensions of its values, which share
// nothing; the cache's bits pass through registers.
//
// Keys go row by row in pieces of PIECE bytes. Of values, which lie transposed, a lane has a
// dimension and a wave 32 rows: 16 bytes of neighbouring positions a load, once for the
// rows that lie in them, and 16 rows that go to a whole unit of 16 positions leave in one
// store of a lane (two for F16). So values of rows far apart cost their whole lines.
//
// That bounds it: of 32 sequences of up to 8,000 positions 2,048 kept, 8 heads of 128 in 8 bits, every list its own,
// 129 us for 283 MB of rows read and written; with the lines around the rows it reads 1.7 times their bytes.
//
// In place, what a chunk reads has to be read before another's rows are written over
// it. A block that has a whole list keeps to it chunk by chunk where every row comes from its own place or from
// behind it, or from before all places that rows go to (an ascending list does): later rows' sources are then
// not among the places of earlier ones. Else it puts all rows by first. Where lists are long and few, their chunks
// are blocks of two launches instead, one that puts rows by and one that brings them back.
enum KeepMode { kWalk, kDirect, kPutBy, kBringBack };
constexpr int kKeepRows = 128;

// A chunk's places. A walk has three of them: the next chunk's are made while this one's rows are on
// their way, and a wave that is a chunk behind still finds its own.
struct KeepPlaces {
  int64_t from[kKeepRows], to[kKeepRows], word_from[kKeepRows], word_to[kKeepRows];
  uint64_t moves[2];  // which of its rows move
};

// A list as a block has it.
struct KeepList {
  int s, kv, part;
  int32_t count, start;
  const int32_t *kept, *table, *into;
};

__device__ __forceinline__ void place_rows(const KeepArgs& a, const KeepList& l, int chunk, KeepPlaces& p) {
  const int thread = threadIdx.x;
  if (thread >= kKeepRows) return;
  const int i = chunk * kKeepRows + thread;
  int64_t page = 0, off = 0, its_page = 0, its_off = 0;
  bool good = i < l.count;
  if (good) {
    good = place_of(a, l.table, a.table_pages, l.kept[i], page, off) &&
           place_of(a, l.into, a.into_pages, (int64_t)l.start + i, its_page, its_off);
    if (!good && a.bad_page) *a.bad_page = 1;
  }
  if (!good) page = off = its_page = its_off = 0;
  if (l.part == 0) {
    p.from[thread] = ((page * a.page_size + off) * a.kv_heads + l.kv) * a.dim;
    p.to[thread] = ((its_page * a.page_size + its_off) * a.kv_heads + l.kv) * a.dim;
    p.word_from[thread] = (page * a.kv_heads + l.kv) * a.page_size + off;
    p.word_to[thread] = (its_page * a.kv_heads + l.kv) * a.page_size + its_off;
  } else {
    p.from[thread] = (page * a.kv_heads + l.kv) * a.dim * a.page_size + off;
    p.to[thread] = (its_page * a.kv_heads + l.kv) * a.dim * a.page_size + its_off;
  }
  const uint64_t rows = __ballot(good);
  if (thread % kWave == 0) p.moves[thread / kWave] = rows;
}

// What a thread has of a chunk of keys: its piece of every `step`-th row from `row0` on, and a row's words.
template <typename E, int PIECE, int PIECES>
struct KeyRows {
  static constexpr int kSlots = PIECES * PIECE / 16 + 1;
  typedef uint32_t Piece __attribute__((ext_vector_type(PIECE / 4)));
  Piece piece[PIECES];
  u32x4 words;
  int step, row0, at;

  __device__ __forceinline__ KeyRows(const KeepArgs& a, const KeepList&) {
    const int pieces = a.dim * (int)sizeof(E) / PIECE;
    step = 256 / pieces, row0 = threadIdx.x / pieces, at = (threadIdx.x - row0 * pieces) * PIECE;
    if (row0 >= step) row0 = kKeepRows;  // (a row's last threads, where rows do not divide the block: none)
  }
  __device__ __forceinline__ bool has(const KeepPlaces& p, int n) const {
    const int row = row0 + n * step;
    return row < kKeepRows && (p.moves[row / 64] >> (row % 64) & 1);
  }
  __device__ __forceinline__ void read(const KeepArgs& a, const KeepList&, const KeepPlaces& p) {
#pragma unroll
    for (int n = 0; n < PIECES; ++n)
      if (has(p, n)) piece[n] = *(const Piece*)((const char*)a.keys + p.from[row0 + n * step] * sizeof(E) + at);
    const int row = threadIdx.x;
    if (row < kKeepRows && (p.moves[row / 64] >> (row % 64) & 1)) {
      if (a.key_scales) words[0] = __float_as_uint(a.key_scales[p.word_from[row]]);
      if (a.value_scales) words[1] = __float_as_uint(a.value_scales[p.word_from[row]]);
      if (a.mass) words[2] = __float_as_uint(a.mass[p.word_from[row]]);
    }
  }
  __device__ __forceinline__ void write(const KeepArgs& a, const KeepList&, const KeepPlaces& p) const {
#pragma unroll
    for (int n = 0; n < PIECES; ++n)
      if (has(p, n)) *(Piece*)((char*)a.keys + p.to[row0 + n * step] * sizeof(E) + at) = piece[n];
    const int row = threadIdx.x;
    if (row < kKeepRows && (p.moves[row / 64] >> (row % 64) & 1)) {
      if (a.key_scales) a.key_scales[p.word_to[row]] = __uint_as_float(words[0]);
      if (a.value_scales) a.value_scales[p.word_to[row]] = __uint_as_float(words[1]);
      if (a.mass) a.mass[p.word_to[row]] = __uint_as_float(words[2]);
    }
  }
  __device__ __forceinline__ void put_by(u32x4* slot) const {
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
      if constexpr (PIECE == 16) slot[n * 256] = piece[n];
      else if (n % 2 == 0) slot[n / 2 * 256] = u32x4{piece[n][0], piece[n][1], piece[n + 1][0], piece[n + 1][1]};
    }
    slot[(kSlots - 1) * 256] = words;
  }
  __device__ __forceinline__ void bring_back(const u32x4* slot) {
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
      if constexpr (PIECE == 16) {
        piece[n] = slot[n * 256];
      } else if (n % 2 == 0) {
        const u32x4 x = slot[n / 2 * 256];
        piece[n] = Piece{x[0], x[1]}, piece[n + 1] = Piece{x[2], x[3]};
      }
    }
    words = slot[(kSlots - 1) * 256];
  }
};

// Of values: a dimension of the wave's 32 rows, as two units.
template <typename E>
struct ValueRows {
  static constexpr int kBytes = sizeof(E), kSlots = 2 * kBytes;
  static constexpr int kRun = 16 / kBytes;  // positions a load
  u32x4 unit[2][kBytes];
  int d, row0;

  __device__ __forceinline__ ValueRows(const KeepArgs&, const KeepList& l) {
    d = (l.part - 1) * 64 + (threadIdx.x & (kWave - 1)), row0 = uniform((int)threadIdx.x / kWave) * 32;
  }
  __device__ __forceinline__ void read(const KeepArgs& a, const KeepList&, const KeepPlaces& p) {
    if (d >= a.dim) return;
    const E* const values = (const E*)a.values + (int64_t)d * a.page_size;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // (places and dimensions are multiples of 16 positions but for `off`, so that a run lies at a multiple of its size)
      int64_t from[16];
      u32x4 run[16], now = {0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        from[n] = uniform(p.from[row0 + u * 16 + n]);
        if (n == 0 || from[n] / kRun != from[n - 1] / kRun) run[n] = *(const u32x4*)(values + from[n] / kRun * kRun);
      }
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        if (n == 0 || from[n] / kRun != from[n - 1] / kRun) now = run[n];
        const int in = (int)(from[n] % kRun) * kBytes;  // bytes
        const uint32_t low = in & 4 ? now[1] : now[0], high = in & 4 ? now[3] : now[2];
        const uint32_t x = (in & 8 ? high : low) >> (in % 4 * 8) & (kBytes == 1 ? 0xffu : 0xffffu);
        const int to = n * kBytes;
        if (to % 4 == 0) unit[u][to / 16][to % 16 / 4] = x;
        else unit[u][to / 16][to % 16 / 4] |= x << (to % 4 * 8);
      }
    }
  }
  __device__ __forceinline__ void write(const KeepArgs& a, const KeepList& l, const KeepPlaces& p) const {
    if (d >= a.dim) return;
    E* const values = (E*)a.values + (int64_t)d * a.page_size;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int first = row0 + u * 16;
      const uint32_t moving = uniform((uint32_t)(p.moves[first / 64] >> (first % 64)) & 0xffffu);
      if (moving == 0) continue;
      if (l.start % 16 == 0 && moving == 0xffffu) {
        u32x4* const to = (u32x4*)(values + uniform(p.to[first]));
#pragma unroll
        for (int n = 0; n < kBytes; ++n) to[n] = unit[u][n];
      } else {
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (moving >> n & 1)
            values[uniform(p.to[first + n])] = (E)(unit[u][n * kBytes / 16][n * kBytes % 16 / 4] >> (n * kBytes % 4 * 8));
      }
    }
  }
  __device__ __forceinline__ void put_by(u32x4* slot) const {
#pragma unroll
    for (int n = 0; n < kSlots; ++n) slot[n * 256] = unit[n / kBytes][n % kBytes];
  }
  __device__ __forceinline__ void bring_back(const u32x4* slot) {
#pragma unroll
    for (int n = 0; n < kSlots; ++n) unit[n / kBytes][n % kBytes] = slot[n * 256];
  }
};

// `slots`: 16-byte places that a thread has in the workspace for a chunk.
template <typename Rows, int MODE>
__device__ __forceinline__ void keep_part(const KeepArgs& a, const KeepList& l, unsigned list, int chunk, int chunks,
                                          int slots, KeepPlaces* sets) {
  Rows rows(a, l);
  auto slot_of = [&](int chunk) { return (u32x4*)a.scratch + (((int64_t)list * chunks + chunk) * slots * 256 + threadIdx.x); };
  if constexpr (MODE != kWalk) {
    if (chunk * kKeepRows >= l.count) return;
    place_rows(a, l, chunk, sets[0]);
    __syncthreads();
    if (MODE == kBringBack) rows.bring_back(slot_of(chunk));
    else rows.read(a, l, sets[0]);
    if (MODE == kPutBy) rows.put_by(slot_of(chunk));
    else rows.write(a, l, sets[0]);
  } else {
    const int all = (l.count + kKeepRows - 1) / kKeepRows;
    if (all == 0) return;
    place_rows(a, l, 0, sets[0]);
    bool by_place = true;
    if (all > 1)
      for (int i = threadIdx.x; i < l.count; i += 256) by_place &= l.kept[i] >= (int64_t)l.start + i || l.kept[i] < l.start;
    if (__syncthreads_and(by_place)) {
      for (int i = 0; i < all; ++i) {
        const KeepPlaces& p = sets[i % 3];
        rows.read(a, l, p);
        if (i + 1 < all) place_rows(a, l, i + 1, sets[(i + 1) % 3]);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's rows have come
        __syncthreads();
        rows.write(a, l, p);
      }
      return;
    }
    for (int back = 0; back < 2; ++back)
      for (int i = 0; i < all; ++i) {
        __syncthreads();
        place_rows(a, l, i, sets[0]);
        __syncthreads();
        if (back) {
          rows.bring_back(slot_of(i));
          rows.write(a, l, sets[0]);
        } else {
          rows.read(a, l, sets[0]);
          rows.put_by(slot_of(i));
        }
      }
  }
}

template <typename E, int PIECE, int PIECES>
constexpr int kKeepSlots = KeyRows<E, PIECE, PIECES>::kSlots > ValueRows<E>::kSlots ? KeyRows<E, PIECE, PIECES>::kSlots
                                                                                    : ValueRows<E>::kSlots;

template <typename E, int PIECE, int PIECES, int MODE>
__global__ void __launch_bounds__(256) keep_rows(KeepArgs a, int chunks) {
  __shared__ KeepPlaces sets[MODE == kWalk ? 3 : 1];
  const int parts = 1 + (a.dim + 63) / 64;
  const unsigned list = MODE == kWalk ? blockIdx.x : blockIdx.x / (unsigned)chunks;
  const int chunk = MODE == kWalk ? 0 : blockIdx.x % (unsigned)chunks;
  KeepList l;
  l.kv = list % (unsigned)a.kv_heads, l.part = list / (unsigned)a.kv_heads % (unsigned)parts;
  l.s = list / (unsigned)a.kv_heads / (unsigned)parts;
  l.count = a.counts ? uniform(a.counts[l.s]) : a.most, l.start = a.starts ? uniform(a.starts[l.s]) : 0;
  if (l.count < 0 || l.count > a.most || l.start < 0) {
    if (a.bad_page) *a.bad_page = 1;
    return;
  }
  l.kept = a.kept + ((int64_t)l.s * a.kept_heads + (a.kept_heads == 1 ? 0 : l.kv)) * a.most;
  l.table = a.tables + (int64_t)l.s * a.table_pages, l.into = a.into + (int64_t)l.s * a.into_pages;
  constexpr int kSlots = kKeepSlots<E, PIECE, PIECES>;
  if (l.part == 0) keep_part<KeyRows<E, PIECE, PIECES>, MODE>(a, l, list, chunk, chunks, kSlots, sets);
  else keep_part<ValueRows<E>, MODE>(a, l, list, chunk, chunks, kSlots, sets);
}

// Bytes of scratch of a row that is put by on its own (move_rows).
int64_t scratch_row(int32_t dim, bool quantized) { return ceil_div((int64_t)dim * 2 * (quantized ? 1 : 2), 4) * 4 + 12; }

int check_keep(const char* entry, int32_t sequences, int32_t most, int32_t kv_heads, int32_t dim) {
  if (sequences < 0 || most < 0 || kv_heads <= 0 || dim <= 0)
    return refuse("%s: %d rows of %d sequences, %d heads of %d values", entry, most, sequences, kv_heads, dim);
  if ((int64_t)sequences * kv_heads > kOneWaveBlocks || (int64_t)sequences * kv_heads * most > kOneWaveBlocks * 4)
    return refuse("%s: %d rows of %d sequences, %d heads in one call", entry, most, sequences, kv_heads);
  return 0;
}

// Pieces of keys that a thread has of a chunk; 0: none that the kernel is made for.
int pieces_of(int32_t dim, bool quantized, int& piece) {
  const int64_t bytes = (int64_t)dim * (quantized ? 1 : 2);
  piece = bytes % 16 == 0 ? 16 : 8;
  if (bytes % piece != 0 || (piece == 8 && !quantized) || bytes / piece > 256) return 0;
  const int64_t pieces = ceil_div(kKeepRows, 256 / (bytes / piece));
  return pieces <= 4 ? 4 : pieces <= 8 ? 8 : pieces <= 16 ? 16 : 0;
}

// Bytes of scratch of a call in place, whichever way it goes: a row each (where the tensors' alignment asks for
// move_rows), or a thread's slots of every chunk.
int64_t keep_bytes(int32_t sequences, int32_t most, int32_t kv_heads, int32_t dim, bool quantized) {
  const int64_t by_rows = (int64_t)sequences * most * kv_heads * scratch_row(dim, quantized);
  int piece;
  const int pieces = pieces_of(dim, quantized, piece), slots = std::max(pieces * piece / 16 + 1, quantized ? 2 : 4);
  // a list of one chunk is read whole before it is written, and by chunks puts nothing by
  if (pieces == 0 || most <= kKeepRows) return ceil_div(by_rows, 16) * 16;
  const int64_t by_chunks = (int64_t)sequences * kv_heads * (1 + ceil_div(dim, 64)) * ceil_div(most, kKeepRows) *
                            slots * 256 * 16;
  return ceil_div(std::max(by_rows, by_chunks), 16) * 16;
}

template <typename E, int PIECE, int PIECES>
int keep_chunks(const char* entry, const KeepArgs& a, bool apart, hipStream_t st) {
  const int chunks = (int)ceil_div(a.most, kKeepRows);
  const int64_t lists = (int64_t)a.sequences * a.kv_heads * (1 + ceil_div(a.dim, 64));
  const dim3 block(256), each((unsigned)(lists * chunks)), walk((unsigned)lists);
  if (apart || chunks == 1) {
    if (chunks == 1) hipLaunchKernelGGL((keep_rows<E, PIECE, PIECES, kWalk>), walk, block, 0, st, a, chunks);
    else hipLaunchKernelGGL((keep_rows<E, PIECE, PIECES, kDirect>), each, block, 0, st, a, chunks);
    return launched(entry);
  }
  // (16 sequences of 8 heads of 128, 384 lists of 4,096 rows, 255 us one way and 277 the other, of 500 31 and 36; 8
  // sequences, 192 lists, 200 and 140; one, 24 lists, 178 and 27)
  if (lists >= 256) {
    hipLaunchKernelGGL((keep_rows<E, PIECE, PIECES, kWalk>), walk, block, 0, st, a, chunks);
    return launched(entry);
  }
  hipLaunchKernelGGL((keep_rows<E, PIECE, PIECES, kPutBy>), each, block, 0, st, a, chunks);
  if (const int bad = launched(entry)) return bad;
  hipLaunchKernelGGL((keep_rows<E, PIECE, PIECES, kBringBack>), each, block, 0, st, a, chunks);
  return launched(entry);
}

template <typename E>
int keep(const char* entry, const KeepArgs& a, bool apart, hipStream_t st) {
  int piece;
  const int pieces = pieces_of(a.dim, sizeof(E) == 1, piece);
  const int64_t blocks = (int64_t)a.sequences * a.kv_heads * (1 + ceil_div(a.dim, 64)) * ceil_div(a.most, kKeepRows);
  if (pieces > 0 && a.cache_pages > 0 && blocks <= kOneWaveBlocks / 4 && aligned16(a.keys) && aligned16(a.values)) {
#define DRIFT_KEEP(PIECE, PIECES) \
  if (piece == PIECE && pieces == PIECES) return keep_chunks<E, PIECE, PIECES>(entry, a, apart, st);
    DRIFT_KEEP(16, 4)
    DRIFT_KEEP(16, 8)
    DRIFT_KEEP(16, 16)
    if constexpr (sizeof(E) == 1) {
      DRIFT_KEEP(8, 4)
      DRIFT_KEEP(8, 8)
      DRIFT_KEEP(8, 16)
    }
#undef DRIFT_KEEP
  }
  const int64_t rows = (int64_t)a.sequences * a.kv_heads * a.most, row_bytes = scratch_row(a.dim, sizeof(E) == 1);
  const dim3 grid((unsigned)ceil_div(rows, 4)), block(256);
  if (apart) {
    hipLaunchKernelGGL((move_rows<E, true, true>), grid, block, 0, st, a, rows, row_bytes);
    return launched(entry);
  }
  hipLaunchKernelGGL((move_rows<E, true, false>), grid, block, 0, st, a, rows, row_bytes);
  if (const int bad = launched(entry)) return bad;
  hipLaunchKernelGGL((move_rows<E, false, true>), grid, block, 0, st, a, rows, row_bytes);
  return launched(entry);
}

bool words_aligned(std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
  return (all & 3) == 0;
}

}  // namespace
}  // namespace drift

using namespace drift;

extern "C" int drift_heaviest(const float* mass, const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                              const int32_t* lengths, int32_t sequences, int32_t kv_heads, int32_t page_size,
                              int32_t sinks, int32_t recent, int32_t keep, int32_t* kept, int32_t* counts,
                              int32_t* bad_page, void* stream) {
  const char* entry = "drift_heaviest";
  clear_error();
  if (sequences < 0 || table_pages < 0 || cache_pages < 0 || kv_heads <= 0)
    return refuse("%s: %d sequences, %d table pages, %d cache pages, %d heads", entry, sequences, table_pages,
                  cache_pages, kv_heads);
  if (page_size <= 0 || page_size % 16 != 0)
    return refuse("%s: pages of %d tokens: not a multiple of 16", entry, page_size);
  if (sinks < 0 || recent < 0 || keep < 0 || (int64_t)sinks + recent > keep)
    return refuse("%s: the first %d and the last %d positions of %d kept", entry, sinks, recent, keep);
  if ((int64_t)sequences * kv_heads > kOneWaveBlocks / kPickWaves)
    return refuse("%s: %d sequences of %d heads in one call", entry, sequences, kv_heads);
  if (sequences == 0) return 0;
  if (!mass || !page_tables || !lengths || !counts || (keep > 0 && !kept)) return refuse("%s: null tensor", entry);
  if (!words_aligned({mass, page_tables, lengths, kept, counts}))
    return refuse("%s: tensors not aligned to their elements", entry);
  const uintptr_t from = reinterpret_cast<uintptr_t>(lengths), to = reinterpret_cast<uintptr_t>(counts);
  if ((from > to ? from - to : to - from) / 4 < (uintptr_t)sequences)
    return refuse("%s: counts overlap lengths", entry);  // (each head's block reads its sequence's length)
  const HeaviestArgs a{mass, page_tables, lengths, sequences, table_pages, cache_pages, page_size, kv_heads,
                       sinks, recent, keep, kept, counts, bad_page, unit_columns(page_size)};
  // (no sequence has more candidates than its page table has room for)
  const int64_t each = ceil_div(std::max<int64_t>((int64_t)table_pages * page_size - sinks - recent, 0), kPickThreads);
  const dim3 grid((unsigned)(sequences * kv_heads)), block(kPickThreads);
  const hipStream_t st = (hipStream_t)stream;
  if (each <= 2) hipLaunchKernelGGL(pick_heaviest<2>, grid, block, 0, st, a);
  else if (each <= 8) hipLaunchKernelGGL(pick_heaviest<8>, grid, block, 0, st, a);
  else if (each <= 16) hipLaunchKernelGGL(pick_heaviest<16>, grid, block, 0, st, a);
  else if (each <= 32) hipLaunchKernelGGL(pick_heaviest<32>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(pick_heaviest<0>, grid, block, 0, st, a);
  return launched(entry);
}

extern "C" int drift_cache_keep_workspace(int32_t sequences, int32_t most, int32_t kv_heads, int32_t head_dim,
                                          int32_t quantized, int64_t* bytes) {
  clear_error();
  if (!bytes) return refuse("drift_cache_keep_workspace: null bytes");
  *bytes = 0;
  if (const int bad = check_keep("drift_cache_keep_workspace", sequences, most, kv_heads, head_dim)) return bad;
  *bytes = keep_bytes(sequences, most, kv_heads, head_dim, quantized != 0);
  return 0;
}

extern "C" int drift_cache_keep(void* keys, void* values, float* key_scales, float* value_scales, float* mass,
                                const int32_t* page_tables, int32_t table_pages, const int32_t* into,
                                int32_t into_pages, int32_t cache_pages, const int32_t* kept, int32_t kept_heads,
                                const int32_t* counts, const int32_t* starts, int32_t sequences, int32_t most,
                                int32_t kv_heads, int32_t head_dim, int32_t page_size, void* workspace,
                                int64_t workspace_bytes, int32_t* bad_page, void* stream) {
  const char* entry = "drift_cache_keep";
  clear_error();
  if (const int bad = check_keep(entry, sequences, most, kv_heads, head_dim)) return bad;
  if (page_size <= 0 || page_size % 16 != 0)
    return refuse("%s: pages of %d tokens: not a multiple of 16", entry, page_size);
  if (table_pages < 0 || into_pages < 0 || cache_pages < 0)
    return refuse("%s: %d table pages, into %d, %d cache pages", entry, table_pages, into_pages, cache_pages);
  if (kept_heads != 1 && kept_heads != kv_heads) return refuse("%s: lists of %d heads for %d", entry, kept_heads, kv_heads);
  if (sequences == 0 || most == 0) return 0;
  if (!keys || !values || !page_tables || !kept) return refuse("%s: null tensor", entry);
  if (!key_scales != !value_scales) return refuse("%s: scales of keys or of values alone", entry);
  if (!words_aligned({key_scales, value_scales, mass, page_tables, into, kept, counts, starts}) ||
      (!key_scales && ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & 1) != 0))
    return refuse("%s: tensors not aligned to their elements", entry);
  const bool apart = into && into != page_tables;
  if (into && !apart && into_pages != table_pages && sequences > 1)  // (a sequence's own pages would be others')
    return refuse("%s: into is page tables of %d pages a sequence as ones of %d", entry, table_pages, into_pages);
  const int64_t bytes = apart ? 0 : keep_bytes(sequences, most, kv_heads, head_dim, key_scales != nullptr);
  if (bytes > 0 && (!workspace || workspace_bytes < bytes || !aligned16(workspace)))
    return refuse("%s: a workspace of %lld bytes, needs %lld at a multiple of 16", entry, (long long)workspace_bytes,
                  (long long)bytes);
  const KeepArgs a{keys, values, key_scales, value_scales, mass, page_tables, apart ? into : page_tables, kept, counts,
                   starts, sequences, table_pages, into ? into_pages : table_pages, cache_pages, page_size, kept_heads,
                   most, kv_heads, head_dim, (char*)workspace, bad_page};
  return key_scales ? keep<uint8_t>(entry, a, apart, (hipStream_t)stream)
                    : keep<uint16_t>(entry, a, apart, (hipStream_t)stream);
}
