// The attention that cached positions gather (paged.hpp has the cache's
// layouts): what a position has been weighed by the rows that see it, of one
// sequence or several in a launch.
//
// Token t of a sequence sits at position P = start + t and sees the positions j <= P
// of its own sequence; query head h reads key head h / (heads / kv_heads). With
//   s_j = scale q.k_j,  p_j = exp(s_j - m) / sum_j exp(s_j - m)
// over the visible j, a position's and key head's mass is the sum of p_j over the
// call's tokens and the heads that read it; where the sequence held the position
// before the call (j < start), added to what it had. The rows' m and sums are needed
// before any p_j is known: a call's few rows keep their scores meanwhile (one pass over
// the keys), many take them twice. Every sum is one wave's or block's in an order of
// its own: no atomics, and the same bits every time.
#include "products.hpp"

#include <algorithm>
#include <type_traits>

namespace drift {
namespace {

constexpr int kMaxHead = 512;
constexpr float kLog2E = 1.44269504088896340736f;

// What the position sums need of a row: its scores' factor, in powers of two (NaN: the
// row is no numbers), its largest score and one over its sum.
typedef f32x4 Row;
enum { kScale, kTop, kInverse };

// What a score by itself needs (a type of its own: the call out of line that gets it by
// reference has a copy in scratch memory, whose size costs every launch).
struct ScoreArgs {
  Paging p;
  int32_t kv_heads, dim;
  float scale;
  UnitColumns columns;
  const void* keys;
  const float* key_scales;
};

struct MassArgs : ScoreArgs {
  int32_t heads, group;
  const float* before;
  float* mass;
  // the workspace: rows' statistics [splits, rows, 2] (largest score and sum), their
  // scores [rows, room] or their queries [rows, terms, padded head] and constants,
  // and positions' partial sums [parts, sequences, kv_heads, summed]
  int64_t rows, room;
  float *statistics, *scores, *partials;
  uint16_t* halves;
  Row* constants;
  // positions in `splits` of at least `chunk` tiles for the statistics; rows in `parts` for the sums, of positions below
  // `summed`, a block every `strides`-th tile of positions
  int32_t splits, chunk, parts, summed, strides;
  int32_t wide;  // masses on 16-byte alignment
};

// Rows of a sequence and key head lie together in the workspace: row r is token r / group, head r % group.
__device__ __forceinline__ int64_t row_place(const MassArgs& a, const Span& span, int kv) {
  return span.first * a.heads + (int64_t)kv * span.rows * a.group;
}

template <typename T>
__device__ __forceinline__ const T* query_of(const T* queries, const MassArgs& a, const Span& span, int kv, uint32_t row) {
  const uint32_t token = row / (uint32_t)a.group;
  return queries + ((span.first + token) * a.heads + kv * a.group + (row - token * (uint32_t)a.group)) * (int64_t)a.dim;
}

// Where position j of a sequence has its numbers [cache_pages, kv_heads, page_size], and its keys; false: nowhere.
struct Place {
  int64_t word, key;
};
__device__ __forceinline__ bool place_of(const ScoreArgs& a, const Span& span, int64_t j, int kv, Place& place) {
  const uint32_t unit = (uint32_t)(j / 16), column = a.columns.of(unit);
  const int64_t page = span.table[column], off = j - (int64_t)column * a.p.page_size;
  if (page < 0 || page >= a.p.cache_pages) {
    flag_bad(a.p);
    return false;
  }
  place.word = (page * a.kv_heads + kv) * (int64_t)a.p.page_size + off;
  place.key = ((page * a.p.page_size + off) * a.kv_heads + kv) * (int64_t)a.dim;
  return true;
}

// Sums of the four positions from j on (a multiple of four: on one page) into their masses.
__device__ __forceinline__ void store_masses(const MassArgs& a, const Span& span, int64_t j, int kv, const float (&sum)[4]) {
  const int64_t length = span.start + span.rows;
  Place place;
  if (j >= length || !place_of(a, span, j, kv, place)) return;
  if (a.wide && j + 4 <= length && (!a.before || j + 4 <= span.start || j >= span.start)) {
    f32x4 x = {sum[0], sum[1], sum[2], sum[3]};
    if (a.before && j < span.start) x += *(const f32x4*)(a.before + place.word);
    *(f32x4*)(a.mass + place.word) = x;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e < length)
      a.mass[place.word + e] = a.before && j + e < span.start ? a.before[place.word + e] + sum[e] : sum[e];
}

// The score of a row and a position, by F32 products one after another.
template <typename T, bool I8>
__device__ __forceinline__ float score_of(const ScoreArgs& a, const T* query, const Place& place) {
  float dot = 0.0f;
  for (int d = 0; d < a.dim; ++d) {
    const float k = I8 ? (float)((const int8_t*)a.keys)[place.key + d] : f16_value(((const uint16_t*)a.keys)[place.key + d]);
    dot = fmaf(load_one(query + d), k, dot);
  }
  if constexpr (I8) dot *= a.key_scales[place.word];
  return dot * a.scale;
}

// ------------------------------------------------------------------ rows and positions one by one

// A row's statistics by one wave, a lane a position.
template <typename T, bool I8>
__global__ void __launch_bounds__(kWave) row_statistics(const T* queries, MassArgs a) {
  __shared__ float query[kMaxHead];
  const int lane = threadIdx.x;
  int64_t nth;
  const int s = locate(a.p, blockIdx.x / (unsigned)a.heads, 1, 0, 1, nth);
  if (s < 0) return;
  const Span span = span_of<true>(a.p, s);
  if (nth >= span.rows) return;
  const int h = blockIdx.x % (unsigned)a.heads, kv = h / a.group;
  const int64_t row = (span.first + nth) * a.heads + h;
  for (int d = lane; d < a.dim; d += kWave) query[d] = load_one(queries + row * a.dim + d);
  wave_sync();
  float top = -kInfinity, total = 0.0f;
  for (int64_t base = 0; base <= span.start + nth; base += kWave) {
    const int64_t j = base + lane;
    Place place;
    const bool seen = j <= span.start + nth && place_of(a, span, j, kv, place);
    const float score = seen ? score_of<float, I8>(a, query, place) : -kInfinity;
    // the running maximum (a NaN stays out of it and reaches the sum by itself)
    const float next = fmaxf(top, group_max<64>(score));
    const float ref = next == -kInfinity ? 0.0f : next;
    float sum = seen ? expf(score - ref) : 0.0f;
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) sum += __shfl_xor(sum, mask, kWave);
    total = fmaf(total, expf(top - ref), sum);
    top = next;
  }
  if (lane == 0) a.statistics[row * 2] = top, a.statistics[row * 2 + 1] = total;
}

// Positions' sums by one wave, a lane a position of a tile of 64; a block every `splits`-th tile of a sequence and key
// head. Its loads bound it, a key's value a lane at a time, again for every row: 64 single tokens at 2,000 positions, 32
// heads over 4 of 512, 25.6 ms, a prompt of 512 tokens, 16 heads over 2 of 512, 176 ms, 2 single tokens over 4 heads of 20
// 46 us.
template <typename T, bool I8>
__global__ void __launch_bounds__(kWave) position_sums(const T* queries, MassArgs a) {
  __shared__ float query[kMaxHead];
  const int lane = threadIdx.x, kv = blockIdx.x % (unsigned)a.kv_heads;
  const unsigned rest = blockIdx.x / (unsigned)a.kv_heads;
  const Span span = span_of<false>(a.p, rest % (unsigned)a.p.sequences);
  if (span.rows == 0) return;
  for (int64_t base = (int64_t)(rest / (unsigned)a.p.sequences) * kWave; base < span.start + span.rows;
       base += (int64_t)a.splits * kWave) {
    const int64_t j = base + lane;
    Place place;
    const bool there = j < span.start + span.rows && place_of(a, span, j, kv, place);
    double sum = 0.0;  // (of small terms and a large sum: 32,768 rows' in F32 were off by 2.7e-5 of their sizes)
    for (int64_t t = max(base - span.start, (int64_t)0); t < span.rows; ++t)
      for (int h = kv * a.group; h < (kv + 1) * a.group; ++h) {
        const int64_t row = (span.first + t) * a.heads + h;
        wave_sync();
        for (int d = lane; d < a.dim; d += kWave) query[d] = load_one(queries + row * a.dim + d);
        wave_sync();
        if (!there || j > span.start + t) continue;
        const float top = a.statistics[row * 2], ref = top == -kInfinity ? 0.0f : top;
        sum += expf(score_of<float, I8>(a, query, place) - ref) / a.statistics[row * 2 + 1];
      }
    if (there) a.mass[place.word] = (float)(a.before && j < span.start ? a.before[place.word] + sum : sum);
  }
}

// ------------------------------------------------------------------ products

// A row's query as a product takes it: a lane's values d_of(k) .. of it, scaled by a power of
// two to below 2^15 (BF16 exactly, down to 2^-32 of the row's largest; F32 as two F16
// terms) and with the scale's sign, lanes l, l + LANES, .. sharing the row. Returns the factor
// that makes its products scores in powers of two: above 0, so that the largest
// product is the largest score and what is masked stays -infinity (a scale of 0, or one that a tiny row
// makes it, is small enough to leave every weight even); NaN where row or scale is no number.
template <typename T, int KS, int TERMS, int LANES, typename At>
__device__ __forceinline__ float take_query(const T* q, const MassArgs& a, At d_of, f16x8 (&query)[KS][TERMS]) {
  float v[KS][8];
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int d = d_of(k);
#pragma unroll
    for (int e = 0; e < 8; e += Chunk<T>::N) {
      float x[Chunk<T>::N];
      Chunk<T>::unpack(cached_load(q + (d < a.dim ? d + e : e)), x);
#pragma unroll
      for (int i = 0; i < Chunk<T>::N; ++i) v[k][e + i] = d < a.dim ? x[i] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[k][e]) & 0x7fffffffu);
  }
#pragma unroll
  for (int mask = LANES; mask < kWave; mask <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, mask, kWave));
  const bool finite = most < 0x7f800000u;
  const int shift = finite && most != 0 ? 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(most)) : 0;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = finite ? ldexpf(v[k][e], shift) : 0.0f;
      if (a.scale < 0.0f) x[e] = -x[e];
    }
    const Halves<TERMS> h = halves_of<TERMS>(x);
#pragma unroll
    for (int t = 0; t < TERMS; ++t) query[k][t] = h.term[t];
  }
  return finite && a.scale == a.scale ? fmaxf(ldexpf(fabsf(a.scale) * kLog2E, -shift), 0x1p-120f) : __builtin_nanf("");
}

// Scores that came out as NaN, taken again by themselves: a term of F16 may have met an
// infinity that the whole number would have made one of.
template <typename T, bool I8>
__device__ __noinline__ float score_again_of(const T* query, const ScoreArgs& a, const Span& span, int kv, int64_t j) {
  Place place;
  if (!place_of(a, span, j, kv, place)) return -kInfinity;
  return score_of<T, I8>(a, query, place) * kLog2E;
}

// Of a lane's scores x[n], of positions at(n), those that are NaN. Copies of the arguments go by
// reference: the kernels' own then stay in scalar registers (passed themselves, every
// use of theirs would read scratch memory).
template <typename T, bool I8, int N, typename At>
__device__ __forceinline__ void scores_again(const T* query, const MassArgs& a, const Span& span, int kv, At at,
                                             float factor, float (&x)[N]) {
  const ScoreArgs args = a;
  const Span rows = span;
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (x[n] != x[n]) x[n] = score_again_of<T, I8>(query, args, rows, kv, at(n)) * factor;
}

// How far, in powers of two, a score may pass what weights are taken against: sums of weights up to 2^kSlack each stay
// numbers, and those 2^-126 of the least.
constexpr float kSlack = 32.0f;

// A row's constants, the weights taken against a number that no score passes: the sum of weights against `top` is no less
// than the largest of them. (Nothing but scores of -infinity seen: 0 / 0, as the formula has it.)
__device__ __forceinline__ Row row_of(float scale, float top, float total) {
  const float most = top + ceilf(log2f(total));
  const float inverse = exp2f(most - top) / total;
  return Row{scale, most, top == -kInfinity || scale != scale ? __builtin_nanf("") : inverse, 0.0f};
}

// Largest scores and sums, in powers of two, of two parts as one's.
__device__ __forceinline__ void join_statistics(float& top, float& total, float top2, float total2) {
  const float high = fmaxf(top, top2), ref = high == -kInfinity ? 0.0f : high;
  total = total * exp2_fast(top - ref) + total2 * exp2_fast(top2 - ref);
  top = high;
}

// ------------------------------------------------------------------ few rows

// The tiles of positions that a split of a unit of 16 rows takes.
struct SplitTiles {
  int each, count;
};
__device__ __forceinline__ SplitTiles split_tiles(const MassArgs& a, uint32_t last, int size) {
  const int tiles = (int)(last / size) + 1;
  const int each = max(a.chunk, (tiles + a.splits - 1) / a.splits);
  return {each, (tiles + each - 1) / each};
}

// Scores of units of 16 rows, kept, and their statistics: positions in tiles of 32 (F16)
// or 64 (8 bits), keys straight from memory into the operands of 16 x 16 x 32
// products, S^T = K Q^T: the result's column (lane % 16) is a row, its rows are
// positions, dealt out so that a lane has TOK / 4 consecutive ones. A block's four waves
// take its split's tiles in turn. Memory bounds it: 64 single tokens at up to 8,000
// positions (304,719 in all), 32 heads over 8 of 128, 160 us for 624 MB of keys and 39 MB of
// scores (4.2 TB/s); without the scores' stores it would be 134 (4.7).
template <typename T, bool I8, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) few_scores(const T* queries, MassArgs a) {
  constexpr int kWaves = 4;
  constexpr int TOK = I8 ? 64 : 32, NT = TOK / 16, TERMS = sizeof(T) == 4 ? 2 : 1, KS = DP / 32;
  __shared__ float stats[kWaves][16][2];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int kv = blockIdx.x % (unsigned)a.kv_heads;
  const unsigned rest = blockIdx.x / (unsigned)a.kv_heads, all_units = gridDim.x / (unsigned)(a.kv_heads * a.splits);
  // a unit's splits lie far apart: where they are neighbours, those that have nothing to do are some dies' alone
  const int split = rest / all_units;
  int64_t nth;
  const int s = locate(a.p, rest % all_units, 16, 0, a.group, nth);
  if (s < 0) return;
  const Span span = span_of<true>(a.p, s);
  const int rows = (int)min((int64_t)span.rows * a.group - nth * 16, (int64_t)16);
  if (rows <= 0) return;
  const uint32_t row0 = (uint32_t)nth * 16, row = row0 + min(col, rows - 1), group = (uint32_t)a.group;
  const uint32_t p0 = (uint32_t)span.start + row0 / group, p1 = (uint32_t)span.start + (row0 + rows - 1) / group;
  const uint32_t position = (uint32_t)span.start + row / group;
  const SplitTiles tiles = split_tiles(a, p1, TOK);
  const int begin = uniform(split * tiles.each), end = uniform(min(begin + tiles.each, (int)(p1 / TOK) + 1));
  if (begin >= end) return;

  f16x8 query[KS][TERMS];
  const float row_scale = take_query<T, KS, TERMS, 16>(
      query_of(queries, a, span, kv, row), a,
      [&](int k) { return I8 ? (k / 2) * 64 + g * 16 + (k % 2) * 8 : k * 32 + g * 8; }, query);
  float* const scores = a.scores + (row_place(a, span, kv) + row) * a.room;

  const int key_unit = (col >> 2) * (TOK / 4) / 16, own_unit = g * (TOK / 4) / 16;
  const uint32_t last_unit = p1 / 16;
  auto page_of = [&](uint32_t u, uint32_t& off) -> int32_t {
    const uint32_t in = min(u, last_unit), column = a.columns.of(in);
    off = (in - column * a.columns.page_units) * 16;
    return span.table[column];
  };
  struct Places {
    int32_t key_page, own_page;
    uint32_t key_off, own_off;
  };
  auto places_of = [&](int i) {
    Places w;
    const uint32_t first = (uint32_t)min(i, end - 1) * NT;
    w.key_page = page_of(first + key_unit, w.key_off);
    w.own_page = page_of(first + own_unit, w.own_off);
    return w;
  };
  constexpr int kKeyLoads = I8 ? KS / 2 : KS;  // 16-byte loads a position
  struct Keys {
    u32x4 raw[NT][kKeyLoads];
    float scale[I8 ? 16 : 1];
  };
  auto load_keys = [&](const Places& w, Keys& to) {
    const int32_t page = (uint32_t)w.key_page < (uint32_t)a.p.cache_pages ? w.key_page : 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t in = w.key_off + ((col >> 2) * (TOK / 4) + 4 * t + (col & 3)) % 16;
      const int64_t at = (((int64_t)page * a.p.page_size + in) * a.kv_heads + kv) * a.dim;
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) {
        if constexpr (I8) {
          const int8_t* key = (const int8_t*)a.keys + at;
          const int d = k * 64 + g * 16;
          if (a.dim == DP) {
            to.raw[t][k] = *(const u32x4_8*)(key + d);
          } else {
            const u32x2 x = *(const u32x2*)(key + (d < a.dim ? d : 0)), y = *(const u32x2*)(key + (d + 8 < a.dim ? d + 8 : 0));
            to.raw[t][k] = u32x4{x.x, x.y, y.x, y.y};
          }
        } else {
          const int d = k * 32 + g * 8;
          to.raw[t][k] = *(const u32x4*)((const uint16_t*)a.keys + at + (d < a.dim ? d : 0));
        }
      }
    }
    if constexpr (I8) {
      const int32_t own = (uint32_t)w.own_page < (uint32_t)a.p.cache_pages ? w.own_page : 0;
      const float* from = a.key_scales + ((int64_t)own * a.kv_heads + kv) * a.p.page_size + w.own_off;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float4 x = *(const float4*)(from + e);
        to.scale[e] = x.x, to.scale[e + 1] = x.y, to.scale[e + 2] = x.z, to.scale[e + 3] = x.w;
      }
    }
  };

  float top = -kInfinity, total = 0.0f;
  auto take_tile = [&](int i, bool okay, const Keys& keys) {
    const uint32_t mine = (uint32_t)i * TOK + g * (TOK / 4);  // the lane's first position
    if (!okay && mine <= p1) flag_bad(a.p);
    f32x4 score[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      score[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        f16x8 key;
        if constexpr (I8) {
          const u32x4 w = keys.raw[t][k / 2];
          key = k % 2 ? codes_f16(w.z, w.w) : codes_f16(w.x, w.y);
        } else {
          key = __builtin_bit_cast(f16x8, keys.raw[t][k]);
        }
#pragma unroll
        for (int m = 0; m < TERMS; ++m)
          score[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, query[k][m], score[t], 0, 0, 0);
      }
    }
    const bool whole = (uint32_t)(i + 1) * TOK - 1 <= p0 && __all(okay);
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = score[t][e] * row_scale;
        if constexpr (I8) x *= keys.scale[4 * t + e];
        if (!whole) x = (okay & (mine + 4 * t + e <= position)) ? x : -kInfinity;
        odd |= x != x;
        score[t][e] = x;
      }
    if (__any(odd && row_scale == row_scale)) {
      float x[4 * NT];
#pragma unroll
      for (int n = 0; n < 4 * NT; ++n) x[n] = score[n / 4][n % 4];
      scores_again<T, I8>(query_of(queries, a, span, kv, row), a, span, kv, [&](int n) { return (int64_t)mine + n; }, 1.0f, x);
#pragma unroll
      for (int n = 0; n < 4 * NT; ++n) score[n / 4][n % 4] = x[n];
    }
    float high = top;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) high = fmaxf(high, score[t][e]);
    const float ref = high == -kInfinity ? 0.0f : high;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += exp2_fast(score[t][e] - ref);
    total = fmaf(total, exp2_fast(top - ref), sum);
    top = high;
    if (col < rows && mine < a.room)
#pragma unroll
      for (int t = 0; t < NT; ++t) *(f32x4*)(scores + mine + 4 * t) = score[t];
  };
  // Keys of two tiles on their way. A tile's places are asked for before the keys of the tile before it are: loads
  // come back in their order, and to wait for the places is then no wait for those keys.
  Keys keys0, keys1;
  int i = begin + wave;
  const Places first0 = places_of(i), first1 = places_of(i + kWaves);
  Places next = places_of(i + 2 * kWaves);
  auto in_cache = [&](const Places& w) { return (uint32_t)w.own_page < (uint32_t)a.p.cache_pages; };
  bool okay0 = in_cache(first0), okay1 = in_cache(first1);
  if (i < end) load_keys(first0, keys0);
  if (i + kWaves < end) load_keys(first1, keys1);
  auto step = [&](Keys& keys, bool& okay) {
    const Places coming = next;
    next = places_of(i + 3 * kWaves);
    take_tile(i, okay, keys);
    okay = in_cache(coming);
    if (i + 2 * kWaves < end) load_keys(coming, keys);
    i += kWaves;
  };
  while (i < end) {
    step(keys0, okay0);
    if (i < end) step(keys1, okay1);
  }
  // the four lanes' of a row, then the waves'
#pragma unroll
  for (int mask = 16; mask < kWave; mask <<= 1)
    join_statistics(top, total, __shfl_xor(top, mask, kWave), __shfl_xor(total, mask, kWave));
  if (g == 0) stats[wave][col][0] = top, stats[wave][col][1] = total;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) join_statistics(top, total, stats[w][col][0], stats[w][col][1]);
  if (g == 0 && col < rows) {
    float* to = a.statistics + (split * a.rows + row_place(a, span, kv) + row) * 2;
    to[0] = top, to[1] = total;
  }
}

// The few rows' positions: a thread four of them, a block 1,024 of a sequence and key
// head; the rows' statistics joined in LDS first, 256 at a time. (19 us of that step: 39 MB of
// scores and 20 MB of masses read and written, 3.1 TB/s, part of it out of the caches: what
// bounds it is each block's chain, tables, statistics, then few loads a thread.)
template <bool I8>
__global__ void __launch_bounds__(256) few_sums(MassArgs a) {
  constexpr int kBatch = 256;
  __shared__ float2 constants[kBatch];
  const int kv = blockIdx.x % (unsigned)a.kv_heads;
  const unsigned rest = blockIdx.x / (unsigned)a.kv_heads;
  const Span span = span_of<false>(a.p, rest / (unsigned)a.strides);
  if (span.rows == 0) return;
  const uint32_t rows = (uint32_t)span.rows * (uint32_t)a.group, group = (uint32_t)a.group;
  const int64_t first = row_place(a, span, kv), length = span.start + span.rows;
  bool staged = false;
  for (int64_t base = (int64_t)(rest % (unsigned)a.strides) * 1024; base < length; base += (int64_t)a.strides * 1024) {
    const int64_t j = base + threadIdx.x * 4;
    float sum[4] = {};
    for (uint32_t row0 = 0; row0 < rows; row0 += kBatch) {
      if (rows > kBatch || !staged) {
        __syncthreads();
        const uint32_t row = row0 + threadIdx.x;
        if (row < rows) {
          const uint32_t end = min((row / 16 + 1) * 16, rows) - 1;
          const int splits = split_tiles(a, (uint32_t)span.start + end / group, I8 ? 64 : 32).count;
          const float* st = a.statistics + (first + row) * 2;
          float top = st[0], total = st[1];
#pragma unroll 4
          for (int i = 1; i < splits; ++i) join_statistics(top, total, st[i * a.rows * 2], st[i * a.rows * 2 + 1]);
          // (nothing but scores of -infinity seen: 0 / 0, as the formula has it)
          constants[threadIdx.x] = make_float2(top, top == -kInfinity ? __builtin_nanf("") : 1.0f / total);
        }
        __syncthreads();
        staged = true;
      }
      if (j >= length) continue;
      const int count = (int)min(rows - row0, (uint32_t)kBatch);
      // rows from `some` on see the first position, from `all` on all four: before their own token rows have no scores
      auto sees = [&](int64_t at) { return (int)min(max((at - span.start) * group - row0, (int64_t)0), (int64_t)count); };
      const int some = sees(j), all = sees(j + 3);
      const float* from = a.scores + (first + row0) * a.room + j;
      for (int r = some; r < all; ++r) {
        const f32x4 x = *(const f32x4*)(from + r * a.room);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r >= sees(j + e)) sum[e] = fmaf(exp2_fast(x[e] - constants[r].x), constants[r].y, sum[e]);
      }
      float part[4] = {};
#pragma unroll 4
      for (int r = all; r < count; ++r) {
        const f32x4 x = *(const f32x4*)(from + r * a.room);
        const float2 c = constants[r];
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] = fmaf(exp2_fast(x[e] - c.x), c.y, part[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += part[e];
    }
    store_masses(a, span, j, kv, sum);
  }
}

// ------------------------------------------------------------------ many rows

// LDS places of 16-byte chunks of rows of DP F16 numbers, moved by an exclusive or with
// the row's number so that the rows of one operand lie on different banks.
template <int DP>
__device__ __forceinline__ int chunk_place(int row, int chunk) {
  return (row * (DP / 8) + (chunk ^ (DP >= 128 ? row & 15 : (row >> 1) & 7))) * 16;
}

// Statistics of many rows: 32 a wave, 128 a block, positions in tiles of 64 that the block stages in LDS once
// for all its rows, by 32 x 32 x 16 products, S^T = K Q^T: the result's column is a row, and its largest score and
// sum stay in its lanes. The queries go to the workspace as the products take them, for many_sums.
//
// The exponentials and what goes with them bound it: a prompt of 8,192 tokens, 32 heads over 8 of 128, 358 us at best and
// 393 at the median of a profiled run (768 and 699 TFLOP/s); vector instructions issue 70% of the time, the products run
// 38%. 64 tokens after 31,936 33 us, of which 128 rows a block leave most to staging.
template <typename T, bool I8, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) many_statistics(const T* queries, MassArgs a) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1, TOK = 64, KS = DP / 16, kThreads = 256;
  constexpr int kTile = TOK * DP * 2, kScales = kTile, kTileBytes = kTile + (I8 ? TOK * 4 : 0);
  constexpr int kLoads = TOK * (DP / 8) / kThreads;
  __shared__ __attribute__((aligned(16))) char tiles[2 * kTileBytes];
  const int thread = threadIdx.x, lane = thread & 63, wave = uniform(thread >> 6), col = lane & 31, h = lane >> 5;
  const int kv = blockIdx.x % (unsigned)a.kv_heads;
  const unsigned rest = blockIdx.x / (unsigned)a.kv_heads, all_units = gridDim.x / (unsigned)(a.kv_heads * a.splits);
  const int split = rest / all_units;
  int64_t nth;
  // the last rows first: they have the most positions
  const int s = locate(a.p, all_units - 1 - rest % all_units, 128, 0, a.group, nth);
  if (s < 0) return;
  const Span span = span_of<true>(a.p, s);
  const int rows = (int)min((int64_t)span.rows * a.group - nth * 128, (int64_t)128);
  if (rows <= 0) return;
  const uint32_t row0 = (uint32_t)nth * 128, group = (uint32_t)a.group, start = (uint32_t)span.start;
  const uint32_t p1 = start + (row0 + rows - 1) / group;
  const SplitTiles split_of = split_tiles(a, p1, TOK);
  const int begin = uniform(split * split_of.each), end = uniform(min(begin + split_of.each, (int)(p1 / TOK) + 1));
  if (begin >= end) return;

  // ---- this wave's rows
  const int wave_row = wave * 32;
  const bool idle = wave_row >= rows;
  const uint32_t w0 = start + (row0 + min(wave_row, rows - 1)) / group;
  const uint32_t w1 = start + (row0 + min(wave_row + 32, rows) - 1) / group;
  const uint32_t row = row0 + min(wave_row + col, rows - 1), position = start + row / group;
  const bool mine = wave_row + col < rows;
  f16x8 query[KS][TERMS];
  const float row_scale = take_query<T, KS, TERMS, 32>(query_of(queries, a, span, kv, row), a,
                                                       [&](int k) { return k * 16 + h * 8; }, query);
  const float row_inverse = 1.0f / row_scale;
  const int64_t place = row_place(a, span, kv) + row;
  if (split == 0 && mine)
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int t = 0; t < TERMS; ++t) *(f16x8*)(a.halves + (place * TERMS + t) * DP + k * 16 + h * 8) = query[k][t];

  // ---- staging: a thread's chunks of a tile. Chunk n of a thread is of a unit that its whole wave shares, so that
  // a load is a scalar base and an offset that stays. A tile's four units are one a lane of four.
  const uint32_t last_unit = p1 / 16;
  constexpr int kBytes = I8 ? 1 : 2;
  const uint32_t position_bytes = (uint32_t)a.kv_heads * a.dim * kBytes, key_head = (uint32_t)kv * a.dim * kBytes;
  struct Entries {
    int32_t page;
    uint32_t off;
  };
  auto entries_of = [&](int i) {
    const uint32_t at = min((uint32_t)min(i, end - 1) * 4 + (lane & 3), last_unit), column = a.columns.of(at);
    return Entries{span.table[column], (at - column * a.columns.page_units) * 16};
  };
  auto at_lane = [](uint64_t x, int u) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, u);
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), u) << 32) | lo;
  };
  constexpr int kTokens = 64 / (DP / 8), kStep = kThreads / (DP / 8);  // positions a wave stages at once, and all four
  const int own_token = lane / (DP / 8) + wave * kTokens, own_chunk = lane % (DP / 8);
  const uint32_t own_at = (uint32_t)(own_token % 16) * position_bytes + key_head +
                          (own_chunk * 8 < a.dim ? own_chunk * 8 * kBytes : 0);
  struct Raw {
    u32x4 chunk[kLoads];
    float scale;
    uint32_t okay;  // which of the tile's units lie in the cache
  };
  auto load_tile = [&](const Entries& units, Raw& raw) {
    const bool okay = (uint32_t)units.page < (uint32_t)a.p.cache_pages;
    if (!okay) flag_bad(a.p);
    const uint64_t page = okay ? units.page : 0;
    const uint64_t from = (page * a.p.page_size + units.off) * position_bytes;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const char* at = (const char*)a.keys + at_lane(from, (n * kStep + wave * kTokens) / 16) +
                       (n * kStep % 16 * position_bytes) + own_at;
      if constexpr (I8) {
        const u32x2 x = *(const u32x2*)at;
        raw.chunk[n].x = x.x, raw.chunk[n].y = x.y;
      } else {
        raw.chunk[n] = *(const u32x4*)at;
      }
    }
    if (I8 && wave == 0) {
      const uint32_t off = (uint32_t)__shfl((int)units.off, lane / 16, kWave);
      const int64_t its = __shfl((int)page, lane / 16, kWave);
      raw.scale = a.key_scales[(its * a.kv_heads + kv) * a.p.page_size + off + lane % 16];
    }
    raw.okay = (uint32_t)__ballot(okay) & 15u;
  };
  const int own_place = chunk_place<DP>(own_token, own_chunk);
  auto store_tile = [&](char* tile, const Raw& raw) {
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      // (16 positions on, and for narrow heads 32, the exclusive or is the same; for wide ones 8 on it has bit 3 turned)
      const int to = kStep % 16 ? chunk_place<DP>(own_token + n * kStep, own_chunk) : own_place + n * kStep * DP * 2;
      *(u32x4*)(tile + to) = I8 ? __builtin_bit_cast(u32x4, codes_f16(raw.chunk[n].x, raw.chunk[n].y)) : raw.chunk[n];
    }
    if (I8 && wave == 0) ((float*)(tile + kScales))[lane] = raw.scale;
  };
  const int key_from = chunk_place<DP>(col, h);

  float top = -kInfinity, total = 0.0f;
  // A tile is asked for two tiles ahead, and its entries before the tile before it is: loads come back in their order,
  // and to wait for the entries is then no wait for that tile.
  Raw raw0, raw1;
  load_tile(entries_of(begin), raw0);
  const Entries second = entries_of(begin + 1);
  Entries next = entries_of(begin + 2);
  uint32_t okay = raw0.okay;
  if (begin + 1 < end) load_tile(second, raw1);
  store_tile(tiles, raw0);
  auto take_tile = [&](int i, Raw& ahead, const Raw& coming) {
    const int now = ((i - begin) & 1) * kTileBytes;
    const Entries units = next;
    next = entries_of(i + 3);
    if (i + 2 < end) load_tile(units, ahead);
    __syncthreads();
    const uint32_t base = (uint32_t)i * TOK;
    if (!idle && base <= w1) {
      const bool whole = okay == 15u && base + TOK - 1 <= w0;
      f32x16 score[2];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 16; ++e) score[half][e] = 0.0f;
      {
        // operands four at a time, the next four on their way while these are multiplied
        f16x8 keys[2][4];
        auto load_keys = [&](int n, f16x8 (&to)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // (the exclusive or with k, in the low bits of places that are multiples of 128, gives them from one)
            const int half = (4 * n + e) / KS, k = (4 * n + e) % KS;
            to[e] = *(const f16x8*)(tiles + ((now + key_from) ^ (k % 8 * 32)) + half * 32 * DP * 2 + k / 8 * 256);
          }
        };
        load_keys(0, keys[0]);
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < KS / 2; ++n) {
          if (n + 1 < KS / 2) load_keys(n + 1, keys[(n + 1) % 2]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int half = (4 * n + e) / KS, k = (4 * n + e) % KS;
#pragma unroll
            for (int m = 0; m < TERMS; ++m)
              score[half] = __builtin_amdgcn_mfma_f32_32x32x16_f16(keys[n % 2][e], query[k][m], score[half], 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
      }
      // score[half][e] is row col, position base + 32 half + 8 (e / 4) + 4 h + e % 4
      if constexpr (I8)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 x = *(const float4*)(tiles + now + kScales + (half * 32 + 2 * e + 4 * h) * 4);
            score[half][e] *= x.x, score[half][e + 1] *= x.y, score[half][e + 2] *= x.z, score[half][e + 3] *= x.w;
          }
      auto mask = [&]() {
#pragma unroll
        for (int n = 0; n < 32; ++n) {
          const int e = n % 16, in = n / 16 * 32 + e / 4 * 8 + e % 4 + 4 * h;
          const bool seen = (bool)(okay >> (in / 16) & 1) & (base + in <= position);
          score[n / 16][e] = seen ? score[n / 16][e] : -kInfinity;
        }
      };
      if (!whole) {
        asm volatile("");  // (a branch, not a choice for every score)
        mask();
      }
      // What weights are taken against is raised only when a score passes it by more than kSlack: while that bound is
      // not below 0, the numbers' bits compare as whole numbers do (a NaN may pass it, or reaches the sum by itself).
      auto raise = [&]() {
        float high = score[0][0];
#pragma unroll
        for (int n = 1; n < 32; ++n) high = fmaxf(high, score[n / 16][n % 16]);
        const float next = fmaxf(top, high * row_scale);
        total *= exp2_fast(top - (next == -kInfinity ? 0.0f : next));
        top = next;
      };
      auto weigh = [&]() {
        const float ref = top == -kInfinity ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < 32; ++n) sum += exp2_fast(fmaf(score[n / 16][n % 16], row_scale, -ref));
        return sum;
      };
      int most = 0;
#pragma unroll
      for (int n = 0; n < 32; ++n) most = max(most, __float_as_int(score[n / 16][n % 16]));
      const float bound = (top + kSlack) * row_inverse;
      if (__any(!(bound >= 0.0f) || most > __float_as_int(bound))) raise();
      float sum = weigh();
      if (__any(sum != sum && row_scale == row_scale)) {
        float x[32];
#pragma unroll
        for (int n = 0; n < 32; ++n) x[n] = score[n / 16][n % 16];
        scores_again<T, I8>(query_of(queries, a, span, kv, row), a, span, kv,
                            [&](int n) { return (int64_t)base + n / 16 * 32 + n % 16 / 4 * 8 + n % 4 + 4 * h; }, row_inverse, x);
#pragma unroll
        for (int n = 0; n < 32; ++n) score[n / 16][n % 16] = x[n];
        raise();
        sum = weigh();
      }
      total += sum;
    }
    if (i + 1 < end) {
      store_tile(tiles + (kTileBytes - now), coming);
      okay = coming.okay;
    }
  };
  for (int i = begin; i < end; i += 2) {
    take_tile(i, raw0, raw1);
    if (i + 1 < end) take_tile(i + 1, raw1, raw0);
  }
  join_statistics(top, total, __shfl_xor(top, 32, kWave), __shfl_xor(total, 32, kWave));
  if (h != 0 || !mine) return;
  if (split == 0) a.constants[place] = row_of(row_scale, top, total);
  if (a.splits > 1) a.statistics[(split * a.rows + place) * 2] = top, a.statistics[(split * a.rows + place) * 2 + 1] = total;
}

// The statistics of many rows' splits joined: a block has the 128 rows of a block of many_statistics.
__global__ void __launch_bounds__(128) many_rows(MassArgs a) {
  const int kv = blockIdx.x % (unsigned)a.kv_heads;
  int64_t nth;
  const int s = locate(a.p, blockIdx.x / (unsigned)a.kv_heads, 128, 0, a.group, nth);
  if (s < 0) return;
  const Span span = span_of<true>(a.p, s);
  const int64_t rows = (int64_t)span.rows * a.group, row = nth * 128 + threadIdx.x;
  if (row >= rows) return;
  const uint32_t last = (uint32_t)min(nth * 128 + 128, rows) - 1;
  const int splits = split_tiles(a, (uint32_t)span.start + last / (uint32_t)a.group, 64).count;
  const int64_t place = row_place(a, span, kv) + row;
  float top = a.statistics[place * 2], total = a.statistics[place * 2 + 1];
#pragma unroll 8
  for (int i = 1; i < splits; ++i) {
    const float* st = a.statistics + (i * a.rows + place) * 2;
    join_statistics(top, total, st[0], st[1]);
  }
  a.constants[place] = row_of(a.constants[place][kScale], top, total);
}

// Many rows' positions: 32 SETS a wave, whose keys stay in its registers, 128 SETS a block, while the
// rows pass through LDS in tiles that all four waves use, by the same products: a result's column is a row, and
// each lane adds up its rows' weights for the positions in its registers, so that rows need no sums across lanes
// until the last. A block has every `parts`-th part of the rows that see its tile of positions.
//
// The prompt's 337 us at best and 365 at the median (815 and 753 TFLOP/s): vector instructions issue 56% of the time, the
// products run 39%, one after the other in each of two waves a SIMD. (Kept instead, its 4.3 GB of scores would have to be
// written and read.) With 256 positions a block each row from LDS is used twice: by 128 the last 64 rows of 32,000
// positions took 82 us for 79.
//
// A score that is NaN where its row is numbers is one of -infinity (a key's infinity met a zero term): had it
// been NaN or infinity the row would not be. So a NaN weight counts as 0, times an inverse that is NaN where the row is.

// The sum over a half of a wave, in every lane of it.
__device__ __forceinline__ float half_sum(float v) {
  v += __int_as_float(dpp_move32<0xb1>(__float_as_int(v)));   // quad_perm [1, 0, 3, 2]
  v += __int_as_float(dpp_move32<0x4e>(__float_as_int(v)));   // quad_perm [2, 3, 0, 1]
  v += __int_as_float(dpp_move32<0x141>(__float_as_int(v)));  // row_half_mirror
  v += __int_as_float(dpp_move32<0x140>(__float_as_int(v)));  // row_mirror
  return v + __shfl_xor(v, 16, kWave);
}

template <int DP>
constexpr int kSets = DP > 128 ? 1 : 2;
template <typename T, int DP>
constexpr int kSumRows = (sizeof(T) == 4 ? 2 : 1) * DP > 256 ? 32 : 64;
// The parts of a tile of positions: `each` tiles of rows, from `from` on; so many of them have any.
struct Parts {
  int from, each, count;
};
__device__ __forceinline__ Parts parts_of(const MassArgs& a, const Span& span, uint32_t j0, int row_tile) {
  const uint32_t rows = (uint32_t)span.rows * (uint32_t)a.group, start = (uint32_t)span.start;
  const int all = (int)((rows + row_tile - 1) / row_tile);
  const int from = j0 > start ? (int)((j0 - start) * (uint32_t)a.group / row_tile) : 0;
  const int each = j0 < (uint32_t)a.summed ? (all - from + a.parts - 1) / a.parts : all;
  return {from, each, (all - from + each - 1) / each};
}

template <typename T, bool I8, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) many_sums(MassArgs a) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1, KS = DP / 16, SETS = kSets<DP>, RT = kSumRows<T, DP>;
  constexpr int kTermBytes = RT * DP * 2, kTileBytes = TERMS * kTermBytes, kPositions = 128 * SETS;
  constexpr int kLoads = kTileBytes / 16 / 256;
  __shared__ __attribute__((aligned(16))) char tiles[2 * kTileBytes];
  const int thread = threadIdx.x, lane = thread & 63, wave = uniform(thread >> 6), col = lane & 31, h = lane >> 5;
  const int kv = blockIdx.x % (unsigned)a.kv_heads;
  const unsigned rest = blockIdx.x / (unsigned)a.kv_heads, in_part = (unsigned)(a.p.sequences * a.strides);
  const int part = rest / in_part, s = rest % in_part / (unsigned)a.strides;
  const Span span = span_of<false>(a.p, s);
  if (span.rows == 0) return;
  const uint32_t rows = (uint32_t)span.rows * (uint32_t)a.group, start = (uint32_t)span.start, group = (uint32_t)a.group;
  const uint32_t length = start + span.rows;
  const int64_t first = row_place(a, span, kv);
  const int all_tiles = (int)((rows + RT - 1) / RT);

  for (int64_t tile = rest % (unsigned)a.strides; tile * kPositions < length; tile += a.strides) {
    const uint32_t j0 = (uint32_t)tile * kPositions;
    // the tiles of rows that see some of the positions, and this part's of them
    const Parts parts = parts_of(a, span, j0, RT);
    if (part >= parts.count) continue;
    const bool parted = j0 < (uint32_t)a.summed;
    const int begin = parts.from + part * parts.each, end = min(begin + parts.each, all_tiles);

    // ---- the rows
    u32x4 raw[kLoads];
    Row constants[RT / 32], coming[RT / 32];
    auto load_tile = [&](int i) {
#pragma unroll
      for (int n = 0; n < kLoads; ++n) {
        const int q = thread + n * 256, row = q / (TERMS * DP / 8), chunk = q % (TERMS * DP / 8);
        raw[n] = *(const u32x4*)(a.halves + (first + min((uint32_t)(i * RT + row), rows - 1)) * (TERMS * DP) + chunk * 8);
      }
#pragma unroll
      for (int r = 0; r < RT / 32; ++r) coming[r] = a.constants[first + min((uint32_t)(i * RT + r * 32 + col), rows - 1)];
    };
    auto store_tile = [&](char* to) {
#pragma unroll
      for (int n = 0; n < kLoads; ++n) {
        const int q = thread + n * 256, row = q / (TERMS * DP / 8), chunk = q % (TERMS * DP / 8);
        *(u32x4*)(to + chunk / (DP / 8) * kTermBytes + chunk_place<DP>(row, chunk % (DP / 8))) = raw[n];
      }
    };
    if (begin < end) load_tile(begin);

    // ---- the wave's positions
    const uint32_t base = j0 + wave * 32 * SETS;
    f16x8 key[SETS][KS];
    float key_scale[SETS][I8 ? 16 : 1];
#pragma unroll
    for (int set = 0; set < SETS; ++set) {
      auto page_of = [&](uint32_t j, uint32_t& off) -> int64_t {
        const uint32_t unit = min(j, length - 1) / 16, column = a.columns.of(unit);
        off = (unit - column * a.columns.page_units) * 16;
        const int32_t page = span.table[column];
        return (uint32_t)page < (uint32_t)a.p.cache_pages ? page : 0;
      };
      uint32_t off;
      const int64_t page = page_of(base + set * 32 + col, off);
      const int64_t at = ((page * a.p.page_size + off + col % 16) * a.kv_heads + kv) * a.dim;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = k * 16 + h * 8 < a.dim ? k * 16 + h * 8 : 0;
        if constexpr (I8) {
          const u32x2 x = *(const u32x2*)((const int8_t*)a.keys + at + d);
          key[set][k] = codes_f16(x.x, x.y);
        } else {
          key[set][k] = __builtin_bit_cast(f16x8, *(const uint4*)((const uint16_t*)a.keys + at + d));
        }
      }
      if constexpr (I8)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int64_t its = page_of(base + set * 32 + 2 * e, off);
          const float4 x = *(const float4*)(a.key_scales + (its * a.kv_heads + kv) * a.p.page_size + off + 2 * e % 16 + 4 * h);
          key_scale[set][e] = x.x, key_scale[set][e + 1] = x.y, key_scale[set][e + 2] = x.z, key_scale[set][e + 3] = x.w;
        }
    }

    const int query_from = chunk_place<DP>(col, h);
    float sum[SETS][16];
#pragma unroll
    for (int set = 0; set < SETS; ++set)
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[set][e] = 0.0f;
    if (begin < end) {
      __syncthreads();  // (the tiles of the positions before are used up)
      store_tile(tiles);
    }
    // WHOLE: every row of the tile sees every position of the block
    auto take_tile = [&](int i, auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      const int now = ((i - begin) & 1) * kTileBytes;
#pragma unroll
      for (int r = 0; r < RT / 32; ++r) constants[r] = coming[r];
      if (i + 1 < end) load_tile(i + 1);
      __syncthreads();
#pragma unroll
      for (int r = 0; r < RT / 32; ++r) {
        const uint32_t row0 = (uint32_t)i * RT + r * 32;
        // (the wave's first position is past the last row's own: nothing is seen)
        if (!WHOLE && (row0 >= rows || base > start + min(row0 + 31, rows - 1) / group)) continue;
        f32x16 score[SETS];
#pragma unroll
        for (int set = 0; set < SETS; ++set)
#pragma unroll
          for (int e = 0; e < 16; ++e) score[set][e] = 0.0f;
        {
          // operands four at a time, as above
          constexpr int kAll = KS * TERMS;
          f16x8 query[2][4];
          auto load_query = [&](int n, f16x8 (&to)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = (4 * n + e) / TERMS, term = (4 * n + e) % TERMS;
              to[e] = *(const f16x8*)(tiles + ((now + query_from) ^ (k % 8 * 32)) + term * kTermBytes + r * 32 * DP * 2 +
                                      k / 8 * 256);
            }
          };
          load_query(0, query[0]);
          __builtin_amdgcn_s_setprio(1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int n = 0; n < kAll / 4; ++n) {
            if (n + 1 < kAll / 4) load_query(n + 1, query[(n + 1) % 2]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int set = 0; set < SETS; ++set)
                score[set] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key[set][(4 * n + e) / TERMS], query[n % 2][e], score[set], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_s_setprio(0);
        }
        const Row c = constants[r];
        // positions base + 32 set + 8 (e / 4) + 4 h + e % 4, of which the row sees those up to its own
        int seen = INT32_MAX;
        if (!WHOLE) seen = row0 + col < rows ? (int)(start + (row0 + col) / group - base) - 4 * h : -1;
#pragma unroll
        for (int set = 0; set < SETS; ++set)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x = score[set][e];
            if constexpr (I8) x *= key_scale[set][e];
            // (at most 1 but for NaN, of which the bounds make 0)
            const float p = __builtin_amdgcn_fmed3f(exp2_fast(fmaf(x, c[kScale], -c[kTop])), 0.0f, 1.0f);
            const float next = fmaf(p, c[kInverse], sum[set][e]);
            sum[set][e] = set * 32 + e / 4 * 8 + e % 4 <= seen ? next : sum[set][e];
          }
      }
      if (i + 1 < end) store_tile(tiles + (kTileBytes - now));
    };
    // rows from token `all` on see all the block's positions; the last tile may have fewer rows
    const uint32_t all = j0 + kPositions > start + 1 ? j0 + kPositions - 1 - start : 0;
    const int first_whole = (int)min(((uint64_t)all * group + RT - 1) / RT, (uint64_t)all_tiles);
    int i = begin;
    for (; i < min(first_whole, end); ++i) take_tile(i, std::false_type());
    for (; i < min((int)(rows / RT), end); ++i) take_tile(i, std::true_type());
    for (; i < end; ++i) take_tile(i, std::false_type());

    // ---- the lanes' rows added up: lanes 0 to 3 of each half have four positions of every set each
#pragma unroll
    for (int set = 0; set < SETS; ++set) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[set][e] = half_sum(sum[set][e]);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (col == q) {
          const uint32_t j = base + set * 32 + 8 * q + 4 * h;
          const float four[4] = {sum[set][4 * q], sum[set][4 * q + 1], sum[set][4 * q + 2], sum[set][4 * q + 3]};
          if (!parted) store_masses(a, span, j, kv, four);
          else if (j < length)
            *(f32x4*)(a.partials + (((int64_t)part * a.p.sequences + s) * a.kv_heads + kv) * a.summed + j) =
                f32x4{four[0], four[1], four[2], four[3]};
        }
    }
  }
}

// Positions' sums over the parts of many rows, four a thread.
__global__ void __launch_bounds__(64) many_parts(MassArgs a, int positions, int row_tile) {
  const int kv = blockIdx.y % (unsigned)a.kv_heads, s = blockIdx.y / (unsigned)a.kv_heads;
  const Span span = span_of<false>(a.p, s);
  const int64_t j = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 4;
  if (span.rows == 0 || j >= min(span.start + span.rows, (int64_t)a.summed)) return;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  const int parts = parts_of(a, span, (uint32_t)(j / positions * positions), row_tile).count;
#pragma unroll 4
  for (int part = 0; part < parts; ++part)
    sum += *(const f32x4*)(a.partials + (((int64_t)part * a.p.sequences + s) * a.kv_heads + kv) * a.summed + j);
  const float four[4] = {sum[0], sum[1], sum[2], sum[3]};
  store_masses(a, span, j, kv, four);
}

// ------------------------------------------------------------------ host side

int check_mass(const char* entry, int32_t heads, int32_t kv_heads, int32_t dim, int64_t room, int64_t longest) {
  if (dim > kMaxHead) return refuse("%s: heads of %d values (at most %d)", entry, dim, kMaxHead);
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return refuse("%s: %d heads over %d key heads", entry, heads, kv_heads);
  if (room < 0 || longest < 0)
    return refuse("%s: room for %lld positions, a longest sequence of %lld", entry, (long long)room, (long long)longest);
  return 0;
}

// How a call's work is laid out, by its numbers alone (the workspace's size
// follows from it before there are tensors).
struct Plan {
  bool few;
  Split split;     // of positions, for the statistics
  int parts;       // of rows, for many rows' sums
  int64_t summed;  // positions that have parts
  int strides;     // blocks of a sequence and key head for the sums
  // bytes of the workspace before each
  int64_t scores, halves, constants, partials, bytes;
};

// Bytes of scores, at most, that are kept rather than taken twice: a cache's keys take eight times as much for
// rows that share a key head by fours. A row has room for every position of its page table, whatever the sequences hold
// (64 sequences of 32 heads at up to 8,000 positions in tables for 65,536: 537 MB of scratch, 164 us for 161; for 131,072
// they are taken twice, 366 us).
constexpr int64_t kMostScores = (int64_t)1 << 29;

int64_t padded(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

Plan plan_of(int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t room,
             int64_t longest, bool by_offsets, bool f32) {
  Plan p{};
  p.split = {1, 1};
  p.strides = p.parts = 1;
  if (sequences <= 0 || tokens <= 0) return p;
  auto at = [&](int64_t bytes) {
    const int64_t from = p.bytes;
    p.bytes += ceil_div(bytes, 16) * 16;
    return from;
  };
  const int64_t rows = tokens * heads, group = heads / kv_heads, units = sequences * kv_heads;
  const int64_t seen = std::max<int64_t>(std::min(longest, room), 1);
  // Up to 32 rows a sequence and key head on average (a decode step's, or some more): their scores are kept (us, kept /
  // taken twice, 16 sequences at up to 4,000 positions, 8 key heads of 128: 8 rows each 31 / 54, 16 34 / 53, 32 47 / 53, 64
  // (at 4,000) 123 / 83; 64 sequences 77 / 186, 96 / 184, 148 / 178, as chunks of every fourth 82 / 184, 116 / 187, 190 /
  // 190). The average is what the host knows: where one sequence has all the rows past the others' single tokens, its
  // units read its keys again and again, and kept scores lose from 16 on average on (64 sequences, 8 rows 117 / 190, 16
  // 223 / 196, 32 482 / 205).
  p.few = tokens * group <= sequences * 32 && rows * room * 4 <= kMostScores;
  if (p.few) {
    p.split = split_of(units, seen, 1024, 4, 16);
    p.strides = (int)std::min(ceil_div(seen, 1024), std::max<int64_t>(kSplitBlocks / units, 1));
  } else {
    p.split = split_of(ceil_div(tokens * group, 128) * kv_heads, seen, 512, 8, 1 << 25);
    const int64_t most_rows = (by_offsets || sequences == 1 ? tokens : 1) * group;
    const int64_t positions = dim <= 128 ? 256 : 128, tiles = ceil_div(seen, positions);
    p.strides = (int)std::min(tiles, std::max<int64_t>(kSplitBlocks / units, 1));
    // Rows in parts until there are some 4,096 blocks: causal rows leave later positions fewer, and chunks among
    // single tokens leave few blocks most of the rows (us, 24 sequences of 1,811 tokens over 8 bits: by 2,048 blocks
    // 108, 4,096 100, 8,192 114, 16,384 141; a prompt of 8,192: 694 by 2,048 and by 8,192).
    p.parts = (int)std::max<int64_t>(std::min({4096 / (units * tiles), ceil_div(most_rows, 256), (int64_t)16}), 1);
    p.summed = p.parts > 1 ? tiles * positions : 0;
  }
  at(p.split.splits * rows * 8);
  if (p.few) {
    p.scores = at(rows * room * 4);
  } else {
    p.halves = at(rows * padded(dim) * (f32 ? 4 : 2));
    p.constants = at(rows * 16);
    p.partials = at(p.parts > 1 ? p.parts * units * p.summed * 4 : 0);
  }
  return p;
}

template <typename T, bool I8, int DP>
int launch_products(const char* entry, const T* queries, const MassArgs& a, const Plan& plan, hipStream_t st) {
  const int64_t units = (int64_t)a.p.sequences * a.kv_heads;
  const dim3 block(256);
  if (plan.few) {
    const int64_t blocks = units_of(a.p, 16, 0, a.group) * a.splits * a.kv_heads;
    hipLaunchKernelGGL((few_scores<T, I8, DP>), dim3((unsigned)blocks), block, 0, st, queries, a);
    if (const int bad = launched(entry)) return bad;
    hipLaunchKernelGGL((few_sums<I8>), dim3((unsigned)(units * a.strides)), block, 0, st, a);
    return launched(entry);
  }
  const int64_t blocks = units_of(a.p, 128, 0, a.group) * a.kv_heads;
  hipLaunchKernelGGL((many_statistics<T, I8, DP>), dim3((unsigned)(blocks * a.splits)), block, 0, st, queries, a);
  if (const int bad = launched(entry)) return bad;
  if (a.splits > 1) {
    hipLaunchKernelGGL(many_rows, dim3((unsigned)blocks), dim3(128), 0, st, a);
    if (const int bad = launched(entry)) return bad;
  }
  hipLaunchKernelGGL((many_sums<T, I8, DP>), dim3((unsigned)(units * a.strides * a.parts)), block, 0, st, a);
  if (const int bad = launched(entry)) return bad;
  if (a.parts > 1) {
    hipLaunchKernelGGL(many_parts, dim3((unsigned)ceil_div(a.summed, 256), (unsigned)units), dim3(64), 0, st, a,
                       128 * kSets<DP>, (kSumRows<T, DP>));
    return launched(entry);
  }
  return 0;
}

template <typename T, bool I8>
int launch_mass(const char* entry, const T* queries, MassArgs a, const Plan& plan, bool aligned, int64_t longest,
                hipStream_t st) {
  const int64_t row_blocks = units_of(a.p, 1, 0, 1) * a.heads, units = (int64_t)a.p.sequences * a.kv_heads;
  if (row_blocks > kOneWaveBlocks || units > kOneWaveBlocks / 16)
    return refuse("%s: %d tokens of %d heads in one call", entry, a.p.tokens, a.heads);
  // (rows of products count in 32 bits)
  const int64_t blocks = (units_of(a.p, plan.few ? 16 : 128, 0, a.group) * a.kv_heads) * plan.split.splits;
  if (aligned && a.dim <= 256 && a.p.cache_pages > 0 && units <= 65535 && blocks <= kOneWaveBlocks / 4 &&
      (int64_t)a.p.tokens * a.group < (int64_t)1 << 31) {
    a.splits = plan.split.splits;
    a.chunk = plan.split.chunk;
    if (I8 == false && plan.few) a.chunk *= 2;  // (tiles of 32)
    a.parts = plan.parts;
    a.summed = (int32_t)plan.summed;
    a.strides = plan.strides;
    char* const from = (char*)a.statistics;
    a.scores = (float*)(from + plan.scores);
    a.halves = (uint16_t*)(from + plan.halves);
    a.constants = (Row*)(from + plan.constants);
    a.partials = (float*)(from + plan.partials);
    if (a.dim <= 64) return launch_products<T, I8, 64>(entry, queries, a, plan, st);
    if (a.dim <= 128) return launch_products<T, I8, 128>(entry, queries, a, plan, st);
    return launch_products<T, I8, 256>(entry, queries, a, plan, st);
  }
  a.splits = (int)std::min<int64_t>(std::max<int64_t>(ceil_div(longest, kWave), 1), std::max<int64_t>(kSplitBlocks / units, 1));
  hipLaunchKernelGGL((row_statistics<T, I8>), dim3((unsigned)row_blocks), dim3(kWave), 0, st, queries, a);
  if (const int bad = launched(entry)) return bad;
  hipLaunchKernelGGL((position_sums<T, I8>), dim3((unsigned)(units * a.splits)), dim3(kWave), 0, st, queries, a);
  return launched(entry);
}

template <typename T>
int attention_mass(const char* entry, const T* queries, MassArgs a, int64_t longest, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  clear_error();
  if (const int bad = check_paging(entry, a.p, a.kv_heads, a.dim)) return bad;
  a.room = std::min((int64_t)a.p.table_pages * a.p.page_size, kMostPositions);
  if (const int bad = check_mass(entry, a.heads, a.kv_heads, a.dim, a.room, longest)) return bad;
  if (a.p.tokens == 0 || a.p.sequences == 0) return 0;
  if (!queries || !a.mass) return refuse("%s: null tensor", entry);
  if (((reinterpret_cast<uintptr_t>(a.mass) | reinterpret_cast<uintptr_t>(a.before)) & 3) != 0 ||
      reinterpret_cast<uintptr_t>(queries) % sizeof(T) != 0)
    return refuse("%s: queries or masses not aligned to their elements", entry);
  if (const int bad = check_cache(entry, a.p, a.keys, a.keys, a.key_scales, a.key_scales)) return bad;
  const uint64_t masses = (uint64_t)a.p.cache_pages * a.kv_heads * a.p.page_size;
  const uintptr_t from = reinterpret_cast<uintptr_t>(a.before), to = reinterpret_cast<uintptr_t>(a.mass);
  if (a.before && from != to && (from > to ? from - to : to - from) / 4 < masses)
    return refuse("%s: mass overlaps before", entry);
  const Plan plan = plan_of(a.p.sequences, a.p.tokens, a.heads, a.kv_heads, a.dim, a.room, longest,
                            a.p.offsets != nullptr, sizeof(T) == 4);
  if (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace))
    return refuse("%s: a workspace of %lld bytes, needs %lld at a multiple of 16", entry, (long long)workspace_bytes,
                  (long long)plan.bytes);
  a.statistics = (float*)workspace;
  a.rows = (int64_t)a.p.tokens * a.heads;
  a.group = a.heads / a.kv_heads;
  a.columns = unit_columns(a.p.page_size);
  a.wide = aligned16(a.mass) && aligned16(a.before);
  const bool aligned = a.dim % 8 == 0 && aligned16(queries) && aligned16(a.keys) && aligned16(a.key_scales);
  return a.key_scales ? launch_mass<T, true>(entry, queries, a, plan, aligned, longest, (hipStream_t)stream)
                      : launch_mass<T, false>(entry, queries, a, plan, aligned, longest, (hipStream_t)stream);
}

}  // namespace
}  // namespace drift

using namespace drift;

extern "C" int drift_attention_mass_workspace(int32_t sequences, int32_t tokens, int32_t heads, int32_t kv_heads,
                                              int32_t head_dim, int32_t room, int32_t longest, int64_t* bytes) {
  clear_error();
  if (!bytes) return refuse("drift_attention_mass_workspace: null bytes");
  *bytes = 0;
  if (const int bad = check_mass("drift_attention_mass_workspace", heads, kv_heads, head_dim, room, longest)) return bad;
  // with offsets or without, in either type
  for (int kind = 0; kind < 4; ++kind)
    *bytes = std::max(*bytes, plan_of(sequences, tokens, heads, kv_heads, head_dim, room, longest, kind & 1, kind & 2).bytes);
  return 0;
}

#define DRIFT_MASS_ARGS                                                                                             \
  MassArgs {                                                                                                        \
    {{page_tables, starts, offsets, sequences, table_pages, cache_pages, page_size, start, tokens, bad_page},       \
     kv_heads, head_dim, scale, {}, keys, key_scales},                                                              \
        heads, 0, before, mass, 0, 0, nullptr, nullptr, nullptr, nullptr, nullptr, 1, 1, 1, 0, 1, 0                 \
  }

extern "C" int drift_attention_mass_f32(const float* queries, const void* keys, const float* key_scales,
                                        const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                        const int32_t* starts, const int32_t* offsets, int32_t sequences, int32_t start,
                                        int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                        int32_t page_size, float scale, int32_t longest, const float* before,
                                        float* mass, void* workspace, int64_t workspace_bytes, int32_t* bad_page,
                                        void* stream) {
  return attention_mass<float>("drift_attention_mass_f32", queries, DRIFT_MASS_ARGS, longest, workspace,
                               workspace_bytes, stream);
}

extern "C" int drift_attention_mass_bf16(const uint16_t* queries, const void* keys, const float* key_scales,
                                         const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                         const int32_t* starts, const int32_t* offsets, int32_t sequences,
                                         int32_t start, int32_t tokens, int32_t heads, int32_t kv_heads,
                                         int32_t head_dim, int32_t page_size, float scale, int32_t longest,
                                         const float* before, float* mass, void* workspace, int64_t workspace_bytes,
                                         int32_t* bad_page, void* stream) {
  return attention_mass<uint16_t>("drift_attention_mass_bf16", queries, DRIFT_MASS_ARGS, longest, workspace,
                                  workspace_bytes, stream);
}
