// Attention of new tokens over the paged key and value cache (paged.hpp has
// its layouts), of one sequence or several in a launch.
//
// Token t of a sequence sits at position P = start + t and sees the positions
// j <= P of its own sequence (its own key, written before, among them); with a
// window only those with j > P - window, or j < sinks. TREE: the tokens are a tree's,
// and of their own positions each sees those whose bits it has; its own P, for
// the window over the positions before them, is start - 1 + their number. Query head h reads key
// head h / (heads / kv_heads):
//   s_j = scale q.k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
// over the visible j, in one pass with the running maximum m and sum, in F32. A
// row that sees nothing is zeros. What is masked has no part in a row, whatever
// it holds (an infinity, a NaN, memory never written); a position whose page
// table entry names no page of the cache is masked, and the flag set.
#include "paged.hpp"
#include "products.hpp"

#include <algorithm>
#include <type_traits>

namespace drift {
namespace {

constexpr int kMaxHead = 512;
// What a row by itself needs. Of arguments that a call out of line gets by reference the kernel
// has a copy in scratch memory, and the size of that memory costs every launch: with 16 or 32
// bytes a lane more than 224 a decode batch took 300 us for 248, an 8-bit chunk 116 for 106. So
// these are apart from the rest, and a tree's from others'.
struct RowArgs {
  Paging p;
  int32_t heads, kv_heads, dim, group;
  float scale;
  int32_t window, sinks;  // window 0: every position up to the row's own
  const void *keys, *values;
  const float *key_scales, *value_scales;
};
// A tree's: what each row sees of its sequence's new tokens, `words` words of 32 bits a token.
struct TreeRowArgs : RowArgs {
  const uint32_t* sees;
  int64_t words;
};
template <bool TREE>
using RowArgsOf = std::conditional_t<TREE, TreeRowArgs, RowArgs>;

template <bool TREE>
struct ArgsOf : RowArgsOf<TREE> {
  // the split over positions: at least `chunk` tiles a split, `splits` of them;
  // where there are several, their maxima and sums [splits, partial_rows, 3] and
  // unscaled results [splits, partial_rows, dim], a row by its place among the
  // call's rows [tokens, heads] or (attend_few's, few_slots) by few_partial
  int32_t splits, chunk;
  int64_t partial_rows;
  float *statistics, *partials;
  int32_t few_slots, few_units;  // attend_few's rows of partials (0: by place), and units, of a sequence and key head
  int32_t few_rows;   // sequences of at most so many rows (tokens times group) are attend_few's, others attend_many's
  UnitColumns columns;
};

// A tree's row's position: start - 1, and one for each of the sequence's new tokens that it sees.
__device__ __forceinline__ int64_t tree_position(const TreeRowArgs& a, const Span& span, int64_t nth) {
  const uint32_t* sees = a.sees + (span.first + nth) * a.words;
  int64_t position = span.start - 1;
  for (int w = 0; (int64_t)w * 32 < span.rows && w < a.words; ++w)
    position += __popc(sees[w] & (uint32_t)bits_below(span.rows - w * 32));
  return position;
}

// What a tree's row sees of the 64 positions from `base` on: of those before `start` the
// ones from `low` on and the first `sinks`, of the others those whose bits it has.
__device__ __forceinline__ uint64_t tree_sees(const TreeRowArgs& a, const Span& span, int64_t nth, int64_t base,
                                              int64_t low, int64_t sinks) {
  uint64_t seen = bits_below(span.start - base) & (~bits_below(low - base) | bits_below(sinks - base));
  const int64_t at = base - span.start;  // the first of the positions among the new tokens
  if (at > -64 && at < span.rows) {
    const uint32_t* sees = a.sees + (span.first + nth) * a.words;
    auto word = [&](int w) -> uint64_t { return w < a.words ? sees[w] : 0; };
    uint64_t bits;
    if (at < 0) {
      bits = (word(0) | word(1) << 32) << -at;
    } else {
      const int w = (int)(at / 32), shift = (int)(at % 32);
      bits = (word(w) | word(w + 1) << 32) >> shift;
      if (shift != 0) bits |= word(w + 2) << (64 - shift);
    }
    seen |= bits & bits_below(span.rows - at);
  }
  return seen;
}

// The first position of a tree's row among those before `start`, but for the sinks.
__device__ __forceinline__ int64_t tree_low(const TreeRowArgs& a, const Span& span, int64_t nth) {
  return a.window ? min(max(tree_position(a, span, nth) - a.window + 1, (int64_t)0), span.start) : 0;
}

// The least position that the rows from token `nth` on may have, and the last that those up to it may see.
template <bool TREE>
__device__ __forceinline__ int64_t first_position(const Span& span, uint32_t nth) {
  return TREE ? max(span.start, (int64_t)1) - 1 : span.start + nth;
}
template <bool TREE>
__device__ __forceinline__ int64_t last_position(const Span& span, uint32_t nth) {
  return span.start + (TREE ? span.rows - 1 : nth);
}

// Where attend_few's row `row` of a sequence and key head, at `place` among the call's, keeps its partials.
template <bool TREE>
__device__ __forceinline__ int64_t few_partial(const ArgsOf<TREE>& a, int s, int kv, uint32_t row, int64_t place) {
  return a.few_slots ? ((int64_t)s * a.kv_heads + kv) * a.few_slots + row : place;
}

// A cache's number `at`, and eight from `at` on (a multiple of eight).
template <bool I8>
__device__ __forceinline__ float row_one(const void* cache, int64_t at) {
  if constexpr (I8) return (float)((const int8_t*)cache)[at];
  else return f16_value(((const uint16_t*)cache)[at]);
}
template <bool I8>
__device__ __forceinline__ void row_eight(const void* cache, int64_t at, float (&v)[8]) {
  if constexpr (I8) {
    const uint2 raw = *(const uint2*)((const int8_t*)cache + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? raw.x : raw.y) >> (8 * (e % 4)));
  } else {
    const uint4 raw = *(const uint4*)((const uint16_t*)cache + at);
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f16_value(word[e / 2] >> (16 * (e % 2)));
  }
}

// ------------------------------------------------------------------ rows one by one

// LDS that one wave's attend_row takes.
struct RowScratch {
  float query[kMaxHead];
  float weight[kWave];
  int64_t place[kWave];  // a value's index at dimension 0, or -1: not visible
};

// A row's state over some of its positions: the sums of a lane's values, lane + 64 i.
struct RowState {
  float sums[kMaxHead / kWave], top, total;
  bool any;  // some position is seen
};

// One row (a token's query head) by one wave over the tiles of 64 positions from,
// from + step, ..: a lane a position for the scores and then a lane a value for the
// sums, every product of F32 values in F32 and one by one. It takes any head size and
// whatever the cache holds. WIDE: keys and values on 16-byte alignment, heads of a
// multiple of 8 values, read in eights; else one by one, at any alignment.
template <typename T, bool I8, bool WIDE, bool TREE>
__device__ __forceinline__ void row_part(const T* queries, const RowArgsOf<TREE>& a, const Span& span, int64_t nth, int h,
                                         int from, int step, RowScratch& r, RowState& state) {
  const int lane = threadIdx.x & (kWave - 1), kv = h / a.group;
  // the last position that may be seen
  const int64_t position = span.start + (TREE ? span.rows - 1 : nth), row = ((span.first + nth) * a.heads + h) * a.dim;
  wave_sync();
  for (int d = lane; d < a.dim; d += kWave) r.query[d] = load_one(queries + row + d);
  wave_sync();
  constexpr int kEach = kMaxHead / kWave;
  float sums[kEach] = {}, top = -kInfinity, total = 0.0f;
  bool any = false;
  int64_t low = 0;
  if constexpr (TREE) low = tree_low(a, span, nth);
  else if (a.window) low = max(position - a.window + 1, (int64_t)0);
  const int64_t sink_end = a.window ? min((int64_t)a.sinks, low) : 0;
  for (int64_t tile = from; tile * kWave <= position; tile += step) {
    if (tile * kWave >= sink_end && (tile + 1) * kWave <= low) {  // what lies between is not seen
      tile += (low / kWave - tile + step - 1) / step * step;
      if (tile * kWave > position) break;
    }
    const int64_t j = tile * kWave + lane;
    bool seen;
    if constexpr (TREE) seen = tree_sees(a, span, nth, tile * kWave, low, sink_end) >> lane & 1;
    else seen = j <= position && (j >= low || j < sink_end);
    int64_t page = 0, off = 0;
    if (seen) {
      page = span.table[j / a.p.page_size];
      off = j % a.p.page_size;
      if (page < 0 || page >= a.p.cache_pages) {
        flag_bad(a.p);
        seen = false;
      }
    }
    float score = -kInfinity, value_scale = 1.0f;
    if (seen) {
      const int64_t key = ((page * a.p.page_size + off) * a.kv_heads + kv) * a.dim;
      float dot = 0.0f;
      if constexpr (WIDE) {
#pragma unroll 4
        for (int d = 0; d < a.dim; d += 8) {
          float k[8];
          row_eight<I8>(a.keys, key + d, k);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot = fmaf(r.query[d + e], k[e], dot);
        }
      } else {
        for (int d = 0; d < a.dim; ++d) dot = fmaf(r.query[d], row_one<I8>(a.keys, key + d), dot);
      }
      if constexpr (I8) {
        const int64_t at = (page * a.kv_heads + kv) * (int64_t)a.p.page_size + off;
        dot *= a.key_scales[at];
        value_scale = a.value_scales[at];
      }
      score = dot * a.scale;
    }
    // the running maximum (a NaN stays out of it and reaches the sum by itself)
    const float next = fmaxf(top, group_max<64>(score));
    const float ref = next == -kInfinity ? 0.0f : next;
    const float keep = expf(top - ref);
    const float p = seen ? expf(score - ref) : 0.0f;
    any |= __any(seen);
    top = next;
    float sum = p;
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) sum += __shfl_xor(sum, mask, kWave);
    total = fmaf(total, keep, sum);
    wave_sync();
    r.weight[lane] = p * value_scale;
    r.place[lane] = seen ? (page * a.kv_heads + kv) * (int64_t)a.dim * a.p.page_size + off : -1;
    wave_sync();
    if constexpr (WIDE) {
      // eight positions from a multiple of eight on lie together in a value's row
      const uint64_t which = __ballot(seen);
#pragma unroll
      for (int i = 0; i < kEach; ++i) sums[i] *= keep;
      for (int n = 0; n < kWave; n += 8) {
        const uint32_t some = (uint32_t)(which >> n) & 255u;
        if (some == 0) continue;
        const int first = __ffs(some) - 1;
        const int64_t at = uniform(r.place[n + first]) - first;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int d = lane + i * kWave;
          if (d >= a.dim) break;
          float v[8];
          row_eight<I8>(a.values, at + (int64_t)d * a.p.page_size, v);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            sums[i] = some >> e & 1 ? fmaf(r.weight[n + e], v[e], sums[i]) : sums[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int d = lane + i * kWave;
        if (d >= a.dim) break;
        float acc = sums[i] * keep;
        for (int n = 0; n < kWave; ++n) {
          const int64_t at = r.place[n];
          if (at < 0) continue;
          acc = fmaf(r.weight[n], row_one<I8>(a.values, at + (int64_t)d * a.p.page_size), acc);
        }
        sums[i] = acc;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) state.sums[i] = sums[i];
  state.top = top, state.total = total, state.any = any;
}

// One row by one wave, for the tile kernels' rows that came out as no numbers: slow,
// and kept small, since its registers count in every kernel that calls it.
template <typename T, bool I8, bool TREE>
__device__ __noinline__ void attend_row_of(const T* queries, T* out, const RowArgsOf<TREE>& a, const Span& span,
                                           int64_t nth, int h, RowScratch& r) {
  RowState state;
  row_part<T, I8, false, TREE>(queries, a, span, nth, h, 0, 1, r, state);
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = ((span.first + nth) * a.heads + h) * a.dim;
  // nothing seen: zeros; nothing but scores of -infinity seen: 0 / 0, as the formula has it
#pragma unroll
  for (int i = 0; i < kMaxHead / kWave; ++i) {
    const int d = lane + i * kWave;
    if (d < a.dim) store_one(out + row + d, state.any ? state.sums[i] / state.total : 0.0f);
  }
}

// Copies of the arguments go by reference: the kernels' own then stay in scalar
// registers (passed themselves, every use of theirs would read scratch memory).
template <typename T, bool I8, bool TREE>
__device__ __forceinline__ void attend_row(const T* queries, T* out, const RowArgsOf<TREE>& a, const Span& span,
                                           int64_t nth, int h, RowScratch& r) {
  const RowArgsOf<TREE> args = a;
  const Span rows = span;
  attend_row_of<T, I8, TREE>(queries, out, args, rows, nth, h, r);
}

// Every row by itself, for what the tile kernels do not take: a block of four waves
// (one, where the grid would not hold them) a row, each with every fourth tile, joined
// in LDS. Loads of a position a lane, and a cache read once a query head, bound it:
// one token of each of 64 sequences at 2,000 positions, 32 heads over 4 of 512 1.65 ms
// (12.6 with a wave a row, value by value), over 8 of 100 1.13 ms (2.56).
constexpr int kRowWaves = 4;

template <typename T, bool I8, bool WIDE, bool TREE>
__global__ void __launch_bounds__(kRowWaves * kWave) attend_rows(const T* queries, T* out, ArgsOf<TREE> a) {
  __shared__ RowScratch scratch[kRowWaves];
  __shared__ float tops[kRowWaves], totals[kRowWaves];
  __shared__ int anys[kRowWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = uniform((int)threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  int64_t nth;
  const int s = locate(a.p, blockIdx.x / (unsigned)a.heads, 1, 0, 1, nth);
  if (s < 0) return;
  const Span span = span_of<true>(a.p, s);
  if (nth >= span.rows) return;
  const int h = blockIdx.x % (unsigned)a.heads;
  RowState state;
  row_part<T, I8, WIDE, TREE>(queries, a, span, nth, h, wave, waves, scratch[wave], state);
  wave_sync();
#pragma unroll
  for (int i = 0; i < kMaxHead / kWave; ++i) scratch[wave].query[lane + i * kWave] = state.sums[i];
  if (lane == 0) tops[wave] = state.top, totals[wave] = state.total, anys[wave] = state.any;
  __syncthreads();
  float top = -kInfinity, total = 0.0f, factor[kRowWaves];
  bool any = false;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w)
    if (w < waves) top = fmaxf(top, tops[w]), any |= anys[w] != 0;
  const float ref = top == -kInfinity ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w)
    if (w < waves) {
      factor[w] = expf(tops[w] - ref);
      total = fmaf(totals[w], factor[w], total);
    }
  const int64_t row = ((span.first + nth) * a.heads + h) * a.dim;
  // nothing seen: zeros; nothing but scores of -infinity seen: 0 / 0, as the formula has it
  for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w)
      if (w < waves) x = fmaf(scratch[w].query[d], factor[w], x);
    store_one(out + row + d, any ? x / total : 0.0f);
  }
}

// ------------------------------------------------------------------ tiles by matrix instructions

// Rows of queries are (token, head of the key head's group) pairs: row r is token
// r / group of the sequence, head r % group, so that heads that share keys
// share their loads, whatever the group. The positions that the rows of tokens t0
// to t1 need, in tiles of `size` of them: `sinks` tiles from position 0, then on
// from `low`.
struct TileList {
  int32_t sinks, low, count;
  __device__ __forceinline__ int tile(int i) const { return i < sinks ? i : low + (i - sinks); }
};

template <bool TREE>
__device__ __forceinline__ TileList tiles_of(const ArgsOf<TREE>& a, int64_t first, int64_t last, int size) {
  TileList t;
  const int64_t low = a.window ? max(first - a.window + 1, (int64_t)0) : 0;
  t.low = (int32_t)(low / size);
  t.sinks = a.window ? min((int32_t)((min((int64_t)a.sinks, low) + size - 1) / size), t.low) : 0;
  t.count = t.sinks + (int32_t)(last / size) - t.low + 1;
  return t;
}

// Tiles a split takes.
template <bool TREE>
__device__ __forceinline__ int split_tiles(const ArgsOf<TREE>& a, int count) {
  return max(a.chunk, (count + a.splits - 1) / a.splits);
}

// Instructions as __builtin_amdgcn_sched_group_barrier counts them.
constexpr int kVectors = 0x2, kProducts = 0x8, kReads = 0x100;

// Weights are exp2 of the score less its row's maximum, times 2^kLift: as F16
// they then keep 11 bits down to 2^-28 of the largest.
constexpr float kLift = 14.0f;

// The few-rows kernel: C tiles of 16 rows by a wave, positions in tiles of 32
// (F16) or 64 (8 bits) that the block's waves take in turn, keys and values
// straight from memory into the operands of the matrix instructions.
//
// The scores are taken transposed, S^T = K Q^T, by 16 x 16 x 32 products: the
// result's column (lane % 16) is a row of queries, its rows positions, four a
// lane and tile. The rows of K are dealt out so that a lane's tiles together hold
// TOK / 4 consecutive positions, from g TOK / 4 on (g = lane / 16): those are the
// positions it has to bring as B operand of O^T = V^T P^T, where its A operand is
// 16 bytes of one value's row of the (transposed) value page. So weights go from
// the softmax into the next product without leaving their lane, no operand is
// staged or shuffled, and each of a row's statistics sits in the lanes of its
// column.
//
// Rows of queries are scaled by a power of two each to below 2^15 (BF16 exactly, down
// to 2^-32 of the row's largest; F32 as two F16 terms, 22 bits, since there are no F32
// products near the F16 ones' rate), their scores scaled back in F32. In 8 bits the
// codes are F16 numbers, a key's scale multiplies its score and a value's is part of
// its weight, which has a running maximum of its own then.
//
// Memory bounds it where there is enough to do: one token of each of 64 sequences of
// 400 to 8,000 positions, 32 heads over 8 of 128, 248 us (1,249 MB, 5.0 TB/s; vector
// instructions issue 17% of the time), in 8 bits 151 us (645 MB; 37%, the codes'
// conversions); one of 517 positions 11 us, a chain of dependent loads. Tiles staged in
// LDS, as attend_many's, gain nothing here: no other wave reads them.
constexpr int kFewWaves = 4;
template <int DP, int C>
struct FewShared {
  float merged[kFewWaves][16][DP + 4], stats[kFewWaves][C * 16][3];
};

template <typename T, bool I8, bool TREE, int DP, int C>
__device__ __forceinline__ void few_block(const T* queries, T* out, const ArgsOf<TREE>& a, unsigned block,
                                          FewShared<DP, C>& shared) {
  constexpr int kWaves = kFewWaves;
  constexpr int TOK = I8 ? 64 : 32, NT = TOK / 16;  // positions a tile, and row tiles of its scores
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  // Over the F16 cache weights have 22 bits for BF16 results too, since memory hides the second term (decode batch 256 us,
  // 259 with one): what is rounded to BF16 is the F32 result. In 8 bits, where the codes' conversions count and the
  // cache's own rounding is 2^-8, they have 11 (heads of 64: 105 us, 117 with two; of 128 159 / 161); trees' have 22
  // everywhere, as many_block says.
  constexpr int kWeightTerms = I8 && !TREE ? TERMS : 2;
  constexpr int KS = DP / 32, DT = DP / 16;         // products along a head, value tiles
  auto& merged = shared.merged;
  auto& stats = shared.stats;
  static_assert(sizeof(RowScratch) <= sizeof(merged) / kWaves, "a wave's part holds a row's scratch");

  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int kv = block % (unsigned)a.kv_heads;
  const unsigned rest = block / (unsigned)a.kv_heads;
  // A unit's splits lie far apart: blocks go to the eight dies in turn, and where splits are neighbours those that have
  // nothing to do are some dies' alone (64 sequences of 400 to 8,000 over 8 bits 155 us, 163 with neighbours).
  const unsigned all_units = (unsigned)(a.p.sequences * a.few_units);
  const int split = rest / all_units;
  const unsigned unit = rest % all_units;
  // (and its later units, of which most sequences have none: 64 single tokens in 4 units each, given by offsets, 244 us,
  // 457 with a sequence's units as neighbours, whose first are all dealt to the same quarter of a die)
  const int s = (int)(unit % (unsigned)a.p.sequences), nth = (int)(unit / (unsigned)a.p.sequences);
  const Span span = span_of<false>(a.p, s);
  const int rows = (int)min((int64_t)span.rows * a.group - nth * (C * 16), (int64_t)(C * 16));
  if (rows <= 0 || (int64_t)span.rows * a.group > a.few_rows) return;
  const uint32_t row0 = (uint32_t)nth * (C * 16), group = (uint32_t)a.group;
  const uint32_t p0 = (uint32_t)first_position<TREE>(span, row0 / group);
  const uint32_t p1 = (uint32_t)last_position<TREE>(span, (row0 + rows - 1) / group);
  const TileList list = tiles_of(a, p0, p1, TOK);
  const int each = split_tiles(a, list.count);
  const int begin = uniform(split * each), end = uniform(min(begin + each, list.count));
  if (begin >= end) return;
  const bool alone = each >= list.count;  // the rows' one split: no others to join

  // the rows' queries as B operands: column col, values 8 g .. of each 32 (8 bits: of each 64, 16 g ..)
  f16x8 query[C][KS][TERMS];
  float row_scale[C];
  uint32_t position[C], low[TREE ? C : 1];  // (TREE: a row's token, and what tree_low has)
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int r = c * 16 + col;
    const uint32_t row = row0 + min(r, rows - 1), token = row / group;
    position[c] = TREE ? token : (uint32_t)span.start + token;
    if constexpr (TREE) low[c] = (uint32_t)tree_low(a, span, token);
    const T* q = queries + ((span.first + token) * a.heads + kv * a.group + (row - token * group)) * (int64_t)a.dim;
    float v[KS][8];
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int d = I8 ? (k / 2) * 64 + g * 16 + (k % 2) * 8 : k * 32 + g * 8;
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
    most = max(most, (uint32_t)__shfl_xor((int)most, 16, kWave));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
    const bool finite = most < 0x7f800000u;
    const int shift = finite && most != 0 ? 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(most)) : 0;
    // a row with a NaN or an infinity: every score NaN
    row_scale[c] = finite ? ldexpf(a.scale * 1.44269504088896340736f, -shift) : __builtin_nanf("");
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = finite ? ldexpf(v[k][e], shift) : 0.0f;
      const Halves<TERMS> h = halves_of<TERMS>(x);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) query[c][k][t] = h.term[t];
    }
  }

  f32x4 acc[C][DT];
  float top[C], value_top[C], total[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    top[c] = value_top[c] = -kInfinity;
    total[c] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[c][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // a lane's unit of 16 positions of a tile, as a row of K and as a part of V
  const int key_unit = (col >> 2) * (TOK / 4) / 16, value_unit = g * (TOK / 4) / 16;
  const uint32_t units = p1 / 16;  // the last unit that a row sees
  // the page of unit u (-1: nothing of it is seen, or it names no page), and the unit's place in it
  auto page_of = [&](uint32_t u, uint32_t& off) -> int32_t {
    const uint32_t in = u > units ? units : u;
    const uint32_t column = a.columns.of(in);
    off = (in - column * a.columns.page_units) * 16;
    const int32_t page = span.table[column];
    return page;
  };
  struct Places {
    int32_t key_page, value_page;
    uint32_t key_off, value_off;
  };
  auto places_of = [&](int i) {
    Places w;
    const uint32_t unit = (uint32_t)list.tile(min(i, end - 1)) * NT;
    w.key_page = page_of(unit + key_unit, w.key_off);
    w.value_page = page_of(unit + value_unit, w.value_off);
    return w;
  };
  using KeyRaw = uint4;
  constexpr int kKeyLoads = I8 ? KS / 2 : KS;  // 16-byte loads a row
  KeyRaw keys[NT][kKeyLoads];
  auto load_keys = [&](const Places& w) {
    const int32_t page = (uint32_t)w.key_page < (uint32_t)a.p.cache_pages ? w.key_page : 0;
    const int r = col & 3;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t in = w.key_off + ((col >> 2) * (TOK / 4) + 4 * t + r) % 16;
      const int64_t at = (((int64_t)page * a.p.page_size + in) * a.kv_heads + kv) * a.dim;
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) {
        const int d = I8 ? k * 64 + g * 16 : k * 32 + g * 8;
        if constexpr (I8) {
          const int8_t* row = (const int8_t*)a.keys + at;
          if (a.dim == DP) {
            keys[t][k] = __builtin_bit_cast(uint4, *(const u32x4_8*)(row + d));
          } else {
            const u32x2 x = *(const u32x2*)(row + (d < a.dim ? d : 0)), y = *(const u32x2*)(row + (d + 8 < a.dim ? d + 8 : 0));
            keys[t][k] = make_uint4(x.x, x.y, y.x, y.y);
          }
        } else {
          keys[t][k] = *(const uint4*)((const uint16_t*)a.keys + at + (d < a.dim ? d : 0));
        }
      }
    }
  };

  // the values, and the scales in 8 bits
  uint4 values[DT];
  float key_scale[I8 ? 16 : 1], value_log[I8 ? 16 : 1];
  auto load_values = [&](const Places& w) {
    const int32_t page = (uint32_t)w.value_page < (uint32_t)a.p.cache_pages ? w.value_page : 0;
    const char* from = (const char*)a.values + (((int64_t)page * a.kv_heads + kv) * a.dim * a.p.page_size +
                                                w.value_off + (g * (TOK / 4)) % 16) * (I8 ? 1 : 2);
    const int64_t stride = (int64_t)a.p.page_size * (I8 ? 1 : 2);
#pragma unroll
    for (int d = 0; d < DT; ++d) values[d] = *(const uint4*)(from + min(d * 16 + col, a.dim - 1) * stride);
    if constexpr (I8) {
      const int64_t at = ((int64_t)page * a.kv_heads + kv) * a.p.page_size + w.value_off;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float4 x = *(const float4*)(a.key_scales + at + e), y = *(const float4*)(a.value_scales + at + e);
        key_scale[e] = x.x, key_scale[e + 1] = x.y, key_scale[e + 2] = x.z, key_scale[e + 3] = x.w;
        value_log[e] = y.x, value_log[e + 1] = y.y, value_log[e + 2] = y.z, value_log[e + 3] = y.w;
      }
    }
  };

  // keys and values of a tile are asked for as soon as the one before it is done with their registers, so that
  // both are on their way for a whole tile's time
  int i = begin + wave;
  Places now = places_of(i), next = places_of(i + kWaves);
  if (i < end) {
    load_keys(now);
    load_values(now);
  }
  for (; i < end; i += kWaves) {
    const uint32_t base = (uint32_t)list.tile(i) * TOK;
    const uint32_t mine = base + g * (TOK / 4);  // the lane's first position
    const bool okay = (uint32_t)now.value_page < (uint32_t)a.p.cache_pages;
    if (!okay && mine <= p1 &&
        (a.window == 0 || mine + TOK / 4 - 1 + (uint32_t)a.window > p0 || mine < (uint32_t)a.sinks))
      flag_bad(a.p);

    // scores: score[c][t][i] is row c 16 + col, position mine + 4 t + i
    f32x4 score[C][NT];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t) score[c][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        f16x8 key;
        if constexpr (I8) {
          const uint4 w = keys[t][k / 2];
          key = k % 2 ? codes_f16(w.z, w.w) : codes_f16(w.x, w.y);
        } else {
          key = __builtin_bit_cast(f16x8, keys[t][k]);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int m = 0; m < TERMS; ++m)
            score[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, query[c][k][m], score[c][t], 0, 0, 0);
      }
    // the next tile's keys on their way, and the places of the one after
    const Places coming = next;
    if (i + kWaves < end) load_keys(coming);
    next = places_of(i + 2 * kWaves);

    if constexpr (I8)
#pragma unroll
      for (int e = 0; e < 16; ++e) value_log[e] = __builtin_amdgcn_logf(value_log[e]);
    // whether every row sees the whole tile
    const bool whole = (TREE ? base + TOK <= (uint32_t)span.start : base + TOK - 1 <= p0) &&
                       (a.window == 0 || base + (uint32_t)a.window > p1 || base + TOK - 1 < (uint32_t)a.sinks) &&
                       __all(okay);
    float weight[C][NT][4];  // TOK / 4 consecutive positions
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float high = -kInfinity, value_high = -kInfinity;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = score[c][t][e] * row_scale[c];
          if constexpr (I8) x *= key_scale[4 * t + e];
          score[c][t][e] = x;
        }
      if constexpr (TREE) {
        if (!whole) {
          const uint32_t sees = okay ? (uint32_t)tree_sees(a, span, position[c], mine, low[TREE ? c : 0], a.sinks) : 0;
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) score[c][t][e] = sees >> (4 * t + e) & 1 ? score[c][t][e] : -kInfinity;
        }
      } else if (!whole) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t j = mine + 4 * t + e;
            const bool seen = okay & (j <= position[c]) &
                              ((a.window == 0) | (j + (uint32_t)a.window > position[c]) | (j < (uint32_t)a.sinks));
            score[c][t][e] = seen ? score[c][t][e] : -kInfinity;
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          high = fmaxf(high, score[c][t][e]);
          if constexpr (I8) {
            // (what is masked stays -infinity whatever its scale)
            const float x = score[c][t][e] + value_log[4 * t + e];
            weight[c][t][e] = !whole && score[c][t][e] == -kInfinity ? -kInfinity : x;
            value_high = fmaxf(value_high, weight[c][t][e]);
          }
        }
      high = fmaxf(column_max(high), top[c]);
      const float ref = high == -kInfinity ? 0.0f : high - kLift;
      const float keep = exp2_fast(top[c] - (high == -kInfinity ? 0.0f : high));
      float value_ref = ref, value_keep = keep;
      if constexpr (I8) {
        value_high = fmaxf(column_max(value_high), value_top[c]);
        value_ref = value_high == -kInfinity ? 0.0f : value_high - kLift;
        value_keep = exp2_fast(value_top[c] - (value_high == -kInfinity ? 0.0f : value_high));
        value_top[c] = value_high;
      }
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = exp2_fast(score[c][t][e] - ref);
          sum += p;
          weight[c][t][e] = I8 ? exp2_fast(weight[c][t][e] - value_ref) : p;
        }
      total[c] = fmaf(total[c], keep, sum);
      top[c] = high;
      if (__any(value_keep != 1.0f))
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[c][d][e] *= value_keep;
    }

    // values that no row of the block sees count as zeros: they may hold anything (in 8 bits every code is a number)
    if (!I8 && !whole) {
      uint32_t keep[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        keep[e] = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t j = mine + 2 * e + half;
          const bool seen = okay & (j <= p1) &
                            ((a.window == 0) | (j + (uint32_t)a.window > p0) | (j < (uint32_t)a.sinks));
          keep[e] |= seen ? 0xffffu << (16 * half) : 0u;
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        values[d].x &= keep[0];
        values[d].y &= keep[1];
        values[d].z &= keep[2];
        values[d].w &= keep[3];
      }
    }
#pragma unroll
    for (int n = 0; n < TOK / 32; ++n) {
      Halves<kWeightTerms> weights[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = weight[c][2 * n + e / 4][e % 4];
        weights[c] = halves_of<kWeightTerms>(x);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f16x8 value;
        if constexpr (I8) value = n ? codes_f16(values[d].z, values[d].w) : codes_f16(values[d].x, values[d].y);
        else value = __builtin_bit_cast(f16x8, values[d]);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int m = 0; m < kWeightTerms; ++m)
            acc[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, weights[c].term[m], acc[c][d], 0, 0, 0);
      }
    }
    if (i + kWaves < end) load_values(coming);
    now = coming;
  }

  // the waves' results joined, 16 rows at a time
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const float sum = column_sum(total[c]);
    if (g == 0) {
      stats[wave][c * 16 + col][0] = top[c];
      stats[wave][c * 16 + col][1] = sum;
      stats[wave][c * 16 + col][2] = I8 ? value_top[c] : top[c];
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) *(f32x4*)&merged[wave][col][d * 16 + g * 4] = acc[c][d];
    __syncthreads();
    uint32_t again = 0;  // rows of this wave that came out as no numbers
    for (int r = wave; r < 16; r += kWaves) {
      if (c * 16 + r >= rows) break;
      float m = -kInfinity, vm = -kInfinity;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        m = fmaxf(m, stats[w][c * 16 + r][0]);
        vm = fmaxf(vm, stats[w][c * 16 + r][2]);
      }
      const float ref = m == -kInfinity ? 0.0f : m, value_ref = vm == -kInfinity ? 0.0f : vm;
      float l = 0.0f, factor[kWaves];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        l = fmaf(stats[w][c * 16 + r][1], exp2_fast(stats[w][c * 16 + r][0] - ref), l);
        factor[w] = exp2_fast(stats[w][c * 16 + r][2] - value_ref);
      }
      const uint32_t row = row0 + c * 16 + r, token = row / group;
      const int h = kv * a.group + (int)(row - token * group);
      const int64_t place = (span.first + token) * a.heads + h;
      const int64_t partial = few_partial(a, s, kv, row, place);
      const float inverse = l == 0.0f ? 0.0f : (I8 ? exp2_fast(value_ref - ref) : 1.0f) / l;
      bool odd = false;
      for (int d = lane; d < a.dim; d += kWave) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x = fmaf(merged[w][r][d], factor[w], x);
        if (alone) {
          x *= inverse;
          odd |= !(fabsf(x) < kInfinity);
          store_one(out + place * a.dim + d, x);
        } else {
          a.partials[((int64_t)split * a.partial_rows + partial) * a.dim + d] = x;
        }
      }
      if (alone) {
        // a row of -infinity alone, as one of NaN, is taken again
        if (__any(odd) || (l == 0.0f && m == -kInfinity)) again |= 1u << r;
      } else if (lane == 0) {
        float* st = a.statistics + ((int64_t)split * a.partial_rows + partial) * 3;
        st[0] = m, st[1] = l, st[2] = vm;
      }
    }
    if (alone) {
      __syncthreads();  // merged is free, and holds the scratch
      RowScratch& scratch = *reinterpret_cast<RowScratch*>(&merged[wave][0][0]);
      for (; again; again &= again - 1) {
        const uint32_t row = row0 + c * 16 + __ffs(again) - 1;
        attend_row<T, I8, TREE>(queries, out, a, span, row / group, kv * a.group + (int)(row % group), scratch);
      }
    }
  }
}

template <typename T, bool I8, bool TREE, int DP, int C>
__global__ void __launch_bounds__(256, C == 1 && DP <= 128 ? 2 : 1) attend_few(const T* queries, T* out, ArgsOf<TREE> a) {
  __shared__ FewShared<DP, C> shared;
  few_block<T, I8, TREE, DP, C>(queries, out, a, blockIdx.x, shared);
}

// The many-rows kernel: 32 rows of queries a wave, four or eight waves a block
// (plan_of says when), positions in tiles of 64 that the block stages in LDS once
// for all its rows, by 32 x 32 x 16 products. As in attend_few
// the scores are taken transposed (the result's column, lane % 32, is a row of
// queries), with the rows of K dealt out so that the 8 weights a lane brings to
// each product of O^T = V^T P^T are those it holds (bits 2 and 3 of the row's
// number trade places).
//
// LDS: keys [64][DP], values [DP][64] in F16 (codes are made F16 numbers as they
// are staged), 16-byte chunks moved by an exclusive or with the row's number so
// that the rows of one operand lie on different banks; twice, so that a block needs
// one barrier a tile. The next tile comes meanwhile: F16 straight into LDS, 8 bits by
// registers.
//
// The maximum that weights are taken against is raised only when a score passes
// it by more than kSlack (in powers of two), which keeps the rescaling of the
// results out of most tiles: weights then reach 2^(kManyLift + kSlack) at most.
//
// What bounds it are the waits between scores, weights and products, which two waves a
// SIMD (by registers; one for heads of 256) cover in part: of the time of 8,192 BF16 tokens
// of a prompt, 32 heads over 8 of 128, 605 us (550 GFLOP, 909 TFLOP/s), vector instructions
// issue 47% and matrix products run 39%; of 4,096 tokens in windows of 1,024, heads of 64,
// 42 us (410 TFLOP/s), 43 and 15%; of 509 F32 tokens after 3,591, 16 heads over 2 of 256, 97
// us with the join (two terms of 32 GFLOP), 25 and 26%; of 1,021 after 2,500 over 8 bits, 106
// us with the join, 44 and 19%.
template <bool I8, int DP>
struct ManyTile {
  static constexpr int kValues = 64 * DP * 2, kScales = 2 * kValues, kExponents = kScales + 2 * 64 * 4;
  static constexpr int kRange = kExponents + 64 * 4;
  static constexpr int kBytes = I8 ? (kRange + 16 + 255) / 256 * 256 : kScales;
};

template <typename T, bool I8, bool TREE, int DP, int WAVES>
__device__ __forceinline__ void many_block(const T* queries, T* out, const ArgsOf<TREE>& a, unsigned block,
                                           unsigned blocks, char (&tiles)[2 * ManyTile<I8, DP>::kBytes]) {
  // BF16's weights have one term, 11 bits: a row's result is then within 2^-11 of its values' sizes before it is rounded
  // to 8 bits, and over many positions their roundings cancel (0.0017 off 64 bits either way, the rounding to BF16's
  // own). A second term costs a fifth to a third: prefill 647 us, 851 with it, window chunk 47 / 56, mixed batch
  // 177 / 225, chunk over 8 bits 120 / 141. Trees' weights have 22 bits: which kernel has a tree's rows depends on the
  // call's other trees, and their precision must not (32 trees of 601 nodes after up to 8,000 positions 175 us, 157
  // with one term, 16 of 811 over 8 bits 125 / 102; of BF16 results one in twelve was another than the F32 one's rounding).
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1, kWeightTerms = TREE ? 2 : TERMS;
  constexpr int kThreads = 64 * WAVES;
  constexpr int kRows = WAVES * 32;  // rows a block
  constexpr int TOK = 64, KS = DP / 16, DT = DP / 32;
  constexpr int kKeyChunks = DP / 8;         // of a position
  constexpr float kSlack = kWeightTerms == 2 ? 1.0f : 8.0f, kManyLift = 15.0f - kSlack;
  constexpr int kLoads = TOK * kKeyChunks / kThreads;  // chunks a thread stages, of keys and of values
  // a tile in LDS: its keys, its values, and in 8 bits their scales, the exponents of the values' (-infinity: no scale
  // above 0) and the most and the least of them
  using Layout = ManyTile<I8, DP>;
  constexpr int kValuesAt = Layout::kValues, kScalesAt = Layout::kScales, kExponentsAt = Layout::kExponents;
  constexpr int kRangeAt = Layout::kRange;
  constexpr int kTileBytes = Layout::kBytes;
  static_assert(sizeof(RowScratch) * WAVES <= sizeof(tiles), "");

  const int thread = threadIdx.x, lane = thread & 63, wave = uniform(thread >> 6), col = lane & 31, h = lane >> 5;
  const int kv = block % (unsigned)a.kv_heads;
  const unsigned rest = block / (unsigned)a.kv_heads;
  // A unit's splits lie far apart, as in attend_few (a mixed batch of 4 key heads in two splits 171 us, 218 with
  // neighbours: half the dies idle); the last rows first: they have the most positions
  const unsigned all_units = blocks / (unsigned)(a.kv_heads * a.splits);
  const int split = rest / all_units;
  const int64_t unit = all_units - 1 - rest % all_units;
  int64_t nth;
  const int s = locate(a.p, unit, kRows, 0, a.group, nth, a.few_rows);
  if (s < 0) return;
  const Span span = span_of<true>(a.p, s);
  const int rows = (int)min((int64_t)span.rows * a.group - nth * kRows, (int64_t)kRows);
  if (rows <= 0 || (int64_t)span.rows * a.group <= a.few_rows) return;
  const uint32_t row0 = (uint32_t)nth * kRows, group = (uint32_t)a.group, start = (uint32_t)span.start;
  const uint32_t p0 = (uint32_t)first_position<TREE>(span, row0 / group);
  const uint32_t p1 = (uint32_t)last_position<TREE>(span, (row0 + rows - 1) / group);
  const TileList list = tiles_of(a, p0, p1, TOK);
  const int each = split_tiles(a, list.count);
  const int begin = uniform(split * each), end = uniform(min(begin + each, list.count));
  if (begin >= end) return;
  const bool alone = each >= list.count;  // the rows' one split: no others to join

  // ---- this wave's rows
  const int wave_row = wave * 32;
  const bool idle = wave_row >= rows;
  const uint32_t w0 = (uint32_t)first_position<TREE>(span, (row0 + min(wave_row, rows - 1)) / group);
  const uint32_t w1 = (uint32_t)last_position<TREE>(span, (row0 + min(wave_row + 32, rows) - 1) / group);
  f16x8 query[KS][TERMS];
  const uint32_t row = row0 + min(wave_row + col, rows - 1), token = row / group;
  const uint32_t position = start + token;
  uint32_t row_low = 0;
  if constexpr (TREE) row_low = (uint32_t)tree_low(a, span, token);
  const T* q = queries + ((span.first + token) * a.heads + kv * a.group + (row - token * group)) * (int64_t)a.dim;
  uint32_t most = 0;
  float v[KS][8];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int d = k * 16 + h * 8;
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
  most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
  const bool finite = most < 0x7f800000u;
  const int shift = finite && most != 0 ? 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(most)) : 0;
  // (above 0, so that the largest score is the largest product: a negative scale turns the query's sign. A scale
  // of 0, or one that a tiny row makes it, is small enough to leave every weight even; a NaN stays one)
  const float row_scale = finite && a.scale == a.scale
                              ? fmaxf(ldexpf(fabsf(a.scale) * 1.44269504088896340736f, -shift), 0x1p-120f)
                              : __builtin_nanf("");
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = finite ? ldexpf(v[k][e], shift) : 0.0f;
      if (a.scale < 0.0f) x[e] = -x[e];
    }
    const Halves<TERMS> half = halves_of<TERMS>(x);
#pragma unroll
    for (int t = 0; t < TERMS; ++t) query[k][t] = half.term[t];
  }
  f32x16 acc[DT];
  const float row_inverse = 1.0f / row_scale;
  float ref = -kInfinity, total = 0.0f;  // what weights are taken against, and their sum so far
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.0f;

  // ---- staging: a thread's chunks of a tile
  // Chunk n of a thread is of a unit that its whole wave shares, so that a load is
  // a scalar base and an offset that stays. Where pages hold whole tiles, eight
  // chunks of a value's row lie together; else two.
  const uint32_t last_unit = p1 / 16;
  const bool wide = a.columns.page_units % 4 == 0;
  constexpr int kUnitThreads = 2 * DP;  // threads that stage a unit's keys, or its values where pages are narrow
  constexpr int kUnits = kThreads >= kUnitThreads ? kThreads / kUnitThreads : 1;  // units that all threads stage at once
  const int wave_unit = kUnits > 1 ? wave / (kUnitThreads / 64) : 0;
  constexpr int kBytes = I8 ? 1 : 2;
  // bytes of a page (the same for keys and values), of a position's keys, and where this head's lie in a page
  const uint32_t page_bytes = (uint32_t)a.p.page_size * a.kv_heads * a.dim * kBytes;
  const uint32_t position_bytes = (uint32_t)a.kv_heads * a.dim * kBytes, key_head = (uint32_t)kv * a.dim * kBytes;
  const uint32_t value_head = (uint32_t)kv * a.dim * a.p.page_size * kBytes;
  // A tile's four units, one a lane of four: the page table's entries, asked for
  // two tiles ahead, and where they lie.
  int32_t entry;
  uint32_t entry_off;
  auto load_entries = [&](int i) {
    const uint32_t at = min((uint32_t)list.tile(min(i, end - 1)) * 4 + (lane & 3), last_unit);
    const uint32_t column = a.columns.of(at);
    entry_off = (at - column * a.columns.page_units) * 16;
    entry = span.table[column];
  };
  struct Pages {
    uint64_t from;  // the unit's page, in bytes from the first
    uint32_t off;   // its first position in the page
    uint32_t page;
    uint32_t okay;  // bit u: unit u's page is one of the cache's
  };
  auto pages_of = [&]() {
    const bool okay = (uint32_t)entry < (uint32_t)a.p.cache_pages;
    const uint32_t page = okay ? entry : 0;
    return Pages{(uint64_t)page * page_bytes, entry_off, page, (uint32_t)__ballot(okay) & 15u};
  };
  auto at_lane = [](uint64_t x, int u) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, u);
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), u) << 32) | lo;
  };
  // the unit of a thread's chunk n of keys
  auto unit_of = [&](int n) { return kUnits == 1 ? n * kThreads / kUnitThreads : (n * kUnits & 3) + wave_unit; };
  // where a tile has chunk `chunk` of position `token`, or of value d
  auto key_place = [](int token, int chunk) {
    return (token * kKeyChunks + (chunk ^ (DP >= 128 ? token & 15 : (token >> 1) & 7))) * 16;
  };
  auto value_place = [](int d, int chunk) { return kValuesAt + (d * 8 + (chunk ^ ((d >> 1) & 7))) * 16; };
  // whether some row of the block sees position j
  auto some_see = [&](uint32_t j) {
    return (j <= p1) & ((a.window == 0) | (j + (uint32_t)a.window > p0) | (j < (uint32_t)a.sinks));
  };
  auto flag_units = [&](uint32_t base, uint32_t okay) {
    if (okay != 15u && thread < TOK && !(okay >> (thread / 16) & 1) && some_see(base + thread)) flag_bad(a.p);
  };

  // F16: straight into LDS. A thread's chunk goes to the place of its number, so it asks for the chunk that belongs there.
  typedef const __attribute__((address_space(1))) void* Global;
  typedef __attribute__((address_space(3))) void* Local;
  auto copy_tile = [&](const Pages& w, int to) {
    const uint64_t key_from = w.from + w.off * position_bytes, value_from = w.from + w.off * kBytes;
    int me = thread;
    asm volatile("" : "+v"(me));  // (or every chunk's offset is kept in registers)
    // the exclusive or is the same for all a thread's chunks, but for bit 3 where a step of n is 8 positions
    constexpr int kStep = kThreads / kKeyChunks;
    const int token = me / kKeyChunks, key_chunk = me % kKeyChunks ^ (DP >= 128 ? token & 15 : (token >> 1) & 7);
    const uint32_t row = (uint32_t)(token % 16) * position_bytes;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int chunk = kStep % 16 ? key_chunk ^ (n * kStep & 8) : key_chunk;
      const char* from = (const char*)a.keys + at_lane(key_from, unit_of(n)) + (key_head + n * kStep % 16 * position_bytes) +
                         (row + (chunk * 8 < a.dim ? chunk * 16 : 0));
      __builtin_amdgcn_global_load_lds((Global)from, (Local)(tiles + to + (wave * 64 + n * kThreads) * 16), 16, 0, 0);
    }
    const int d = me >> 3, value_chunk = (me & 7) ^ ((d >> 1) & 7);
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)value_from, value_chunk >> 1, kWave);
    const uint64_t from = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(value_from >> 32), value_chunk >> 1, kWave) << 32) | lo;
    const char* head = (const char*)a.values + from + (value_head + (value_chunk & 1) * 16);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const uint32_t at = (uint32_t)min(d + n * (kThreads / 8), a.dim - 1) * a.p.page_size * 2;
      __builtin_amdgcn_global_load_lds((Global)(head + at), (Local)(tiles + to + kValuesAt + (wave * 64 + n * kThreads) * 16), 16, 0, 0);
    }
  };
  // Values that no row of the block sees count as zeros: they may hold anything. Each thread mends the chunks it asked
  // for, once they have come.
  auto mend_tile = [&](int at, int i, uint32_t okay) {
    const uint32_t base = (uint32_t)list.tile(i) * TOK;
    if (okay == 15u && base + TOK - 1 <= p1 &&
        (a.window == 0 || base + (uint32_t)a.window > p0 || base + TOK - 1 < (uint32_t)a.sinks))
      return;
    flag_units(base, okay);
    const int chunk = (thread & 7) ^ ((thread >> 4) & 7);
    uint32_t keep[4] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      keep[e / 2] |= (bool)(okay >> (chunk / 2) & 1) & some_see(base + chunk * 8 + e) ? e % 2 ? 0xffff0000u : 0xffffu : 0u;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      uint4* place = (uint4*)(tiles + at + kValuesAt + (thread + n * kThreads) * 16);
      const uint4 x = *place;
      *place = make_uint4(x.x & keep[0], x.y & keep[1], x.z & keep[2], x.w & keep[3]);
    }
  };

  // 8 bits: by registers, made F16 numbers on the way.
  uint2 key_raw[I8 ? kLoads : 1], value_raw[I8 ? kLoads : 1];
  float scale_raw = 0.0f;
  auto load_tile = [&](const Pages& w) {
    const uint64_t key_from = w.from + w.off * position_bytes, value_from = w.from + w.off * kBytes;
    int me = thread;
    asm volatile("" : "+v"(me));
    const int chunk0 = me % kKeyChunks * 8;
    const uint32_t key_at = (uint32_t)(me / kKeyChunks % 16) * position_bytes + (chunk0 < a.dim ? chunk0 : 0);
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      key_raw[n] = *(const uint2*)((const char*)a.keys + at_lane(key_from, unit_of(n)) +
                                   (key_head + n * kThreads / kKeyChunks % 16 * position_bytes) + key_at);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int q = me + kThreads * n, d = min(wide ? q >> 3 : (q >> 1) % DP, a.dim - 1);
      const uint32_t value_at = (uint32_t)d * a.p.page_size + (wide ? me & 7 : me & 1) * 8;
      value_raw[n] = *(const uint2*)((const char*)a.values + at_lane(value_from, wide ? 0 : unit_of(n)) + value_head + value_at);
    }
    // wave 0 brings the keys' scales, wave 1 the values'
    if (wave < 2) {
      const uint32_t row = (uint32_t)__shfl((int)(w.page * (uint32_t)a.kv_heads + kv), lane / 16, kWave);
      const uint32_t off = (uint32_t)__shfl((int)w.off, lane / 16, kWave);
      scale_raw = (wave == 0 ? a.key_scales : a.value_scales)[(uint64_t)row * a.p.page_size + off + lane % 16];
    }
  };
  constexpr int kNone = -1000;  // no scale above 0
  auto store_tile = [&](char* tile, int i, uint32_t okay) {
    const uint32_t base = (uint32_t)list.tile(i) * TOK;
    flag_units(base, okay);
    int me = thread;
    asm volatile("" : "+v"(me));
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int q = me + kThreads * n;
      *(uint4*)(tile + key_place(q / kKeyChunks, q % kKeyChunks)) =
          __builtin_bit_cast(uint4, codes_f16(key_raw[n].x, key_raw[n].y));
    }
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int q = me + kThreads * n, d = wide ? q >> 3 : (q >> 1) % DP;
      *(uint4*)(tile + value_place(d, wide ? q & 7 : q / kUnitThreads * 2 + (q & 1))) =
          __builtin_bit_cast(uint4, codes_f16(value_raw[n].x, value_raw[n].y));
    }
    // (every code is a number: what no row sees needs a scale of 0 alone)
    float* scales = (float*)(tile + kScalesAt);
    if (wave == 0) scales[lane] = scale_raw;
    else if (wave == 1) {
      const float x = (bool)(okay >> (lane / 16) & 1) & some_see(base + lane) ? scale_raw : 0.0f;
      scales[TOK + lane] = x;
      const bool counts = x > 0.0f && x < kInfinity;
      const float exponent = (float)__builtin_amdgcn_frexp_expf(x);
      ((float*)(tile + kExponentsAt))[lane] = counts ? exponent : -kInfinity;
      const float most = group_max<64>(counts ? exponent : (float)kNone);
      const float least = -group_max<64>(counts ? -exponent : (float)kNone);
      if (lane == 0) *(int2*)(tile + kRangeAt) = make_int2((int)most, (int)least);
    }
  };
  // operands: chunk 2 k + h of the lane's position, and chunk 2 n + h of its value: the exclusive or with k and n
  // (chunks of 16 bytes, in the low bits of places that are multiples of 128) gives them from one place each
  const int key_row = (col & ~12) | ((col & 4) << 1) | ((col & 8) >> 1);
  const int key_from = key_place(key_row, h), value_from = value_place(col, h);
  // In 8 bits weights are taken times the values' scales over 2^value_exponent: an F16 number keeps that for scales
  // within 2^kNear of the largest so far, whose exponent it then is. Where scales lie further apart (a row of a value
  // next to 0 among others) it is a row's own from there on: that of its largest weight times scale, so that a row keeps
  // its bits whatever scales it hardly weighs (1,024 tokens after 6,000, 16 heads over 4 of 128, one value row 2^-30 of
  // the others: 144 us, 132 without that row).
  constexpr int kNear = 16, kLeastExponent = -100;  // (a scale below 2^28 over 2^kLeastExponent is a number)
  int most_exponent = kNone, least_exponent = -kNone;  // of the values' scales so far
  int value_exponent = kNone;
  // A tile comes while the one before it is used (8 bits: is written then, and is in registers a tile before that).
  load_entries(begin);
  Pages pages = pages_of();
  uint32_t okay = pages.okay, okay_now = okay;
  if constexpr (I8) load_tile(pages);
  else copy_tile(pages, 0);
  load_entries(begin + 1);
  if constexpr (I8) {
    store_tile(tiles, begin, okay);
    if (begin + 1 < end) {
      pages = pages_of();
      load_tile(pages);
      okay = pages.okay;
      load_entries(begin + 2);
    }
  }
  for (int i = begin; i < end; ++i) {
    int now = uniform(((i - begin) & 1) * kTileBytes);
    asm volatile("" : "+s"(now));  // (or both buffers' every address is kept in registers)
    char* tile = tiles + now;
    if constexpr (!I8) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the tile has come
      mend_tile(now, i, okay_now);
    }
    __syncthreads();
    const uint32_t okay_then = okay_now;
    if (i + 1 < end) {
      if constexpr (I8) {
        store_tile(tiles + (kTileBytes - now), i + 1, okay);
        okay_now = okay;
        if (i + 2 < end) {
          pages = pages_of();
          load_tile(pages);
          okay = pages.okay;
          load_entries(i + 3);
        }
      } else {
        pages = pages_of();
        copy_tile(pages, kTileBytes - now);
        okay_now = pages.okay;
        load_entries(i + 2);
      }
    }
    const uint32_t base = (uint32_t)list.tile(i) * TOK;
    // whether any, and whether every row of the wave sees the tile
    if (idle || base > w1) continue;
    if (a.window && base + TOK - 1 + (uint32_t)a.window <= w0 && base >= (uint32_t)a.sinks) continue;
    const bool whole = okay_then == 15u && (TREE ? base + TOK <= start : base + TOK - 1 <= w0) &&
                       (a.window == 0 || base + (uint32_t)a.window > w1 || base + TOK - 1 < (uint32_t)a.sinks);
    bool apart = false, change = false;
    float factor = 1.0f;  // what the results so far are multiplied by, where there is a change
    if constexpr (I8) {
      const int2 range = *(const int2*)(tile + kRangeAt);
      const int most = max(uniform(range.x), -126);
      least_exponent = min(least_exponent, uniform(range.y));
      const int before = most_exponent;
      most_exponent = max(most_exponent, most);
      apart = most_exponent - least_exponent > kNear;
      if (!apart && most > before) {
        factor = before == kNone ? 0.0f : exp2_fast((float)(before - most));
        value_exponent = most;
        change = true;
      }
    }
    // scores: score[half][e] is row col, position base + 32 half + 16 (e / 8) + 8 h + e % 8
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
    }
    if constexpr (I8) {
      const float* scales = (const float*)(tile + kScalesAt) + h * 8;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 x = *(const float4*)(scales + half * 32 + e / 8 * 16 + e % 8);
          score[half][e] *= x.x, score[half][e + 1] *= x.y;
          score[half][e + 2] *= x.z, score[half][e + 3] *= x.w;
        }
    }
    if (!whole) {
      if constexpr (TREE) {
        const uint64_t sees = tree_sees(a, span, token, base, row_low, a.sinks) >> (h * 8);
#pragma unroll
        for (int n = 0; n < 32; ++n)
          score[n / 16][n % 16] = sees >> (n / 8 * 16 + n % 8) & 1 ? score[n / 16][n % 16] : -kInfinity;
      } else {
        int mine = (int)base + h * 8;
        asm volatile("" : "+v"(mine));  // (or what depends on it alone is kept for every tile)
        const int last = (int)position, low = a.window ? last - a.window + 1 : INT32_MIN;
#pragma unroll
        for (int n = 0; n < 32; ++n) {
          const int j = mine + n / 8 * 16 + n % 8;
          const bool seen = (j <= last) & ((j >= low) | (j < a.sinks));
          score[n / 16][n % 16] = seen ? score[n / 16][n % 16] : -kInfinity;
        }
      }
      if (okay_then != 15u)
#pragma unroll
        for (int n = 0; n < 32; ++n)
          if (!(okay_then >> (n / 8) & 1)) score[n / 16][n % 16] = -kInfinity;
    }
    __builtin_amdgcn_s_setprio(0);
    // Whether a score passes what weights are taken against by more than kSlack: while that bound is not below 0,
    // the numbers' bits compare as whole numbers do (a NaN among them passes it), which takes half the
    // instructions of a maximum that must quieten NaN. The maximum itself is taken only then, by whole numbers too (a
    // row with a NaN is NaN whatever its weights are taken against).
    const float bound = (ref + kSlack) * row_inverse;
    int most = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      most = max(most, max(__float_as_int(score[0][e]), __float_as_int(score[1][e])));
    if (__any(!(bound >= 0.0f) || most > __float_as_int(bound))) {
      // (the bits of numbers as whole numbers in order: those of negative ones turned)
      auto ordered = [](float x) { const int b = __float_as_int(x); return b ^ (int)((uint32_t)(b >> 31) >> 1); };
      int top = ordered(score[0][0]);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, max(ordered(score[0][e]), ordered(score[1][e])));
      const float high = __int_as_float(top ^ (int)((uint32_t)(top >> 31) >> 1));
      const float next = fmaxf(ref, fmaxf(high, __shfl_xor(high, 32, kWave)) * row_scale);
      const float to = next == -kInfinity ? 0.0f : next;
      total *= exp2_fast(ref - to);
      float down = 0.0f;
      if constexpr (I8)
        if (apart) {  // the results keep their size (up to doubled), and weights to come are taken times 2^down
          const float room = (float)max(value_exponent - kLeastExponent, 0);
          down = ceilf(fminf(fmaxf(next - ref, 0.0f), room));
          value_exponent -= (int)down;
        }
      factor *= exp2_fast(ref + down - to);
      ref = next;
      change = true;
    }
    const float lift = kManyLift - (ref == -kInfinity ? 0.0f : ref);
    if constexpr (I8)
      if (apart) {
        // a power of two that is no less than the row's largest weight times scale, over 2^kManyLift
        float high = -kInfinity;
#pragma unroll
        for (int n = 0; n < 32; n += 4) {
          const float4 x = *(const float4*)((const float*)(tile + kExponentsAt) + h * 8 + n / 8 * 16 + n % 8);
          const float exponent[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            high = fmaxf(high, fmaf(score[n / 16][n % 16 + e], row_scale, lift - kManyLift) + exponent[e]);
          __builtin_amdgcn_sched_barrier(0);
        }
        high = fmaxf(high, __shfl_xor(high, 32, kWave));
        const int next = max(value_exponent, (int)ceilf(fminf(fmaxf(high, (float)kLeastExponent), 126.0f)));
        factor = ldexpf(factor, max(value_exponent - next, -200));
        value_exponent = next;
        change = true;
      }
    if (change)
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] *= factor;
    // 16 positions at a time, the next ones' weights made between the products of these
    Halves<kWeightTerms> weights[2];
    auto weigh = [&](int n, Halves<kWeightTerms>& to) {
      float value_scale[I8 ? 8 : 1];
      if constexpr (I8) {
        const float* scales = (const float*)(tile + kScalesAt) + TOK + h * 8 + n * 16;
#pragma unroll
        for (int e = 0; e < 8; ++e) value_scale[e] = ldexpf(scales[e], -value_exponent);
      }
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = exp2_fast(fmaf(score[n / 2][n % 2 * 8 + e], row_scale, lift));
        total += p;
        w[e] = I8 ? p * value_scale[e] : p;
      }
      to = halves_of<kWeightTerms>(w);
    };
    f16x8 values[2][DT];
    auto load_values = [&](int n, f16x8 (&to)[DT]) {
#pragma unroll
      for (int d = 0; d < DT; ++d) to[d] = *(const f16x8*)(tiles + ((now + value_from) ^ (n * 32)) + d * 4096);
    };
    load_values(0, values[0]);
    weigh(0, weights[0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n < 3) {
        load_values(n + 1, values[(n + 1) % 2]);
        weigh(n + 1, weights[(n + 1) % 2]);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int m = 0; m < kWeightTerms; ++m)
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(values[n % 2][d], weights[n % 2].term[m], acc[d], 0, 0, 0);
      if (n < 3) {
        constexpr int kVector = (I8 ? 48 : 32) + (kWeightTerms == 2 ? 24 : 0);  // about what the weights take
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          __builtin_amdgcn_sched_group_barrier(kProducts, kWeightTerms, 0);
          __builtin_amdgcn_sched_group_barrier(kReads, 1, 0);
          __builtin_amdgcn_sched_group_barrier(kVectors, kVector / DT, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  if (value_exponent == kNone) value_exponent = 0;
  uint64_t again;
  const int r = wave_row + col;
  const bool there = r < rows;
  const int64_t place = (span.first + token) * a.heads + kv * a.group + (row - token * group);
  const float sum = total + __shfl_xor(total, 32, kWave);
  bool odd = sum == 0.0f && ref == -kInfinity;
  if (alone) {
    const float inverse = sum == 0.0f ? 0.0f : (I8 ? exp2_fast((float)value_exponent) : 1.0f) / sum;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int at = d * 32 + 2 * e + 4 * h;
        float x[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          x[n] = acc[d][e + n] * inverse;
          odd |= !(fabsf(x[n]) < kInfinity);
        }
        if (there && at < a.dim) {
          if constexpr (TERMS == 2) *(float4*)(out + place * a.dim + at) = make_float4(x[0], x[1], x[2], x[3]);
          else *(uint2*)(out + place * a.dim + at) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        }
      }
    again = __ballot(odd && there);
  } else {
    const int64_t at = (int64_t)split * a.partial_rows + place;
    if (there) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (d * 32 + 2 * e + 4 * h < a.dim)
            *(f32x4*)(a.partials + at * a.dim + d * 32 + 2 * e + 4 * h) =
                f32x4{acc[d][e], acc[d][e + 1], acc[d][e + 2], acc[d][e + 3]};
      if (h == 0) {
        a.statistics[at * 3] = ref;
        a.statistics[at * 3 + 1] = sum;
        a.statistics[at * 3 + 2] = ref + (float)value_exponent;
      }
    }
    again = 0;
  }
  __syncthreads();  // the tiles are free, and hold the scratch
  RowScratch& scratch = reinterpret_cast<RowScratch*>(tiles)[wave];
  for (uint32_t rest_rows = (uint32_t)again | (uint32_t)(again >> 32); rest_rows; rest_rows &= rest_rows - 1) {
    const uint32_t row = row0 + wave_row + __ffs(rest_rows) - 1;
    attend_row<T, I8, TREE>(queries, out, a, span, row / group, kv * a.group + (int)(row % group), scratch);
  }
}

template <typename T, bool I8, bool TREE, int DP, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, DP > 128 ? 1 : 2) attend_many(const T* queries, T* out, ArgsOf<TREE> a) {
  __shared__ __attribute__((aligned(16))) char tiles[2 * ManyTile<I8, DP>::kBytes];
  many_block<T, I8, TREE, DP, WAVES>(queries, out, a, blockIdx.x, gridDim.x, tiles);
}

// Both in one launch: the chunks' blocks, then the single tokens', whose reads fill the
// time that the last chunks' products leave. 6 chunks (1,793 tokens) and 18 single tokens
// over up to 6,000 positions, 28 heads over 4 of 128: 162 us, 226 in launches of their
// own. The longest chunk's blocks bound it.
template <typename T, bool I8, bool TREE, int DP>
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) attend_both(const T* queries, T* out, ArgsOf<TREE> few,
                                                                     ArgsOf<TREE> many, unsigned many_blocks) {
  constexpr size_t kMany = 2 * ManyTile<I8, DP>::kBytes, kFew = sizeof(FewShared<DP, 1>);
  __shared__ __attribute__((aligned(16))) char shared[kMany > kFew ? kMany : kFew];
  if (blockIdx.x < many_blocks)
    many_block<T, I8, TREE, DP, 4>(queries, out, many, blockIdx.x, many_blocks, reinterpret_cast<char (&)[kMany]>(shared));
  else
    few_block<T, I8, TREE, DP, 1>(queries, out, few, blockIdx.x - many_blocks, reinterpret_cast<FewShared<DP, 1>&>(shared));
}

// Joins the splits of attend_few (FEW) or attend_many: a block takes up to
// kJoinRows rows of one unit (`rows` of them, tiles of `tile` positions, which say
// how many splits it had), a row by as many lanes as hold its values in fours.
template <bool FEW>
constexpr int kJoinRows = FEW ? 16 : 32;

template <typename T, bool I8, bool TREE, bool FEW, int DP>
__device__ __forceinline__ void join_block(const T* queries, T* out, const ArgsOf<TREE>& a, unsigned block, int rows,
                                           int tile, RowScratch (&scratch)[4]) {
  // (many rows have few splits: two fours a lane let each wave have twice the rows on the way; 2 splits of 32,672 rows
  // of 128 values 9.4 us, 11.5 by one)
  constexpr int V = FEW ? 1 : 2, N = FEW ? 8 : 4;  // fours of values a lane, splits at a time
  constexpr int L = DP / 4 / V, kRows = kJoinRows<FEW>;  // lanes a row, rows a block
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), in = lane % L;
  const int parts = rows / kRows;
  const int kv = block % (unsigned)a.kv_heads, part = block / (unsigned)a.kv_heads % (unsigned)parts;
  const unsigned unit = block / (unsigned)a.kv_heads / (unsigned)parts;
  int s;
  int64_t nth;
  if constexpr (FEW) s = (int)(unit % (unsigned)a.p.sequences), nth = unit / (unsigned)a.p.sequences;
  else s = locate(a.p, unit, rows, 0, a.group, nth, a.few_rows);
  if (s < 0) return;
  const Span span = span_of<!FEW>(a.p, s);
  const uint32_t all = (uint32_t)span.rows * (uint32_t)a.group, group = (uint32_t)a.group;
  const uint32_t row0 = (uint32_t)nth * rows;
  if (row0 + part * kRows >= all || (all <= (uint32_t)a.few_rows) != FEW) return;
  const uint32_t last = min(row0 + rows, all) - 1, end = min(row0 + (part + 1) * kRows, last + 1);
  const TileList list = tiles_of(a, first_position<TREE>(span, row0 / group), last_position<TREE>(span, last / group), tile);
  const int each = split_tiles(a, list.count), splits = (list.count + each - 1) / each;
  if (splits == 1) return;
  for (uint32_t first = row0 + part * kRows + wave * (64 / L); first < end; first += 4 * (64 / L)) {
    const uint32_t mine = first + lane / L, row = min(mine, end - 1), token = row / group;
    const int h = kv * a.group + (int)(row - token * group);
    const int64_t place = (span.first + token) * a.heads + h;
    const int64_t partial = FEW ? few_partial(a, s, kv, row, place) : place;
    const float* st = a.statistics + partial * 3;
    const float* from = a.partials + partial * a.dim;
    const int64_t st_step = a.partial_rows * 3, step = a.partial_rows * a.dim;
    float m = -kInfinity, vm = -kInfinity, l = 0.0f;
    // a lane's values: fours in + k L of the row
    int d[V];
    f32x4 x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) d[k] = (in + k * L) * 4, x[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // N splits at a time, their loads on the way together
    for (int i = 0; i < splits; i += N) {
      float sm[N], sl[N], sv[N];
      f32x4 v[N][V];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int64_t at = min(i + n, splits - 1);
        sm[n] = st[at * st_step], sl[n] = st[at * st_step + 1], sv[n] = st[at * st_step + 2];
#pragma unroll
        for (int k = 0; k < V; ++k) v[n][k] = *(const f32x4*)(from + at * step + min(d[k], a.dim - 4));
      }
      float next = m, value_next = vm;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (i + n >= splits) {
          sm[n] = sv[n] = -kInfinity, sl[n] = 0.0f;
#pragma unroll
          for (int k = 0; k < V; ++k) v[n][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        next = fmaxf(next, sm[n]), value_next = fmaxf(value_next, sv[n]);
      }
      const float ref = next == -kInfinity ? 0.0f : next, value_ref = value_next == -kInfinity ? 0.0f : value_next;
      l *= exp2_fast(m - ref);
      const float keep = exp2_fast(vm - value_ref);
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] *= keep;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        l = fmaf(sl[n], exp2_fast(sm[n] - ref), l);
        const float factor = exp2_fast(sv[n] - value_ref);
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k][e] = fmaf(v[n][k][e], factor, x[k][e]);
      }
      m = next, vm = value_next;
    }
    const float apart = (vm == -kInfinity ? 0.0f : vm) - (m == -kInfinity ? 0.0f : m);
    const float inverse = l == 0.0f ? 0.0f : (I8 ? exp2_fast(apart) : 1.0f) / l;
    bool odd = l == 0.0f && m == -kInfinity;
    const bool there = mine < end;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      x[k] *= inverse;
      if (!there || d[k] >= a.dim) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= !(fabsf(x[k][e]) < kInfinity);
      if constexpr (sizeof(T) == 4) *(f32x4*)(out + place * a.dim + d[k]) = x[k];
      else *(uint2*)(out + place * a.dim + d[k]) = make_uint2(pack_bf16(x[k][0], x[k][1]), pack_bf16(x[k][2], x[k][3]));
    }
    // rows that came out as no numbers are taken again
    for (uint64_t again = __ballot(there && odd); again;) {
      const int which = (__ffsll((unsigned long long)again) - 1) / L;
      const uint32_t r = first + which, t = r / group;
      attend_row<T, I8, TREE>(queries, out, a, span, t, kv * a.group + (int)(r - t * group), scratch[wave]);
      again &= L == 64 ? 0 : ~(((1ull << (L % 64)) - 1) << (which * L));
    }
  }
}

template <typename T, bool I8, bool TREE, bool FEW, int DP>
__global__ void __launch_bounds__(256) attend_join(const T* queries, T* out, ArgsOf<TREE> a, int rows, int tile) {
  __shared__ RowScratch scratch[4];
  join_block<T, I8, TREE, FEW, DP>(queries, out, a, blockIdx.x, rows, tile, scratch);
}

// Both kernels' splits in one launch, many rows' first (each a launch of its own: 5 us of a call's).
template <typename T, bool I8, bool TREE, int DP>
__global__ void __launch_bounds__(256) attend_joins(const T* queries, T* out, ArgsOf<TREE> few, ArgsOf<TREE> many,
                                                    int few_rows, int many_rows, unsigned many_blocks) {
  __shared__ RowScratch scratch[4];
  if (blockIdx.x < many_blocks)
    join_block<T, I8, TREE, false, DP>(queries, out, many, blockIdx.x, many_rows, 64, scratch);
  else join_block<T, I8, TREE, true, DP>(queries, out, few, blockIdx.x - many_blocks, few_rows, I8 ? 64 : 32, scratch);
}

// ------------------------------------------------------------------ host side

int check_attention(const char* entry, int32_t heads, int32_t kv_heads, int32_t dim, int32_t window, int32_t sinks,
                    int64_t longest) {
  if (dim > kMaxHead) return refuse("%s: heads of %d values (at most %d)", entry, dim, kMaxHead);
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return refuse("%s: %d heads over %d key heads", entry, heads, kv_heads);
  if (window < 0 || sinks < 0 || (sinks > 0 && window == 0))
    return refuse("%s: a window of %d positions with %d sinks", entry, window, sinks);
  if (longest < 0) return refuse("%s: a longest sequence of %lld positions", entry, (long long)longest);
  return 0;
}

// How a call's work is laid out, by its numbers alone (the workspace's size
// follows from it before there are tensors).
struct Plan {
  int few_rows;     // rows of a sequence and key head up to which it is attend_few's, where both run
  bool few16;       // attend_few's sequences have at most 16 rows
  int many_rows;    // rows a block of attend_many
  Split few, many;  // attend_few, attend_many
  bool both;                // in one launch
  int64_t few_most;                               // rows of a sequence and key head that attend_few may have
  int64_t few_slots, few_partials, many_partials;  // ArgsOf::few_slots, partial_rows
  // floats of the workspace before attend_few's partials, and before either's statistics
  int64_t few_at, few_statistics, many_statistics;
  int64_t bytes;
};

// Rows of queries of a sequence and key head up to which attend_few takes it, at most.
constexpr int kFewRows = 64;

Plan plan_of(int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t window,
             int64_t sinks, int64_t longest, bool by_offsets, bool quantized, bool f32, bool tree) {
  Plan p{0, true, 128, {0, 1}, {0, 1}, false, 0, 0, 0, 0, 0, 0, 0, 0};
  if (sequences <= 0 || tokens <= 0) return p;
  const int64_t group = heads / kv_heads, each = by_offsets ? tokens : ceil_div(tokens, sequences);
  const int64_t seen = window ? std::min(longest, window + sinks + std::min(each, (int64_t)kFewRows)) : longest;
  // (16 rows a unit while a sequence has no more on average: 64 sequences of 24 rows at 4,000 positions 311 us in
  // units of 64, 419 in two of 16 each)
  // Where sequences have more than kFewRows rows on average, those with few are single tokens for the most part, and a
  // chunk's few rows are better off among attend_many's: a mixed batch of 24 sequences, 18 of one token, 162 us, 251
  // with units of 64 rows for all up to 64 (in launches of their own; 226 with 16).
  p.few_rows = by_offsets && tokens * group > sequences * kFewRows ? 16 : kFewRows;
  // Trees have 16 to some hundred rows each, of positions that memory has to bring for all of them: in units of 16 by
  // waves two a SIMD, and past 16 rows among attend_many's, whose tiles serve 128 (us, as above / so: 8 nodes of one
  // sequence, 32 rows, 29 / 15, 8 sequences of 12 nodes at 3,000 positions 103 / 45, 32 of 16 at 4,000 223 / 145, 64 of 8
  // 358 / 251, 16 of 20 rows over 24 heads of their own 259 / 207). Over 8 bits, whose second reading is half as dear and
  // whose codes attend_many converts for rows that a tile has not, units of 16 up to kFewRows where trees have up to 40
  // rows on average (us, among attend_many's / so: 64 of 32 rows at 4,000 281 / 238, 16 of 20 240 / 170, 4 of 32 at 1,000
  // 41 / 21, though 8 of 32 at 4,000 51 / 58 and 16 of 35 56 / 74; with more rows 8 of 48 59 / 74, 32 of 48 at 1,000 62 / 80).
  if (tree && each * group > kFewRows) p.few_rows = quantized && tokens * group <= sequences * 40 ? kFewRows : 16;
  p.few16 = p.few_rows == 16 || tree ? true : by_offsets ? tokens * group <= sequences * 16 : each * group <= 16;
  // Up to 768 positions a second launch takes longer than it saves (one token at 517 12.5 us, 14.2 in splits, at 767 13.5
  // and 13.8, at 1,023 15.9 and 14.3; heads of 256 over 8 bits at 500 16.4 and 17.7, at 760 20.1 and 17.7). Splits of
  // 1,024 positions at most even out sequences of unlike lengths (64 of 400 to 8,000 251 us, in splits of 512 259, of 2,048
  // 249, of 4,096 271; over 8 bits 155, 173, 154 and 160).
  if (by_offsets || each * group <= kFewRows)
    p.few = seen <= 768 ? Split{1, 1} : split_of(sequences * kv_heads, seen, 1024, 4, 16);
  if (each * group > kFewRows) {
    // Blocks of 256 rows read keys and values (and make codes F16 numbers) half as often; blocks of 128 leave fewer
    // rows idle, two of them on a compute unit wait at barriers of their own, and single tokens share their launch. So
    // one sequence's go by blocks times positions; us, 128 / 256, 32 heads over 8 of 128, tokens after positions:
    //   BF16: 64 after 500 27.8 / 29.8, 256 after 0 20.5 / 18.8, 1,021 after 0 48 / 38, 8,192 619 / 584
    //   F32: 512 after 0 37.4 / 38.8, 512 after 500 53 / 47, 1,021 after 4,000 199 / 179
    //   8 bits, BF16: 512 after 500 42.7 / 45.1, 256 after 1,000 39.7 / 42.7, 512 after 1,000 51 / 46, 1,021 after
    //   2,500 122 / 107
    // and several sequences' by blocks alone: BF16, 24 sequences of 1,811 tokens 198 / 267, 4 of 4,096 215 / 221,
    // 8 of 8,192 515 / 522; in 8 bits 276 / 310, 302 / 269, 726 / 683.
    const int64_t rows = tokens * group;
    bool large;
    if (!by_offsets && sequences == 1) {
      const int64_t blocks = ceil_div(rows, 256) * kv_heads;
      large = blocks * seen > (quantized ? 3 << 15 : f32 ? 1 << 15 : 1 << 13) && blocks >= (quantized ? 24 : 1);
    } else {
      large = rows / 256 * kv_heads >= (quantized ? 384 : 768);
    }
    p.many_rows = large && dim > 64 && dim <= 128 ? 256 : 128;
    const int64_t blocks = ceil_div(rows, p.many_rows) * kv_heads, wanted = dim > 128 || p.many_rows == 256 ? 256 : 512;
    // (a tile of wide heads takes long enough for splits of 4: us, 2 heads of 256, splits of 8 / of 4, 5 trees in a window
    // of 1,024 57 / 48, over 8 bits 71 / 51, 4 trees of 20 nodes at 700 positions 55 / 43, one of 200 at 1,500 62 / 55,
    // 8 of 40 at 3,000 108 / 107, 2 of 100 at 8,000 and 32 of 20 at 6,000 alike)
    p.many = blocks * 4 >= wanted * 3 ? Split{1, 1} : split_of(blocks, seen, wanted, tree && dim > 128 ? 4 : 8, 1 << 25);
  }
  p.few_most = std::min(each * group, (int64_t)p.few_rows);
  // single tokens' blocks after the chunks' in one launch: the mixed batch 162 us, 226 in two, 203 the other way round
  p.both = p.few.splits > 0 && p.many.splits > 0 && p.few16 && p.many_rows == 128;
  // Partials by a row's place suit both kernels at once, since a row is one kernel's: attend_few has slots of its own
  // only where those are fewer (a few sequences' few rows beside long chunks).
  const int64_t rows = tokens * heads, slots = sequences * kv_heads * p.few_most;
  p.few_slots = slots < rows ? p.few_most : 0;
  p.few_partials = std::min(slots, rows);
  p.many_partials = rows;
  const int64_t few = p.few.splits > 1 ? p.few.splits * p.few_partials : 0;
  const int64_t many = p.many.splits > 1 ? p.many.splits * p.many_partials : 0;
  const int64_t by_place = p.few_slots ? many : std::max(few, many), by_slot = p.few_slots ? few : 0;
  p.many_statistics = by_place * dim;
  p.few_at = p.few_slots ? ceil_div(by_place * (dim + 3), 4) * 4 : 0;
  p.few_statistics = p.few_at + (p.few_slots ? by_slot : by_place) * dim;
  p.bytes = (p.few_slots ? p.few_at + by_slot * (dim + 3) : by_place * (dim + 3)) * 4;
  return p;
}

// Tiles of 16 rows that a wave of attend_few takes where there are more rows: as
// many as leave their results and queries in its 512 registers.
template <typename T, bool I8, int DP>
constexpr int kManyTiles = DP > 128 ? 1 : DP <= 64 || (sizeof(T) == 2 && !I8) ? 4 : 2;

template <typename T, bool I8, bool TREE, int DP>
int launch_tiles(const char* entry, const T* queries, T* out, const ArgsOf<TREE>& a, const Plan& plan, hipStream_t st) {
  ArgsOf<TREE> few = a, many = a;
  const int few_tiles = plan.few16 ? 1 : kManyTiles<T, I8, DP>, few_rows = 16 * few_tiles;
  int64_t few_units = 0, many_units = 0;
  if (plan.few.splits > 0) {
    few.splits = plan.few.splits;
    few.chunk = I8 ? plan.few.chunk : plan.few.chunk * 2;
    few.few_slots = (int)plan.few_slots;
    few.few_units = (int)ceil_div(plan.few_most, few_rows);
    few.partial_rows = plan.few_partials;
    few.partials = a.partials + plan.few_at;
    few.statistics = a.partials + plan.few_statistics;
    few_units = (int64_t)a.p.sequences * few.few_units;
  }
  if (plan.many.splits > 0) {
    many.splits = plan.many.splits;
    many.chunk = plan.many.chunk;
    many.partial_rows = plan.many_partials;
    many.statistics = a.partials + plan.many_statistics;
    many_units = units_of(a.p, plan.many_rows, 0, a.group, a.few_rows);
  }
  const unsigned few_blocks = (unsigned)(few_units * few.splits * a.kv_heads);
  const unsigned many_blocks = (unsigned)(many_units * many.splits * a.kv_heads);
  const dim3 block(256);
  if (plan.both) {
    hipLaunchKernelGGL((attend_both<T, I8, TREE, DP>), dim3(many_blocks + few_blocks), block, 0, st, queries, out, few, many,
                       many_blocks);
  } else {
    if (few_blocks > 0) {
      if (plan.few16) hipLaunchKernelGGL((attend_few<T, I8, TREE, DP, 1>), dim3(few_blocks), block, 0, st, queries, out, few);
      else hipLaunchKernelGGL((attend_few<T, I8, TREE, DP, kManyTiles<T, I8, DP>>), dim3(few_blocks), block, 0, st, queries, out, few);
    }
    if (many_blocks > 0) {
      if constexpr (DP == 128) {
        if (plan.many_rows == 256)
          hipLaunchKernelGGL((attend_many<T, I8, TREE, DP, 8>), dim3(many_blocks), dim3(512), 0, st, queries, out, many);
        else hipLaunchKernelGGL((attend_many<T, I8, TREE, DP, 4>), dim3(many_blocks), block, 0, st, queries, out, many);
      } else {
        hipLaunchKernelGGL((attend_many<T, I8, TREE, DP, 4>), dim3(many_blocks), block, 0, st, queries, out, many);
      }
    }
  }
  if (const int bad = launched(entry)) return bad;
  const unsigned few_joins = few_blocks > 0 && few.splits > 1 ? (unsigned)(few_units * a.kv_heads * (few_rows / kJoinRows<true>)) : 0;
  const unsigned many_joins = many_blocks > 0 && many.splits > 1 ? (unsigned)(many_units * a.kv_heads * (plan.many_rows / kJoinRows<false>)) : 0;
  if (few_joins > 0 && many_joins > 0)
    hipLaunchKernelGGL((attend_joins<T, I8, TREE, DP>), dim3(many_joins + few_joins), block, 0, st, queries, out, few, many,
                       few_rows, plan.many_rows, many_joins);
  else if (few_joins > 0)
    hipLaunchKernelGGL((attend_join<T, I8, TREE, true, DP>), dim3(few_joins), block, 0, st, queries, out, few, few_rows,
                       I8 ? 64 : 32);
  else if (many_joins > 0)
    hipLaunchKernelGGL((attend_join<T, I8, TREE, false, DP>), dim3(many_joins), block, 0, st, queries, out, many,
                       plan.many_rows, 64);
  return few_joins + many_joins > 0 ? launched(entry) : 0;
}

template <typename T, bool I8, bool TREE>
int attend(const char* entry, const T* queries, T* out, ArgsOf<TREE> a, const Plan& plan, bool aligned, hipStream_t st) {
  const int64_t row_blocks = units_of(a.p, 1, 0, 1) * a.heads;
  if (row_blocks > kOneWaveBlocks) return refuse("%s: %d tokens of %d heads in one call", entry, a.p.tokens, a.heads);
  const int64_t blocks = ((int64_t)a.p.sequences * 4 * std::max(plan.few.splits, 4) +
                          units_of(a.p, 128, 0, a.group) * std::max(plan.many.splits, 16)) * a.kv_heads;
  // (the tile kernels' offsets within a page, and rows of scales, have 32 bits)
  const bool small = (int64_t)a.p.page_size * a.kv_heads * a.dim * 2 < (int64_t)1 << 31 &&
                     (int64_t)a.p.cache_pages * a.kv_heads < (int64_t)1 << 31;
  if (!aligned || !small || a.dim > 256 || a.p.cache_pages == 0 || blocks > kOneWaveBlocks / 4) {
    const dim3 grid((unsigned)row_blocks), block(kWave * (row_blocks * kRowWaves > kOneWaveBlocks ? 1 : kRowWaves));
    const bool wide = a.dim % 8 == 0 && aligned16(a.keys) && aligned16(a.values);
    if (wide) hipLaunchKernelGGL((attend_rows<T, I8, true, TREE>), grid, block, 0, st, queries, out, a);
    else hipLaunchKernelGGL((attend_rows<T, I8, false, TREE>), grid, block, 0, st, queries, out, a);
    return launched(entry);
  }
  a.few_rows = plan.few.splits == 0 ? 0 : plan.many.splits == 0 ? INT32_MAX : plan.few_rows;
  if (a.dim <= 64) return launch_tiles<T, I8, TREE, 64>(entry, queries, out, a, plan, st);
  if (a.dim <= 128) return launch_tiles<T, I8, TREE, 128>(entry, queries, out, a, plan, st);
  return launch_tiles<T, I8, TREE, 256>(entry, queries, out, a, plan, st);
}

template <typename T, bool TREE>
int paged_attention(const char* entry, const T* queries, T* out, const RowArgsOf<TREE>& rows, int64_t longest, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  clear_error();
  ArgsOf<TREE> a{rows};
  a.splits = a.chunk = 1;
  if (const int bad = check_paging(entry, a.p, a.kv_heads, a.dim)) return bad;
  if (const int bad = check_attention(entry, a.heads, a.kv_heads, a.dim, a.window, a.sinks, longest)) return bad;
  if (a.p.tokens == 0 || a.p.sequences == 0) return 0;
  if (!queries || !out) return refuse("%s: null tensor", entry);
  if constexpr (TREE) {
    if (!a.sees) return refuse("%s: null tensor", entry);
    if (a.words <= 0) return refuse("%s: %d words of what a row sees", entry, (int)a.words);
    if ((reinterpret_cast<uintptr_t>(a.sees) & 3) != 0)
      return refuse("%s: what the rows see not aligned to its elements", entry);
  }
  if ((const void*)queries == (const void*)out) return refuse("%s: out is queries", entry);
  if ((reinterpret_cast<uintptr_t>(queries) | reinterpret_cast<uintptr_t>(out)) % sizeof(T) != 0)
    return refuse("%s: queries or out not aligned to their elements", entry);
  if (const int bad = check_cache(entry, a.p, a.keys, a.values, a.key_scales, a.value_scales)) return bad;
  const uintptr_t from = reinterpret_cast<uintptr_t>(queries), to = reinterpret_cast<uintptr_t>(out);
  if ((from > to ? from - to : to - from) / sizeof(T) < (uint64_t)a.p.tokens * a.heads * a.dim)
    return refuse("%s: out overlaps queries", entry);
  a.group = a.heads / a.kv_heads;
  a.columns = unit_columns(a.p.page_size);
  const Plan plan = plan_of(a.p.sequences, a.p.tokens, a.heads, a.kv_heads, a.dim, a.window, a.sinks, longest,
                            a.p.offsets != nullptr, a.key_scales != nullptr, sizeof(T) == 4, TREE);
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace)))
    return refuse("%s: a workspace of %lld bytes, needs %lld at a multiple of 16", entry, (long long)workspace_bytes,
                  (long long)plan.bytes);
  a.partials = (float*)workspace;
  // (the tile kernels load the one and store the other 8 or 16 bytes at a time)
  const bool aligned = a.dim % 8 == 0 && aligned16(queries) && aligned16(out) && aligned16(a.keys) && aligned16(a.values) &&
                       (!a.key_scales || (aligned16(a.key_scales) && aligned16(a.value_scales)));
  const hipStream_t st = (hipStream_t)stream;
  return a.key_scales ? attend<T, true, TREE>(entry, queries, out, a, plan, aligned, st)
                      : attend<T, false, TREE>(entry, queries, out, a, plan, aligned, st);
}

}  // namespace
}  // namespace drift

using namespace drift;

namespace {
int attention_workspace(const char* entry, int32_t sequences, int32_t tokens, int32_t heads, int32_t kv_heads,
                        int32_t head_dim, int32_t window, int32_t sinks, int32_t longest, bool tree, int64_t* bytes) {
  clear_error();
  if (!bytes) return refuse("%s: null bytes", entry);
  *bytes = 0;
  if (const int bad = check_attention(entry, heads, kv_heads, head_dim, window, sinks, longest)) return bad;
  // with offsets or without, over either cache, in either type
  for (int kind = 0; kind < 8; ++kind)
    *bytes = std::max(*bytes, plan_of(sequences, tokens, heads, kv_heads, head_dim, window, sinks, longest, kind & 1,
                                      kind & 2, kind & 4, tree).bytes);
  return 0;
}
}  // namespace

extern "C" int drift_paged_attention_workspace(int32_t sequences, int32_t tokens, int32_t heads, int32_t kv_heads,
                                               int32_t head_dim, int32_t window, int32_t sinks, int32_t longest,
                                               int64_t* bytes) {
  return attention_workspace("drift_paged_attention_workspace", sequences, tokens, heads, kv_heads, head_dim, window,
                             sinks, longest, false, bytes);
}

extern "C" int drift_tree_attention_workspace(int32_t sequences, int32_t tokens, int32_t heads, int32_t kv_heads,
                                              int32_t head_dim, int32_t window, int32_t sinks, int32_t longest,
                                              int64_t* bytes) {
  return attention_workspace("drift_tree_attention_workspace", sequences, tokens, heads, kv_heads, head_dim, window,
                             sinks, longest, true, bytes);
}

#define DRIFT_ROW_ARGS                                                                                              \
  RowArgs {                                                                                                         \
    {page_tables, starts, offsets, sequences, table_pages, cache_pages, page_size, start, tokens, bad_page}, heads, \
        kv_heads, head_dim, 0, scale, window, sinks, keys, values, key_scales, value_scales                         \
  }

extern "C" int drift_paged_attention_f32(const float* queries, const void* keys, const void* values,
                                         const float* key_scales, const float* value_scales,
                                         const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                         const int32_t* starts, const int32_t* offsets, int32_t sequences,
                                         int32_t start, int32_t tokens, int32_t heads, int32_t kv_heads,
                                         int32_t head_dim, int32_t page_size, float scale, int32_t window,
                                         int32_t sinks, int32_t longest, float* out, void* workspace,
                                         int64_t workspace_bytes, int32_t* bad_page, void* stream) {
  return paged_attention<float, false>("drift_paged_attention_f32", queries, out, DRIFT_ROW_ARGS, longest, workspace,
                                workspace_bytes, stream);
}

extern "C" int drift_paged_attention_bf16(const uint16_t* queries, const void* keys, const void* values,
                                          const float* key_scales, const float* value_scales,
                                          const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                          const int32_t* starts, const int32_t* offsets, int32_t sequences,
                                          int32_t start, int32_t tokens, int32_t heads, int32_t kv_heads,
                                          int32_t head_dim, int32_t page_size, float scale, int32_t window,
                                          int32_t sinks, int32_t longest, uint16_t* out, void* workspace,
                                          int64_t workspace_bytes, int32_t* bad_page, void* stream) {
  return paged_attention<uint16_t, false>("drift_paged_attention_bf16", queries, out, DRIFT_ROW_ARGS, longest,
                                   workspace, workspace_bytes, stream);
}

extern "C" int drift_tree_attention_f32(const float* queries, const void* keys, const void* values,
                                        const float* key_scales, const float* value_scales,
                                        const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                        const int32_t* starts, const int32_t* offsets, int32_t sequences, int32_t start,
                                        int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                        int32_t page_size, float scale, int32_t window, int32_t sinks, int32_t longest,
                                        const int32_t* sees, int32_t words, float* out, void* workspace,
                                        int64_t workspace_bytes, int32_t* bad_page, void* stream) {
  return paged_attention<float, true>("drift_tree_attention_f32", queries, out, (TreeRowArgs{DRIFT_ROW_ARGS, (const uint32_t*)sees, words}),
                                      longest, workspace, workspace_bytes, stream);
}

extern "C" int drift_tree_attention_bf16(const uint16_t* queries, const void* keys, const void* values,
                                         const float* key_scales, const float* value_scales,
                                         const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                         const int32_t* starts, const int32_t* offsets, int32_t sequences,
                                         int32_t start, int32_t tokens, int32_t heads, int32_t kv_heads,
                                         int32_t head_dim, int32_t page_size, float scale, int32_t window,
                                         int32_t sinks, int32_t longest, const int32_t* sees, int32_t words,
                                         uint16_t* out, void* workspace, int64_t workspace_bytes, int32_t* bad_page,
                                         void* stream) {
  return paged_attention<uint16_t, true>("drift_tree_attention_bf16", queries, out, (TreeRowArgs{DRIFT_ROW_ARGS, (const uint32_t*)sees, words}),
                                         longest, workspace, workspace_bytes, stream);
}
