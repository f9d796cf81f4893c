// Attention of new tokens over the paged key and value cache (paged.hpp has
// its layouts), of one sequence or several in a launch.
//
// Token t of a sequence sits at position P = start + t and sees the positions
// j <= P of its own sequence (its own key, written before, among them); with a
// window only those with j > P - window, or j < sinks. Query head h reads key
// head h / (heads / kv_heads):
//   s_j = scale q.k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
// over the visible j, in one pass with the running maximum m and sum, in F32. A
// row that sees nothing is zeros. What is masked has no part in a row, whatever
// it holds (an infinity, a NaN, memory never written); a position whose page
// table entry names no page of the cache is masked, and the flag set.
#include "paged.hpp"

#include <algorithm>

namespace drift {
namespace {

constexpr int kMaxHead = 512;
constexpr float kInfinity = __builtin_huge_valf();

struct AttentionArgs {
  Paging p;
  int32_t heads, kv_heads, dim, group;
  float scale;
  int32_t window, sinks;  // window 0: every position up to the row's own
  const void *keys, *values;
  const float *key_scales, *value_scales;
  // the split over positions: at least `chunk` tiles a split, `splits` of them;
  // their maxima and sums [splits, tokens, heads, 2] and unscaled results
  // [splits, tokens, heads, dim] where there are several
  int32_t splits, chunk;
  float *statistics, *partials;
  int32_t page_units, unit_shift;  // page_size / 16, and its logarithm where it is a power of two (else -1)
};

__device__ __forceinline__ float f16_value(uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// ------------------------------------------------------------------ rows one by one

// LDS that one wave's attend_row takes.
struct RowScratch {
  float query[kMaxHead];
  float weight[kWave];
  int64_t place[kWave];  // a value's index at dimension 0, or -1: not visible
};

// One row (a token's query head) by one wave: 64 positions at a time, a lane a
// position for the scores and then a lane a value for the sums, every product of
// F32 values in F32 and one by one. It takes any head size and alignment and
// whatever the cache holds, and is slow: the vector unit and its narrow loads
// bound it.
template <typename T, bool I8>
__device__ __noinline__ void attend_row(const T* queries, T* out, const AttentionArgs& a, const Span& span, int64_t nth,
                                        int h, RowScratch& r) {
  const int lane = threadIdx.x & (kWave - 1), kv = h / a.group;
  const int64_t position = span.start + nth, row = ((span.first + nth) * a.heads + h) * a.dim;
  wave_sync();
  for (int d = lane; d < a.dim; d += kWave) r.query[d] = load_one(queries + row + d);
  wave_sync();
  constexpr int kEach = kMaxHead / kWave;
  float sums[kEach] = {}, top = -kInfinity, total = 0.0f;
  bool any = false;
  const int64_t low = a.window ? max(position - a.window + 1, (int64_t)0) : 0;
  const int64_t sink_end = a.window ? min((int64_t)a.sinks, low) : 0;
  for (int64_t base = 0; base <= position; base += kWave) {
    if (base >= sink_end && base + kWave <= low) base = low / kWave * kWave;  // what lies between is not seen
    const int64_t j = base + lane;
    bool seen = j <= position && (j >= low || j < sink_end);
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
      for (int d = 0; d < a.dim; ++d) {
        float k;
        if constexpr (I8) k = (float)((const int8_t*)a.keys)[key + d];
        else k = f16_value(((const uint16_t*)a.keys)[key + d]);
        dot = fmaf(r.query[d], k, dot);
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
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int d = lane + i * kWave;
      if (d >= a.dim) break;
      float acc = sums[i] * keep;
      for (int n = 0; n < kWave; ++n) {
        const int64_t at = r.place[n];
        if (at < 0) continue;
        float v;
        if constexpr (I8) v = (float)((const int8_t*)a.values)[at + (int64_t)d * a.p.page_size];
        else v = f16_value(((const uint16_t*)a.values)[at + (int64_t)d * a.p.page_size]);
        acc = fmaf(r.weight[n], v, acc);
      }
      sums[i] = acc;
    }
  }
  // nothing seen: zeros; nothing but scores of -infinity seen: 0 / 0, as the formula has it
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int d = lane + i * kWave;
    if (d < a.dim) store_one(out + row + d, any ? sums[i] / total : 0.0f);
  }
}

template <typename T, bool I8>
__global__ void __launch_bounds__(64) attend_rows(const T* queries, T* out, AttentionArgs a) {
  __shared__ RowScratch scratch;
  int64_t nth;
  const int s = locate(a.p, blockIdx.x / (unsigned)a.heads, 1, 0, 1, nth);
  if (s < 0) return;
  const Span span = span_of(a.p, s);
  if (nth >= span.rows) return;
  attend_row<T, I8>(queries, out, a, span, nth, blockIdx.x % (unsigned)a.heads, scratch);
}

// ------------------------------------------------------------------ tiles by matrix instructions

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at an address of 8-byte multiples
typedef unsigned int u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// Rows of queries are (token, head of the key head's group) pairs: row r is token
// r / group of the sequence, head r % group, so that heads that share keys
// share their loads, whatever the group. The positions that the rows of tokens t0
// to t1 need, in tiles of `size` of them: `sinks` tiles from position 0, then on
// from `low`.
struct TileList {
  int32_t sinks, low, count;
  __device__ __forceinline__ int tile(int i) const { return i < sinks ? i : low + (i - sinks); }
};

__device__ __forceinline__ TileList tiles_of(const AttentionArgs& a, int64_t first, int64_t last, int size) {
  TileList t;
  const int64_t low = a.window ? max(first - a.window + 1, (int64_t)0) : 0;
  t.low = (int32_t)(low / size);
  t.sinks = a.window ? min((int32_t)((min((int64_t)a.sinks, low) + size - 1) / size), t.low) : 0;
  t.count = t.sinks + (int32_t)(last / size) - t.low + 1;
  return t;
}

// Tiles a split takes.
__device__ __forceinline__ int split_tiles(const AttentionArgs& a, int count) {
  return max(a.chunk, (count + a.splits - 1) / a.splits);
}

// Moves across the four lanes l, l + 16, l + 32, l + 48 that share a column.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// Four int8 codes (a dword) as F16, exactly: the code with its sign bit turned is
// 0 .. 255 as c + 128, and 0x6400 | (c + 128) is the F16 number 1024 + c + 128.
__device__ __forceinline__ void codes_f16(uint32_t word, f16x2& lo, f16x2& hi) {
  word ^= 0x80808080u;
  const f16x2 base = {(_Float16)1152.0f, (_Float16)1152.0f};
  lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, word, 0x04010400u)) - base;
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, word, 0x04030402u)) - base;
}

__device__ __forceinline__ f16x8 join(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
  return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ f16x8 codes_f16(uint32_t w0, uint32_t w1) {
  f16x2 a, b, c, d;
  codes_f16(w0, a, b);
  codes_f16(w1, c, d);
  return join(a, b, c, d);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A lane's eight weights as the product takes them: F16, and for F32 results the
// F16 remainder too.
template <int TERMS>
struct Halves {
  f16x8 term[TERMS];
};
template <int TERMS>
__device__ __forceinline__ Halves<TERMS> halves_of(const float (&v)[8]) {
  Halves<TERMS> h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h.term[0][i] = (_Float16)v[i];
  if constexpr (TERMS == 2)
#pragma unroll
    for (int i = 0; i < 8; ++i) h.term[1][i] = (_Float16)(v[i] - (float)h.term[0][i]);
  return h;
}

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
// Rows of queries are scaled by a power of two each to below 2^15 (exactly; F32
// rows as two F16 terms, 22 bits), their scores scaled back in F32. In 8 bits the
// codes are F16 numbers, a key's scale multiplies its score and a value's is part of
// its weight, which has a running maximum of its own then.
template <typename T, bool I8, int DP, int C>
__global__ void __launch_bounds__(256, C == 1 && DP <= 128 ? 2 : 1) attend_few(const T* queries, T* out, AttentionArgs a) {
  constexpr int kWaves = 4;
  constexpr int TOK = I8 ? 64 : 32, NT = TOK / 16;  // positions a tile, and row tiles of its scores
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  constexpr int KS = DP / 32, DT = DP / 16;         // products along a head, value tiles
  constexpr int kStride = DP + 4;
  __shared__ float merged[kWaves][16][kStride];
  __shared__ float stats[kWaves][C * 16][3];
  static_assert(sizeof(RowScratch) <= sizeof(merged) / kWaves, "a wave's part holds a row's scratch");

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int kv = blockIdx.x % (unsigned)a.kv_heads;
  const unsigned rest = blockIdx.x / (unsigned)a.kv_heads;
  const int split = rest % (unsigned)a.splits;
  int64_t nth;
  const int s = locate(a.p, rest / (unsigned)a.splits, C * 16, 0, a.group, nth);
  if (s < 0) return;
  const Span span = span_of(a.p, s);
  const int rows = (int)min((int64_t)span.rows * a.group - nth * (C * 16), (int64_t)(C * 16));
  if (rows <= 0) return;
  const uint32_t row0 = (uint32_t)nth * (C * 16), group = (uint32_t)a.group;
  const uint32_t p0 = (uint32_t)span.start + row0 / group, p1 = (uint32_t)span.start + (row0 + rows - 1) / group;
  const TileList list = tiles_of(a, p0, p1, TOK);
  const int each = split_tiles(a, list.count);
  const int begin = split * each, end = min(begin + each, list.count);
  if (begin >= end) return;

  // the rows' queries as B operands: column col, values 8 g .. of each 32 (8 bits: of each 64, 16 g ..)
  f16x8 query[C][KS][TERMS];
  float row_scale[C];
  uint32_t position[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int r = c * 16 + col;
    const uint32_t row = row0 + min(r, rows - 1), token = row / group;
    position[c] = (uint32_t)span.start + token;
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
    const uint32_t column = a.unit_shift >= 0 ? in >> a.unit_shift : in / (uint32_t)a.page_units;
    off = (in - column * (uint32_t)a.page_units) * 16;
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

  int i = begin + wave;
  Places now = places_of(i), next = places_of(i + kWaves);
  if (i < end) load_keys(now);
  for (; i < end; i += kWaves) {
    const uint32_t base = (uint32_t)list.tile(i) * TOK;
    const uint32_t mine = base + g * (TOK / 4);  // the lane's first position
    const bool okay = (uint32_t)now.value_page < (uint32_t)a.p.cache_pages;
    const int32_t value_page = okay ? now.value_page : 0;
    if (!okay && mine <= p1 &&
        (a.window == 0 || mine + TOK / 4 - 1 + (uint32_t)a.window > p0 || mine < (uint32_t)a.sinks))
      flag_bad(a.p);

    // the values, and the scales in 8 bits
    uint4 values[DT];
    {
      const char* from = (const char*)a.values + (((int64_t)value_page * a.kv_heads + kv) * a.dim * a.p.page_size +
                                                  now.value_off + (g * (TOK / 4)) % 16) * (I8 ? 1 : 2);
      const int64_t stride = (int64_t)a.p.page_size * (I8 ? 1 : 2);
#pragma unroll
      for (int d = 0; d < DT; ++d) values[d] = *(const uint4*)(from + min(d * 16 + col, a.dim - 1) * stride);
    }
    float key_scale[I8 ? 16 : 1], value_log[I8 ? 16 : 1];
    if constexpr (I8) {
      const int64_t at = ((int64_t)value_page * a.kv_heads + kv) * a.p.page_size + now.value_off;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float4 x = *(const float4*)(a.key_scales + at + e), y = *(const float4*)(a.value_scales + at + e);
        key_scale[e] = x.x, key_scale[e + 1] = x.y, key_scale[e + 2] = x.z, key_scale[e + 3] = x.w;
        value_log[e] = y.x, value_log[e + 1] = y.y, value_log[e + 2] = y.z, value_log[e + 3] = y.w;
      }
    }

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
    const bool whole = base + TOK - 1 <= p0 &&
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
      if (!whole)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t j = mine + 4 * t + e;
            const bool seen = okay && j <= position[c] &&
                              (a.window == 0 || j + (uint32_t)a.window > position[c] || j < (uint32_t)a.sinks);
            score[c][t][e] = seen ? score[c][t][e] : -kInfinity;
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
          const bool seen = okay && j <= p1 &&
                            (a.window == 0 || j + (uint32_t)a.window > p0 || j < (uint32_t)a.sinks);
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
      Halves<TERMS> weights[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = weight[c][2 * n + e / 4][e % 4];
        weights[c] = halves_of<TERMS>(x);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f16x8 value;
        if constexpr (I8) value = n ? codes_f16(values[d].z, values[d].w) : codes_f16(values[d].x, values[d].y);
        else value = __builtin_bit_cast(f16x8, values[d]);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int m = 0; m < TERMS; ++m)
            acc[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, weights[c].term[m], acc[c][d], 0, 0, 0);
      }
    }
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
      const float inverse = l == 0.0f ? 0.0f : (I8 ? exp2_fast(value_ref - ref) : 1.0f) / l;
      bool odd = false;
      for (int d = lane; d < a.dim; d += kWave) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x = fmaf(merged[w][r][d], factor[w], x);
        if (a.splits == 1) {
          x *= inverse;
          odd |= !(fabsf(x) < kInfinity);
          store_one(out + place * a.dim + d, x);
        } else {
          a.partials[((int64_t)split * a.p.tokens * a.heads + place) * a.dim + d] = x;
        }
      }
      if (a.splits == 1) {
        // a row of -infinity alone, as one of NaN, is taken again
        if (__any(odd) || (l == 0.0f && m == -kInfinity)) again |= 1u << r;
      } else if (lane == 0) {
        float* st = a.statistics + ((int64_t)split * a.p.tokens * a.heads + place) * 3;
        st[0] = m, st[1] = l, st[2] = vm;
      }
    }
    if (a.splits == 1) {
      __syncthreads();  // merged is free, and holds the scratch
      RowScratch& scratch = *reinterpret_cast<RowScratch*>(&merged[wave][0][0]);
      for (; again; again &= again - 1) {
        const uint32_t row = row0 + c * 16 + __ffs(again) - 1;
        attend_row<T, I8>(queries, out, a, span, row / group, kv * a.group + (int)(row % group), scratch);
      }
    }
  }
}

// Joins the splits of attend_few (ROWS rows of TOK-position tiles a unit) row by row, a
// wave a row.
template <typename T, bool I8>
__global__ void __launch_bounds__(64) attend_join(const T* queries, T* out, AttentionArgs a, int rows, int tile) {
  __shared__ RowScratch scratch;
  const int lane = threadIdx.x, h = blockIdx.x % (unsigned)a.heads;
  int64_t nth;
  const int s = locate(a.p, blockIdx.x / (unsigned)a.heads, 1, 0, 1, nth);
  if (s < 0) return;
  const Span span = span_of(a.p, s);
  if (nth >= span.rows) return;
  // the unit the row was in, its tiles and so its splits
  const int64_t row0 = (nth * a.group + h % a.group) / rows * rows;
  const int64_t last = min(row0 + rows, (int64_t)span.rows * a.group) - 1;
  const TileList list = tiles_of(a, span.start + row0 / a.group, span.start + last / a.group, tile);
  const int each = split_tiles(a, list.count), splits = (list.count + each - 1) / each;
  const int64_t place = (span.first + nth) * a.heads + h, stride = (int64_t)a.p.tokens * a.heads;
  float m = -kInfinity, vm = -kInfinity;
  for (int i = lane; i < splits; i += kWave) {
    const float* st = a.statistics + (i * stride + place) * 3;
    m = fmaxf(m, st[0]);
    vm = fmaxf(vm, st[2]);
  }
  m = group_max<64>(m);
  vm = group_max<64>(vm);
  const float ref = m == -kInfinity ? 0.0f : m, value_ref = vm == -kInfinity ? 0.0f : vm;
  float l = 0.0f;
  constexpr int kEach = kMaxHead / kWave;
  float x[kEach] = {};
  for (int i = 0; i < splits; ++i) {
    const float* st = a.statistics + (i * stride + place) * 3;
    l = fmaf(st[1], exp2_fast(st[0] - ref), l);
    const float factor = exp2_fast(st[2] - value_ref);
    const float* part = a.partials + (i * stride + place) * a.dim;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (lane + e * kWave < a.dim) x[e] = fmaf(part[lane + e * kWave], factor, x[e]);
  }
  const float inverse = l == 0.0f ? 0.0f : (I8 ? exp2_fast(value_ref - ref) : 1.0f) / l;
  bool odd = l == 0.0f && m == -kInfinity;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int d = lane + e * kWave;
    if (d >= a.dim) break;
    x[e] *= inverse;
    odd |= !(fabsf(x[e]) < kInfinity);
    store_one(out + place * a.dim + d, x[e]);
  }
  if (__any(odd)) attend_row<T, I8>(queries, out, a, span, nth, h, scratch);
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
  bool few;    // at most 16 rows of queries a sequence and key head
  int splits;  // over positions
  int chunk;   // tiles of 32 positions that a split has at least
  int64_t bytes;
};

Plan plan_of(int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t window,
             int64_t sinks, int64_t longest) {
  Plan p{true, 1, 1, 0};
  if (sequences <= 0 || tokens <= 0) return p;
  const int64_t group = heads / kv_heads, each = ceil_div(tokens, sequences);
  p.few = each * group <= 16;
  const int64_t seen = window ? std::min(longest, window + sinks + each) : longest;
  const int64_t tiles = std::max<int64_t>(ceil_div(seen, 32), 1);
  const int64_t blocks = (sequences + tokens * group / (p.few ? 16 : 64)) * kv_heads;
  int64_t chunk = tiles * blocks / 1024;
  chunk = std::min<int64_t>(std::max<int64_t>(chunk, 8), 64);
  p.chunk = (int)chunk;
  p.splits = (int)std::min<int64_t>(ceil_div(tiles, chunk), 1024);
  if (p.splits > 1) p.bytes = (int64_t)p.splits * tokens * heads * (dim + 3) * 4;
  return p;
}

// Tiles of 16 rows that a wave of attend_few takes where there are more rows: as
// many as leave their results and queries in its 512 registers.
template <typename T, bool I8, int DP>
constexpr int kManyTiles = DP > 128 ? 1 : DP <= 64 || (sizeof(T) == 2 && !I8) ? 4 : 2;

template <typename T, bool I8, int DP>
int launch_few(const char* entry, const T* queries, T* out, const AttentionArgs& a, bool few, hipStream_t st) {
  constexpr int kMany = kManyTiles<T, I8, DP>;
  const int rows = 16 * (few ? 1 : kMany);
  const dim3 grid((unsigned)(units_of(a.p, rows, 0, a.group) * a.splits * a.kv_heads)), block(256);
  if (few) hipLaunchKernelGGL((attend_few<T, I8, DP, 1>), grid, block, 0, st, queries, out, a);
  else hipLaunchKernelGGL((attend_few<T, I8, DP, kMany>), grid, block, 0, st, queries, out, a);
  const int bad = launched(entry);
  if (bad || a.splits == 1) return bad;
  hipLaunchKernelGGL((attend_join<T, I8>), dim3((unsigned)(units_of(a.p, 1, 0, 1) * a.heads)), dim3(kWave), 0, st,
                     queries, out, a, rows, I8 ? 64 : 32);
  return launched(entry);
}

template <typename T, bool I8>
int attend(const char* entry, const T* queries, T* out, AttentionArgs a, const Plan& plan, bool aligned, hipStream_t st) {
  const int64_t row_blocks = units_of(a.p, 1, 0, 1) * a.heads;
  if (row_blocks > kOneWaveBlocks) return refuse("%s: %d tokens of %d heads in one call", entry, a.p.tokens, a.heads);
  const int64_t blocks = units_of(a.p, 16, 0, a.group) * plan.splits * a.kv_heads;  // at most
  if (!aligned || a.dim > 256 || a.p.cache_pages == 0 || blocks > kOneWaveBlocks / 4) {
    hipLaunchKernelGGL((attend_rows<T, I8>), dim3((unsigned)row_blocks), dim3(kWave), 0, st, queries, out, a);
    return launched(entry);
  }
  a.splits = plan.splits;
  a.chunk = I8 ? plan.chunk / 2 : plan.chunk;
  if (a.dim <= 64) return launch_few<T, I8, 64>(entry, queries, out, a, plan.few, st);
  if (a.dim <= 128) return launch_few<T, I8, 128>(entry, queries, out, a, plan.few, st);
  return launch_few<T, I8, 256>(entry, queries, out, a, plan.few, st);
}

template <typename T>
int paged_attention(const char* entry, const T* queries, T* out, AttentionArgs a, int64_t longest, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  clear_error();
  if (const int bad = check_paging(entry, a.p, a.kv_heads, a.dim)) return bad;
  if (const int bad = check_attention(entry, a.heads, a.kv_heads, a.dim, a.window, a.sinks, longest)) return bad;
  if (a.p.tokens == 0 || a.p.sequences == 0) return 0;
  if (!queries || !out) return refuse("%s: null tensor", entry);
  if ((const void*)queries == (const void*)out) return refuse("%s: out is queries", entry);
  if ((reinterpret_cast<uintptr_t>(queries) | reinterpret_cast<uintptr_t>(out)) % sizeof(T) != 0)
    return refuse("%s: queries or out not aligned to their elements", entry);
  if (const int bad = check_cache(entry, a.p, a.keys, a.values, a.key_scales, a.value_scales)) return bad;
  a.group = a.heads / a.kv_heads;
  a.page_units = a.p.page_size / 16;
  a.unit_shift = (a.page_units & (a.page_units - 1)) == 0 ? __builtin_ctz((unsigned)a.page_units) : -1;
  const Plan plan = plan_of(a.p.sequences, a.p.tokens, a.heads, a.kv_heads, a.dim, a.window, a.sinks, longest);
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace)))
    return refuse("%s: a workspace of %lld bytes, needs %lld at a multiple of 16", entry, (long long)workspace_bytes,
                  (long long)plan.bytes);
  a.partials = (float*)workspace;
  a.statistics = a.partials + (int64_t)plan.splits * a.p.tokens * a.heads * a.dim;
  const bool aligned = a.dim % 8 == 0 && aligned16(queries) && aligned16(a.keys) && aligned16(a.values) &&
                       (!a.key_scales || (aligned16(a.key_scales) && aligned16(a.value_scales)));
  const hipStream_t st = (hipStream_t)stream;
  return a.key_scales ? attend<T, true>(entry, queries, out, a, plan, aligned, st)
                      : attend<T, false>(entry, queries, out, a, plan, aligned, st);
}

}  // namespace
}  // namespace drift

using namespace drift;

extern "C" int drift_paged_attention_workspace(int32_t sequences, int32_t tokens, int32_t heads, int32_t kv_heads,
                                               int32_t head_dim, int32_t window, int32_t sinks, int32_t longest,
                                               int64_t* bytes) {
  clear_error();
  if (!bytes) return refuse("drift_paged_attention_workspace: null bytes");
  *bytes = 0;
  if (const int bad = check_attention("drift_paged_attention_workspace", heads, kv_heads, head_dim, window, sinks,
                                      longest))
    return bad;
  *bytes = plan_of(sequences, tokens, heads, kv_heads, head_dim, window, sinks, longest).bytes;
  return 0;
}

#define DRIFT_ATTENTION_ARGS                                                                                        \
  AttentionArgs {                                                                                                   \
    {page_tables, starts, offsets, sequences, table_pages, cache_pages, page_size, start, tokens, bad_page}, heads, \
        kv_heads, head_dim, 0, scale, window, sinks, keys, values, key_scales, value_scales, 1, 1, nullptr, nullptr, 0, 0 \
  }

extern "C" int drift_paged_attention_f32(const float* queries, const void* keys, const void* values,
                                         const float* key_scales, const float* value_scales,
                                         const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                         const int32_t* starts, const int32_t* offsets, int32_t sequences,
                                         int32_t start, int32_t tokens, int32_t heads, int32_t kv_heads,
                                         int32_t head_dim, int32_t page_size, float scale, int32_t window,
                                         int32_t sinks, int32_t longest, float* out, void* workspace,
                                         int64_t workspace_bytes, int32_t* bad_page, void* stream) {
  return paged_attention<float>("drift_paged_attention_f32", queries, out, DRIFT_ATTENTION_ARGS, longest, workspace,
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
  return paged_attention<uint16_t>("drift_paged_attention_bf16", queries, out, DRIFT_ATTENTION_ARGS, longest,
                                   workspace, workspace_bytes, stream);
}
