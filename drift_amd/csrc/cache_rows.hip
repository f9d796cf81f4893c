// Rows into and out of the paged key and value cache, of one sequence or
// several in a launch: the F16 cache, and the cache in 8 bits, quantised as it
// is written (paged.hpp has both layouts).
//
// A row x (a position's key or value of one head, D values) is kept as codes
// round-half-away(x / d), at most 127 in size, and d = max |x| / 127 rounded to
// F32. The quotient decides as the exact one would: x and d have 24 bits, so x / d
// is a half or at least 2^-27 from one, and the double product x * (1 / d), within
// 2^-51 relative of it, with 2^-40 added in the direction away from 0 falls on
// the exact quotient's side. A row of zeros has d = 0 and codes 0. A row with a
// NaN or an infinity has d = NaN and codes 0: it reads back as NaN throughout,
// and so does what attends to it. One scale a row (128 + 4 bytes for 128 values,
// where blocks of 32 would take 144) because a row's scale can be applied to its
// score, and its value's to its weight, after the products of whole rows.
#include "paged.hpp"

namespace drift {

int check_paging(const char* entry, const Paging& p, int32_t kv_heads, int32_t head_dim) {
  if (p.tokens < 0 || kv_heads <= 0 || head_dim <= 0)
    return refuse("%s: %d tokens of %d heads of %d values", entry, p.tokens, kv_heads, head_dim);
  if (p.page_size <= 0 || p.page_size % 16 != 0)
    return refuse("%s: pages of %d tokens: not a multiple of 16", entry, p.page_size);
  if (p.start < 0 || p.table_pages < 0 || p.cache_pages < 0 || p.sequences < 0)
    return refuse("%s: start %d, %d table pages, %d cache pages, %d sequences", entry, p.start, p.table_pages,
                  p.cache_pages, p.sequences);
  if (!p.starts) {
    if (p.sequences > 1) return refuse("%s: %d sequences without starts", entry, p.sequences);
    if (p.sequences == 1 && (int64_t)p.table_pages * p.page_size < (int64_t)p.start + p.tokens)
      return refuse("%s: a page table of %d pages for %lld positions", entry, p.table_pages,
                    (long long)p.start + p.tokens);
    if (p.sequences == 1 && (int64_t)p.start + p.tokens > kMostPositions)
      return refuse("%s: %lld positions (at most %lld)", entry, (long long)p.start + p.tokens, (long long)kMostPositions);
  }
  if (!p.offsets && p.sequences > 1 && p.sequences != p.tokens)
    return refuse("%s: %d sequences of %d tokens without offsets", entry, p.sequences, p.tokens);
  return 0;
}

int check_cache(const char* entry, const Paging& p, const void* keys, const void* values, const float* key_scales,
                const float* value_scales) {
  if (!keys || !values || !p.tables) return refuse("%s: null tensor", entry);
  if (!key_scales != !value_scales) return refuse("%s: scales of keys or of values alone", entry);
  const uintptr_t wide = key_scales ? 0 : 1;
  if (((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & wide) != 0 ||
      ((reinterpret_cast<uintptr_t>(key_scales) | reinterpret_cast<uintptr_t>(value_scales) |
        reinterpret_cast<uintptr_t>(p.tables) | reinterpret_cast<uintptr_t>(p.starts) |
        reinterpret_cast<uintptr_t>(p.offsets)) & 3) != 0)
    return refuse("%s: cache, scales or tables not aligned to their elements", entry);
  return 0;
}

namespace {

constexpr int kTile = 16;  // positions a tile; pages hold whole tiles

struct CacheRows {
  Paging p;
  int32_t kv_heads, dim;
  void *keys, *values;
  float *key_scales, *value_scales;
  int32_t extra;  // tiles a sequence past ceil(rows / 16): its first row may lie inside a tile
};

__device__ __forceinline__ uint32_t f16_bits(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ float f16_value(uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// A tile of a launch: 16 aligned positions of a sequence and one key head, of
// which [lo, hi) are the sequence's rows here.
struct Tile {
  int64_t first, lo, hi;
  int64_t row;        // the token row of position lo
  int64_t page, off;  // where it lies
  int kv;
};

__device__ __forceinline__ bool tile_of(const CacheRows& c, Tile& t) {
  const int64_t unit = blockIdx.x / (unsigned)c.kv_heads;
  t.kv = blockIdx.x % (unsigned)c.kv_heads;
  int64_t nth;
  const int s = locate(c.p, unit, kTile, c.extra, 1, nth);
  if (s < 0) return false;
  const Span span = span_of<true>(c.p, s);
  t.first = (span.start / kTile + nth) * kTile;
  t.lo = max(t.first, span.start);
  t.hi = min(t.first + kTile, span.start + span.rows);
  if (t.lo >= t.hi) return false;
  t.row = span.first + t.lo - span.start;
  t.page = span.table[t.first / c.p.page_size];
  t.off = t.first % c.p.page_size;
  if (t.page < 0 || t.page >= c.p.cache_pages) {
    flag_bad(c.p);
    return false;
  }
  return true;
}

// Max over the 16 lanes of a row of the values' magnitude bits: as whole
// numbers a NaN is above an infinity and that above every number.
__device__ __forceinline__ uint32_t row_max_bits(uint32_t v) {
  v = max(v, (uint32_t)dpp_move32<0xb1>((int)v));
  v = max(v, (uint32_t)dpp_move32<0x4e>((int)v));
  v = max(v, (uint32_t)dpp_move32<0x141>((int)v));
  return max(v, (uint32_t)dpp_move32<0x140>((int)v));
}

struct RowScale {
  float d;
  double inverse;  // 0 where every code is 0
};

__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
  RowScale r;
  if (max_bits >= 0x7f800000u) {
    r.d = __builtin_nanf("");
    r.inverse = 0.0;
  } else {
    r.d = __uint_as_float(max_bits) / 127.0f;
    r.inverse = r.d == 0.0f ? 0.0 : 1.0 / (double)r.d;
  }
  return r;
}

__device__ __forceinline__ int code_of(float x, double inverse) {
  const double size = inverse == 0.0 ? 0.0 : fabs((double)x);  // (an infinity times 0 is no number)
  const int code = min((int)fma(size, inverse, 0.5 + 0x1p-40), 127);
  return x < 0.0f ? -code : code;
}

// The LDS word of a staged tile of values that holds positions 4 q to 4 q + 3
// of value d (WORDS words hold 4 of them): four words of padding a chunk of N
// values let the 64 lanes of a write land on 64 banks.
template <int N, int WORDS>
__device__ __forceinline__ int staged_word(int d, int q) {
  return d * 4 * WORDS + q * WORDS + (d / N) * 4 * WORDS;
}
template <int N, int WORDS>
constexpr int kStagedWords(int chunks) {
  return chunks * (N + 1) * 4 * WORDS;
}

// One tile a one-wave block. Lane l has chunks l % 16 + 16 i of the four
// positions 4 (l / 16) + j, for keys and then for values, so a load covers 256
// bytes of four rows, a row's maximum takes four steps across 16 lanes, and a
// value's four positions are one word (F16: two) of the transposed tile, which
// leaves through LDS as 16-byte stores.
//
// Memory bounds it: 8,192 F32 rows of 8 heads of 128 into 8 bits 21.8 us (3.9 TB/s),
// 64 BF16 ones, a decode step's, 6.5 us (a launch's chain). A block for the keys and
// one for the values: 23.3 and 5.6 us.
template <typename T, bool I8, int CPL>
__global__ void __launch_bounds__(64) write_tiles(const T* k, const T* v, CacheRows c) {
  constexpr int N = Chunk<T>::N, W = I8 ? 1 : 2;
  __shared__ uint32_t staged[kStagedWords<N, W>(16 * CPL)];
  Tile t;
  if (!tile_of(c, t)) return;
  const int lane = threadIdx.x, q = lane / 16, ci = lane % 16, chunks = c.dim / N;
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    const T* x = what ? v : k;
    typename Chunk<T>::Raw raw[4][CPL];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // positions and chunks past the rows' are clamped to ones of theirs
      const int64_t position = min(max(t.first + 4 * q + j, t.lo), t.hi - 1);
      const T* row = x + ((t.row + position - t.lo) * c.kv_heads + t.kv) * c.dim;
#pragma unroll
      for (int i = 0; i < CPL; ++i) raw[j][i] = Chunk<T>::load_raw(row + min(ci + 16 * i, chunks - 1) * N);
    }
    RowScale scale[4];
    if constexpr (I8) {
      float* scales = (what ? c.value_scales : c.key_scales) +
                      (t.page * c.kv_heads + t.kv) * (int64_t)c.p.page_size + t.off;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
          float x1[N];
          Chunk<T>::unpack(raw[j][i], x1);
#pragma unroll
          for (int e = 0; e < N; ++e) most = max(most, __float_as_uint(x1[e]) & 0x7fffffffu);
        }
        scale[j] = row_scale(row_max_bits(most));
        const int64_t position = t.first + 4 * q + j;
        if (ci == 0 && position >= t.lo && position < t.hi) scales[4 * q + j] = scale[j].d;
      }
    }
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const int chunk = ci + 16 * i;
      if (chunk >= chunks) break;
      uint32_t words[N][W] = {};  // the chunk's values, four positions each
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x1[N];
        Chunk<T>::unpack(raw[j][i], x1);
        uint32_t bits[N];
#pragma unroll
        for (int e = 0; e < N; ++e)
          bits[e] = I8 ? (uint32_t)code_of(x1[e], scale[j].inverse) & 0xffu : f16_bits(x1[e]);
        if (what == 0) {  // a key's chunk goes as it is
          uint32_t packed[N * (I8 ? 1 : 2) / 4] = {};
#pragma unroll
          for (int e = 0; e < N; ++e)
            if constexpr (I8) packed[e / 4] |= bits[e] << (8 * (e % 4));
            else packed[e / 2] |= bits[e] << (16 * (e % 2));
          const int64_t position = t.first + 4 * q + j;
          if (position >= t.lo && position < t.hi) {
            char* at = (char*)c.keys +
                       (((t.page * c.p.page_size + t.off + 4 * q + j) * c.kv_heads + t.kv) * c.dim + chunk * N) * (I8 ? 1 : 2);
            if constexpr (sizeof(packed) == 4) *(uint32_t*)at = packed[0];
            else if constexpr (sizeof(packed) == 8) *(uint2*)at = make_uint2(packed[0], packed[1]);
            else *(uint4*)at = make_uint4(packed[0], packed[1], packed[2], packed[3]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if constexpr (I8) words[e][0] |= bits[e] << (8 * j);
            else words[e][j / 2] |= bits[e] << (16 * (j % 2));
        }
      }
      if (what == 1)
#pragma unroll
        for (int e = 0; e < N; ++e)
#pragma unroll
          for (int w = 0; w < W; ++w) staged[staged_word<N, W>(chunk * N + e, q) + w] = words[e][w];
    }
  }
  wave_sync();
  constexpr int kBytes = I8 ? 1 : 2;
  char* tile = (char*)c.values + ((t.page * c.kv_heads + t.kv) * (int64_t)c.dim * c.p.page_size + t.off) * kBytes;
  const int64_t stride = (int64_t)c.p.page_size * kBytes;
  if (t.hi - t.lo == kTile) {
    for (int i = lane; i < c.dim * W; i += kWave) {
      const int d = i / W, half = i % W;
      *(uint4*)(tile + d * stride + half * 16) = *(const uint4*)&staged[staged_word<N, W>(d, half * 2)];
    }
  } else {
    const int skip = (int)(t.lo - t.first), width = (int)(t.hi - t.lo);
    for (int i = lane; i < c.dim * width; i += kWave) {
      const int d = i / width, position = skip + i % width;
      const uint32_t* word = &staged[staged_word<N, W>(d, position / 4)];
      if constexpr (I8) ((uint8_t*)(tile + d * stride))[position] = (uint8_t)(word[0] >> (8 * (position % 4)));
      else ((uint16_t*)(tile + d * stride))[position] = (uint16_t)(word[position % 4 / 2] >> (16 * (position % 2)));
    }
  }
}

// Any head size and alignment: a wave a row of a head, value by value.
template <typename T, bool I8>
__global__ void __launch_bounds__(64) write_rows(const T* k, const T* v, CacheRows c) {
  const int64_t unit = blockIdx.x / (unsigned)c.kv_heads;
  const int kv = blockIdx.x % (unsigned)c.kv_heads, lane = threadIdx.x;
  int64_t nth;
  const int s = locate(c.p, unit, 1, 0, 1, nth);
  if (s < 0) return;
  const Span span = span_of<true>(c.p, s);
  if (nth >= span.rows) return;
  const int64_t position = span.start + nth, page = span.table[position / c.p.page_size];
  const int64_t off = position % c.p.page_size;
  if (page < 0 || page >= c.p.cache_pages) {
    flag_bad(c.p);
    return;
  }
  const int64_t row = ((span.first + nth) * c.kv_heads + kv) * c.dim;
  for (int what = 0; what < 2; ++what) {
    const T* x = (what ? v : k) + row;
    const int64_t at = what ? (page * c.kv_heads + kv) * (int64_t)c.dim * c.p.page_size + off
                            : ((page * c.p.page_size + off) * c.kv_heads + kv) * c.dim;
    const int64_t stride = what ? c.p.page_size : 1;
    RowScale scale;
    if constexpr (I8) {
      uint32_t most = 0;
      for (int d = lane; d < c.dim; d += kWave) most = max(most, __float_as_uint(load_one(x + d)) & 0x7fffffffu);
#pragma unroll
      for (int mask = 1; mask < kWave; mask <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, mask, kWave));
      scale = row_scale(most);
      if (lane == 0)
        (what ? c.value_scales : c.key_scales)[(page * c.kv_heads + kv) * (int64_t)c.p.page_size + off] = scale.d;
    }
    for (int d = lane; d < c.dim; d += kWave) {
      if constexpr (I8) ((int8_t*)(what ? c.values : c.keys))[at + d * stride] = (int8_t)code_of(load_one(x + d), scale.inverse);
      else ((uint16_t*)(what ? c.values : c.keys))[at + d * stride] = (uint16_t)f16_bits(load_one(x + d));
    }
  }
}

// The tiles read back: keys by rows, values through LDS, their transpose
// undone. 9,192 positions of 8 heads of 128 out of 8 bits as F32 15.1 us (6.2 TB/s).
template <typename T, bool I8, int CPL>
__global__ void __launch_bounds__(64) read_tiles(T* k, T* v, CacheRows c) {
  constexpr int N = Chunk<T>::N, W = I8 ? 1 : 2, kBytes = I8 ? 1 : 2;
  __shared__ uint32_t staged[kStagedWords<N, W>(16 * CPL)];
  Tile t;
  if (!tile_of(c, t)) return;
  const int lane = threadIdx.x, q = lane / 16, ci = lane % 16, chunks = c.dim / N;
  const char* tile = (const char*)c.values + ((t.page * c.kv_heads + t.kv) * (int64_t)c.dim * c.p.page_size + t.off) * kBytes;
  const int64_t stride = (int64_t)c.p.page_size * kBytes;
#pragma unroll 4
  for (int i = lane; i < c.dim * W; i += kWave) {
    const int d = i / W, half = i % W;
    *(uint4*)&staged[staged_word<N, W>(d, half * 2)] = *(const uint4*)(tile + d * stride + half * 16);
  }
  float key_scale[4], value_scale[4];
  if constexpr (I8) {
    const int64_t at = (t.page * c.kv_heads + t.kv) * (int64_t)c.p.page_size + t.off + 4 * q;
#pragma unroll
    for (int j = 0; j < 4; ++j) key_scale[j] = c.key_scales[at + j], value_scale[j] = c.value_scales[at + j];
  }
  uint32_t keys[4][CPL][N * kBytes / 4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const char* row = (const char*)c.keys + ((t.page * c.p.page_size + t.off + 4 * q + j) * c.kv_heads + t.kv) * (int64_t)c.dim * kBytes;
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const char* at = row + min(ci + 16 * i, chunks - 1) * N * kBytes;
#pragma unroll
      for (int w = 0; w < N * kBytes / 4; ++w) keys[j][i][w] = ((const uint32_t*)at)[w];
    }
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    const int chunk = ci + 16 * i;
    if (chunk >= chunks) break;
    uint32_t words[N][W];
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int w = 0; w < W; ++w) words[e][w] = staged[staged_word<N, W>(chunk * N + e, q) + w];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t position = t.first + 4 * q + j;
      if (position < t.lo || position >= t.hi) continue;
      const int64_t row = ((t.row + position - t.lo) * c.kv_heads + t.kv) * (int64_t)c.dim + chunk * N;
      float key[N], value[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (I8) {
          key[e] = (float)(int8_t)(keys[j][i][e / 4] >> (8 * (e % 4))) * key_scale[j];
          value[e] = (float)(int8_t)(words[e][0] >> (8 * j)) * value_scale[j];
        } else {
          key[e] = f16_value((keys[j][i][e / 2] >> (16 * (e % 2))) & 0xffffu);
          value[e] = f16_value((words[e][j / 2] >> (16 * (j % 2))) & 0xffffu);
        }
      }
      Chunk<T>::store(k + row, key);
      Chunk<T>::store(v + row, value);
    }
  }
}

template <typename T, bool I8>
__global__ void __launch_bounds__(64) read_rows(T* k, T* v, CacheRows c) {
  const int64_t unit = blockIdx.x / (unsigned)c.kv_heads;
  const int kv = blockIdx.x % (unsigned)c.kv_heads, lane = threadIdx.x;
  int64_t nth;
  const int s = locate(c.p, unit, 1, 0, 1, nth);
  if (s < 0) return;
  const Span span = span_of<true>(c.p, s);
  if (nth >= span.rows) return;
  const int64_t position = span.start + nth, page = span.table[position / c.p.page_size];
  const int64_t off = position % c.p.page_size;
  if (page < 0 || page >= c.p.cache_pages) {
    flag_bad(c.p);
    return;
  }
  const int64_t row = ((span.first + nth) * c.kv_heads + kv) * c.dim;
  for (int what = 0; what < 2; ++what) {
    const int64_t at = what ? (page * c.kv_heads + kv) * (int64_t)c.dim * c.p.page_size + off
                            : ((page * c.p.page_size + off) * c.kv_heads + kv) * c.dim;
    const int64_t stride = what ? c.p.page_size : 1;
    const float scale = I8 ? (what ? c.value_scales : c.key_scales)[(page * c.kv_heads + kv) * (int64_t)c.p.page_size + off] : 1.0f;
    for (int d = lane; d < c.dim; d += kWave) {
      float x;
      if constexpr (I8) x = (float)((const int8_t*)(what ? c.values : c.keys))[at + d * stride] * scale;
      else x = f16_value(((const uint16_t*)(what ? c.values : c.keys))[at + d * stride]);
      store_one((what ? v : k) + row + d, x);
    }
  }
}

// Chunks a lane of a head of `chunks`: 1, 2, 4 or 8 (0: more, or cut chunks).
int chunks_a_lane(int dim, int n) {
  if (dim % n != 0) return 0;
  const int each = (dim / n + 15) / 16;
  return each <= 1 ? 1 : each <= 2 ? 2 : each <= 4 ? 4 : each <= 8 ? 8 : 0;
}

template <typename T, bool WRITE, bool I8>
int launch_rows(const char* entry, T* k, T* v, CacheRows c, bool aligned, hipStream_t st) {
  // a call that names its rows by themselves (no offsets, a row a sequence) needs no further tile
  const bool single = !c.p.offsets && c.p.sequences == c.p.tokens;
  c.extra = single ? 0 : 1;
  const int each = aligned ? chunks_a_lane(c.dim, Chunk<T>::N) : 0;
  const int64_t blocks = (each ? units_of(c.p, kTile, c.extra, 1) : units_of(c.p, 1, 0, 1)) * c.kv_heads;
  if (blocks > kOneWaveBlocks) return refuse("%s: %d tokens of %d heads in one call", entry, c.p.tokens, c.kv_heads);
  const dim3 grid((unsigned)blocks), block(kWave);
#define DRIFT_ROWS(CPL)                                                                     \
  case CPL:                                                                                 \
    if constexpr (WRITE) hipLaunchKernelGGL((write_tiles<T, I8, CPL>), grid, block, 0, st, k, v, c); \
    else hipLaunchKernelGGL((read_tiles<T, I8, CPL>), grid, block, 0, st, k, v, c);         \
    break;
  switch (each) {
    DRIFT_ROWS(1)
    DRIFT_ROWS(2)
    DRIFT_ROWS(4)
    DRIFT_ROWS(8)
    default:
      if constexpr (WRITE) hipLaunchKernelGGL((write_rows<T, I8>), grid, block, 0, st, k, v, c);
      else hipLaunchKernelGGL((read_rows<T, I8>), grid, block, 0, st, k, v, c);
  }
#undef DRIFT_ROWS
  return launched(entry);
}

template <typename T, bool WRITE>
int cache_rows(const char* entry, T* k, T* v, void* keys, void* values, float* key_scales, float* value_scales,
               const Paging& p, int32_t kv_heads, int32_t dim, void* stream) {
  clear_error();
  if (const int bad = check_paging(entry, p, kv_heads, dim)) return bad;
  if (p.tokens == 0 || p.sequences == 0) return 0;
  if (!k || !v) return refuse("%s: null tensor", entry);
  if (const int bad = check_cache(entry, p, keys, values, key_scales, value_scales)) return bad;
  const CacheRows c{p, kv_heads, dim, keys, values, key_scales, value_scales, 0};
  const bool aligned = aligned16(k) && aligned16(v) && aligned16(keys) && aligned16(values);
  return key_scales ? launch_rows<T, WRITE, true>(entry, k, v, c, aligned, (hipStream_t)stream)
                    : launch_rows<T, WRITE, false>(entry, k, v, c, aligned, (hipStream_t)stream);
}

}  // namespace
}  // namespace drift

using namespace drift;

#define DRIFT_PAGING Paging{page_tables, starts, offsets, sequences, table_pages, cache_pages, page_size, start, tokens, bad_page}

extern "C" int drift_paged_write_f32(const float* k, const float* v, void* keys, void* values, float* key_scales,
                                     float* value_scales, const int32_t* page_tables, int32_t table_pages,
                                     int32_t cache_pages, const int32_t* starts, const int32_t* offsets,
                                     int32_t sequences, int32_t start, int32_t tokens, int32_t kv_heads,
                                     int32_t head_dim, int32_t page_size, int32_t* bad_page, void* stream) {
  return cache_rows<float, true>("drift_paged_write_f32", const_cast<float*>(k), const_cast<float*>(v), keys, values,
                                 key_scales, value_scales, DRIFT_PAGING, kv_heads, head_dim, stream);
}

extern "C" int drift_paged_write_bf16(const uint16_t* k, const uint16_t* v, void* keys, void* values,
                                      float* key_scales, float* value_scales, const int32_t* page_tables,
                                      int32_t table_pages, int32_t cache_pages, const int32_t* starts,
                                      const int32_t* offsets, int32_t sequences, int32_t start, int32_t tokens,
                                      int32_t kv_heads, int32_t head_dim, int32_t page_size, int32_t* bad_page,
                                      void* stream) {
  return cache_rows<uint16_t, true>("drift_paged_write_bf16", const_cast<uint16_t*>(k), const_cast<uint16_t*>(v), keys,
                                    values, key_scales, value_scales, DRIFT_PAGING, kv_heads, head_dim, stream);
}

extern "C" int drift_paged_read_f32(float* k, float* v, const void* keys, const void* values, const float* key_scales,
                                    const float* value_scales, const int32_t* page_tables, int32_t table_pages,
                                    int32_t cache_pages, const int32_t* starts, const int32_t* offsets,
                                    int32_t sequences, int32_t start, int32_t tokens, int32_t kv_heads,
                                    int32_t head_dim, int32_t page_size, int32_t* bad_page, void* stream) {
  return cache_rows<float, false>("drift_paged_read_f32", k, v, const_cast<void*>(keys), const_cast<void*>(values),
                                  const_cast<float*>(key_scales), const_cast<float*>(value_scales), DRIFT_PAGING,
                                  kv_heads, head_dim, stream);
}

extern "C" int drift_paged_read_bf16(uint16_t* k, uint16_t* v, const void* keys, const void* values,
                                     const float* key_scales, const float* value_scales, const int32_t* page_tables,
                                     int32_t table_pages, int32_t cache_pages, const int32_t* starts,
                                     const int32_t* offsets, int32_t sequences, int32_t start, int32_t tokens,
                                     int32_t kv_heads, int32_t head_dim, int32_t page_size, int32_t* bad_page,
                                     void* stream) {
  return cache_rows<uint16_t, false>("drift_paged_read_bf16", k, v, const_cast<void*>(keys), const_cast<void*>(values),
                                     const_cast<float*>(key_scales), const_cast<float*>(value_scales), DRIFT_PAGING,
                                     kv_heads, head_dim, stream);
}
