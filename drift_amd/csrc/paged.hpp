// The paged key and value cache as several sequences' calls see it: the page
// tables, where each sequence's token rows lie and at which positions, and
// the checks that the entry points over it share.
//
// The cache (ops/KvCache.scala:5-22): keys [pages, page_size, kv_heads,
// head_dim], values [pages, kv_heads, head_dim, page_size] (transposed within
// a page), in F16; or in 8 bits, the same two of int8 codes with F32 scales
// [pages, kv_heads, page_size], one a position and key head: a value is its
// code times its row's scale.
#pragma once

#include "common.hpp"

#include <algorithm>

namespace drift {

// Several sequences' token rows, packed: sequence s has rows offsets[s] up to
// offsets[s + 1] of the token tensors, at positions starts[s] and on, in the
// pages of tables[s]. All three are read on the device, so a captured launch
// serves as sequences grow. Without offsets there is one sequence of all
// rows, or a row a sequence; without starts one sequence at `start`.
struct Paging {
  const int32_t* tables;   // [sequences, table_pages]
  const int32_t* starts;   // nullable
  const int32_t* offsets;  // nullable
  int32_t sequences, table_pages, cache_pages, page_size, start, tokens;
  int32_t* bad_page;  // nullable
};

// A value that every lane of a wave holds alike, in scalar registers: what comes
// from memory or across lanes the compiler takes for different otherwise, and
// then masks every branch and loop on it.
template <typename T>
__device__ __forceinline__ T uniform(T v) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "");
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
  } else {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)bits);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(bits >> 32));
    return __builtin_bit_cast(T, ((uint64_t)hi << 32) | lo);
  }
}

// Positions a sequence can have: a tile past its last still counts in 32 bits.
constexpr int64_t kMostPositions = INT32_MAX - 127;

struct Span {
  int64_t first;         // its first token row
  int32_t rows;          // 0 where the sequence is not described rightly
  int64_t start;         // the first row's position
  const int32_t* table;  // its pages
};

__device__ __forceinline__ void flag_bad(const Paging& p) {
  if (p.bad_page) *p.bad_page = 1;
}

// Sequence s as the device's arrays describe it. Rows outside the token
// tensors or before the end of an earlier sequence, or with rows a start below 0
// or an end past the page table, make it a sequence of no rows and set the flag:
// nothing is read or written for it. (Offsets that go back would else give rows to two
// sequences, and more units than a launch has; LOCATED: locate has seen to that.)
// Whole waves call, every lane with the same s.
template <bool LOCATED>
__device__ __forceinline__ Span span_of(const Paging& p, int s) {
  Span span;
  bool behind = false;
  int64_t from = p.sequences == 1 ? 0 : s, to = p.sequences == 1 ? p.tokens : s + 1;
  if (p.offsets) {
    const int begin = p.offsets[s], end = p.offsets[s + 1];
    if constexpr (!LOCATED) {
      int l = threadIdx.x & (kWave - 1), before = p.offsets[min(l, s)];  // (asked for together with the others)
      for (;;) {
        behind |= before > begin && before <= p.tokens;
        if ((l += kWave) >= s) break;
        before = p.offsets[l];
      }
      behind = __any(behind);
    }
    from = uniform(begin);
    to = uniform(end);
  }
  span.start = p.starts ? uniform(p.starts[s]) : p.start;
  span.first = from;
  span.table = p.tables + (int64_t)s * p.table_pages;
  const bool good = from >= 0 && to >= from && to <= p.tokens && !behind &&
                    (to == from || (span.start >= 0 && span.start + (to - from) <=
                                                           min((int64_t)p.table_pages * p.page_size, kMostPositions)));
  if (!good) flag_bad(p);
  span.rows = good ? (int32_t)(to - from) : 0;
  return span;
}

// Work in units of `per` items, a row having `scale` of them: ceil(rows scale /
// per) + extra units a sequence, by offsets none where there are `least` items or
// fewer. The sequence that unit `unit` of the launch belongs to (-1: none), and
// which of its units it is. Whole waves call, every lane with the same unit.
__device__ __forceinline__ int locate(const Paging& p, int64_t unit, int per, int extra, int64_t scale, int64_t& nth,
                                          int64_t least = 0) {
  if (!p.offsets) {
    if (p.sequences == 1) {
      nth = unit;
      return 0;
    }
    const int64_t each = (scale + per - 1) / per + extra;
    nth = unit % each;
    const int64_t s = unit / each;
    return s < p.sequences ? (int)s : -1;
  }
  const int lane = threadIdx.x & (kWave - 1);
  int passed = INT32_MIN;  // the largest offset of the groups of sequences before, of those that name a row
  for (int base = 0; base < p.sequences; base += kWave) {
    const int s = base + lane;
    int64_t units = 0;
    const int from = p.offsets[min(s, p.sequences)], to = p.offsets[min(s + 1, p.sequences)];
    int most = from;  // of the offsets up to and with this lane's
    if (__any(to < from || to > p.tokens)) {
      most = from <= p.tokens ? from : INT32_MIN;
#pragma unroll
      for (int step = 1; step < kWave; step <<= 1) {
        const int before = __shfl_up(most, step, kWave);
        if (lane >= step) most = max(most, before);
      }
    }
    most = max(most, passed);
    if (s < p.sequences) {
      const bool good = from >= most && from >= 0 && to >= from && to <= p.tokens;
      if (!good) flag_bad(p);  // and no units, so that the others' are all in the launch
      const int64_t rows = (int64_t)to - from;
      units = good && rows * scale > least ? (rows * scale + per - 1) / per + extra : 0;
    }
    int64_t end = units;  // units of this group of sequences, up to and with this lane's
#pragma unroll
    for (int step = 1; step < kWave; step <<= 1) {
      const int64_t before = __shfl_up(end, step, kWave);
      if (lane >= step) end += before;
    }
    const uint64_t past = __ballot(unit < end);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      nth = unit - uniform(__shfl(end, at, kWave) - __shfl(units, at, kWave));
      return base + at;
    }
    unit -= uniform(__shfl(end, kWave - 1, kWave));
    passed = uniform(__shfl(most, kWave - 1, kWave));
  }
  return -1;
}

// ---------------------------------------------------------------- host side

// Units a launch needs for every sequence's (locate), whatever the offsets hold: a part of one is left over in as
// many sequences as can have more than `least` items, and one unit more looks through every sequence's offsets.
inline int64_t units_of(const Paging& p, int64_t per, int64_t extra, int64_t scale, int64_t least = 0) {
  if (p.offsets) {
    const int64_t items = (int64_t)p.tokens * scale;
    return items / per + std::min((int64_t)p.sequences, items / (least + 1)) * (1 + extra) + (p.sequences > kWave);
  }
  if (p.sequences == 1) return ceil_div((int64_t)p.tokens * scale, per) + extra;
  return p.sequences * (ceil_div(scale, per) + extra);
}

// The checks of a call over the paged cache; nonzero (refused) if bad.
int check_paging(const char* entry, const Paging& p, int32_t kv_heads, int32_t head_dim);
// Its tensors: the cache's, and the page tables.
int check_cache(const char* entry, const Paging& p, const void* keys, const void* values, const float* key_scales,
                const float* value_scales);

}  // namespace drift
