// The attention that cached positions gather (paged.hpp has the cache's
// layouts): what a position has been weighed by the rows that see it, of one
// sequence or several in a launch.
//
// Token t of a sequence sits at position P = start + t and sees the positions j <= P
// of its own sequence; query head h reads key head h / (heads / kv_heads). With
//   s_j = scale q.k_j,  p_j = exp(s_j - m) / sum_j exp(s_j - m)
// over the visible j, a position's and key head's mass is the sum of p_j over the
// call's tokens and the heads that read it; where the sequence held the position
// before the call (j < start), added to what it had. Scores are taken twice, for the
// rows' statistics and, these known, for the positions' sums, which one wave each
// takes in the rows' order: no atomics, and the same bits every time.
#include "paged.hpp"

#include <algorithm>

namespace drift {
namespace {

constexpr int kMaxHead = 512;
constexpr float kInfinity = __builtin_huge_valf();

struct MassArgs {
  Paging p;
  int32_t heads, kv_heads, dim, group;
  float scale;
  const void* keys;
  const float *key_scales, *before;
  float* mass;
  float* statistics;  // [tokens, heads, 2]: a row's largest score, and the sum of exp(score - that)
  int32_t splits;
  UnitColumns columns;
};

__device__ __forceinline__ float f16_value(uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Where position j of a sequence has its numbers [cache_pages, kv_heads, page_size], and its keys; false: nowhere.
struct Place {
  int64_t word, key;
};
__device__ __forceinline__ bool place_of(const MassArgs& a, const Span& span, int64_t j, int kv, Place& place) {
  const int64_t page = span.table[j / a.p.page_size], off = j % a.p.page_size;
  if (page < 0 || page >= a.p.cache_pages) {
    flag_bad(a.p);
    return false;
  }
  place.word = (page * a.kv_heads + kv) * (int64_t)a.p.page_size + off;
  place.key = ((page * a.p.page_size + off) * a.kv_heads + kv) * (int64_t)a.dim;
  return true;
}

// The score of a row (its query in LDS) and a position, by F32 products one after another.
template <bool I8>
__device__ __forceinline__ float score_of(const MassArgs& a, const float* query, const Place& place) {
  float dot = 0.0f;
  for (int d = 0; d < a.dim; ++d) {
    const float k = I8 ? (float)((const int8_t*)a.keys)[place.key + d] : f16_value(((const uint16_t*)a.keys)[place.key + d]);
    dot = fmaf(query[d], k, dot);
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
    const float score = seen ? score_of<I8>(a, query, place) : -kInfinity;
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
// head.
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
        sum += expf(score_of<I8>(a, query, place) - ref) / a.statistics[row * 2 + 1];
      }
    if (there) a.mass[place.word] = (float)(a.before && j < span.start ? a.before[place.word] + sum : sum);
  }
}

// ------------------------------------------------------------------ host side

int check_mass(const char* entry, int32_t heads, int32_t kv_heads, int32_t dim, int64_t longest) {
  if (dim > kMaxHead) return refuse("%s: heads of %d values (at most %d)", entry, dim, kMaxHead);
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return refuse("%s: %d heads over %d key heads", entry, heads, kv_heads);
  if (longest < 0) return refuse("%s: a longest sequence of %lld positions", entry, (long long)longest);
  return 0;
}

struct Plan {
  int64_t bytes;
};

Plan plan_of(int64_t sequences, int64_t tokens, int64_t heads) {
  if (sequences <= 0 || tokens <= 0) return {0};
  return {ceil_div(tokens * heads * 2, 4) * 16};
}

template <typename T, bool I8>
int launch_mass(const char* entry, const T* queries, MassArgs a, int64_t longest, hipStream_t st) {
  const int64_t row_blocks = units_of(a.p, 1, 0, 1) * a.heads, units = (int64_t)a.p.sequences * a.kv_heads;
  if (row_blocks > kOneWaveBlocks || units > kOneWaveBlocks / 16)
    return refuse("%s: %d tokens of %d heads in one call", entry, a.p.tokens, a.heads);
  a.splits = (int)std::min<int64_t>(std::max<int64_t>(ceil_div(longest, kWave), 1),
                                    std::max<int64_t>(16384 / units, 1));
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
  if (const int bad = check_mass(entry, a.heads, a.kv_heads, a.dim, longest)) return bad;
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
  const Plan plan = plan_of(a.p.sequences, a.p.tokens, a.heads);
  if (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace))
    return refuse("%s: a workspace of %lld bytes, needs %lld at a multiple of 16", entry, (long long)workspace_bytes,
                  (long long)plan.bytes);
  a.statistics = (float*)workspace;
  a.group = a.heads / a.kv_heads;
  a.columns = unit_columns(a.p.page_size);
  return a.key_scales ? launch_mass<T, true>(entry, queries, a, longest, (hipStream_t)stream)
                      : launch_mass<T, false>(entry, queries, a, longest, (hipStream_t)stream);
}

}  // namespace
}  // namespace drift

using namespace drift;

extern "C" int drift_attention_mass_workspace(int32_t sequences, int32_t tokens, int32_t heads, int32_t kv_heads,
                                              int32_t head_dim, int32_t longest, int64_t* bytes) {
  clear_error();
  if (!bytes) return refuse("drift_attention_mass_workspace: null bytes");
  *bytes = 0;
  if (const int bad = check_mass("drift_attention_mass_workspace", heads, kv_heads, head_dim, longest)) return bad;
  *bytes = plan_of(sequences, tokens, heads).bytes;
  return 0;
}

#define DRIFT_MASS_ARGS                                                                                             \
  MassArgs {                                                                                                        \
    {page_tables, starts, offsets, sequences, table_pages, cache_pages, page_size, start, tokens, bad_page}, heads, \
        kv_heads, head_dim, 0, scale, keys, key_scales, before, mass, nullptr, 1, {}                                \
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
