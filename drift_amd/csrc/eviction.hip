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
__global__ void __launch_bounds__(kPickThreads) pick_heaviest(HeaviestArgs a) {
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t sums[2][kPickWaves];
  __shared__ uint32_t found[2];
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
  auto order_at = [&](uint32_t candidate) -> uint32_t {
    const uint32_t j = candidate + a.sinks, unit = j / 16, column = a.columns.of(unit);
    const int32_t page = table[column];
    if (page < 0 || page >= a.cache_pages) {
      if (a.bad_page) *a.bad_page = 1;
      return 0;
    }
    return order_of(a.mass[((int64_t)page * a.kv_heads + kv) * a.page_size + (j - column * a.columns.page_units * 16)]);
  };

  uint32_t digits = 0, known = 0, left = wanted;  // the threshold's digits so far, and how many are wanted of those that share them
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 1024 : 2048;
    for (int i = thread; i < kBins; i += kPickThreads) bins[i] = 0;
    __syncthreads();
    for (uint32_t i = thread; i < candidates; i += kPickThreads) {
      const uint32_t order = order_at(i);
      if ((order & known) == digits) atomicAdd(&bins[order >> shift & (width - 1)], 1u);
    }
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
    if (above < left && left <= above + high) found[0] = bin + 1, found[1] = above;
    else if (above + high < left && left <= above + high + low) found[0] = bin, found[1] = above + high;
    __syncthreads();
    digits |= found[0] << shift;
    known |= (uint32_t)(width - 1) << shift;
    left -= found[1];
    __syncthreads();
  }

  // a wave's candidates lie together, so that their places follow from the waves' before
  const uint32_t each = (candidates + kPickThreads - 1) / kPickThreads * kWave;
  const uint32_t begin = min(wave * each, candidates), end = min(begin + each, candidates);
  uint32_t more = 0, equal = 0;
  for (uint32_t i = begin; i < end; i += kWave) {
    const uint32_t order = i + lane < end ? order_at(i + lane) : 0;
    const bool in = i + lane < end;
    more += __popcll(__ballot(in && order > digits));
    equal += __popcll(__ballot(in && order == digits));
  }
  if (lane == 0) sums[0][wave] = more, sums[1][wave] = equal;
  __syncthreads();
  uint32_t more_before = 0, equal_before = 0;
  for (int w = 0; w < wave; ++w) more_before += sums[0][w], equal_before += sums[1][w];
  uint32_t place = a.sinks + more_before + min(equal_before, left);
  const uint64_t below = (1ull << lane) - 1;
  for (uint32_t i = begin; i < end; i += kWave) {
    const bool in = i + lane < end;
    const uint32_t order = in ? order_at(i + lane) : 0;
    const uint64_t ties = __ballot(in && order == digits);
    const bool taken = in && (order > digits || (order == digits && equal_before + __popcll(ties & below) < left));
    const uint64_t all = __ballot(taken);
    if (taken) kept[place + __popcll(all & below)] = (int32_t)(i + lane + a.sinks);
    place += __popcll(all);
    equal_before += __popcll(ties);
  }
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

// A wave a row. READ: from the cache, else from the scratch; WRITE: to the cache, else to the
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

int64_t scratch_row(int32_t dim, bool quantized) { return ceil_div((int64_t)dim * 2 * (quantized ? 1 : 2), 4) * 4 + 12; }

int check_keep(const char* entry, int32_t sequences, int32_t most, int32_t kv_heads, int32_t dim) {
  if (sequences < 0 || most < 0 || kv_heads <= 0 || dim <= 0)
    return refuse("%s: %d rows of %d sequences, %d heads of %d values", entry, most, sequences, kv_heads, dim);
  if ((int64_t)sequences * kv_heads > kOneWaveBlocks || (int64_t)sequences * kv_heads * most > kOneWaveBlocks * 4)
    return refuse("%s: %d rows of %d sequences, %d heads in one call", entry, most, sequences, kv_heads);
  return 0;
}

int64_t keep_bytes(int32_t sequences, int32_t most, int32_t kv_heads, int32_t dim, bool quantized) {
  return (int64_t)sequences * most * kv_heads * scratch_row(dim, quantized);
}

template <typename E>
int keep(const char* entry, const KeepArgs& a, bool apart, hipStream_t st) {
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
  hipLaunchKernelGGL(pick_heaviest, dim3((unsigned)(sequences * kv_heads)), dim3(kPickThreads), 0, (hipStream_t)stream, a);
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
