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

struct AttentionArgs {
  Paging p;
  int32_t heads, kv_heads, dim, group;
  float scale;
  int32_t window, sinks;  // window 0: every position up to the row's own
  const void *keys, *values;
  const float *key_scales, *value_scales;
};

__device__ __forceinline__ float f16_value(uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

__device__ __forceinline__ bool visible(const AttentionArgs& a, int64_t j, int64_t position) {
  return j <= position && (a.window == 0 || j > position - a.window || j < a.sinks);
}

// Any head size and alignment: a wave a row (a token's query head), 64
// positions at a time, a lane a position for the scores and then a lane a value
// for the sums. Every product is of F32 values in F32, one by one: what bounds it
// is the vector unit and the unaligned loads.
template <typename T, bool I8>
__global__ void __launch_bounds__(64) attend_rows(const T* queries, T* out, AttentionArgs a) {
  __shared__ float query[kMaxHead];
  __shared__ float weight[kWave];
  __shared__ int64_t place[kWave];  // the value's index at dimension 0, or -1: not visible
  const int lane = threadIdx.x, h = blockIdx.x % (unsigned)a.heads, kv = h / a.group;
  int64_t nth;
  const int s = locate(a.p, blockIdx.x / (unsigned)a.heads, 1, 0, 1, nth);
  if (s < 0) return;
  const Span span = span_of(a.p, s);
  if (nth >= span.rows) return;
  const int64_t position = span.start + nth, row = ((span.first + nth) * a.heads + h) * a.dim;
  for (int d = lane; d < a.dim; d += kWave) query[d] = load_one(queries + row + d);
  wave_sync();
  constexpr int kEach = kMaxHead / kWave;
  float sums[kEach] = {}, top = -__builtin_huge_valf(), total = 0.0f;
  bool any = false;
  const int64_t low = a.window ? max(position - a.window + 1, (int64_t)0) : 0;
  const int64_t sink_end = a.window ? min((int64_t)a.sinks, low) : 0;
  for (int64_t base = 0; base <= position; base += kWave) {
    if (base >= sink_end && base + kWave <= low) base = low / kWave * kWave;  // what lies between is not seen
    const int64_t j = base + lane;
    bool seen = visible(a, j, position);
    int64_t page = 0, off = 0;
    if (seen) {
      page = span.table[j / a.p.page_size];
      off = j % a.p.page_size;
      if (page < 0 || page >= a.p.cache_pages) {
        flag_bad(a.p);
        seen = false;
      }
    }
    float score = -__builtin_huge_valf(), value_scale = 1.0f;
    if (seen) {
      const int64_t key = ((page * a.p.page_size + off) * a.kv_heads + kv) * a.dim;
      float dot = 0.0f;
      for (int d = 0; d < a.dim; ++d) {
        float k;
        if constexpr (I8) k = (float)((const int8_t*)a.keys)[key + d];
        else k = f16_value(((const uint16_t*)a.keys)[key + d]);
        dot = fmaf(query[d], k, dot);
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
    const float ref = next == -__builtin_huge_valf() ? 0.0f : next;
    const float keep = expf(top - ref);
    const float p = seen ? expf(score - ref) : 0.0f;
    any |= __any(seen);
    top = next;
    float sum = p;
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) sum += __shfl_xor(sum, mask, kWave);
    total = fmaf(total, keep, sum);
    wave_sync();
    weight[lane] = p * value_scale;
    place[lane] = seen ? (page * a.kv_heads + kv) * (int64_t)a.dim * a.p.page_size + off : -1;
    wave_sync();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int d = lane + i * kWave;
      if (d >= a.dim) break;
      float acc = sums[i] * keep;
      for (int n = 0; n < kWave; ++n) {
        const int64_t at = place[n];
        if (at < 0) continue;
        float v;
        if constexpr (I8) v = (float)((const int8_t*)a.values)[at + (int64_t)d * a.p.page_size];
        else v = f16_value(((const uint16_t*)a.values)[at + (int64_t)d * a.p.page_size]);
        acc = fmaf(weight[n], v, acc);
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
  const hipStream_t st = (hipStream_t)stream;
  const int64_t blocks = units_of(a.p, 1, 0, 1) * a.heads;
  if (blocks > kOneWaveBlocks) return refuse("%s: %d tokens of %d heads in one call", entry, a.p.tokens, a.heads);
  const dim3 grid((unsigned)blocks), block(kWave);
  if (a.key_scales) hipLaunchKernelGGL((attend_rows<T, true>), grid, block, 0, st, queries, out, a);
  else hipLaunchKernelGGL((attend_rows<T, false>), grid, block, 0, st, queries, out, a);
  return launched(entry);
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
  return 0;
}

extern "C" int drift_paged_attention_f32(const float* queries, const void* keys, const void* values,
                                         const float* key_scales, const float* value_scales,
                                         const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                         const int32_t* starts, const int32_t* offsets, int32_t sequences,
                                         int32_t start, int32_t tokens, int32_t heads, int32_t kv_heads,
                                         int32_t head_dim, int32_t page_size, float scale, int32_t window,
                                         int32_t sinks, int32_t longest, float* out, void* workspace,
                                         int64_t workspace_bytes, int32_t* bad_page, void* stream) {
  const AttentionArgs a{{page_tables, starts, offsets, sequences, table_pages, cache_pages, page_size, start, tokens,
                         bad_page}, heads, kv_heads, head_dim, 0, scale, window, sinks, keys, values, key_scales,
                        value_scales};
  return paged_attention<float>("drift_paged_attention_f32", queries, out, a, longest, workspace, workspace_bytes,
                                stream);
}

extern "C" int drift_paged_attention_bf16(const uint16_t* queries, const void* keys, const void* values,
                                          const float* key_scales, const float* value_scales,
                                          const int32_t* page_tables, int32_t table_pages, int32_t cache_pages,
                                          const int32_t* starts, const int32_t* offsets, int32_t sequences,
                                          int32_t start, int32_t tokens, int32_t heads, int32_t kv_heads,
                                          int32_t head_dim, int32_t page_size, float scale, int32_t window,
                                          int32_t sinks, int32_t longest, uint16_t* out, void* workspace,
                                          int64_t workspace_bytes, int32_t* bad_page, void* stream) {
  const AttentionArgs a{{page_tables, starts, offsets, sequences, table_pages, cache_pages, page_size, start, tokens,
                         bad_page}, heads, kv_heads, head_dim, 0, scale, window, sinks, keys, values, key_scales,
                        value_scales};
  return paged_attention<uint16_t>("drift_paged_attention_bf16", queries, out, a, longest, workspace,
                                   workspace_bytes, stream);
}
