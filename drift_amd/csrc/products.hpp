// Shared pieces of the kernels that take scores of rows and cached positions by
// matrix instructions: their operands' types, the 8-bit cache's codes as F16
// numbers, and F32 values as F16 terms. (How a row of queries is scaled is each
// kernel's own: those that compare products before they are scores turn a negative
// scale's sign into the query and keep the factor above 0, attend_few, which scales
// every product at once, needs neither.)
#pragma once

#include "paged.hpp"

namespace drift {
namespace {

constexpr float kInfinity = __builtin_huge_valf();

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
// 16 bytes at an address of 8-byte multiples
typedef unsigned int u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// Bits 0 .. n - 1.
__device__ __forceinline__ uint64_t bits_below(int64_t n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }

__device__ __forceinline__ float f16_value(uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
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

// Eight of a lane's values as a product takes them: F16, and with two terms the
// F16 remainder too.
template <int TERMS>
struct Halves {
  f16x8 term[TERMS];
};
template <int TERMS>
__device__ __forceinline__ Halves<TERMS> halves_of(const float (&v)[8]) {
  Halves<TERMS> h;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float x = v[i];
    // one F32 value for both terms: left to itself the compiler rounds a product once, to F16, for the first and
    // twice for the second, and at a tie the two then belong to different neighbours
    if constexpr (TERMS == 2) asm volatile("" : "+v"(x));
    h.term[0][i] = (_Float16)x;
    if constexpr (TERMS == 2) h.term[1][i] = (_Float16)(x - (float)h.term[0][i]);
  }
  return h;
}

// ---------------------------------------------------------------- host side

// How positions are split among blocks.
struct Split {
  int splits;  // over positions; 0: nothing is to be done this way
  int chunk;   // tiles of 64 positions that a split has at least
};

// Blocks with their splits, at most, where sequences are split evenly whatever the chip
// has room for: 32 times 512 places even out any lengths, and what the splits leave in
// the workspace stays within so many blocks' rows however wide the page tables are.
constexpr int64_t kSplitBlocks = 16384;

// `blocks` blocks before the split, over `positions` positions, towards `wanted`
// of them.
inline Split split_of(int64_t blocks, int64_t positions, int64_t wanted, int64_t least, int64_t most) {
  const int64_t tiles = std::max<int64_t>(ceil_div(positions, 64), 1);
  const int64_t chunk = std::min(std::max(ceil_div(tiles * blocks, wanted), least), most);
  const int64_t room = std::min<int64_t>(std::max<int64_t>(kSplitBlocks / blocks, 1), 1024);
  return {(int)std::min(ceil_div(tiles, chunk), room), (int)std::min<int64_t>(chunk, INT32_MAX)};
}

}  // namespace
}  // namespace drift
