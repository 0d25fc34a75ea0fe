// 8-bit floating point matrices (E4M3: four exponent bits, three mantissa bits,
// up to 448, no infinities) with an fp32 scale for each block of 128, and the
// slots of tokens routed to experts.  Layout and conversions shared by the
// kernels.
//
// A packed matrix of R rows and K columns is two arrays:
//   Q[R][pitch(K)]  one element a byte, rows of whole 128-byte lines, zero behind
//                   column K;
//   S[ceil(K / 128)][ceil(R / block)]  the scale of 128 columns of `block` rows,
//                   1 or 128.  Columns first: the scales of a tile's rows in one
//                   step of a product are beside each other.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "dbg_checks.hpp"
#include "miaie_internal.hpp"
#include "mxfp4.hpp"

namespace miaie {
namespace fp8 {

using mx::abs_bits;
using mx::At;
using mx::v4bf;
using mx::v8i;
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

__host__ __device__ constexpr size_t blocks(long n) { return ((size_t)n + 127) / 128; }
__host__ __device__ constexpr size_t pitch(int K) { return blocks(K) * 128; }

// Exponent field of the scale of a block whose largest magnitude has the fp32 bits
// `amax` (sign cleared): the smallest power of two that amax is at most 448 =
// 1.75 x 2^8 times, at least 2^-126 so that its reciprocal is finite too.  Powers
// of two make x / S exact: an element is rounded once, and every implementation
// gets the same codes.  They are also what the matrix instructions scale by.
// 255: the block holds an infinity or NaN, and all of it becomes NaN.
__device__ __forceinline__ uint32_t scale_of(uint32_t amax) {
  const int e = (int)((amax + 0x1fffff) >> 23) - 8;
  return amax >= 0x7f800000 ? 255u : (uint32_t)max(e, 1);
}
__device__ __forceinline__ float scale_f32(uint32_t e) { return __uint_as_float(e == 255 ? 0x7fc00000u : e << 23); }
__device__ __forceinline__ float inverse_f32(uint32_t e) { return __uint_as_float((254 - min(e, 253u)) << 23); }

// Four values times inv to four codes, the first in the low byte; halves go to the
// even code.  (Magnitudes up to 448 x (1 / inv) by the scale's choice.)
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float inv) {
  int q = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, q, true);
}

// a of lanes 32.. with b of lanes 0..31, and a of odd sixteens with b of even ones
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
// Largest of the four lanes 16 apart.
__device__ __forceinline__ uint32_t max_over_16s(uint32_t v) {
  uint32_t w = v;
  swap32(v, w);
  w = v = max(v, w);
  swap16(v, w);
  return max(v, w);
}

// s = 1 / (1 + e^-g) and 1 - s, from e^-|g|, which does not overflow; the reciprocal is
// good to a unit in the last place
struct Sigmoid {
  float s, rest;
  __device__ __forceinline__ explicit Sigmoid(float g) {
    const float x = expf(-fabsf(g)), big = __builtin_amdgcn_rcpf(1.f + x), small = x * big;
    s = g < 0.f ? small : big, rest = g < 0.f ? big : small;
  }
};
// silu(g) u
__device__ __forceinline__ float swiglu(float g, float u) { return g * Sigmoid(g).s * u; }

// ---- slots: the (token, choice) pairs of T tokens with k choices each, sorted by
// expert, every expert's from a multiple of 128 on.  One array of ints.
struct Slots {
  const int* start;      // [E + 1]: first slot of each expert; the last: slots in use, a multiple of 128
  const int* count;      // [E]
  const int* slot_of;    // [T k]: slot of a pair, -1 without an expert
  const int* row_of;     // [rows]: pair of a slot (t k + choice), -1 in padding
  const int* expert_of;  // [rows / 128], -1 behind the last slot in use (for callers; the kernels go by the counts)
  int tokens, top_k, experts, rows;
};

constexpr size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// Most slots that the pairs can take: E' = min(E, T k) experts with 127 slots of
// padding each, where the pairs allow that.
constexpr long slot_rows(long tokens, long top_k, long experts) {
  const long n = tokens * top_k, used = experts < n ? experts : n;
  return 128 * (used + (n - used) / 128);
}
constexpr size_t slot_ints(long tokens, long top_k, long experts) {
  const size_t rows = (size_t)slot_rows(tokens, top_k, experts);
  return round16(2 * experts + 1) + round16((size_t)tokens * top_k) + rows + rows / 128;
}
inline Slots slots_of(const int* order, int tokens, int top_k, int experts) {
  Slots s;
  s.tokens = tokens, s.top_k = top_k, s.experts = experts, s.rows = (int)slot_rows(tokens, top_k, experts);
  s.start = order;
  s.count = order + experts + 1;
  s.slot_of = order + round16(2 * (size_t)experts + 1);
  s.row_of = s.slot_of + round16((size_t)tokens * top_k);
  s.expert_of = s.row_of + s.rows;
  return s;
}

}  // namespace fp8
}  // namespace miaie
