// MXFP4 matrices: 4-bit floats (E2M1) in blocks of 32 along a row that share
// one power of two (E8M0), as in the OCP Microscaling Formats specification
// v1.0.  Layout and conversions shared by the kernels.
//
// A packed matrix of R rows and K columns is two arrays:
//   Q[R][q_pitch(K)]  two elements a byte, the even column in the low four
//                     bits; a row is a whole number of 128-byte lines (256
//                     columns), zero behind column K;
//   S[ceil(K / 512)][R][16]  biased exponents: the scale of row r and block b
//                     (columns 32 b .. 32 b + 31) is byte s_byte(b) of entry
//                     [b / 16][r], zero behind column K.
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 128 columns: lane l supplies 32 of
// row l % 16, those of block 4 t + l / 16 of its 512 columns in step t, and
// their scale in a byte of a register chosen by the instruction.  s_byte puts
// the scales that one lane needs in the four steps of 512 columns into one
// dword, and those of the 16 rows of a fragment into 256 contiguous bytes: a
// lane loads one dword for four steps and spends no instruction on
// rearranging it (with the blocks of a row in order it takes a byte of each of
// four dwords).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "dbg_checks.hpp"
#include "miaie_internal.hpp"

namespace miaie {
namespace mx {

__host__ __device__ constexpr size_t q_pitch(int K) { return ((size_t)K + 255) / 256 * 128; }  // bytes of a row of Q
__host__ __device__ constexpr int s_groups(int K) { return (int)(((long)K + 511) / 512); }     // entries [b / 16]
__host__ __device__ constexpr int s_byte(int b) { return (b & 3) * 4 + ((b >> 2) & 3); }

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v8f __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));

// V at any address that is a multiple of T's size (gfx950's unaligned access mode)
template <class V, class T>
struct __attribute__((packed, aligned(alignof(T)))) At {
  V v;
};

// Scale byte of a block whose largest magnitude has the fp32 bits `amax`
// (sign cleared): 2^(floor(log2(amax)) - 2) puts that value into [4, 8), where
// E2M1 ends at 6.  Below 2^-127 (all-zero blocks among them) the scale stays at
// 2^-127; a block that holds an infinity or NaN becomes NaN (255).
__device__ __forceinline__ uint32_t scale_of(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e == 255 ? 255u : max(e, 2u) - 2;
}

// The power of two as the conversions take it: they read the exponent field
// alone, so 0 is 2^-127 (checked on the device for every scale and rounding
// boundary; halves go to the even code, magnitudes beyond 6 to 6).
__device__ __forceinline__ float scale_f32(uint32_t s) { return __uint_as_float(s << 23); }

// Eight values to eight codes, the first in the low four bits.
__device__ __forceinline__ uint32_t pack8(const float (&x)[8], float scale) {
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[0], x[1], scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[2], x[3], scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[4], x[5], scale, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, x[6], x[7], scale, 3);
  return q;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// v of another lane of the same four (CTRL: two bits of source lane for each)
template <int CTRL>
__device__ __forceinline__ uint32_t quad_swap(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}

// Eight consecutive elements as they are in memory, n of them inside the row (n >= 1; the rest 0).
template <class T>
struct Raw8 {
  typedef T V __attribute__((ext_vector_type(8)));
  V v;
  __device__ __forceinline__ void clear() { v = V{}; }
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= 8) {
      using P = At<V, T>;
      v = MIAIE_LD(reinterpret_cast<const P*>(p)).v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? MIAIE_LD(p + i) : (T)0.f;
    }
  }
  // The values are in the registers from here on: a load is waited for here, not
  // where the compiler first uses it.
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(V) / 16; ++i) {
      v4i w;
      __builtin_memcpy(&w, reinterpret_cast<const char*>(&v) + 16 * i, 16);
      asm volatile("" : "+v"(w));
      __builtin_memcpy(reinterpret_cast<char*>(&v) + 16 * i, &w, 16);
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};

// The same as fp32.
template <class T>
__device__ __forceinline__ void load8(const T* p, int n, float (&x)[8]) {
  typedef T V __attribute__((ext_vector_type(8)));
  if (n >= 8) {
    using P = At<V, T>;
    const V v = MIAIE_LD(reinterpret_cast<const P*>(p)).v;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? (float)MIAIE_LD(p + i) : 0.f;
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, int n, const float (&x)[8]) {
  typedef T V __attribute__((ext_vector_type(8)));
  V v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
  if (n >= 8) {
    using P = At<V, T>;
    MIAIE_ST(reinterpret_cast<P*>(p), P{v});
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) MIAIE_ST(p + i, v[i]);
  }
}

}  // namespace mx
}  // namespace miaie
