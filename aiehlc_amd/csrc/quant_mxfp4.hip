// Conversion of fp32 / bf16 matrices to MXFP4 (mxfp4.hpp) along their rows and
// along their columns, and back.
//
// The columns' form is the packed transpose: a product contracts along the
// packed axis, so the gradients dX = dY . W and dW = dY^T . X of a linear
// layer take dY, W and X packed along the other axis than Y = X . W^T does.
#include <algorithm>

#include "mxfp4.hpp"

namespace miaie {
namespace {

using namespace mx;

// One wave packs 512 columns of a row: lane l has columns 8 l .. 8 l + 7, four
// lanes a block.  Bound by memory: 8192 x 8192 bf16 in 39.6 us, 4.3 TB/s read and
// written (a copy of 1 GiB reaches 5.2); four pieces a wave, their loads in
// flight together, took 43.6.
template <class T>
__global__ __launch_bounds__(256) void quant_rows(const T* __restrict__ X, uint8_t* __restrict__ Q,
                                                  uint8_t* __restrict__ S, int R, int C, int ldx, int units,
                                                  int stride) {
  const int lane = threadIdx.x & 63;
  const int groups = s_groups(C);
  const size_t pitch = q_pitch(C);
  for (int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); unit < units; unit += stride) {
    const int row = unit / groups, g = unit % groups;
    const int c0 = 512 * g + 8 * lane;
    float x[8] = {};
    if (c0 < C) load8(X + (size_t)row * ldx + c0, C - c0, x);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, abs_bits(x[i]));
    amax = max(amax, quad_swap<0xB1>(amax));  // lanes 1 0 3 2
    amax = max(amax, quad_swap<0x4E>(amax));  // lanes 2 3 0 1
    const uint32_t s = scale_of(amax);
    const uint32_t q = pack8(x, scale_f32(s));
    if ((size_t)c0 < 2 * pitch) MIAIE_ST(reinterpret_cast<uint32_t*>(Q + row * pitch + c0 / 2), q);
    if ((lane & 3) == 0) MIAIE_ST(S + ((size_t)g * R + row) * 16 + s_byte(lane >> 2), (uint8_t)s);
  }
}

typedef uint16_t v2us __attribute__((ext_vector_type(2)));

// Two adjacent columns of one row; the second is absent in the last column of
// an odd matrix.
template <class T>
struct Pair;
template <>
struct Pair<float> {
  v2f v;
  __device__ __forceinline__ void load(const float* p, bool two) {
    using P = At<v2f, float>;
    if (two)
      v = MIAIE_LD(reinterpret_cast<const P*>(p)).v;
    else
      v = v2f{MIAIE_LD(p), 0.f};
  }
  // exponents of the larger of a row's two magnitudes, two rows
  __device__ __forceinline__ static uint32_t exponents(const Pair& a, const Pair& b) {
    return max(abs_bits(a.v[0]), abs_bits(a.v[1])) >> 23 | max(abs_bits(b.v[0]), abs_bits(b.v[1])) >> 23 << 16;
  }
  template <int BYTE>
  __device__ __forceinline__ uint32_t codes(uint32_t q, float scale) const {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, BYTE);
  }
  __device__ __forceinline__ static void pack(const Pair (&x)[32], uint32_t (&s)[2], uint32_t (&q)[2][4]) {
    uint32_t a0 = 0, a1 = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) a0 = max(a0, abs_bits(x[i].v[0])), a1 = max(a1, abs_bits(x[i].v[1]));
    s[0] = scale_of(a0), s[1] = scale_of(a1);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      float c0[8], c1[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c0[i] = x[8 * d + i].v[0], c1[i] = x[8 * d + i].v[1];
      q[0][d] = pack8(c0, scale_f32(s[0]));
      q[1][d] = pack8(c1, scale_f32(s[1]));
    }
  }
};
template <>
struct Pair<__bf16> {
  uint32_t v;
  __device__ __forceinline__ void load(const __bf16* p, bool two) {
    using P = At<uint32_t, __bf16>;
    if (two)
      v = MIAIE_LD(reinterpret_cast<const P*>(p)).v;
    else
      v = MIAIE_LD(reinterpret_cast<const uint16_t*>(p));
  }
  // (magnitudes are compared as 16-bit integers, two in one instruction)
  __device__ __forceinline__ static uint32_t exponents(const Pair& a, const Pair& b) {
    const v2us c0 = __builtin_bit_cast(v2us, __builtin_amdgcn_perm(b.v, a.v, 0x05040100u) & 0x7fff7fffu);
    const v2us c1 = __builtin_bit_cast(v2us, __builtin_amdgcn_perm(b.v, a.v, 0x07060302u) & 0x7fff7fffu);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(c0, c1) >> 7);
  }
  template <int BYTE>
  __device__ __forceinline__ uint32_t codes(uint32_t q, float scale) const {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(v2bf, v), scale, BYTE);
  }
  __device__ __forceinline__ static void pack(const Pair (&x)[32], uint32_t (&s)[2], uint32_t (&q)[2][4]) {
    v2us a = {0, 0};
#pragma unroll
    for (int i = 0; i < 32; ++i) a = __builtin_elementwise_max(a, __builtin_bit_cast(v2us, x[i].v & 0x7fff7fffu));
    s[0] = scale_of((uint32_t)a[0] << 16), s[1] = scale_of((uint32_t)a[1] << 16);
    const float f0 = scale_f32(s[0]), f1 = scale_f32(s[1]);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t q0 = 0, q1 = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = x[8 * d + 2 * k].v, hi = x[8 * d + 2 * k + 1].v;
        const v2bf c0 = __builtin_bit_cast(v2bf, __builtin_amdgcn_perm(hi, lo, 0x05040100u));
        const v2bf c1 = __builtin_bit_cast(v2bf, __builtin_amdgcn_perm(hi, lo, 0x07060302u));
        switch (k) {  // (the byte is part of the instruction)
          case 0: q0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q0, c0, f0, 0), q1 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q1, c1, f1, 0); break;
          case 1: q0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q0, c0, f0, 1), q1 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q1, c1, f1, 1); break;
          case 2: q0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q0, c0, f0, 2), q1 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q1, c1, f1, 2); break;
          default: q0 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q0, c0, f0, 3), q1 = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q1, c1, f1, 3); break;
        }
      }
      q[0][d] = q0, q[1][d] = q1;
    }
  }
};

// A workgroup of four waves packs 256 rows of 64 columns along the rows' axis:
// each lane has two columns of a block of 32 rows, the other lanes of its half
// wave the columns beside them, so every load of a half wave is one row's 128
// (bf16) or 256 bytes, all 32 are in flight, and no lane needs another's values.
// The packed rows (128 bytes of 64 columns) leave through LDS in whole lines.  A
// workgroup loads, packs and stores once; 256 rows rather than 512 or 128 leave
// the fewest idle (4096 x 4096 bf16: 13.2 us, 14.0, 13.7; 1023 x 2049 fp32 along
// both axes 6.9, 8.4, 7.6).
//
// ROWS: along the columns' axis too, from the same registers.  A block of 32
// columns is the 16 lanes of a half wave's half, whose maxima come from four lane
// permutations, for two rows at a time (only the exponents are needed); the codes
// leave through LDS, 32 bytes of a row.  (2048 x 4096 bf16: 10.7 us, 14 in two
// launches that each read x.)
constexpr int RB = 8;  // blocks of 32 rows
__host__ __device__ inline int row_tiles(int R) { return s_groups(R) * (16 / RB); }

template <class T, bool ROWS>
__global__ __launch_bounds__(32 * RB) void quant_cols(const T* __restrict__ X, uint8_t* __restrict__ Qt,
                                                      uint8_t* __restrict__ St, uint8_t* __restrict__ Q,
                                                      uint8_t* __restrict__ S, int R, int C, int ldx, int tiles_c) {
  constexpr int P = 16 * RB + 16, PR = 36;  // bytes of a packed column, and of 64 columns of a packed row, in LDS
  __shared__ __attribute__((aligned(16))) uint8_t lq[64 * P], ls[64 * RB];
  __shared__ __attribute__((aligned(16))) uint8_t rq[ROWS ? 32 * RB * PR : 16], rs[ROWS ? 2 * 32 * RB : 16];
  const int tid = threadIdx.x, pair = tid & 31, rb = tid >> 5;  // column pair, block of rows
  int tile = blockIdx.x;
  if constexpr (ROWS) {
    // The eight tiles of 512 columns, which write parts of the same lines, on one XCD
    // (workgroups go round the eight).
    tile = (tile & ~63) + 8 * (tile & 7) + (tile >> 3 & 7);
    if (tile >= row_tiles(R) * tiles_c) return;
  }
  const int first = 32 * RB * (tile / tiles_c), c0 = 64 * (tile % tiles_c), c = c0 + 2 * pair;
  const int g = first / 512, b0 = first % 512 / 32, r0 = first + 32 * rb;
  Pair<T> x[32];
  const T* p = X + (size_t)r0 * ldx + c;
  if (first + 32 * RB <= R && c0 + 64 <= C) {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i].load(p + (size_t)i * ldx, true);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      x[i] = Pair<T>{};
      if (r0 + i < R && c < C) x[i].load(p + (size_t)i * ldx, c + 1 < C);
    }
  }
  uint32_t s[2], q[2][4];
  Pair<T>::pack(x, s, q);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    *reinterpret_cast<uint4*>(lq + (2 * pair + k) * P + 16 * rb) = make_uint4(q[k][0], q[k][1], q[k][2], q[k][3]);
    ls[(2 * pair + k) * RB + 2 * (rb & 3) + (rb >> 2)] = (uint8_t)s[k];  // (as in s_byte)
  }
  if constexpr (ROWS) {
    uint32_t scales[8];  // of the block's 32 rows, a byte each
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      uint32_t pairs[2], codes = 0;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v2us e = __builtin_bit_cast(v2us, Pair<T>::exponents(x[4 * d + 2 * k], x[4 * d + 2 * k + 1]));
        auto widen = [&](auto ctrl) {
          e = __builtin_elementwise_max(e, __builtin_bit_cast(v2us, quad_swap<decltype(ctrl)::value>(__builtin_bit_cast(uint32_t, e))));
        };
        widen(std::integral_constant<int, 0xB1>{});   // 1 0 3 2 of a four
        widen(std::integral_constant<int, 0x4E>{});   // 2 3 0 1
        widen(std::integral_constant<int, 0x141>{});  // the other four of eight
        widen(std::integral_constant<int, 0x140>{});  // the other eight of sixteen
        // scale_of: e - 2 from 2 on, 255 for 255
        const v2us two = {2, 2}, top = {254, 254};
        const v2us nan = __builtin_elementwise_max(e, top) - top;
        pairs[k] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(e, two) - two + nan + nan);
      }
      codes = x[4 * d].template codes<0>(codes, scale_f32(pairs[0] & 255));
      codes = x[4 * d + 1].template codes<1>(codes, scale_f32(pairs[0] >> 16));
      codes = x[4 * d + 2].template codes<2>(codes, scale_f32(pairs[1] & 255));
      codes = x[4 * d + 3].template codes<3>(codes, scale_f32(pairs[1] >> 16));
#pragma unroll
      for (int k = 0; k < 4; ++k) rq[(32 * rb + 4 * d + k) * PR + pair] = (uint8_t)(codes >> (8 * k));
      scales[d] = __builtin_amdgcn_perm(pairs[1], pairs[0], 0x06040200u);
    }
    if ((pair & 15) == 0) {
      uint4* to = reinterpret_cast<uint4*>(rs + 32 * RB * (pair >> 4) + 32 * rb);
      to[0] = make_uint4(scales[0], scales[1], scales[2], scales[3]);
      to[1] = make_uint4(scales[4], scales[5], scales[6], scales[7]);
    }
  }
  __syncthreads();
  const size_t pitch = q_pitch(R);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int col = 32 * k + tid / RB, ch = tid % RB;
    const size_t off = first / 2 + 16 * ch;
    if (c0 + col < C && off < pitch)
      MIAIE_ST(reinterpret_cast<uint4*>(Qt + (size_t)(c0 + col) * pitch + off), *reinterpret_cast<const uint4*>(lq + col * P + 16 * ch));
  }
  const int col = c0 + tid / 4;  // two blocks' scales of a column a thread
  if (col < C)
    MIAIE_ST(reinterpret_cast<uint16_t*>(St + ((size_t)g * C + col) * 16 + 4 * (tid & 3) + b0 / 4),
             *reinterpret_cast<const uint16_t*>(ls + 2 * tid));
  if constexpr (ROWS) {
    const int row = first + tid;
    if (row < R) {
      const size_t row_pitch = q_pitch(C);
      const uint32_t* from = reinterpret_cast<const uint32_t*>(rq + tid * PR);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if ((size_t)c0 / 2 + 16 * k < row_pitch)
          MIAIE_ST(reinterpret_cast<uint4*>(Q + row * row_pitch + c0 / 2 + 16 * k),
                   make_uint4(from[4 * k], from[4 * k + 1], from[4 * k + 2], from[4 * k + 3]));
        const int block = c0 / 32 + k;
        MIAIE_ST(S + ((size_t)(block >> 4) * R + row) * 16 + s_byte(block), rs[32 * RB * k + tid]);
      }
    }
  }
}

// One wave unpacks 512 columns of a row (8192 x 8192 to bf16: 25.6 us).
template <class T>
__global__ __launch_bounds__(256) void dequant(const uint8_t* __restrict__ Q, const uint8_t* __restrict__ S,
                                               T* __restrict__ Y, int R, int C, int ldy, int units, int stride) {
  const int lane = threadIdx.x & 63;
  const int groups = s_groups(C);
  for (int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); unit < units; unit += stride) {
    const int row = unit / groups, g = unit % groups;
    const int c0 = 512 * g + 8 * lane;
    if (c0 >= C) continue;
    const uint32_t q = MIAIE_LD(reinterpret_cast<const uint32_t*>(Q + row * q_pitch(C) + c0 / 2));
    const float scale = scale_f32(MIAIE_LD(S + ((size_t)g * R + row) * 16 + s_byte(lane >> 2)));
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1),
              c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
    const float x[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    store8(Y + (size_t)row * ldy + c0, C - c0, x);
  }
}

// Workgroups of four waves for one piece a wave (more than a launch takes: several turns a wave).
int wave_grid(int units) { return std::min((units - 1) / 4 + 1, 1 << 22); }

}  // namespace

int launch_quant_mxfp4(miaie_ctx* ctx, const void* X, int dtype, int R, int C, int ldx, uint8_t* Q, uint8_t* S,
                       uint8_t* Qt, uint8_t* St) {
  hipError_t e = hipSuccess;
  auto go = [&](auto t) {
    using T = typename decltype(t)::type;
    const T* x = static_cast<const T*>(X);
    if (Q && Qt) {  // (the rows' form has zeros up to the end of its last 512 columns)
      const int tiles_c = 8 * s_groups(C);
      e = launch<quant_cols<T, true>>(ctx->device, dim3(((unsigned)row_tiles(R) * tiles_c + 63) / 64 * 64), dim3(32 * RB), 0,
                                      ctx->stream, x, Qt, St, Q, S, R, C, ldx, tiles_c);
    } else if (Q) {
      const int units = R * s_groups(C), grid = wave_grid(units);
      e = launch<quant_rows<T>>(ctx->device, dim3(grid), dim3(256), 0, ctx->stream, x, Q, S, R, C, ldx, units, 4 * grid);
    } else {
      const int tiles_c = (C + 63) / 64;
      e = launch<quant_cols<T, false>>(ctx->device, dim3((unsigned)row_tiles(R) * tiles_c), dim3(32 * RB), 0, ctx->stream, x,
                                       Qt, St, nullptr, nullptr, R, C, ldx, tiles_c);
    }
  };
  if (dtype == MIAIE_BF16)
    go(type_t<__bf16>{});
  else
    go(type_t<float>{});
  return check_launch(ctx, e, "quant_mxfp4");
}

int launch_dequant_mxfp4(miaie_ctx* ctx, const uint8_t* Q, const uint8_t* S, void* Y, int dtype, int R, int C,
                         int ldy) {
  const int units = R * s_groups(C), grid = wave_grid(units);
  const hipError_t e =
      dtype == MIAIE_BF16
          ? launch<dequant<__bf16>>(ctx->device, dim3(grid), dim3(256), 0, ctx->stream, Q, S, static_cast<__bf16*>(Y), R, C,
                                    ldy, units, 4 * grid)
          : launch<dequant<float>>(ctx->device, dim3(grid), dim3(256), 0, ctx->stream, Q, S, static_cast<float*>(Y), R, C,
                                   ldy, units, 4 * grid);
  return check_launch(ctx, e, "dequant_mxfp4");
}

}  // namespace miaie
