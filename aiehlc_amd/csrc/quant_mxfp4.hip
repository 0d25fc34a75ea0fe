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
// lanes a block.
template <class T>
__global__ __launch_bounds__(256) void quant_rows(const T* __restrict__ X, uint8_t* __restrict__ Q,
                                                  uint8_t* __restrict__ S, int R, int C, int ldx, int units,
                                                  int stride) {
  const int lane = threadIdx.x & 63;
  const int groups = s_groups(C);
  for (int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); unit < units; unit += stride) {
    const int row = unit / groups, g = unit % groups;
    const size_t pitch = q_pitch(C);
    const int c0 = 512 * g + 8 * lane;
    float x[8] = {};
    if (c0 < C) load8(X + (size_t)row * ldx + c0, C - c0, x);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, abs_bits(x[i]));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 1));
    amax = max(amax, (uint32_t)__shfl_xor((int)amax, 2));
    const uint32_t s = scale_of(amax);
    const uint32_t q = pack8(x, scale_f32(s));
    if ((size_t)c0 < 2 * pitch) MIAIE_ST(reinterpret_cast<uint32_t*>(Q + row * pitch + c0 / 2), q);
    if ((lane & 3) == 0) MIAIE_ST(S + ((size_t)g * R + row) * 16 + s_byte(lane >> 2), (uint8_t)s);
  }
}

// A workgroup of 8 waves packs 512 rows of 64 columns along the rows' axis:
// each lane has two columns of a block of 32 rows, the other lanes of its half
// wave the columns beside them, so every load of a half wave is one row's 128
// (bf16) or 256 bytes and no lane needs another's values.
template <class T>
__global__ __launch_bounds__(512) void quant_cols(const T* __restrict__ X, uint8_t* __restrict__ Q,
                                                  uint8_t* __restrict__ S, int R, int C, int ldx, int tiles_c) {
  const int tid = threadIdx.x, pair = tid & 31, rb = tid >> 5;  // column pair, block of rows
  const int g = blockIdx.x / tiles_c, c0 = 64 * (blockIdx.x % tiles_c) + 2 * pair;
  const int r0 = 512 * g + 32 * rb;
  const size_t pitch = q_pitch(R);
  float x[2][32];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const T* p = X + (size_t)(r0 + i) * ldx + c0;
    x[0][i] = r0 + i < R && c0 < C ? (float)MIAIE_LD(p) : 0.f;
    x[1][i] = r0 + i < R && c0 + 1 < C ? (float)MIAIE_LD(p + 1) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (c0 + k >= C) break;
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = max(amax, abs_bits(x[k][i]));
    const uint32_t s = scale_of(amax);
    const float scale = scale_f32(s);
    uint32_t q[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const float(&v)[8] = *reinterpret_cast<const float(*)[8]>(&x[k][8 * d]);
      q[d] = pack8(v, scale);
    }
    if ((size_t)r0 < 2 * pitch)
      MIAIE_ST(reinterpret_cast<uint4*>(Q + (size_t)(c0 + k) * pitch + r0 / 2), make_uint4(q[0], q[1], q[2], q[3]));
    MIAIE_ST(S + ((size_t)g * C + c0 + k) * 16 + s_byte(rb), (uint8_t)s);
  }
}

// One wave unpacks 512 columns of a row.
template <class T>
__global__ __launch_bounds__(256) void dequant(const uint8_t* __restrict__ Q, const uint8_t* __restrict__ S,
                                               T* __restrict__ Y, int R, int C, int ldy, int units,
                                               int stride) {
  const int lane = threadIdx.x & 63;
  const int groups = s_groups(C);
  for (int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); unit < units; unit += stride) {
    const int row = unit / groups, g = unit % groups;
    const int c0 = 512 * g + 8 * lane;
    if (c0 >= C) continue;
    const uint32_t q = MIAIE_LD(reinterpret_cast<const uint32_t*>(Q + row * q_pitch(C) + c0 / 2));
    const float scale = scale_f32(MIAIE_LD(S + ((size_t)g * R + row) * 16 + s_byte(lane >> 2)));
    float x[8];
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1),
              c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
    store8(Y + (size_t)row * ldy + c0, C - c0, x);
  }
}

// Workgroups of four waves for one unit a wave (more units than a launch takes: several a wave).
int wave_grid(int units) { return std::min((units - 1) / 4 + 1, 1 << 23); }

}  // namespace

int launch_quant_mxfp4(miaie_ctx* ctx, const void* X, int dtype, int R, int C, int ldx, uint8_t* Q, uint8_t* S,
                       uint8_t* Qt, uint8_t* St) {
  hipError_t e = hipSuccess;
  auto go = [&](auto t) {
    using T = typename decltype(t)::type;
    const T* x = static_cast<const T*>(X);
    if (Q) {
      const int units = R * s_groups(C), grid = wave_grid(units);
      e = launch<quant_rows<T>>(ctx->device, dim3(grid), dim3(256), 0, ctx->stream, x, Q, S, R, C, ldx, units, 4 * grid);
    }
    if (Qt && e == hipSuccess) {
      const int tiles_c = (C + 63) / 64;
      e = launch<quant_cols<T>>(ctx->device, dim3((unsigned)s_groups(R) * tiles_c), dim3(512), 0, ctx->stream, x, Qt,
                                St, R, C, ldx, tiles_c);
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
          ? launch<dequant<__bf16>>(ctx->device, dim3(grid), dim3(256), 0, ctx->stream, Q, S, static_cast<__bf16*>(Y), R, C, ldy, units,
                                    4 * grid)
          : launch<dequant<float>>(ctx->device, dim3(grid), dim3(256), 0, ctx->stream, Q, S, static_cast<float*>(Y), R, C, ldy, units,
                                    4 * grid);
  return check_launch(ctx, e, "dequant_mxfp4");
}

}  // namespace miaie
