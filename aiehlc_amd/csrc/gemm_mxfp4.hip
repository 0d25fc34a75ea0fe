// Products of MXFP4 matrices (mxfp4.hpp): C[m][n] = sum_k A[m][k] B[n][k], both
// packed along k, on v_mfma_scale_f32_16x16x128_f8f6f4.
//
// An instruction multiplies four blocks of 32 k: lane l holds the 16 bytes of
// block l / 16 of row l % 16 of each operand, and their scales.  A block's sum
// is exact (the products are multiples of 1/4 up to 36); the four block sums
// and the accumulator are added in fp32.
//
// Operand roles: srcA is the B fragment and srcB the A fragment, so lane l of
// the result has row m = l % 16 and the four consecutive columns
// n = 4 (l / 16) + 0..3 of its 16 x 16 block: whole vectors of a row of C, and
// for a packed result the eight lanes' values of a block of 32 columns are one
// row's.
#include <type_traits>

#include "gfx950_ops.hpp"
#include "mxfp4.hpp"

namespace miaie {
namespace {

using namespace mx;

// What becomes of a row's four columns.
enum Out { OUT_F32, OUT_BF16, OUT_MX, OUT_MX_RELU };

__device__ __forceinline__ v8i wide(v4i x) { return v8i{x[0], x[1], x[2], x[3], 0, 0, 0, 0}; }

// acc += B fragment x A fragment, scales in byte T of sb and sa
template <int T>
__device__ __forceinline__ v4f mfma(v4i b, v4i a, v4f acc, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(b), wide(a), acc, 4, 4, T, sb, T, sa);
}

struct Args {
  const uint8_t *Aq, *As, *Bq, *Bs;
  void* C;      // OUT_F32, OUT_BF16
  uint8_t* Yq;  // OUT_MX
  uint8_t* Ys;
  int M, N, K, ldc;
};

template <class T>
__device__ __forceinline__ void store4(T* C, size_t ldc, int m, int n, int M, int N, v4f v) {
  if (m >= M || n >= N) return;
  typedef T V __attribute__((ext_vector_type(4)));
  const V r = __builtin_convertvector(v, V);
  T* p = C + (size_t)m * ldc + n;
  if (n + 4 <= N) {
    using P = At<V, T>;
    MIAIE_ST(reinterpret_cast<P*>(p), P{r});
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (n + e < N) MIAIE_ST(p + e, r[e]);
  }
}

// Block nb (columns 32 nb ..) of row m, of which this lane holds columns
// 32 nb + 4 fg + e (lo) and 32 nb + 16 + 4 fg + e (hi); the row's other lanes
// are 16, 32 and 48 away.  Columns from N on become zeros.
template <bool RELU>
__device__ __forceinline__ void store_block(const Args& p, int m, int nb, int fg, v4f lo, v4f hi) {
  float x[8];
  uint32_t amax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int n = 32 * nb + (e >> 2) * 16 + 4 * fg + (e & 3);
    float v = e < 4 ? lo[e & 3] : hi[e & 3];
    if (RELU) v = v < 0.f ? 0.f : v;  // (keeps NaN)
    x[e] = n < p.N ? v : 0.f;
    amax = max(amax, abs_bits(x[e]));
  }
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
  amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
  if (m >= p.M) return;
  const uint32_t s = scale_of(amax);
  const uint32_t q = pack8(x, scale_f32(s));
  const size_t pitch = q_pitch(p.N);
  if (16 * (size_t)nb < pitch) {
    uint8_t* d = p.Yq + m * pitch + 16 * (size_t)nb + 2 * fg;
    MIAIE_ST(reinterpret_cast<uint16_t*>(d), (uint16_t)q);
    MIAIE_ST(reinterpret_cast<uint16_t*>(d + 8), (uint16_t)(q >> 16));
  }
  if (fg == 0) MIAIE_ST(p.Ys + ((size_t)(nb >> 4) * p.M + m) * 16 + s_byte(nb), (uint8_t)s);
}

// ---------------------------------------------------------------- few rows
// A workgroup of W waves owns 16 MI rows and 32 columns; the waves share out
// the 512-column groups of k and add their sums in LDS.  Fragments come
// straight from memory: a wave reads 256 contiguous bytes of 16 rows of each
// operand per group.
template <int MI, int W, Out OUT>
__global__ __launch_bounds__(64 * W) void gemm_mx_rows(Args p, int tiles_n) {
  constexpr int NJ = 2;
  __shared__ v4f part[W > 1 ? W - 1 : 1][MI * NJ][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int m0 = 16 * MI * (blockIdx.x / tiles_n), n0 = 32 * (blockIdx.x % tiles_n);
  const size_t pitch = q_pitch(p.K);
  const int groups = s_groups(p.K), tiles_k = (int)(pitch / 64);  // 128-column steps: an even number
  v4f acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint8_t *aq[MI], *bq[NJ], *as[MI], *bs[NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const size_t m = min(m0 + 16 * i + fr, p.M - 1);
    aq[i] = p.Aq + m * pitch + 16 * fg;
    as[i] = p.As + m * 16 + 4 * fg;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const size_t n = min(n0 + 16 * j + fr, p.N - 1);
    bq[j] = p.Bq + n * pitch + 16 * fg;
    bs[j] = p.Bs + n * 16 + 4 * fg;
  }
  if (n0 < p.N) {
    for (int g = wave; g < groups; g += W) {
      int sa[MI], sb[NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i) sa[i] = MIAIE_LD(reinterpret_cast<const int*>(as[i] + (size_t)g * p.M * 16));
#pragma unroll
      for (int j = 0; j < NJ; ++j) sb[j] = MIAIE_LD(reinterpret_cast<const int*>(bs[j] + (size_t)g * p.N * 16));
      auto step = [&](auto t_c) {
        constexpr int t = decltype(t_c)::value;
        const size_t off = 256 * (size_t)g + 64 * t;
        v4i a[MI], b[NJ];
#pragma unroll
        for (int i = 0; i < MI; ++i) a[i] = MIAIE_LD(reinterpret_cast<const v4i*>(aq[i] + off));
#pragma unroll
        for (int j = 0; j < NJ; ++j) b[j] = MIAIE_LD(reinterpret_cast<const v4i*>(bq[j] + off));
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = mfma<t>(b[j], a[i], acc[i][j], sb[j], sa[i]);
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
      if (4 * g + 2 < tiles_k) {
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
      }
    }
  }
  if constexpr (W > 1) {
    if (wave > 0) {
#pragma unroll
      for (int f = 0; f < MI * NJ; ++f) part[wave - 1][f][lane] = acc[f / NJ][f % NJ];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < W - 1; ++w)
#pragma unroll
      for (int f = 0; f < MI * NJ; ++f) acc[f / NJ][f % NJ] += part[w][f][lane];
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + 16 * i + fr;
    if constexpr (OUT == OUT_F32 || OUT == OUT_BF16) {
      using T = std::conditional_t<OUT == OUT_F32, float, __bf16>;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        store4(static_cast<T*>(p.C), p.ldc, m, n0 + 16 * j + 4 * fg, p.M, p.N, acc[i][j]);
    } else {
      store_block<OUT == OUT_MX_RELU>(p, m, n0 / 32, fg, acc[i][0], acc[i][1]);
    }
  }
}

template <Out OUT>
int run(miaie_ctx* ctx, const Args& p) {
  // (a packed result has zeros up to the end of its last 512 columns)
  const int cols = OUT == OUT_MX || OUT == OUT_MX_RELU ? 512 * s_groups(p.N) : p.N;
  const int tiles_n = (cols + 31) / 32;
  const long tiles_m = (p.M + 31l) / 32;
  if (tiles_m * tiles_n >= 1l << 24) return fail(ctx, MIAIE_EINVAL, "gemm_mxfp4: M=%d N=%d too large", p.M, p.N);
  const hipError_t e = launch<gemm_mx_rows<2, 4, OUT>>(ctx->device, dim3((unsigned)(tiles_m * tiles_n)), dim3(256), 0,
                                                       ctx->stream, p, tiles_n);
  return check_launch(ctx, e, "gemm_mx_rows");
}

}  // namespace

int launch_gemm_mxfp4(miaie_ctx* ctx, const uint8_t* Aq, const uint8_t* As, const uint8_t* Bq, const uint8_t* Bs,
                      void* C, int dtype, int M, int N, int K, int ldc) {
  const Args p{Aq, As, Bq, Bs, C, nullptr, nullptr, M, N, K, ldc};
  return dtype == MIAIE_BF16 ? run<OUT_BF16>(ctx, p) : run<OUT_F32>(ctx, p);
}

int launch_gemm_mxfp4_rq(miaie_ctx* ctx, const uint8_t* Aq, const uint8_t* As, const uint8_t* Bq, const uint8_t* Bs,
                         uint8_t* Yq, uint8_t* Ys, int M, int N, int K, int relu) {
  const Args p{Aq, As, Bq, Bs, nullptr, Yq, Ys, M, N, K, 0};
  return relu ? run<OUT_MX_RELU>(ctx, p) : run<OUT_MX>(ctx, p);
}

}  // namespace miaie
