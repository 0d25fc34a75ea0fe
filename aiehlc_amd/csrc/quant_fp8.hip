// Conversion to 8-bit floating point with a scale for each block of 128
// (fp8.hpp): of a matrix, of rows gathered into slots, and of what SwiGLU and
// its gradient make of the slots' projections; along rows, along columns (the
// packed transpose) or both; and back.
//
// A product contracts along the packed axis, so a linear layer's gradients take
// dY along both axes and X along its columns; the transpose of weights packed in
// blocks of 128 x 128 has the same codes and scales.
#include <algorithm>
#include <type_traits>

#include "fp8.hpp"

namespace miaie {
namespace {

using namespace fp8;

// ---- where a tile's values come from: eight columns c .. c + 7 of a row.  A source
// says in turn what a row is (row), loads its columns (fetch) and makes their values
// (values); a thread does each for its rows before the next, so that all loads
// are in flight together.  (A load and its use in one branch a row wait for each
// other: 2048 x 4096 bf16 10.3 us.)  fetch takes rows that do not exist, or are
// padding, from where there is one, and values makes them zero.
template <class T, bool WHOLE>
struct Eight {  // all eight columns exist, of any thread of the workgroup
  typedef T V __attribute__((ext_vector_type(8)));
  V v;
  __device__ __forceinline__ void load(const T* p, int = 8, int = 8) {
    using P = At<V, T>;
    v = MIAIE_LD(reinterpret_cast<const P*>(p)).v;
  }
  __device__ __forceinline__ void place() {}
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};

// n columns from p on exist of a row of C.  Where that is fewer than eight, the row's
// last eight are loaded, one vector like the others', and shifted to their places (eight
// loads and conditions of their own: 333 x 1000 bf16 6.4 us for 3.8, most of the difference
// the way of so many instructions into the cache).
template <class T>
struct Eight<T, false> {
  typedef T V __attribute__((ext_vector_type(8)));
  typedef uint32_t W __attribute__((ext_vector_type(2 * sizeof(T))));
  V v;
  int shift;
  __device__ __forceinline__ void load(const T* p, int n, int C) {
    if (C >= 8) {
      using P = At<V, T>;
      v = MIAIE_LD(reinterpret_cast<const P*>(p + min(0, n - 8))).v;
      shift = 8 - n;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? MIAIE_LD(p + i) : (T)0.f;
      shift = 0;
    }
  }
  // (what is behind the last column is anything)
  __device__ __forceinline__ void place() {
    if (shift <= 0) return;
    constexpr int K = 2 * sizeof(T);  // words
    W w = __builtin_bit_cast(W, v);
#pragma unroll
    for (int by = 4; by > 0; by /= 2) {
      const int words = by * K / 8;
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const uint32_t from = words ? w[min(i + words, K - 1)] : __builtin_amdgcn_alignbit(w[min(i + 1, K - 1)], w[i], 16);
        w[i] = shift & by ? from : w[i];
      }
    }
    v = __builtin_bit_cast(V, w);
  }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};

template <class T>
struct FromMatrix {
  const T* X;
  int R, C, ldx;
  static constexpr bool TAILS = true;  // tiles whose last columns do not exist
  using Row = int;
  template <bool WHOLE>
  using Raw = Eight<T, WHOLE>;
  __device__ __forceinline__ bool tile(int) const { return true; }
  __device__ __forceinline__ Row row(int r) const { return r; }
  template <bool WHOLE>
  __device__ __forceinline__ Raw<WHOLE> fetch(Row r, int c) const {
    Raw<WHOLE> raw;
    raw.load(X + (size_t)min(r, R - 1) * ldx + c, C - c, C);
    return raw;
  }
  template <bool WHOLE>
  __device__ __forceinline__ void values(Row r, int c, Raw<WHOLE> raw, float (&x)[8]) const {
    raw.place();
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r < R && (WHOLE || c + i < C) ? raw[i] : 0.f;
  }
};

// A slot's token, times its weight where there are weights; padding is zero.
template <class T>
struct FromTokens {
  const T* X;
  const float* w;
  Slots s;
  int R, C, ldx;
  static constexpr bool TAILS = true;
  using Row = int;  // pair
  template <bool WHOLE>
  struct Raw {
    Eight<T, WHOLE> x;
    float f;
  };
  __device__ __forceinline__ bool tile(int r0) const { return r0 < MIAIE_LD(s.start + s.experts); }
  __device__ __forceinline__ Row row(int r) const { return MIAIE_LD(s.row_of + r); }
  template <bool WHOLE>
  __device__ __forceinline__ Raw<WHOLE> fetch(Row pair, int c) const {
    Raw<WHOLE> raw;
    raw.x.load(X + (size_t)(max(pair, 0) / s.top_k) * ldx + c, C - c, C);
    raw.f = w ? MIAIE_LD(w + max(pair, 0)) : 1.f;
    return raw;
  }
  template <bool WHOLE>
  __device__ __forceinline__ void values(Row pair, int c, Raw<WHOLE> raw, float (&x)[8]) const {
    raw.x.place();
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = pair >= 0 && (WHOLE || c + i < C) ? raw.x[i] * raw.f : 0.f;  // (no -0 or NaN behind the last column)
  }
};

// silu(gate) up of a slot's projections, gate in columns [0, F), up in [F, 2 F).
template <class T>
struct FromSwiglu {
  const T* GU;
  Slots s;
  int R, C, ldx;  // C = F
  static constexpr bool TAILS = false;
  struct Row {
    int r, pair;
  };
  template <bool WHOLE>
  struct Raw {
    Eight<T, WHOLE> g, u;
  };
  __device__ __forceinline__ bool tile(int r0) const { return r0 < MIAIE_LD(s.start + s.experts); }
  __device__ __forceinline__ Row row(int r) const { return Row{r, MIAIE_LD(s.row_of + r)}; }
  template <bool WHOLE>
  __device__ __forceinline__ Raw<WHOLE> fetch(Row r, int c) const {
    static_assert(WHOLE, "F is a multiple of 128");
    Raw<WHOLE> raw;
    raw.g.load(GU + (size_t)r.r * ldx + c);
    raw.u.load(GU + (size_t)r.r * ldx + C + c);
    return raw;
  }
  template <bool WHOLE>
  __device__ __forceinline__ void values(Row r, int, const Raw<WHOLE>& raw, float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r.pair >= 0 ? swiglu(raw.g[i], raw.u[i]) : 0.f;
  }
};

// Its gradient: with s = 1 / (1 + e^-g), dg = dh u s (1 + g (1 - s)) in columns
// [0, F) and du = dh g s in [F, 2 F).
template <class T>
struct FromSwigluGrad {
  const T* GU;
  const float* dH;
  Slots s;
  int R, C, ldx, ldh;  // C = 2 F
  static constexpr bool TAILS = false;
  struct Row {
    int r, pair;
  };
  template <bool WHOLE>
  struct Raw {
    Eight<T, WHOLE> g, u;
    Eight<float, WHOLE> d;
  };
  __device__ __forceinline__ bool tile(int r0) const { return r0 < MIAIE_LD(s.start + s.experts); }
  __device__ __forceinline__ Row row(int r) const { return Row{r, MIAIE_LD(s.row_of + r)}; }
  template <bool WHOLE>
  __device__ __forceinline__ Raw<WHOLE> fetch(Row r, int c) const {
    static_assert(WHOLE, "F is a multiple of 128");
    const int F = C / 2, f = c < F ? c : c - F;
    Raw<WHOLE> raw;
    raw.g.load(GU + (size_t)r.r * ldx + f);
    if (c < F) raw.u.load(GU + (size_t)r.r * ldx + F + f);  // (the same for the workgroup)
    raw.d.load(dH + (size_t)r.r * ldh + f);
    return raw;
  }
  template <bool WHOLE>
  __device__ __forceinline__ void values(Row r, int c, const Raw<WHOLE>& raw, float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float g = raw.g[i];
      const Sigmoid y(g);
      const float v = c < C / 2 ? raw.d[i] * raw.u[i] * y.s * (1.f + g * y.rest) : raw.d[i] * g * y.s;
      x[i] = r.pair >= 0 ? v : 0.f;
    }
  }
};

// A workgroup of 512 threads packs 128 rows of 128 columns, whole blocks along
// either axis: thread t has columns 8 (t % 16) .. + 7 of rows 4 (t / 16) .. + 3 (eight
// rows of half as many threads take 137 to 165 registers along both axes, and a CU
// has fewer waves of them).
// A row's block is 16 neighbouring lanes, whose maxima come from four lane
// permutations; a column's are joined through LDS, and the codes of the transpose
// leave through LDS as whole lines.  Columns behind C are zero.
template <class Src, int BLOCK, bool ROWS, bool COLS>
__global__ __launch_bounds__(512) void quant_tile(Src src, uint8_t* __restrict__ Q, float* __restrict__ S,
                                                  uint8_t* __restrict__ Qt, float* __restrict__ St, int tiles_c) {
  __shared__ __attribute__((aligned(16))) uint8_t lq[COLS ? 128 * 128 : 16];
  constexpr int N = 4;  // rows of a thread
  __shared__ uint32_t lmax[8][COLS ? 128 : 1];
  const int tid = threadIdx.x, cl = tid & 15, rg = tid >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tr = blockIdx.x / tiles_c, tc = blockIdx.x % tiles_c;
  const int r0 = 128 * tr + N * rg, c = 128 * tc + 8 * cl;
  if (!src.tile(128 * tr)) return;
  auto over_waves = [&](int k) __attribute__((always_inline)) {
    uint32_t m = lmax[0][k];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = max(m, lmax[w][k]);
    return m;
  };
  float x[N][8];
  {
    typename Src::Row row[N];
#pragma unroll
    for (int p = 0; p < N; ++p) row[p] = src.row(r0 + p);
    auto take = [&](auto whole_c) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole_c)::value;
      typename Src::template Raw<WHOLE> raw[N];
#pragma unroll
      for (int p = 0; p < N; ++p) raw[p] = src.template fetch<WHOLE>(row[p], c);
#pragma unroll
      for (int p = 0; p < N; ++p) src.template values<WHOLE>(row[p], c, raw[p], x[p]);
    };
    if constexpr (Src::TAILS) {
      if (128 * tc + 128 <= src.C)
        take(std::true_type{});
      else
        take(std::false_type{});
    } else {
      take(std::true_type{});
    }
  }
  uint32_t e_row[N], e_all = 0;
  if constexpr (BLOCK == 128) {
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, abs_bits(x[p][i]));
    m = max(m, mx::quad_swap<0xB1>(m));   // lanes 1 0 3 2
    m = max(m, mx::quad_swap<0x4E>(m));   // lanes 2 3 0 1
    m = max(m, mx::quad_swap<0x141>(m));  // the other four of eight
    m = max(m, mx::quad_swap<0x140>(m));  // the other eight of sixteen
    m = max_over_16s(m);
    if ((tid & 63) == 0) lmax[wave][0] = m;
    __syncthreads();
    e_all = scale_of(over_waves(0));
    if (tid == 0) {
      const size_t tiles_r = blocks(src.R);
      if (ROWS) MIAIE_ST(S + tc * tiles_r + tr, scale_f32(e_all));
      if (COLS) MIAIE_ST(St + (size_t)tr * blocks(src.C) + tc, scale_f32(e_all));
    }
  }
  if constexpr (ROWS) {
    const size_t row_pitch = pitch(src.C);
#pragma unroll
    for (int p = 0; p < N; ++p) {
      uint32_t e = e_all;
      if constexpr (BLOCK == 1) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, abs_bits(x[p][i]));
        m = max(m, mx::quad_swap<0xB1>(m));
        m = max(m, mx::quad_swap<0x4E>(m));
        m = max(m, mx::quad_swap<0x141>(m));
        m = max(m, mx::quad_swap<0x140>(m));
        e = scale_of(m);
      }
      const float inv = inverse_f32(e);
      const v2u q = {pack4(x[p][0], x[p][1], x[p][2], x[p][3], inv), pack4(x[p][4], x[p][5], x[p][6], x[p][7], inv)};
      if (r0 + p < src.R) MIAIE_ST(reinterpret_cast<v2u*>(Q + (size_t)(r0 + p) * row_pitch + c), q);
      e_row[p] = e;
    }
    if constexpr (BLOCK == 1) {  // lane cl of a row group writes row cl's scale
      uint32_t e = e_row[0];
#pragma unroll
      for (int p = 1; p < N; ++p) e = cl == p ? e_row[p] : e;
      if (cl < N && r0 + cl < src.R) MIAIE_ST(S + (size_t)tc * src.R + r0 + cl, scale_f32(e));
    }
  }
  if constexpr (COLS) {
    uint32_t e_col[8];
    if constexpr (BLOCK == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int p = 0; p < N; ++p) m = max(m, abs_bits(x[p][i]));
        m = max_over_16s(m);
        if ((tid & 48) == 0) lmax[wave][8 * cl + i] = m;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = 8 * cl + i;
        e_col[i] = scale_of(over_waves(k));
      }
      if (tid < 16) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < src.C) MIAIE_ST(St + (size_t)tr * src.C + c + i, scale_f32(e_col[i]));
      }
    }
    // four rows of a column are four bytes, at their place xor the column's eight: the
    // lanes beside each other write different banks
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float inv = inverse_f32(BLOCK == 128 ? e_all : e_col[i]);
      *reinterpret_cast<uint32_t*>(lq + 128 * (8 * cl + i) + 4 * (rg ^ 4 * (cl & 7))) = pack4(x[0][i], x[1][i], x[2][i], x[3][i], inv);
    }
    __syncthreads();
    const size_t col_pitch = pitch(src.R);
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int k = 64 * it + (tid >> 3), m = tid & 7;
      const v4u q = *reinterpret_cast<const v4u*>(lq + 128 * k + 16 * (m ^ (k >> 3 & 7)));
      if (128 * tc + k < src.C) MIAIE_ST(reinterpret_cast<v4u*>(Qt + (size_t)(128 * tc + k) * col_pitch + 128 * tr + 16 * m), q);
    }
  }
}

// Eight columns a thread.
template <class T>
__global__ __launch_bounds__(256) void dequant(const uint8_t* __restrict__ Q, const float* __restrict__ S,
                                               T* __restrict__ Y, int R, int C, int ldy, int block, long units, long stride) {
  const int per_row = (int)(pitch(C) / 8);
  for (long u = blockIdx.x * 256l + threadIdx.x; u < units; u += stride) {
    const int row = (int)(u / per_row), c = 8 * (int)(u % per_row);
    if (c >= C) continue;
    const v2u q = MIAIE_LD(reinterpret_cast<const v2u*>(Q + (size_t)row * pitch(C) + c));
    const float s = MIAIE_LD(S + (size_t)(c / 128) * (block == 1 ? (size_t)R : blocks(R)) + (block == 1 ? row : row / 128));
    float x[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const mx::v2f a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
      x[4 * h] = a[0] * s, x[4 * h + 1] = a[1] * s, x[4 * h + 2] = b[0] * s, x[4 * h + 3] = b[1] * s;
    }
    mx::store8(Y + (size_t)row * ldy + c, C - c, x);
  }
}

template <int BLOCK, class Src>
int run(miaie_ctx* ctx, const char* what, const Src& src, uint8_t* Q, float* S, uint8_t* Qt, float* St) {
  const int tiles_c = (int)blocks(src.C);
  const dim3 grid((unsigned)(blocks(src.R) * tiles_c));
  hipError_t e = hipSuccess;
  auto go = [&](auto k) {
    e = launch<decltype(k)::value>(ctx->device, grid, dim3(512), 0, ctx->stream, src, Q, S, Qt, St, tiles_c);
  };
  if (Q && Qt)
    go(kernel_t<quant_tile<Src, BLOCK, true, true>>{});
  else if (Q)
    go(kernel_t<quant_tile<Src, BLOCK, true, false>>{});
  else
    go(kernel_t<quant_tile<Src, BLOCK, false, true>>{});
  return check_launch(ctx, e, what);
}

template <class F>
int with_type(int dtype, F&& f) {
  return dtype == MIAIE_BF16 ? f(type_t<__bf16>{}) : f(type_t<float>{});
}

}  // namespace

int launch_quant_fp8(miaie_ctx* ctx, const void* X, int dtype, int R, int C, int ldx, int block, uint8_t* Q, float* S,
                     uint8_t* Qt, float* St) {
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    const FromMatrix<T> src{static_cast<const T*>(X), R, C, ldx};
    return block == 1 ? run<1>(ctx, "quant_fp8", src, Q, S, Qt, St) : run<128>(ctx, "quant_fp8", src, Q, S, Qt, St);
  });
}

int launch_dequant_fp8(miaie_ctx* ctx, const uint8_t* Q, const float* S, int block, void* Y, int dtype, int R, int C,
                       int ldy) {
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    const long units = (long)R * (long)(pitch(C) / 8), grid = std::min((units + 255) / 256, 1l << 22);
    const hipError_t e = launch<dequant<T>>(ctx->device, dim3((unsigned)grid), dim3(256), 0, ctx->stream, Q, S,
                                            static_cast<T*>(Y), R, C, ldy, block, units, 256 * grid);
    return check_launch(ctx, e, "dequant_fp8");
  });
}

int launch_experts_quant_fp8(miaie_ctx* ctx, const fp8::Slots& s, const void* X, int dtype, const float* w, int C,
                             int ldx, uint8_t* Q, float* S, uint8_t* Qt, float* St) {
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    const FromTokens<T> src{static_cast<const T*>(X), w, s, s.rows, C, ldx};
    return run<1>(ctx, "experts_quant_fp8", src, Q, S, Qt, St);
  });
}

int launch_experts_swiglu_fp8(miaie_ctx* ctx, const fp8::Slots& s, const void* GU, int dtype, int F, int ldgu, uint8_t* Q,
                              float* S, uint8_t* Qt, float* St) {
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    const FromSwiglu<T> src{static_cast<const T*>(GU), s, s.rows, F, ldgu};
    return run<1>(ctx, "experts_swiglu_fp8", src, Q, S, Qt, St);
  });
}

int launch_experts_swiglu_grad_fp8(miaie_ctx* ctx, const fp8::Slots& s, const void* GU, int dtype, const float* dH, int F,
                                   int ldgu, int ldh, uint8_t* Q, float* S, uint8_t* Qt, float* St) {
  return with_type(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    const FromSwigluGrad<T> src{static_cast<const T*>(GU), dH, s, s.rows, 2 * F, ldgu, ldh};
    return run<1>(ctx, "experts_swiglu_grad_fp8", src, Q, S, Qt, St);
  });
}

}  // namespace miaie
