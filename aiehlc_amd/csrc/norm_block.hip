// The norms around a block of a residual network, fused with its gate and the
// residual's scale, and their gradients:
//
//   r = alpha x + gate * w_after * b / rms(b)      (after the block b = f(y))
//   y = w_before * r / rms(r)                      (before the next block)
//   rms(v) = sqrt(mean(v^2) + eps) over a row
//
// One read of x and b, one write of r and y.  Everything between is fp32; r is
// rounded to its stored type first and the second norm reads the rounded
// values, as a separate call would.  1 / rms of both norms is kept for the
// gradient, in which, with n = b / rms(b), m = r / rms(r):
//
//   t  = dy * w_before           dr = dout + (t - m mean(t m)) / rms(r)
//   dx = alpha dr                u  = dr * gate * w_after
//   db = (u - n mean(u n)) / rms(b)
//   dw_before = sum dy * m       dw_after = sum dr * gate * n       over rows
//   dgate = sum dr * w_after * n                        over a gate's rows
//
// The sums over rows are taken in a fixed order: each workgroup sums its rows
// in registers and writes one partial row; a second launch adds those.
#include <algorithm>

#include "mxfp4.hpp"

namespace miaie {
namespace {

using mx::load8;
using mx::store8;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

// Sum over a row of THREADS threads: a wave, or the workgroup (red: one float
// per wave; every thread of the workgroup calls it the same number of times).
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* red, int tid) {
  v = wave_sum(v);
  if constexpr (THREADS > 64) {
    __syncthreads();  // the last sum has been read
    if ((tid & 63) == 0) red[tid >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v += red[w];
  }
  return v;
}

template <class T>
__device__ __forceinline__ float rounded(float v) {
  return (float)(T)v;
}

struct Fwd {
  const void *x, *b, *gate;
  const float *w_after, *w_before;
  void *out, *y;
  float* rstd;
  int rows, cols, ldx, ldb, gate_rows;
  int stride;  // rows that all workgroups together take at a time
  float alpha, eps;
};

// TPR threads hold a row, 8 NC columns each; a workgroup of max(TPR, 256)
// threads has one row (TPR >= 256) or four (TPR = 64).  ST: x and out, BT: b,
// gate and y.
template <class ST, class BT, int TPR, int NC>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_fwd(Fwd p) {
  constexpr int RPW = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  const int tid = threadIdx.x, t = tid % TPR;
  // (the threads that share a barrier have the same row)
  for (int row = blockIdx.x * RPW + tid / TPR; row < p.rows; row += p.stride) {
    const ST* x = static_cast<const ST*>(p.x) + (size_t)row * p.ldx;
    float r[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[c][e] = 0.f;
      if (k < p.cols) load8(x + k, p.cols - k, r[c]);
    }
    if (p.b) {
      const BT* b = static_cast<const BT*>(p.b) + (size_t)row * p.ldb;
      float v[NC][8], ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
        if (k < p.cols) load8(b + k, p.cols - k, v[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[c][e], v[c][e], ss);
      }
      const float ra = 1.f / sqrtf(row_sum<TPR>(ss, red, tid) / (float)p.cols + p.eps);
      if (p.rstd && t == 0) MIAIE_ST(p.rstd + row, ra);
      const BT* gate = p.gate ? static_cast<const BT*>(p.gate) + (size_t)(row / p.gate_rows) * p.cols : nullptr;
      ST* out = static_cast<ST*>(p.out) + (size_t)row * p.ldx;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c);
        if (k < p.cols) {
          float w[8], g[8];
          load8(p.w_after + k, p.cols - k, w);
          if (gate) load8(gate + k, p.cols - k, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float n = v[c][e] * ra * w[e];
            if (gate) n *= g[e];
            r[c][e] = rounded<ST>(fmaf(p.alpha, r[c][e], n));
          }
          store8(out + k, p.cols - k, r[c]);
        }
      }
    }
    if (p.y) {
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * (t + TPR * c) + e < p.cols) ss = fmaf(r[c][e], r[c][e], ss);
      const float rb = 1.f / sqrtf(row_sum<TPR>(ss, red, tid) / (float)p.cols + p.eps);
      if (p.rstd && t == 0) MIAIE_ST(p.rstd + p.rows + row, rb);
      BT* y = static_cast<BT*>(p.y) + (size_t)row * p.ldb;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c);
        if (k < p.cols) {
          float w[8];
          load8(p.w_before + k, p.cols - k, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] *= r[c][e] * rb;
          store8(y + k, p.cols - k, w);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ gradient
struct Bwd {
  const void *r, *b, *gate;
  const float *w_after, *w_before, *rstd;
  const void *dout, *dy;
  void *dx, *db;
  float* dgate;           // written here where a gate's rows are one workgroup's (parts == 0)
  float* work;            // [workgroups][3][cols]: partial sums of dw_before, dw_after, dgate
  int rows, cols, ldx, ldb, gate_rows;
  int groups;             // gate rows in all: ceil(rows / gate_rows)
  int workgroups;
  int parts;              // workgroups that share a gate's rows; 0: each row lane takes whole gates
  int want;               // bit 0: dw_before, bit 1: dw_after, bit 2: dgate
  float alpha;
};

// parts > 0: workgroup i has the rows of part i % parts of gate i / parts.
// parts == 0: the row lanes of all workgroups take gates in turn.
template <class ST, class BT, int TPR, int NC>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_bwd(Bwd p) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPW = THREADS / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  __shared__ float lanes[RPW > 1 ? (RPW - 1) * TPR * 8 : 1];
  const int tid = threadIdx.x, t = tid % TPR, lane_row = tid / TPR;
  const size_t cols = p.cols;
  float dwb[NC][8] = {}, dwa[NC][8] = {}, dg[NC][8] = {};

  auto row_grad = [&](int row) {
    const float ra = p.b ? MIAIE_LD(p.rstd + row) : 0.f, rb = p.dy ? MIAIE_LD(p.rstd + p.rows + row) : 0.f;
    float dr[NC][8], m[NC][8], tt[NC][8], c1 = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) dr[c][e] = m[c][e] = tt[c][e] = 0.f;
      if (k >= p.cols) continue;
      if (p.dout) load8(static_cast<const ST*>(p.dout) + (size_t)row * p.ldx + k, p.cols - k, dr[c]);
      if (p.dy) {
        float w[8], d[8];
        load8(static_cast<const ST*>(p.r) + (size_t)row * p.ldx + k, p.cols - k, m[c]);
        load8(static_cast<const BT*>(p.dy) + (size_t)row * p.ldb + k, p.cols - k, d);
        load8(p.w_before + k, p.cols - k, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m[c][e] *= rb;
          tt[c][e] = e < p.cols - k ? d[e] * w[e] : 0.f;
          if (e < p.cols - k) dwb[c][e] = fmaf(d[e], m[c][e], dwb[c][e]);
          c1 = fmaf(tt[c][e], m[c][e], c1);
        }
      }
    }
    if (p.dy) {
      c1 = row_sum<TPR>(c1, red, tid) / (float)p.cols;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) dr[c][e] = fmaf(rb, tt[c][e] - m[c][e] * c1, dr[c][e]);
    }
    if (p.dx) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c);
        float d[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = p.alpha * dr[c][e];
        if (k < p.cols) store8(static_cast<ST*>(p.dx) + (size_t)row * p.ldx + k, p.cols - k, d);
      }
    }
    if (!p.b) return;
    float c2 = 0.f;
    const BT* gate = p.gate ? static_cast<const BT*>(p.gate) + (size_t)(row / p.gate_rows) * cols : nullptr;
    // (m becomes n, dr becomes u)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) m[c][e] = 0.f;
      if (k >= p.cols) continue;
      float w[8], g[8];
      load8(static_cast<const BT*>(p.b) + (size_t)row * p.ldb + k, p.cols - k, m[c]);
      load8(p.w_after + k, p.cols - k, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = 1.f;
      if (gate) load8(gate + k, p.cols - k, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[c][e] *= ra;
        const float dn = dr[c][e] * m[c][e];
        if (e < p.cols - k) {
          dwa[c][e] = fmaf(dn, g[e], dwa[c][e]);
          dg[c][e] = fmaf(dn, w[e], dg[c][e]);
        }
        dr[c][e] = e < p.cols - k ? dr[c][e] * g[e] * w[e] : 0.f;
        c2 = fmaf(dr[c][e], m[c][e], c2);
      }
    }
    if (!p.db) return;
    c2 = row_sum<TPR>(c2, red, tid) / (float)p.cols;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = ra * (dr[c][e] - m[c][e] * c2);
      if (k < p.cols) store8(static_cast<BT*>(p.db) + (size_t)row * p.ldb + k, p.cols - k, d);
    }
  };

  if (p.parts > 0) {
    const int gate = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const int first = gate * p.gate_rows, n = min(p.gate_rows, p.rows - first);
    const int r0 = first + (int)((long)n * part / p.parts), r1 = first + (int)((long)n * (part + 1) / p.parts);
    for (int row = r0 + lane_row; row < r1; row += RPW) row_grad(row);
  } else {
    for (int gate = blockIdx.x * RPW + lane_row; gate < p.groups; gate += p.workgroups * RPW) {
      const int first = gate * p.gate_rows, last = min(first + p.gate_rows, p.rows);
      for (int row = first; row < last; ++row) row_grad(row);
      if (p.want & 4) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int k = 8 * (t + TPR * c);
          if (k < p.cols) store8(p.dgate + gate * cols + k, p.cols - k, dg[c]);
#pragma unroll
          for (int e = 0; e < 8; ++e) dg[c][e] = 0.f;
        }
      }
    }
  }

  // the workgroup's partial sums
  auto put = [&](float(&v)[NC][8], int which) {
    float* dst = p.work + ((size_t)blockIdx.x * 3 + which) * cols;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
      if constexpr (RPW > 1) {
        __syncthreads();
        if (lane_row > 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) lanes[((lane_row - 1) * 8 + e) * TPR + t] = v[c][e];
        }
        __syncthreads();
        if (lane_row == 0) {
#pragma unroll
          for (int l = 0; l < RPW - 1; ++l)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] += lanes[(l * 8 + e) * TPR + t];
        }
      }
      if (lane_row == 0 && k < p.cols) store8(dst + k, p.cols - k, v[c]);
    }
  };
  if (p.want & 1) put(dwb, 0);
  if (p.want & 2) put(dwa, 1);
  if ((p.want & 4) && p.parts > 0) put(dg, 2);
}

// Sums of partial rows: workgroup (x, y) adds 64 columns of output row y (0:
// dw_before, 1: dw_after, 2 + g: dgate row g), its four waves a quarter of the
// partial rows each.
__global__ __launch_bounds__(256) void norm_join(const float* __restrict__ work, float* __restrict__ dw_before,
                                                 float* __restrict__ dw_after, float* __restrict__ dgate, int cols,
                                                 int workgroups, int parts) {
  __shared__ float sum[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.x * 64 + lane;
  const int out = blockIdx.y;
  float* dst = out == 0 ? dw_before : out == 1 ? dw_after : dgate;
  if (!dst) return;
  const int first = out < 2 ? 0 : (out - 2) * parts, n = out < 2 ? workgroups : parts;
  const int which = min(out, 2);
  float s = 0.f;
  if (k < cols)
    for (int i = wave; i < n; i += 4) s += MIAIE_LD(work + ((size_t)(first + i) * 3 + which) * cols + k);
  sum[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && k < cols) {
    s = sum[0][lane] + sum[1][lane] + sum[2][lane] + sum[3][lane];
    MIAIE_ST(dst + (out < 2 ? 0 : (size_t)(out - 2) * cols) + k, s);
  }
}

// go(threads per row, 8-column chunks per thread) for rows of `cols` columns
template <class F>
void with_row(int cols, F&& go) {
  if (cols <= 512)
    go(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  else if (cols <= 1024)
    go(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  else if (cols <= 2048)
    go(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
  else if (cols <= 4096)
    go(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  else if (cols <= 8192)
    go(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
  else
    go(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
}

template <class F>
void with_types(int stream_dtype, int branch_dtype, F&& go) {
  if (stream_dtype == MIAIE_F32) {
    if (branch_dtype == MIAIE_F32)
      go(type_t<float>{}, type_t<float>{});
    else
      go(type_t<float>{}, type_t<__bf16>{});
  } else {
    if (branch_dtype == MIAIE_F32)
      go(type_t<__bf16>{}, type_t<float>{});
    else
      go(type_t<__bf16>{}, type_t<__bf16>{});
  }
}

}  // namespace

int launch_norm_block(miaie_ctx* ctx, const void* x, const void* b, const void* gate, const float* w_after,
                      const float* w_before, void* out, void* y, float* rstd, int rows, int cols, int ldx, int ldb,
                      int gate_rows, int stream_dtype, int branch_dtype, float alpha, float eps) {
  Fwd p{x, b, gate, w_after, w_before, out, y, rstd, rows, cols, ldx, ldb, gate_rows, 0, alpha, eps};
  hipError_t e = hipSuccess;
  with_types(stream_dtype, branch_dtype, [&](auto st, auto bt) {
    with_row(cols, [&](auto tpr, auto nc) {
      constexpr int TPR = decltype(tpr)::value, NC = decltype(nc)::value, RPW = TPR < 256 ? 256 / TPR : 1;
      const int workgroups = std::min((rows + RPW - 1) / RPW, 1 << 20);
      p.stride = workgroups * RPW;
      e = launch<norm_fwd<typename decltype(st)::type, typename decltype(bt)::type, TPR, NC>>(
          ctx->device, dim3(workgroups), dim3(TPR < 256 ? 256 : TPR), 0, ctx->stream, p);
    });
  });
  return check_launch(ctx, e, "norm_fwd");
}

int launch_norm_block_grad(miaie_ctx* ctx, const void* r, const void* b, const void* gate, const float* w_after,
                           const float* w_before, const float* rstd, const void* dout, const void* dy, void* dx,
                           void* db, float* dgate, float* dw_after, float* dw_before, float* work, int rows, int cols,
                           int ldx, int ldb, int gate_rows, int stream_dtype, int branch_dtype, float alpha) {
  Bwd p{r,    b,    gate, w_after, w_before,  rstd, dout, dy, dx, db, dgate, work, rows, cols, ldx, ldb, gate_rows,
        0,    0,    0,    0,       alpha};
  p.groups = (int)(((long)rows + gate_rows - 1) / gate_rows);
  p.want = (dw_before ? 1 : 0) | (dw_after ? 2 : 0) | (dgate ? 4 : 0);
  hipError_t e = hipSuccess;
  with_types(stream_dtype, branch_dtype, [&](auto st, auto bt) {
    with_row(cols, [&](auto tpr, auto nc) {
      constexpr int TPR = decltype(tpr)::value, NC = decltype(nc)::value, RPW = TPR < 256 ? 256 / TPR : 1;
      // at most 256 workgroups (the work buffer holds 341 partial rows of
      // three sums), each with at least one row for every row lane
      constexpr int kMost = 256;
      if (p.groups <= kMost / 2) {
        p.parts = (int)std::min<long>(kMost / p.groups, ((long)gate_rows + RPW - 1) / RPW);
        p.workgroups = p.groups * p.parts;
      } else {
        p.parts = 0;
        p.workgroups = (int)std::min<long>(kMost, ((long)p.groups + RPW - 1) / RPW);
      }
      e = launch<norm_bwd<typename decltype(st)::type, typename decltype(bt)::type, TPR, NC>>(
          ctx->device, dim3(p.workgroups), dim3(TPR < 256 ? 256 : TPR), 0, ctx->stream, p);
    });
  });
  if (e == hipSuccess && (dw_before || dw_after || (dgate && p.parts > 0)))
    e = launch<norm_join>(ctx->device, dim3((cols + 63) / 64, dgate && p.parts > 0 ? 2 + p.groups : 2), dim3(256), 0,
                          ctx->stream, work, dw_before, dw_after, dgate, cols, p.workgroups, p.parts);
  return check_launch(ctx, e, "norm_bwd");
}

}  // namespace miaie
