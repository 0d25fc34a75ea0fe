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
using mx::Raw8;
using mx::store8;

// Sum over a wave, in every lane: within sixteens by lane permutations that are
// part of the addition, then across them.
template <int CTRL>
__device__ __forceinline__ float add_lane(float v) {
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = add_lane<0xB1>(v);   // lane 1 0 3 2 of a four
  v = add_lane<0x4E>(v);   // 2 3 0 1
  v = add_lane<0x141>(v);  // the other four of eight (mirrored)
  v = add_lane<0x140>(v);  // the other eight of sixteen
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r16[0]) + __uint_as_float(r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r32[0]) + __uint_as_float(r32[1]);
}

// Sum over a row of TPR threads, a wave or several (red: one float for each
// wave of the workgroup, all of whose threads call it the same number of times).
// Two sums that take turns each have a red: behind the barrier of the one all
// have read the other's.  A sum by itself waits first until its last is read.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red, int tid, bool alone) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    if (alone) __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = v;
    __syncthreads();
    const float* mine = red + tid / TPR * (TPR / 64);
    v = mine[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) v += mine[w];
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
// threads takes one row (TPR >= 256) or several.  ST: x and out, BT: b, gate and
// y.  Everything a row needs is loaded before its first sum: a single row waits
// for memory once (1 x 4096 bf16 3.6 us, 5.4 with the weights and the gate loaded
// where they are used).  Bound by memory: 8192 x 4096, fp32 stream, bf16 branch in
// 76 us, 5.3 TB/s.
template <class ST, class BT, int TPR, int NC>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_fwd(Fwd p) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPW = THREADS / TPR;
  __shared__ float red[2][THREADS / 64];
  const bool alone = !(p.b && p.y);
  const int tid = threadIdx.x, t = tid % TPR;
  Raw8<float> w_after[NC], w_before[NC];
  // (every thread makes the same number of turns: a row's sum is a barrier)
  for (int row0 = blockIdx.x * RPW; row0 < p.rows; row0 += p.stride) {
    const int row = row0 + tid / TPR;
    const bool active = row < p.rows;
    const size_t xo = (size_t)row * p.ldx, bo = (size_t)row * p.ldb;
    const BT* gate = p.gate && active ? static_cast<const BT*>(p.gate) + (size_t)(row / p.gate_rows) * p.cols : nullptr;
    Raw8<BT> b[NC], g[NC];
    Raw8<ST> x[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c), n = p.cols - k;
      b[c].clear(), x[c].clear(), g[c].clear();
      if (n <= 0 || !active) continue;
      if (p.b) b[c].load(static_cast<const BT*>(p.b) + bo + k, n);
      x[c].load(static_cast<const ST*>(p.x) + xo + k, n);
      if (gate) g[c].load(gate + k, n);
    }
    if (row0 == blockIdx.x * RPW) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c), n = p.cols - k;
        w_after[c].clear(), w_before[c].clear();
        if (n <= 0) continue;
        if (p.b) w_after[c].load(p.w_after + k, n);
        if (p.y) w_before[c].load(p.w_before + k, n);
      }
    }
    float r[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) r[c][e] = x[c][e];
    if (p.b) {
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(b[c][e], b[c][e], ss);
      const float ra = 1.f / sqrtf(row_sum<TPR>(ss, red[0], tid, alone) / (float)p.cols + p.eps);
      if (p.rstd && t == 0 && active) MIAIE_ST(p.rstd + row, ra);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c), n = p.cols - k;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v = b[c][e] * ra * w_after[c][e];
          if (gate) v *= g[c][e];
          r[c][e] = rounded<ST>(fmaf(p.alpha, r[c][e], v));
        }
        if (n > 0 && active) store8(static_cast<ST*>(p.out) + xo + k, n, r[c]);
      }
    }
    if (p.y) {
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(r[c][e], r[c][e], ss);  // (0 behind the last column)
      const float rb = 1.f / sqrtf(row_sum<TPR>(ss, red[1], tid, alone) / (float)p.cols + p.eps);
      if (p.rstd && t == 0 && active) MIAIE_ST(p.rstd + p.rows + row, rb);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c), n = p.cols - k;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = r[c][e] * rb * w_before[c][e];
        if (n > 0 && active) store8(static_cast<BT*>(p.y) + bo + k, n, y);
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
//
// 1024 threads, TPR of them to a row: 1024 / TPR rows at a time, so that a CU has
// 16 waves' loads in flight although the partial sums allow only about one
// workgroup a CU (four waves a CU took more than twice the time).  4095 x 4096
// bf16: 47 us, 4.3 TB/s; its six tensors once at the rate of a large copy are 39.
constexpr int BWD_THREADS = 1024;

template <class ST, class BT, int TPR, int NC>
__global__ __launch_bounds__(BWD_THREADS) void norm_bwd(Bwd p) {
  constexpr int RPW = BWD_THREADS / TPR;
  __shared__ float red[2][BWD_THREADS / 64];
  const bool alone = !(p.dy && p.b && p.db);
  // Rows of two chunks a thread keep the norms' sums in LDS, each thread its own
  // columns', and fetch no row ahead, so that of one row only 14 to 16 registers a
  // thread (56 to 60 bytes) are in scratch memory.  1024 x 16384 bf16: 68 us with
  // every tensor from beyond the caches, of which a copy's rate takes 39, and 57 with
  // those of the call before (143 with the sums and the next row in scratch memory
  // too); fp32 stream 89 and 84 us.  The rest have none, but for two registers of
  // fp32 rows of 513 to 4096 columns.
  constexpr bool WIDE = NC > 1;
  __shared__ float kept[WIDE ? 2 * NC * 8 * TPR : 1];
  __shared__ __attribute__((aligned(16))) float weights[WIDE ? 4 : 2 * 8 * TPR];
  __shared__ __attribute__((aligned(16))) float gates[WIDE ? 4 : 8 * BWD_THREADS];  // (and the partial sums at the end)
  const int tid = threadIdx.x, t = tid % TPR, lane_row = tid / TPR;
  const size_t cols = p.cols;
  float dwb[NC][8] = {}, dwa[NC][8] = {}, dg[NC][8] = {};
  auto in_lds = [&](int which, int c, int e) -> float& { return kept[((which * NC + c) * 8 + e) * TPR + t]; };
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < 2 * NC * 8; ++i) kept[i * TPR + t] = 0.f;
  }

  auto weight8 = [&](int which, int c, float(&w)[8]) {
    const int k = 8 * (t + TPR * c);
    if constexpr (WIDE) {
      load8((which ? p.w_after : p.w_before) + k, p.cols - k, w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = weights[((2 * which + e / 4) * TPR + t) * 4 + e % 4];
    }
  };

  // The next row's tensors, on their way while a row is computed, which itself
  // loads nothing: loads return in order, and one of a row's own would wait for all
  // of the next row's (4095 x 4096 bf16: 47 us, 52 with the gate, the weights and the
  // reciprocal roots loaded where they are used).
  Raw8<ST> x_r[NC], x_dout[NC];
  Raw8<BT> x_dy[NC], x_b[NC];
  float x_ra = 0.f, x_rb = 0.f;
  auto fetch = [&](int row, bool active) {
    if (active) {
      if (p.b) x_ra = MIAIE_LD(p.rstd + row);
      if (p.dy) x_rb = MIAIE_LD(p.rstd + p.rows + row);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
      x_r[c].clear(), x_dout[c].clear(), x_dy[c].clear(), x_b[c].clear();
      if (k >= p.cols || !active) continue;
      const size_t xo = (size_t)row * p.ldx + k, bo = (size_t)row * p.ldb + k;
      if (p.dy) {
        x_r[c].load(static_cast<const ST*>(p.r) + xo, p.cols - k);
        x_dy[c].load(static_cast<const BT*>(p.dy) + bo, p.cols - k);
      }
      if (p.dout) x_dout[c].load(static_cast<const ST*>(p.dout) + xo, p.cols - k);
      if (p.b) x_b[c].load(static_cast<const BT*>(p.b) + bo, p.cols - k);
    }
  };

  // A gate's values, each thread its own columns'.
  auto load_gate = [&](int gate, bool active) {
    Raw8<BT> g;
    g.clear();
    if (!WIDE && p.gate && active && 8 * t < p.cols)
      g.load(static_cast<const BT*>(p.gate) + gate * cols + 8 * t, p.cols - 8 * t);
    return g;
  };
  auto keep_gate = [&](const Raw8<BT>& g) {
    if (WIDE || !p.gate) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) gates[(e / 4 * BWD_THREADS + tid) * 4 + e % 4] = g[e];
  };
  auto gate8 = [&](int gate, int c, float(&g)[8]) {
    const int k = 8 * (t + TPR * c);
    if constexpr (WIDE) {
      load8(static_cast<const BT*>(p.gate) + gate * cols + k, p.cols - k, g);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = gates[(e / 4 * BWD_THREADS + tid) * 4 + e % 4];
    }
  };

  // The norms' weights in LDS, before's and after's: [which][half of 8][thread][4]
  // (zeros behind the last column).
  auto keep_weights = [&] {
    if (WIDE) return;
    for (int i = tid; i < 2 * TPR; i += BWD_THREADS) {
      const int which = i / TPR, col = i % TPR, k = 8 * col;
      const float* w = which ? p.w_after : p.w_before;
      float v[8] = {};
      if (w && k < p.cols) load8(w + k, p.cols - k, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) weights[((2 * which + e / 4) * TPR + col) * 4 + e % 4] = v[e];
    }
    __syncthreads();
  };
  auto arrive = [&] {
#pragma unroll
    for (int c = 0; c < NC; ++c) x_r[c].arrive(), x_dout[c].arrive(), x_dy[c].arrive(), x_b[c].arrive();
    asm volatile("" : "+v"(x_ra), "+v"(x_rb));
  };

  // (a lane without a row takes part in the sums' barriers, and adds nothing to the
  // sums over rows: its 0 times an infinite weight would make them NaN)
  auto row_grad = [&](int row, int gate, bool active, int next, bool next_active) {
    if constexpr (WIDE) fetch(row, active);
    if constexpr (!WIDE) arrive();
    const float ra = active ? x_ra : 0.f, rb = active ? x_rb : 0.f;
    float dr[NC][8], m[NC][8], tt[NC][8], v[NC][8], c1 = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) dr[c][e] = x_dout[c][e], m[c][e] = x_r[c][e], tt[c][e] = x_dy[c][e], v[c][e] = x_b[c][e];
    if constexpr (!WIDE) fetch(next, next_active);
    if (p.dy) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c);
        if (k >= p.cols || !active) continue;
        float w[8];
        weight8(0, c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // (what is behind the last column is zero)
          m[c][e] *= rb;
          float& sum = WIDE ? in_lds(0, c, e) : dwb[c][e];
          sum = fmaf(tt[c][e], m[c][e], sum);
          tt[c][e] *= w[e];
          c1 = fmaf(tt[c][e], m[c][e], c1);
        }
      }
      c1 = row_sum<TPR>(c1, red[0], tid, alone) / (float)p.cols;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) dr[c][e] = fmaf(rb, tt[c][e] - m[c][e] * c1, dr[c][e]);
    }
    if (p.dx && active) {
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
    // (v becomes n, dr becomes u)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
      if (k >= p.cols || !active) continue;
      float w[8], g[8];
      weight8(1, c, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = 1.f;
      if (p.gate) gate8(gate, c, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] *= ra;
        const float dn = dr[c][e] * v[c][e];
        float& sum = WIDE ? in_lds(1, c, e) : dwa[c][e];
        sum = fmaf(dn, g[e], sum);
        dg[c][e] = fmaf(dn, w[e], dg[c][e]);
        dr[c][e] *= g[e] * w[e];
        c2 = fmaf(dr[c][e], v[c][e], c2);
      }
    }
    if (!p.db) return;
    c2 = row_sum<TPR>(c2, red[1], tid, alone) / (float)p.cols;
    // (ahead of the last store, for which the next row need not wait)
    if constexpr (!WIDE) arrive();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = 8 * (t + TPR * c);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = ra * (dr[c][e] - v[c][e] * c2);
      if (k < p.cols && active) store8(static_cast<BT*>(p.db) + (size_t)row * p.ldb + k, p.cols - k, d);
    }
  };

  if (p.parts > 0) {
    const int gate = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const int first = gate * p.gate_rows, n = min(p.gate_rows, p.rows - first);
    const int r0 = first + (int)((long)n * part / p.parts), r1 = first + (int)((long)n * (part + 1) / p.parts);
    if constexpr (!WIDE) fetch(r0 + lane_row, r0 + lane_row < r1);
    const Raw8<BT> g = load_gate(gate, true);
    keep_weights();
    keep_gate(g);
    for (int row = r0 + lane_row, i = r0; i < r1; i += RPW, row += RPW) row_grad(row, gate, row < r1, row + RPW, row + RPW < r1);
  } else {
    // (every row lane makes the same number of turns; a gate's last row fetches the
    // first of the lane's next gate)
    const int step = p.workgroups * RPW;
    auto rows_of = [&](int gate) { return gate < p.groups ? min(p.gate_rows, p.rows - gate * p.gate_rows) : 0; };
    int gate = blockIdx.x * RPW + lane_row, n = rows_of(gate);
    if constexpr (!WIDE) fetch(gate * p.gate_rows, n > 0);
    keep_weights();
    for (int g0 = blockIdx.x * RPW; g0 < p.groups; g0 += step) {
      const int first = gate * p.gate_rows, then = gate < p.groups - step ? gate + step : p.groups, n_then = rows_of(then);
      keep_gate(load_gate(gate, n > 0));
      for (int i = 0; i < p.gate_rows; ++i) {
        const bool last = i == p.gate_rows - 1;
        row_grad(first + i, gate, i < n, last ? then * p.gate_rows : first + i + 1, last ? n_then > 0 : i + 1 < n);
      }
      if (p.want & 4) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int k = 8 * (t + TPR * c);
          if (k < p.cols && n > 0) store8(p.dgate + gate * cols + k, p.cols - k, dg[c]);
#pragma unroll
          for (int e = 0; e < 8; ++e) dg[c][e] = 0.f;
        }
      }
      gate = then, n = n_then;
    }
  }

  // the workgroup's partial sums: its row lanes' added through LDS, a column a thread
  auto put = [&](float(&v)[NC][8], int which) {
    float* dst = p.work + ((size_t)blockIdx.x * 3 + which) * cols;
    if constexpr (RPW == 1) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int k = 8 * (t + TPR * c);
        if (k < p.cols) store8(dst + k, p.cols - k, v[c]);
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) gates[8 * tid + e] = v[0][e];
      __syncthreads();
      for (int k = tid; k < min(p.cols, 8 * TPR); k += BWD_THREADS) {
        float s = gates[k];
#pragma unroll
        for (int r = 1; r < RPW; ++r) s += gates[8 * TPR * r + k];
        MIAIE_ST(dst + k, s);
      }
    }
  };
  if constexpr (WIDE) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) dwb[c][e] = in_lds(0, c, e), dwa[c][e] = in_lds(1, c, e);
  }
  if (p.want & 1) put(dwb, 0);
  if (p.want & 2) put(dwa, 1);
  if ((p.want & 4) && p.parts > 0) put(dg, 2);
}

// Sums of partial rows: workgroup (x, y) adds 64 columns of output row y (0:
// dw_before, 1: dw_after, 2 + g: dgate row g), its 16 waves a sixteenth of the
// partial rows each, eight loads in flight (256 partial rows of 3 x 4096: 4.7 us,
// half of them the launch).
__global__ __launch_bounds__(1024) void norm_join(const float* __restrict__ work, float* __restrict__ dw_before,
                                                  float* __restrict__ dw_after, float* __restrict__ dgate, int cols,
                                                  int workgroups, int parts) {
  __shared__ float sum[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.x * 64 + lane;
  const int out = blockIdx.y;
  float* dst = out == 0 ? dw_before : out == 1 ? dw_after : dgate;
  if (!dst) return;
  const int first = out < 2 ? 0 : (out - 2) * parts, n = out < 2 ? workgroups : parts;
  const int which = min(out, 2);
  float s = 0.f;
  if (k < cols) {
    const float* p = work + ((size_t)first * 3 + which) * cols + k;
    for (int i = wave; i < n; i += 128) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i + 16 * u < n ? MIAIE_LD(p + (size_t)(i + 16 * u) * 3 * cols) : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  }
  sum[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && k < cols) {
#pragma unroll
    for (int w = 1; w < 16; ++w) s += sum[w][lane];
    MIAIE_ST(dst + (out < 2 ? 0 : (size_t)(out - 2) * cols) + k, s);
  }
}

// go(threads per row, 8-column chunks per thread) for rows of `cols` columns
template <class F>
void with_row(int cols, F&& go) {
  using One = std::integral_constant<int, 1>;
  if (cols <= 512)
    go(std::integral_constant<int, 64>{}, One{});
  else if (cols <= 1024)
    go(std::integral_constant<int, 128>{}, One{});
  else if (cols <= 2048)
    go(std::integral_constant<int, 256>{}, One{});
  else if (cols <= 4096)
    go(std::integral_constant<int, 512>{}, One{});
  else if (cols <= 8192)
    go(std::integral_constant<int, 1024>{}, One{});
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
      // (at most 16 workgroups a CU, which load the weights once for all their rows)
      const int turns = (rows + RPW - 1) / RPW, workgroups = (int)std::min<long>(turns, 16l * ctx->cus);
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
      constexpr int TPR = decltype(tpr)::value, NC = decltype(nc)::value, RPW = BWD_THREADS / TPR;
      // At most 256 workgroups (the work buffer holds 341 partial rows of three
      // sums).  Up to 128 gates share them out, each with at least a row of a gate's
      // gate_rows (there or not) for every row lane; of more, every row lane takes
      // whole gates, so that few long gates leave CUs idle: 16512 rows of 512 columns
      // take 20 us in 128 gates and 232 us in 129.
      constexpr int kMost = 256;
      if (p.groups <= kMost / 2) {
        p.parts = (int)std::min<long>(kMost / p.groups, ((long)gate_rows + RPW - 1) / RPW);
        p.workgroups = p.groups * p.parts;
      } else {
        p.parts = 0;
        p.workgroups = (int)std::min<long>(kMost, ((long)p.groups + RPW - 1) / RPW);
      }
      e = launch<norm_bwd<typename decltype(st)::type, typename decltype(bt)::type, TPR, NC>>(
          ctx->device, dim3(p.workgroups), dim3(BWD_THREADS), 0, ctx->stream, p);
    });
  });
  if (e == hipSuccess && (dw_before || dw_after || (dgate && p.parts > 0)))
    e = launch<norm_join>(ctx->device, dim3((cols + 63) / 64, dgate && p.parts > 0 ? 2 + p.groups : 2), dim3(1024), 0,
                          ctx->stream, work, dw_before, dw_after, dgate, cols, p.workgroups, p.parts);
  return check_launch(ctx, e, "norm_bwd");
}

}  // namespace miaie
