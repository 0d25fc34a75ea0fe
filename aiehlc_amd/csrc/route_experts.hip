// Routing of tokens to experts and its gradient, the order of the routed tokens'
// slots, and the weighted sum over a token's slots with its gradient.
#include <algorithm>

#include "fp8.hpp"

namespace miaie {
namespace {

using namespace fp8;

// ---- reductions over a wave, the result in every lane
template <class V>
__device__ __forceinline__ V from_dpp(V v, int step) {
  uint32_t w[sizeof(V) / 4];
  __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
  for (uint32_t& x : w) {
    switch (step) {
      case 0: x = mx::quad_swap<0xB1>(x); break;   // lanes 1 0 3 2
      case 1: x = mx::quad_swap<0x4E>(x); break;   // lanes 2 3 0 1
      case 2: x = mx::quad_swap<0x141>(x); break;  // the other four of eight
      default: x = mx::quad_swap<0x140>(x); break; // the other eight of sixteen
    }
  }
  V r;
  __builtin_memcpy(&r, w, sizeof(V));
  return r;
}
template <class V, class Op>
__device__ __forceinline__ V over_wave(V v, Op op) {
#pragma unroll
  for (int step = 0; step < 4; ++step) v = op(v, from_dpp(v, step));
  // the other sixteen, then the other half: swapping a copy leaves one value in each
#pragma unroll
  for (int step = 0; step < 2; ++step) {
    uint32_t a[sizeof(V) / 4], b[sizeof(V) / 4];
    __builtin_memcpy(a, &v, sizeof(V));
    __builtin_memcpy(b, &v, sizeof(V));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
      if (step == 0)
        swap16(a[i], b[i]);
      else
        swap32(a[i], b[i]);
    }
    V x, y;
    __builtin_memcpy(&x, a, sizeof(V));
    __builtin_memcpy(&y, b, sizeof(V));
    v = op(x, y);
  }
  return v;
}
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ double operator()(double a, double b) const { return fmax(a, b); }
};
struct Add {
  __device__ float operator()(float a, float b) const { return a + b; }
  __device__ double operator()(double a, double b) const { return a + b; }
};

constexpr float kNone = -INFINITY;

// v of a lane that is the same for the whole wave
template <class V>
__device__ __forceinline__ V at_lane(V v, int lane) {
  uint32_t w[sizeof(V) / 4];
  __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
  for (uint32_t& x : w) x = (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
  V r;
  __builtin_memcpy(&r, w, sizeof(V));
  return r;
}

// What the wave's lanes have written to LDS before, each of them reads behind.  (A wave's
// LDS instructions stay in order; the compiler is kept from moving or splitting them.)
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <class T>
__device__ __forceinline__ float load1(const T* p) {
  return (float)MIAIE_LD(p);
}

// A score in 64 bits: two experts' may be next to each other, and the choice
// between them must not depend on how an exponential is rounded.
template <bool SIGMOID>
__device__ __forceinline__ double score_of(float l, float largest, double total) {
  if (SIGMOID) return 1.0 / (1.0 + exp(-(double)l));
  return exp((double)l - (double)largest) / total;
}

struct RouteArgs {
  const float* bias;
  int* idx;
  float* w;
  int T, E, k, ld, groups, kept, group_top, renormalize;
  float scale;
};

// A wave a token, expert lane + 64 p in a lane's p-th place: the experts that equal
// the largest are found by a ballot a place, the lowest index first.  BY_SCORE: the
// choice is score + bias in 64 bits, or groups are compared by sums of two; without
// either the order of the logits is that of the scores, and only the chosen
// experts' exponentials are needed.
template <class T, int PER, bool SIGMOID, bool BY_SCORE>
__global__ __launch_bounds__(256) void route_tokens(const T* __restrict__ logits, RouteArgs a) {
  using V = std::conditional_t<BY_SCORE, double, float>;
  __shared__ double lds[BY_SCORE ? 4 * 64 * PER : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x * 4 + wave;
  if (t >= a.T) return;  // (no barriers: a wave's LDS is its own)
  const T* row = logits + (size_t)t * a.ld;
  float l[PER], largest = kNone;
  bool nan = false;
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int e = lane + 64 * p;
    l[p] = e < a.E ? load1(row + e) : kNone;
  }
  float bias[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) bias[p] = BY_SCORE && a.bias && lane + 64 * p < a.E ? MIAIE_LD(a.bias + lane + 64 * p) : 0.f;
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    nan |= l[p] != l[p];
    largest = fmaxf(largest, l[p]);
  }
  largest = over_wave(largest, Max{});
  V c[PER], of[PER];  // what is compared, and what the weight comes from: the score, or the logit
  double total = 1.0;
  // (without renormalisation a softmax weight needs the sum too)
  if (!SIGMOID && (BY_SCORE || !a.renormalize)) {
    double sum = 0.0;
#pragma unroll
    for (int p = 0; p < PER; ++p) sum += l[p] > kNone ? exp((double)l[p] - (double)largest) : 0.0;
    total = over_wave(sum, Add{});
  }
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    if constexpr (BY_SCORE) {
      of[p] = score_of<SIGMOID>(l[p], largest, total);
      c[p] = of[p] + (double)bias[p];
      const bool allowed = l[p] > kNone;  // (not NaN)
      if (allowed && c[p] != c[p]) nan = true;
      if (!allowed || c[p] != c[p]) c[p] = -(double)INFINITY;
    } else {
      of[p] = c[p] = l[p] == l[p] ? l[p] : kNone;
    }
  }
  // such a token's weights are all NaN (a sum over its slots is, too)
  nan = __ballot(nan) != 0 || (!SIGMOID && largest == INFINITY);
  if constexpr (BY_SCORE) {
    if (a.groups > 1) {
      double* mine = lds + wave * 64 * PER;
      const int size = a.E / a.groups;
#pragma unroll
      for (int p = 0; p < PER; ++p) mine[lane + 64 * p] = c[p];
      wave_lds_order();
      // `shared` lanes a group, the largest power of two that leaves lanes for all of
      // them; each takes every shared-th member, and their best two are merged
      int shared = 64;
      while (shared * a.groups > 64) shared >>= 1;
      const int g = lane / shared;
      double of = -(double)INFINITY, second = -(double)INFINITY;
      if (g < a.groups)
        for (int m = lane % shared; m < size; m += shared) {
          const double v = mine[g * size + m];
          second = fmax(second, fmin(of, v));
          of = fmax(of, v);
        }
      for (int d = 1; d < shared; d *= 2) {
        const double v = __shfl_xor(of, d), w = __shfl_xor(second, d);
        second = fmax(fmin(of, v), fmax(second, w));
        of = fmax(of, v);
      }
      if (a.group_top > 1 && second != -(double)INFINITY) of += second;
      int better = 0;
      for (int x = 0; x < a.groups; ++x) {
        const double v = at_lane(of, x * shared);
        better += v > of || (v == of && x < g);
      }
      const unsigned long long keep = __ballot(g < a.groups && better < a.kept);
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const int e = lane + 64 * p;
        if (e < a.E && !(keep >> (e / size * shared) & 1)) c[p] = -(double)INFINITY;
      }
    }
  }
  int chosen = -1;  // of lane j: the j-th expert
  V from = 0;
  for (int j = 0; j < a.k; ++j) {
    V best = c[0];
#pragma unroll
    for (int p = 1; p < PER; ++p) best = Max{}(best, c[p]);
    best = over_wave(best, Max{});
    if (best == (V)-INFINITY) break;
    int e = -1;
    V v = 0;
#pragma unroll
    for (int p = PER - 1; p >= 0; --p) {
      const unsigned long long has = __ballot(c[p] == best);
      if (has) {
        const int l = __builtin_ctzll(has);
        e = 64 * p + l;
        v = at_lane(of[p], l);
      }
    }
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (e == lane + 64 * p) c[p] = (V)-INFINITY;
    if (lane == j) chosen = e, from = v;
  }
  double s = 0.0;
  if (chosen >= 0) s = BY_SCORE ? (double)from : score_of<SIGMOID>((float)from, largest, total);
  if (a.renormalize) s /= over_wave(s, Add{}) + 1e-20;
  if (lane < a.k) {
    MIAIE_ST(a.idx + (size_t)t * a.k + lane, chosen);
    MIAIE_ST(a.w + (size_t)t * a.k + lane, nan ? NAN : (float)(a.scale * s));
  }
}

struct RouteGradArgs {
  const int* idx;
  const float* dw;
  float* dlogits;
  int T, E, k, ld, ldd, renormalize;
  float scale;
};

// A wave a token.  With p the scores, w_j = scale p_j / P, P = sum of the chosen p
// + 1e-20 (without renormalisation P = 1):
//   dp_j = scale (dw_j - sum_i dw_i p_i / P) / P,
//   sigmoid: dl_e = dp_e p_e (1 - p_e); softmax: dl_e = p_e (dp_e - sum_j dp_j p_j),
// dp_e the sum over the choices of e.  The k choices are computed in 64 bits (their
// differences cancel), the E experts in 32.
template <class T, int PER, bool SIGMOID>
__global__ __launch_bounds__(256) void route_tokens_grad(const T* __restrict__ logits, RouteGradArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x * 4 + wave;
  if (t >= a.T) return;
  const T* row = logits + (size_t)t * a.ld;
  float l[PER], p[PER], largest = kNone;
#pragma unroll
  for (int i = 0; i < PER; ++i) l[i] = lane + 64 * i < a.E ? load1(row + lane + 64 * i) : kNone;
  int e = -1;
  float dw = 0.f, le = kNone;
  if (lane < a.k) {
    e = MIAIE_LD(a.idx + (size_t)t * a.k + lane);
    if (e >= a.E) e = -1;
    if (e >= 0) {
      dw = MIAIE_LD(a.dw + (size_t)t * a.k + lane);
      le = load1(row + e);
    }
  }
  double total = 1.0;
  if (SIGMOID) {
#pragma unroll
    for (int i = 0; i < PER; ++i) p[i] = 1.f / (1.f + expf(-l[i]));
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) largest = fmaxf(largest, l[i]);
    largest = over_wave(largest, Max{});
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      p[i] = l[i] == kNone ? 0.f : expf(l[i] - largest);
      sum += p[i];
    }
    total = over_wave((double)sum, Add{});
#pragma unroll
    for (int i = 0; i < PER; ++i) p[i] = l[i] == kNone ? 0.f : p[i] / (float)total;
  }
  const double pe = e >= 0 && le != kNone ? score_of<SIGMOID>(le, largest, total) : 0.0;
  double dp = a.scale * (double)dw;
  if (a.renormalize) {
    const double sum = over_wave(pe, Add{}) + 1e-20, dot = over_wave(dw * pe, Add{});
    dp = a.scale * (dw - dot / sum) / sum;
  }
  if (e < 0) dp = 0.0;
  const float inner = SIGMOID ? 0.f : (float)over_wave(dp * pe, Add{});
  float d[PER] = {};
  for (int j = 0; j < a.k; ++j) {
    const int ej = __shfl(e, j);
    const float dj = __shfl((float)dp, j);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (ej == lane + 64 * i) d[i] += dj;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (lane + 64 * i >= a.E) continue;
    float dl;
    if (SIGMOID) {  // p (1 - p) = x / (1 + x)^2, x = e^-|l|
      const float x = expf(-fabsf(l[i]));
      dl = d[i] * (x / ((1.f + x) * (1.f + x)));
    } else {
      dl = p[i] * (d[i] - inner);
    }
    MIAIE_ST(a.dlogits + (size_t)t * a.ldd + lane + 64 * i, dl);
  }
}

// ---------------------------------------------------------------- the slots' order
// A stable counting sort.  Every workgroup counts all pairs by expert, those before
// its own run and those behind it, and so knows where each expert's slots begin and
// where its own pairs go without waiting for another; then each of its waves places
// its part of the run in turn, 64 pairs at a time, a pair behind those of the same
// expert in lower lanes.  (16384 pairs of 64 experts by one workgroup: 17.4 us, most
// of it the placing; by 16 of them 6.4.)  Up to some 10^5 pairs the launch is most of the
// time; beyond, that every workgroup counts all: 131072 pairs of 64 experts 21 us, 2^23 of
// them 1.2 ms, and 115 us and 7.1 ms where all have one expert, whose count the 64 lanes
// of a wave raise one by one.
constexpr int kOrderWaves = 16, kOrderThreads = 64 * kOrderWaves, kOrderGroups = 64;
__global__ __launch_bounds__(kOrderThreads) void order_slots(const int* __restrict__ idx, int* __restrict__ start,
                                                             int* __restrict__ count, int* __restrict__ slot_of,
                                                             int* __restrict__ row_of, int* __restrict__ expert_of, int pairs,
                                                             int experts, int rows, int bits, int run) {
  extern __shared__ int at[];  // [waves + 2][experts]: a wave's count of an expert, then its next slot; pairs before and behind
  __shared__ int wave_sum[kOrderWaves];
  __shared__ int2 ends[MIAIE_MAX_EXPERTS];  // an expert's last slot in use and in all
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int begin = blockIdx.x * run, end = min(pairs, begin + run);
  const int first = begin + wave * (run / kOrderWaves), last = min(end, first + run / kOrderWaves);
  int* const before = at + kOrderWaves * experts;
  for (int i = tid; i < (kOrderWaves + 2) * experts; i += kOrderThreads) at[i] = 0;
  __syncthreads();
  constexpr int PANEL = 8;  // loads in flight together
  int e[PANEL];
  auto load = [&](int i0, int step, int to) {
#pragma unroll
    for (int u = 0; u < PANEL; ++u) {
      const int i = i0 + step * u;
      e[u] = i < to ? MIAIE_LD(idx + i) : -1;
    }
#pragma unroll
    for (int u = 0; u < PANEL; ++u)
      if (e[u] >= experts) e[u] = -1;
  };
  for (int i0 = tid; i0 < pairs; i0 += kOrderThreads * PANEL) {
    load(i0, kOrderThreads, pairs);
#pragma unroll
    for (int u = 0; u < PANEL; ++u) {
      const int i = i0 + kOrderThreads * u;
      if (e[u] < 0) continue;
      if (i < begin)
        atomicAdd(before + e[u], 1);
      else if (i >= end)
        atomicAdd(before + experts + e[u], 1);
      else
        atomicAdd(at + (i - begin) / (run / kOrderWaves) * experts + e[u], 1);
    }
  }
  __syncthreads();
  // thread e: the expert's pairs, and its place among the experts
  int n = 0, of_wave[kOrderWaves] = {};
  if (tid < experts) {
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) of_wave[w] = at[w * experts + tid];
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) n += of_wave[w];
    n += before[tid] + before[experts + tid];
  }
  const int padded = (n + 127) / 128 * 128;
  int upto = padded;
  for (int d = 1; d < 64; d *= 2) {
    const int v = __shfl_up(upto, d);
    if (lane >= d) upto += v;
  }
  if (lane == 63) wave_sum[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) upto += wave_sum[w];
  if (tid < experts) {
    const int slot = upto - padded;
    if (blockIdx.x == 0) {
      MIAIE_ST(start + tid, slot);
      MIAIE_ST(count + tid, n);
      if (tid == experts - 1) MIAIE_ST(start + experts, upto);
    }
    ends[tid] = make_int2(slot + n, upto);
    int next = slot + before[tid];
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) {
      at[w * experts + tid] = next;
      next += of_wave[w];
    }
  }
  __syncthreads();
  // padding and the blocks' experts, shared out over all waves
  const int waves = gridDim.x * kOrderWaves;
  for (int x = blockIdx.x * kOrderWaves + wave; x < experts; x += waves) {
    const int2 to = ends[x];
    const int from = x ? ends[x - 1].y : 0;
    for (int r = to.x + lane; r < to.y; r += 64) MIAIE_ST(row_of + r, -1);
    for (int b = from / 128 + lane; b < to.y / 128; b += 64) MIAIE_ST(expert_of + b, x);
  }
  for (int b = ends[experts - 1].y / 128 + blockIdx.x * kOrderThreads + tid; b < rows / 128; b += gridDim.x * kOrderThreads)
    MIAIE_ST(expert_of + b, -1);
  for (int i0 = first; i0 < last; i0 += 64 * PANEL) {
    load(i0 + lane, 64, last);
#pragma unroll
    for (int u = 0; u < PANEL; ++u) {
      if (i0 + 64 * u >= last) break;
      const int i = i0 + 64 * u + lane;
      unsigned long long same = __ballot(e[u] >= 0);
      for (int b = 0; b < bits; ++b) {
        const unsigned long long has = __ballot(e[u] >> b & 1);
        same &= (e[u] >> b & 1) ? has : ~has;
      }
      int slot = -1;
      const int ahead = __popcll(same & ((1ull << lane) - 1)), base = e[u] >= 0 ? at[wave * experts + e[u]] : 0;
      wave_lds_order();  // every lane has read its expert's place, which the first of them moves on
      if (e[u] >= 0) {
        slot = base + ahead;
        MIAIE_ST(row_of + slot, i);
        if (ahead == 0) at[wave * experts + e[u]] = base + __popcll(same);
      }
      wave_lds_order();
      if (i < last) MIAIE_ST(slot_of + i, slot);
    }
  }
}

// out[t] = sum over the choices j, in their order, of w[t][j] Y[slot]: eight columns
// a thread.  Sums are fp32; with Y in bf16 each term has been rounded once before, which
// the caller chooses.
template <class TY, class T>
__global__ __launch_bounds__(256) void combine(const TY* __restrict__ Y, const float* __restrict__ w, T* __restrict__ out,
                                               Slots s, int C, int ldy, int ldo, int per_row, long units, long stride) {
  for (long u = blockIdx.x * 256l + threadIdx.x; u < units; u += stride) {
    const int t = (int)(u / per_row), c = 8 * (int)(u % per_row);
    float sum[8] = {};
    for (int j0 = 0; j0 < s.top_k; j0 += 4) {
      float y[4][8] = {}, f[4] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j0 + j >= s.top_k) continue;
        const size_t pair = (size_t)t * s.top_k + j0 + j;
        const int slot = MIAIE_LD(s.slot_of + pair);
        f[j] = w ? MIAIE_LD(w + pair) : 1.f;  // (NaN without a slot too)
        if (slot >= 0) mx::load8(Y + (size_t)slot * ldy + c, C - c, y[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = __builtin_fmaf(f[j], y[j][i], sum[i]);
    }
    mx::store8(out + (size_t)t * ldo + c, C - c, sum);
  }
}

// dw[t][j] = <dout[t], Y[slot]>, a wave a pair; 0 without an expert.
template <class TY, class T>
__global__ __launch_bounds__(256) void combine_grad(const TY* __restrict__ Y, const T* __restrict__ dout,
                                                    float* __restrict__ dw, Slots s, int C, int ldy, int ldo, int pairs) {
  const int lane = threadIdx.x & 63;
  const int pair = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (pair >= pairs) return;
  const int slot = MIAIE_LD(s.slot_of + pair);
  float sum = 0.f;
  if (slot >= 0)
    for (int c = 8 * lane; c < C; c += 512) {
      float y[8], d[8];
      mx::load8(Y + (size_t)slot * ldy + c, C - c, y);
      mx::load8(dout + (size_t)(pair / s.top_k) * ldo + c, C - c, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(y[i], d[i], sum);
    }
  sum = over_wave(sum, Add{});
  if (lane == 0) MIAIE_ST(dw + pair, sum);
}

// f(type of Y, type of the result or its gradient): the same, or fp32 and bf16
template <class F>
int with_slot_types(int y_dtype, int dtype, F&& f) {
  if (dtype != MIAIE_BF16) return f(type_t<float>{}, type_t<float>{});
  return y_dtype == MIAIE_BF16 ? f(type_t<__bf16>{}, type_t<__bf16>{}) : f(type_t<float>{}, type_t<__bf16>{});
}

// f(type of the logits, number of a lane's places)
template <class F>
int with_experts(int dtype, int E, F&& f) {
  auto go = [&](auto t) {
    if (E <= 64) return f(t, std::integral_constant<int, 1>{});
    if (E <= 128) return f(t, std::integral_constant<int, 2>{});
    if (E <= 256) return f(t, std::integral_constant<int, 4>{});
    if (E <= 512) return f(t, std::integral_constant<int, 8>{});
    return f(t, std::integral_constant<int, 16>{});
  };
  return dtype == MIAIE_BF16 ? go(type_t<__bf16>{}) : go(type_t<float>{});
}

}  // namespace

int launch_route_experts(miaie_ctx* ctx, const void* logits, int dtype, const float* bias, int* idx, float* w, int tokens,
                         int experts, int top_k, int ld, int scoring, int groups, int groups_kept, int group_top,
                         int renormalize, float scale) {
  const RouteArgs a{bias, idx, w, tokens, experts, top_k, ld, groups, groups_kept, group_top, renormalize, scale};
  return with_experts(dtype, experts, [&](auto t, auto per) {
    using T = typename decltype(t)::type;
    constexpr int PER = decltype(per)::value;
    hipError_t e = hipSuccess;
    auto go = [&](auto k) {
      e = launch<decltype(k)::value>(ctx->device, dim3((tokens + 3u) / 4), dim3(256), 0, ctx->stream,
                                     static_cast<const T*>(logits), a);
    };
    const bool by_score = bias || groups > 1;
    if (scoring == MIAIE_SIGMOID) {
      if (by_score)
        go(kernel_t<route_tokens<T, PER, true, true>>{});
      else
        go(kernel_t<route_tokens<T, PER, true, false>>{});
    } else {
      if (by_score)
        go(kernel_t<route_tokens<T, PER, false, true>>{});
      else
        go(kernel_t<route_tokens<T, PER, false, false>>{});
    }
    return check_launch(ctx, e, "route_tokens");
  });
}

int launch_route_experts_grad(miaie_ctx* ctx, const void* logits, int dtype, const int* idx, const float* dw, float* dlogits,
                              int tokens, int experts, int top_k, int ld, int ldd, int scoring, int renormalize,
                              float scale) {
  const RouteGradArgs a{idx, dw, dlogits, tokens, experts, top_k, ld, ldd, renormalize, scale};
  return with_experts(dtype, experts, [&](auto t, auto per) {
    using T = typename decltype(t)::type;
    constexpr int PER = decltype(per)::value;
    const dim3 grid((tokens + 3u) / 4);
    const T* l = static_cast<const T*>(logits);
    const hipError_t e = scoring == MIAIE_SIGMOID
                             ? launch<route_tokens_grad<T, PER, true>>(ctx->device, grid, dim3(256), 0, ctx->stream, l, a)
                             : launch<route_tokens_grad<T, PER, false>>(ctx->device, grid, dim3(256), 0, ctx->stream, l, a);
    return check_launch(ctx, e, "route_tokens_grad");
  });
}

int launch_experts_order(miaie_ctx* ctx, const fp8::Slots& s, const int* idx) {
  int bits = 0;
  while (1 << bits < s.experts) ++bits;
  const int pairs = s.tokens * s.top_k;
  // a run a workgroup: whole 64s a wave
  const int groups = std::min(kOrderGroups, (pairs + kOrderThreads - 1) / kOrderThreads);
  const int run = ((pairs + groups - 1) / groups + kOrderThreads - 1) / kOrderThreads * kOrderThreads;
  const hipError_t e = launch<order_slots>(ctx->device, dim3((pairs + run - 1) / run), dim3(kOrderThreads),
                                           sizeof(int) * (kOrderWaves + 2) * s.experts, ctx->stream, idx,
                                           const_cast<int*>(s.start), const_cast<int*>(s.count), const_cast<int*>(s.slot_of),
                                           const_cast<int*>(s.row_of), const_cast<int*>(s.expert_of), pairs, s.experts, s.rows,
                                           bits, run);
  return check_launch(ctx, e, "order_slots");
}

int launch_experts_combine(miaie_ctx* ctx, const fp8::Slots& s, const void* Y, int y_dtype, const float* w, void* out,
                           int dtype, int C, int ldy, int ldo) {
  const int per_row = (C + 7) / 8;
  const long units = (long)s.tokens * per_row, grid = std::min((units + 255) / 256, 1l << 22);
  return with_slot_types(y_dtype, dtype, [&](auto ty, auto t) {
    using TY = typename decltype(ty)::type;
    using T = typename decltype(t)::type;
    return check_launch(ctx,
                        launch<combine<TY, T>>(ctx->device, dim3((unsigned)grid), dim3(256), 0, ctx->stream,
                                               static_cast<const TY*>(Y), w, static_cast<T*>(out), s, C, ldy, ldo, per_row,
                                               units, 256 * grid),
                        "experts_combine");
  });
}

int launch_experts_combine_grad(miaie_ctx* ctx, const fp8::Slots& s, const void* Y, int y_dtype, const void* dout, float* dw,
                                int dtype, int C, int ldy, int ldo) {
  const int pairs = s.tokens * s.top_k;
  return with_slot_types(y_dtype, dtype, [&](auto ty, auto t) {
    using TY = typename decltype(ty)::type;
    using T = typename decltype(t)::type;
    return check_launch(ctx,
                        launch<combine_grad<TY, T>>(ctx->device, dim3((pairs + 3u) / 4), dim3(256), 0, ctx->stream,
                                                    static_cast<const TY*>(Y), static_cast<const T*>(dout), dw, s, C, ldy,
                                                    ldo, pairs),
                        "experts_combine_grad");
  });
}

}  // namespace miaie
