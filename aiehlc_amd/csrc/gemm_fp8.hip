// Products of 8-bit floating point matrices with a scale for each block of 128
// (fp8.hpp) on v_mfma_f32_16x16x128_f8f6f4:
//   C[m][n] = sum over blocks b of k: Sa[b][m] Sb[b][n] sum_{k in b} A[m][k] B[n][k]
// dense, over the slots of routed tokens (each expert's rows with its own B), and
// over each expert's slots as k (the gradients of the experts' weights).
//
// An instruction multiplies 128 k, one block: lane l holds 32 of row l % 16 of
// each operand, the 16-byte chunks l / 16 and 4 + l / 16 (any order of k does that
// both operands share).  Scales:
//   B in blocks of 128 x 128 (weights, whose scales may be any fp32): the block's
//     product starts from zero and is added by a multiply-add per value, with one
//     factor Sa Sb for a lane's four values;
//   B with a scale for each row (both operands packed by this library): both
//     scales are powers of two, the instruction applies them and adds to the
//     accumulator itself.  In multiply-adds their eight a fragment (a factor a
//     column) would take as long as the instruction.
//
// Operand roles: srcA is the B fragment and srcB the A fragment, so lane l of the
// result has row m = l % 16 and the four consecutive columns n = 4 (l / 16) + 0..3
// of its 16 x 16 block: vectors of a row of C, and one scale of A a lane.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fp8.hpp"
#include "gfx950_ops.hpp"

namespace miaie {
namespace {

using namespace fp8;

enum Mode { DENSE, SLOTS, WGRAD };
enum Out { OUT_F32, OUT_BF16, OUT_GLU };  // OUT_GLU: silu(gate) up, packed along its rows

struct Args {
  const uint8_t* Aq;
  const float* As;
  const uint8_t* Bq;
  const float* Bs;
  void* C;      // OUT_F32, OUT_BF16
  uint8_t* Hq;  // OUT_GLU
  float* Hs;
  int M, N, K, ldc;  // OUT_GLU: N = F, B has 2 F rows; SLOTS: M = the slots' rows; WGRAD: K = those
  int a_rows;        // rows of A (the stride of its scales)
  int gather;        // SLOTS: A's rows are tokens
  Slots s;
};

__device__ __forceinline__ v4f mfma0(v8i b, v8i a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma_scaled(v8i b, v8i a, v4f acc, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 0, 0, 0, sb, 0, sa);
}
__device__ __forceinline__ v8i join(v4i lo, v4i hi) { return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}; }

// The same two as the large tiles issue them, in the order that the program has them:
// the compiler keeps neither a product's place (it starts every product of a step
// before it adds any, in more registers than there are) nor an accumulator's.  A
// result is there 8 passes and 3 wait states after its instruction's issue, which the
// next one's waits 8 passes for: who reads it issues two others before, or waits
// (tests/test_fp8_asm.py checks the distances in the assembly).
__device__ __forceinline__ void issue_mfma0(v4f& p, v8i b, v8i a) {
#if MIAIE_DEVICE_CHECKS
  p = mfma0(b, a);
#else
  asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, 0" : "=&v"(p) : "v"(b), "v"(a));
#endif
}
__device__ __forceinline__ void issue_mfma_scaled(v4f& acc, v8i b, v8i a, int sb, int sa) {
#if MIAIE_DEVICE_CHECKS
  acc = mfma_scaled(b, a, acc, sb, sa);
#else
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+v"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa));
#endif
}
__device__ __forceinline__ void wait_results() { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory"); }

// 16-byte chunk c of a row's 128 bytes lies at c ^ swz(row): the 16 rows of a
// fragment read cover all banks.
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }

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

// ---------------------------------------------------------------- large tiles
// A workgroup of eight waves owns a BM x BN tile, a wave NI x NJ blocks of 16 x 16.
// A step is 128 k: whole 128-byte lines of BM + BN rows and their scales, copied
// into one of STAGES stages of LDS with no registers in between.  A wave keeps its
// rows' fragments of A through a step and takes those of B column by column.
//
// Waves 0-3 (group 0, one on each SIMD) have the first half of B's columns, waves
// 4-7 the second, half a step behind: while the one group begins a step, with all of
// A's fragments to read, the matrix units have the middle of the other's.  (All eight
// in step: 3200 cycles a step of 256 x 256 for 2062 of matrix instructions, whichever
// number of workgroups runs.)  Two barriers a step:
//   E0(t), group 0 at the end of its step t, group 1 in the middle of its own: all of
//     A and the first half of B of step t + 1 are there, B's first half of step t has
//     been read, and A of step t by both groups, so both take the copies of step
//     t + STAGES;
//   E1(t), group 0 in the middle of step t + 1, group 1 at the end of t: the same of
//     B's second half.
template <int BM_, int BN_, int WAVES_M_, int STAGES_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WAVES_M = WAVES_M_, WAVES_N = 8 / WAVES_M, STAGES = STAGES_;
  static constexpr int WAVES = 8, THREADS = 512;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, NI = WM / 16, NJ = WN / 16;
  static constexpr int A = 0, B = BM * 128, S = B + BN * 128, STAGE = S + 4 * (BM + BN);
  static constexpr int A_CP = BM / 64, B_CP = BN / 128;  // a wave's copies of A, and of half of B
  static constexpr int C0 = A_CP + B_CP + 1, C1 = B_CP + 1;  // ... sent after E0 and E1, one of scales in each
  static constexpr int LDS = STAGES * STAGE;
  static_assert(BM % 64 == 0 && BN % 128 == 0 && WAVES_N % 2 == 0 && BM / 64 + BN / 128 <= 8 && STAGE % 128 == 0, "copies of whole waves");
  static_assert(LDS <= 163840, "LDS of a CU");
  // group 1 has the second half of the columns
  __device__ static __forceinline__ int wm(int wave) { return (wave & 3) % WAVES_M; }
  __device__ static __forceinline__ int wn(int wave) { return (wave >> 2) * (WAVES_N / 2) + (wave & 3) / WAVES_M; }
};

template <int BM_, int BN_, int STAGES_>
struct SmallTile {
  static constexpr int BM = BM_, BN = BN_, WAVES_M = 2, WAVES_N = 2, STAGES = STAGES_;
  static constexpr int WAVES = 4, THREADS = 256;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, NI = WM / 16, NJ = WN / 16;
  static constexpr int A = 0, B = BM * 128, S = B + BN * 128, STAGE = S + 4 * (BM + BN);
  static constexpr int A_CP = BM / 8 / WAVES, B_CP = BN / 8 / WAVES;  // copies of a wave in a step
  static constexpr int S_CP = ((BM + BN) / 64 + WAVES - 1) / WAVES, CP = A_CP + B_CP + S_CP;
  static constexpr int LDS = STAGES * STAGE;
  static_assert(A_CP >= 1 && B_CP >= 1 && BM % 64 == 0 && BN % 64 == 0 && STAGE % 128 == 0, "copies of whole waves");
  __device__ static __forceinline__ int wm(int wave) { return wave / WAVES_N; }
  __device__ static __forceinline__ int wn(int wave) { return wave % WAVES_N; }
};

// Waits for what an event makes visible; `left` steps follow the one it is about
// (t + 1).  Copies that may still be in flight: those sent after it.
template <class G, int EVENT, int LEFT = G::STAGES - 1>
__device__ __forceinline__ void wait_event(int left) {
  constexpr int S = G::STAGES;
  if constexpr (LEFT > 0) {
    if (left < LEFT) return wait_event<G, EVENT, LEFT - 1>(left);
  }
  constexpr int a = LEFT < S - 2 ? LEFT : S - 2, b = LEFT + (EVENT == 0) < S - 1 ? LEFT + (EVENT == 0) : S - 1;
  dev::wait_vmcnt<EVENT == 0 ? a * G::C0 + b * G::C1 : b * G::C0 + a * G::C1>();
}

// Where a tile's operands are: wave-uniform addresses of step 0, a row's offset for
// each of a wave's copies.
struct Operands {
  const uint8_t *a, *b;
  const float *as, *bs;
  size_t as_step, bs_step;  // floats from one step's scales to the next's
  int steps;
  int rows, cols;  // of the tile that exist
};

template <class G, int BBLOCK, bool GLU, class RowA, class RowB, class ScaleB>
__device__ __forceinline__ void multiply(int8_t* lds, const Operands& o, uint32_t a_pitch, uint32_t b_pitch, RowA row_a, RowB row_b,
                                         ScaleB scale_b, const dbg::Span& aq_span, const dbg::Span& as_span,
                                         const dbg::Span& bq_span, const dbg::Span& bs_span, v4f (&acc)[G::NI][G::NJ]) {
  constexpr int NI = G::NI, NJ = G::NJ;
  const uint32_t lds0 = dev::lds_addr(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = G::wm(wave), wn = G::wn(wave), fr = lane & 15, fg = lane >> 4;

  uint32_t a_off[G::A_CP], b_off[2][G::B_CP], s_off[2];
#pragma unroll
  for (int x = 0; x < G::A_CP; ++x) {
    const int r = 8 * (8 * x + wave) + (lane >> 3);
    a_off[x] = row_a(r) * a_pitch + 16 * ((lane & 7) ^ swz(r));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int x = 0; x < G::B_CP; ++x) {
      const int r = h * (G::BN / 2) + 8 * (8 * x + wave) + (lane >> 3);
      b_off[h][x] = row_b(r) * b_pitch + 16 * ((lane & 7) ^ swz(r));
    }
  // (scales of 64 rows a wave; every wave makes a copy, some of them the same)
  int s_row[2];
  s_row[0] = 64 * (wave % (G::BM / 64 + G::BN / 128));
  if (s_row[0] >= G::BM) {
    s_off[0] = 4 * scale_b(s_row[0] - G::BM + lane);
  } else {
    s_off[0] = 4 * row_a(s_row[0] + lane);
  }
  s_row[1] = G::BM + G::BN / 2 + 64 * (wave % (G::BN / 128));
  s_off[1] = 4 * scale_b(s_row[1] - G::BM + lane);
  const uint8_t *a_src = o.a, *b_src[2] = {o.b, o.b};
  const float *as_src = o.as, *bs_src[2] = {o.bs, o.bs};
  // Copy c of the next step's operands that follow E0 (0 .. C0 - 1) and E1 (0 .. C1 - 1).
  auto copy_b = [&](uint32_t st, int h, int x) __attribute__((always_inline)) {
    dev::gload_lds16(b_src[h], b_off[h][x], lds0 + st + G::B + h * (G::BN / 2 * 128) + 1024 * (8 * x + wave), bq_span);
  };
  auto copy0 = [&](uint32_t st, int c) __attribute__((always_inline)) {
    if (c < G::A_CP) {
      dev::gload_lds16(a_src, a_off[c], lds0 + st + G::A + 1024 * (8 * c + wave), aq_span);
    } else if (c < G::A_CP + G::B_CP) {
      copy_b(st, 0, c - G::A_CP);
    } else {
      if (s_row[0] < G::BM)
        dev::gload_lds4(as_src, s_off[0], lds0 + st + G::S + 4 * s_row[0], as_span);
      else
        dev::gload_lds4(bs_src[0], s_off[0], lds0 + st + G::S + 4 * s_row[0], bs_span);
      a_src += 128, b_src[0] += 128, as_src += o.as_step, bs_src[0] += o.bs_step;
    }
  };
  auto copy1 = [&](uint32_t st, int c) __attribute__((always_inline)) {
    if (c < G::B_CP) {
      copy_b(st, 1, c);
    } else {
      dev::gload_lds4(bs_src[1], s_off[1], lds0 + st + G::S + 4 * s_row[1], bs_span);
      b_src[1] += 128, bs_src[1] += o.bs_step;
    }
  };

  const uint32_t a_fo = G::A + (wm * G::WM + fr) * 128 + ((fg ^ swz(fr)) << 4);
  const uint32_t b_fo = G::B + (wn * G::WN + fr) * 128 + ((fg ^ swz(fr)) << 4);
  auto read = [&](uint32_t at, int block) __attribute__((always_inline)) -> v8i {
    return join(*reinterpret_cast<const v4i*>(lds + at + 2048 * block), *reinterpret_cast<const v4i*>(lds + (at ^ 64) + 2048 * block));
  };
  auto scale = [&](uint32_t st, int row) __attribute__((always_inline)) -> float {
    return *reinterpret_cast<const float*>(lds + st + G::S + 4 * row);
  };
  const int KT = o.steps;
  constexpr int X = NI * NJ, P = 4, BEHIND = 2;  // a step's products; one is added when two more have been issued
  static_assert(X % P == 0 && NJ % 2 == 0, "a step begins where the one before began");
  v8i a[NI], b[2];
  v4f p[P];
  float sa[NI], sb[2], s[GLU ? 2 : 1][NI], s_last[BEHIND];
  int ea[NI], eb[2];
#pragma unroll
  for (int k = 0; k < P; ++k) p[k] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < BEHIND; ++k) s_last[k] = 0.f;
  auto read_scales = [&](uint32_t st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i) sa[i] = scale(st, wm * G::WM + 16 * i + fr);
    if constexpr (BBLOCK != 1) {
      sb[0] = scale(st, G::BM + wn * G::WN);
      if constexpr (GLU) sb[1] = scale(st, G::BM + wn * G::WN + G::WN / 2);
    }
  };
  auto read_b = [&](uint32_t st, int j) __attribute__((always_inline)) {
    b[j & 1] = read(b_fo + st, j);
    if constexpr (BBLOCK == 1) sb[j & 1] = scale(st, G::BM + wn * G::WN + 16 * j + fr);
  };
  auto add = [&](int x, float f) __attribute__((always_inline)) {  // a step's x-th product
    v4f& to = acc[dev::snake_j<NI>(x)][x / NI];
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = __builtin_fmaf(p[x % P][e], f, to[e]);
    asm volatile("" : "+v"(to));  // (added here and not later)
  };
  auto factor = [&](int x) __attribute__((always_inline)) { return s[GLU && x / NI >= NJ / 2][dev::snake_j<NI>(x)]; };
#pragma unroll
  for (int k = 0; k < G::STAGES; ++k) {
    if (k < KT)
#pragma unroll
      for (int c = 0; c < G::C0; ++c) copy0(k * G::STAGE, c);
    if (k < G::STAGES - 1 && k < KT)
#pragma unroll
      for (int c = 0; c < G::C1; ++c) copy1(k * G::STAGE, c);
  }
  if (KT >= G::STAGES)
    dev::wait_vmcnt<(G::STAGES - 1) * (G::C0 + G::C1)>();
  else
    dev::wait_vmcnt<0>();
  dev::barrier();  // A and the first half of B of step 0
  uint32_t st = 0;
  auto event1 = [&](int t) __attribute__((always_inline)) {  // E1(t)
    if (t + 1 < KT) wait_event<G, 1>(KT - 2 - t);
    dev::barrier();
  };
  auto event0 = [&](int t) __attribute__((always_inline)) {
    if (t + 1 < KT) wait_event<G, 0>(KT - 2 - t);
    dev::barrier();
  };
  auto begin = [&](uint32_t st) __attribute__((always_inline)) {
    read_scales(st);
#pragma unroll
    for (int i = 0; i < NI; ++i) a[i] = read(a_fo + st, i);
    read_b(st, 0);
  };
  // A step; its first half sends the copies that follow the event at the end of the
  // step before (FIRST), its second those that follow the event in the middle, one
  // now and then: all at once the waves wait for each other's.
  uint32_t last = (G::STAGES - 1) * G::STAGE;  // stage of step t - 1
  auto step = [&](auto group_c, auto first_c, auto second_c, int t) __attribute__((always_inline)) {
    constexpr int GROUP = decltype(group_c)::value;
    constexpr bool FIRST = decltype(first_c)::value, SECOND = decltype(second_c)::value;
    constexpr int CF = GROUP == 0 ? G::C0 : G::C1, CS = GROUP == 0 ? G::C1 : G::C0;
    const uint32_t next = st + G::STAGE == G::LDS ? 0 : st + G::STAGE;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if constexpr (BBLOCK == 1) {
        ea[i] = (int)(__float_as_uint(sa[i]) >> 23);
        asm volatile("" : "+v"(ea[i]));
      } else {
        s[0][i] = sa[i] * sb[0];
        if constexpr (GLU) s[1][i] = sa[i] * sb[1];
      }
    }
    dev::sched_fence();
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const int j = x / NI, i = dev::snake_j<NI>(x);
      if (x % NI == 0) {
        if constexpr (BBLOCK == 1) {  // (three wait states from a scale's shift to its use)
          eb[j & 1] = (int)(__float_as_uint(sb[j & 1]) >> 23);
          asm volatile("s_nop 2" : "+v"(eb[j & 1]));
        }
        if (j == NJ / 2) {
          if constexpr (GROUP == 0)
            event1(t - 1);
          else
            event0(t);
        }
        if (j + 1 < NJ) {
          read_b(st, j + 1);
        } else {
          dev::waitcnt<63, 0>();  // this step's last fragments are in registers
          if constexpr (GROUP == 0)
            event0(t);
          else
            event1(t);
          read_scales(next);
          read_b(next, 0);
        }
        dev::sched_fence();
      }
      if constexpr (BBLOCK == 1)
        issue_mfma_scaled(acc[i][j], b[j & 1], a[i], eb[j & 1], ea[i]);
      else
        issue_mfma0(p[x % P], b[j & 1], a[i]);
      dev::sched_fence();
      if (j == NJ - 1) a[i] = read(a_fo + next, i);
      if constexpr (FIRST) {
#pragma unroll
        for (int c = 0; c < CF; ++c)
          if (x == c * (X / 2) / CF) GROUP == 0 ? copy0(last, c) : copy1(last, c);
      }
      if constexpr (SECOND) {  // (not with the reads of the last column)
        constexpr int ROOM = X / 2 - NI;
#pragma unroll
        for (int c = 0; c < CS; ++c)
          if (x == X / 2 + c * ROOM / CS) GROUP == 0 ? copy1(last, c) : copy0(st, c);
      }
      if constexpr (BBLOCK != 1) {
        if (x < BEHIND)
          add(X - BEHIND + x, s_last[x]);  // (of the step before)
        else
          add(x - BEHIND, factor(x - BEHIND));
      }
      dev::sched_fence();
    }
    if constexpr (BBLOCK != 1) {
#pragma unroll
      for (int k = 0; k < BEHIND; ++k) s_last[k] = factor(X - BEHIND + k);
    }
    last = st;
    st = next;
  };
  using Yes = std::true_type;
  using No = std::false_type;
  auto loop = [&](auto group_c) __attribute__((always_inline)) {
    constexpr int GROUP = decltype(group_c)::value;
    int t = 0;
    if constexpr (GROUP == 0) {  // A and B's first half up to step STAGES - 1 are on their way
      if (G::STAGES - 1 < KT)
        step(group_c, No{}, Yes{}, t);
      else
        step(group_c, No{}, No{}, t);
      for (t = 1; t - 1 + G::STAGES < KT; ++t) step(group_c, Yes{}, Yes{}, t);
    } else {
      for (; t + G::STAGES < KT; ++t) step(group_c, Yes{}, Yes{}, t);
      if (t - 1 + G::STAGES < KT) step(group_c, Yes{}, No{}, t), ++t;
    }
    for (; t < KT; ++t) step(group_c, No{}, No{}, t);
  };
  if (wave < 4) {
    begin(0);
    loop(std::integral_constant<int, 0>{});
    dev::barrier();  // E1 of the last step
  } else {
    event1(-1);
    begin(0);
    loop(std::integral_constant<int, 1>{});
  }
  dev::sched_fence();
  wait_results();
#pragma unroll
  for (int k = 0; k < P; ++k) asm volatile("" : "+v"(p[k]));  // (read behind the wait)
  if constexpr (BBLOCK != 1) {
#pragma unroll
    for (int k = 0; k < BEHIND; ++k) add(X - BEHIND + k, s_last[k]);
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) asm volatile("" : "+v"(acc[i][j]));
  }
  dev::sched_fence();
}

// Tiles of few workgroups and short steps: four waves, one on each SIMD, all in step,
// with one barrier; a workgroup of its own fits beside it.
template <class G, int BBLOCK, bool GLU, class RowA, class RowB, class ScaleB>
__device__ __forceinline__ void multiply_small(int8_t* lds, const Operands& o, uint32_t a_pitch, uint32_t b_pitch, RowA row_a, RowB row_b,
                                         ScaleB scale_b, const dbg::Span& aq_span, const dbg::Span& as_span,
                                         const dbg::Span& bq_span, const dbg::Span& bs_span, v4f (&acc)[G::NI][G::NJ]) {
  constexpr int NI = G::NI, NJ = G::NJ;
  const uint32_t lds0 = dev::lds_addr(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = G::wm(wave), wn = G::wn(wave), fr = lane & 15, fg = lane >> 4;

  uint32_t a_off[G::A_CP], b_off[G::B_CP], s_off[G::S_CP];
#pragma unroll
  for (int x = 0; x < G::A_CP; ++x) {
    const int r = 8 * (G::WAVES * x + wave) + (lane >> 3);
    a_off[x] = row_a(r) * a_pitch + 16 * ((lane & 7) ^ swz(r));
  }
#pragma unroll
  for (int x = 0; x < G::B_CP; ++x) {
    const int r = 8 * (G::WAVES * x + wave) + (lane >> 3);
    b_off[x] = row_b(r) * b_pitch + 16 * ((lane & 7) ^ swz(r));
  }
  // (scales: every wave makes the same number of copies, the last ones again)
  int s_row[G::S_CP];
#pragma unroll
  for (int x = 0; x < G::S_CP; ++x) {
    s_row[x] = 64 * ((G::WAVES * x + wave) % ((G::BM + G::BN) / 64));
    s_off[x] = 4 * (s_row[x] < G::BM ? row_a(s_row[x] + lane) : scale_b(s_row[x] - G::BM + lane));
  }
  const uint8_t *a_src = o.a, *b_src = o.b;
  const float *as_src = o.as, *bs_src = o.bs;
  auto copy = [&](uint32_t st) __attribute__((always_inline)) {  // the next step's operands
#pragma unroll
    for (int x = 0; x < G::A_CP; ++x)
      dev::gload_lds16(a_src, a_off[x], lds0 + st + G::A + 1024 * (G::WAVES * x + wave), aq_span);
#pragma unroll
    for (int x = 0; x < G::B_CP; ++x)
      dev::gload_lds16(b_src, b_off[x], lds0 + st + G::B + 1024 * (G::WAVES * x + wave), bq_span);
#pragma unroll
    for (int x = 0; x < G::S_CP; ++x) {
      if (s_row[x] < G::BM)
        dev::gload_lds4(as_src, s_off[x], lds0 + st + G::S + 4 * s_row[x], as_span);
      else
        dev::gload_lds4(bs_src, s_off[x], lds0 + st + G::S + 4 * s_row[x], bs_span);
    }
    a_src += 128, b_src += 128, as_src += o.as_step, bs_src += o.bs_step;
  };

  const uint32_t a_fo = G::A + (wm * G::WM + fr) * 128 + ((fg ^ swz(fr)) << 4);
  const uint32_t b_fo = G::B + (wn * G::WN + fr) * 128 + ((fg ^ swz(fr)) << 4);
  auto read = [&](uint32_t at, int block) __attribute__((always_inline)) -> v8i {
    return join(*reinterpret_cast<const v4i*>(lds + at + 2048 * block), *reinterpret_cast<const v4i*>(lds + (at ^ 64) + 2048 * block));
  };
  auto scale = [&](uint32_t st, int row) __attribute__((always_inline)) -> float {
    return *reinterpret_cast<const float*>(lds + st + G::S + 4 * row);
  };
  const int KT = o.steps;
  constexpr int X = NI * NJ, P = 4, BEHIND = 2;  // a step's products; one is added when two more have been issued
  static_assert(X % P == 0 && NJ % 2 == 0, "a step begins where the one before began");
  v8i a[NI], b[2];
  v4f p[P];
  float sa[NI], sb[2], s[GLU ? 2 : 1][NI], s_last[BEHIND];
  int ea[NI], eb[2];
#pragma unroll
  for (int k = 0; k < P; ++k) p[k] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < BEHIND; ++k) s_last[k] = 0.f;
  auto read_scales = [&](uint32_t st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i) sa[i] = scale(st, wm * G::WM + 16 * i + fr);
    if constexpr (BBLOCK != 1) {
      sb[0] = scale(st, G::BM + wn * G::WN);
      if constexpr (GLU) sb[1] = scale(st, G::BM + wn * G::WN + G::WN / 2);
    }
  };
  auto read_b = [&](uint32_t st, int j) __attribute__((always_inline)) {
    b[j & 1] = read(b_fo + st, j);
    if constexpr (BBLOCK == 1) sb[j & 1] = scale(st, G::BM + wn * G::WN + 16 * j + fr);
  };
  auto add = [&](int x, float f) __attribute__((always_inline)) {  // a step's x-th product
    v4f& to = acc[dev::snake_j<NI>(x)][x / NI];
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = __builtin_fmaf(p[x % P][e], f, to[e]);
    asm volatile("" : "+v"(to));  // (added here and not later)
  };
  auto factor = [&](int x) __attribute__((always_inline)) { return s[GLU && x / NI >= NJ / 2][dev::snake_j<NI>(x)]; };
#pragma unroll
  for (int k = 0; k < G::STAGES; ++k)
    if (k < KT) copy(k * G::STAGE);
  dev::wait_tiles_behind<G::CP, G::STAGES>(min(KT, G::STAGES));
  dev::barrier();
  uint32_t st = 0;
  read_scales(0);
#pragma unroll
  for (int i = 0; i < NI; ++i) a[i] = read(a_fo, i);
  read_b(0, 0);

  for (int t = 0; t < KT; ++t) {
    const uint32_t next = st + G::STAGE == G::LDS ? 0 : st + G::STAGE;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if constexpr (BBLOCK == 1) {
        ea[i] = (int)(__float_as_uint(sa[i]) >> 23);
        asm volatile("" : "+v"(ea[i]));
      } else {
        s[0][i] = sa[i] * sb[0];
        if constexpr (GLU) s[1][i] = sa[i] * sb[1];
      }
    }
    dev::sched_fence();
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const int j = x / NI, i = dev::snake_j<NI>(x);
      if (x % NI == 0) {
        if constexpr (BBLOCK == 1) {  // (three wait states from a scale's shift to its use)
          eb[j & 1] = (int)(__float_as_uint(sb[j & 1]) >> 23);
          asm volatile("s_nop 2" : "+v"(eb[j & 1]));
        }
        if (j + 1 < NJ) {
          read_b(st, j + 1);
        } else {
          // This step's last fragments are in registers: once every wave is here, and
          // the next step's operands too, its stage takes the copies of step t + STAGES.
          dev::waitcnt<63, 0>();
          if (t + 1 < KT) dev::wait_tiles_behind<G::CP, G::STAGES - 1>(min(KT - 1 - t, G::STAGES - 1));
          dev::barrier();
          if (t + G::STAGES < KT) copy(st);
          read_scales(next);
          read_b(next, 0);
        }
        dev::sched_fence();
      }
      if constexpr (BBLOCK == 1)
        issue_mfma_scaled(acc[i][j], b[j & 1], a[i], eb[j & 1], ea[i]);
      else
        issue_mfma0(p[x % P], b[j & 1], a[i]);
      dev::sched_fence();
      if (j == NJ - 1) a[i] = read(a_fo + next, i);
      if constexpr (BBLOCK != 1) {
        if (x < BEHIND)
          add(X - BEHIND + x, s_last[x]);  // (of the step before)
        else
          add(x - BEHIND, factor(x - BEHIND));
      }
      dev::sched_fence();
    }
    if constexpr (BBLOCK != 1) {
#pragma unroll
      for (int k = 0; k < BEHIND; ++k) s_last[k] = factor(X - BEHIND + k);
    }
    st = next;
  }
  dev::sched_fence();
  wait_results();
#pragma unroll
  for (int k = 0; k < P; ++k) asm volatile("" : "+v"(p[k]));  // (read behind the wait)
  if constexpr (BBLOCK != 1) {
#pragma unroll
    for (int k = 0; k < BEHIND; ++k) add(X - BEHIND + k, s_last[k]);
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) asm volatile("" : "+v"(acc[i][j]));
  }
  dev::sched_fence();
}

// A wave's part at row 0 and column n0 of C (m < M rows, n0 + .. < N columns of it
// exist).  In bf16 two blocks beside each other are exchanged between the lanes of a
// row, so that each holds eight columns of one: 16 bytes a lane in either type.
template <class T, int NI, int NJ>
__device__ __forceinline__ void store_part(T* C, size_t ldc, int m0, int n0, int M, int N, const v4f (&acc)[NI][NJ]) {
  const int lane = threadIdx.x & 63, fr = lane & 15, fg = lane >> 4;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int m = m0 + 16 * i + fr;
#pragma unroll
    for (int j = 0; j < NJ; j += 2) {
      if constexpr (sizeof(T) == 4) {
        store4(C, ldc, m, n0 + 16 * j + 4 * fg, M, N, acc[i][j]);
        store4(C, ldc, m, n0 + 16 * j + 16 + 4 * fg, M, N, acc[i][j + 1]);
      } else {
        v2u a = __builtin_bit_cast(v2u, __builtin_convertvector(acc[i][j], v4bf));
        v2u b = __builtin_bit_cast(v2u, __builtin_convertvector(acc[i][j + 1], v4bf));
        uint32_t a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];
        swap16(a0, b0);
        swap16(a1, b1);
        const v8bf v = __builtin_bit_cast(v8bf, v4u{a0, a1, b0, b1});
        const int n = n0 + 16 * j + 16 * (fg & 1) + 8 * (fg >> 1);
        if (m < M) {
          T* p = C + (size_t)m * ldc + n;
          if (n + 8 <= N) {
            using P = At<v8bf, T>;
            MIAIE_ST(reinterpret_cast<P*>(p), P{v});
          } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
              if (n + e < N) MIAIE_ST(p + e, v[e]);
          }
        }
      }
    }
    dev::sched_fence();  // (more rows at once take more registers than there are)
  }
}

// H = silu(gate) up of a wave's rows, columns j < NJ / 2 gate and the others up of
// the same H columns; packed along its rows.  A block of 128 columns of H is the
// workgroup's, so the rows' maxima are joined through LDS.
template <class G>
__device__ __forceinline__ void store_glu(const Args& p, int8_t* lds, int slot0, int rows, int f0, v4f (&acc)[G::NI][G::NJ]) {
  constexpr int NI = G::NI, HJ = G::NJ / 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = G::wm(wave), wn = G::wn(wave), fr = lane & 15, fg = lane >> 4;
  uint32_t* const lmax = reinterpret_cast<uint32_t*>(lds);
  uint32_t mine[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < HJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float h = swiglu(acc[i][j][e], acc[i][j + HJ][e]);
        acc[i][j][e] = h;
        m = max(m, abs_bits(h));
      }
    mine[i] = max_over_16s(m);
  }
  __syncthreads();  // (the last fragments have been read)
#pragma unroll
  for (int i = 0; i < NI; ++i)
    if (fg == 0) lmax[wn * G::BM + wm * G::WM + 16 * i + fr] = mine[i];
  __syncthreads();
  const size_t h_pitch = pitch(p.N);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = wm * G::WM + 16 * i + fr;
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < G::WAVES_N; ++w) m = max(m, lmax[w * G::BM + r]);
    const uint32_t e = scale_of(m);
    const float inv = inverse_f32(e);
    uint32_t q[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < HJ; ++j) q[j] = pack4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], inv);
    uint8_t* row = p.Hq + (size_t)(slot0 + r) * h_pitch + f0 + wn * (G::WN / 2);
    if constexpr (HJ == 4) {  // the lanes' 4 x 4 dwords transposed: 16 columns of one block a lane
      swap32(q[0], q[2]);
      swap32(q[1], q[3]);
      swap16(q[0], q[1]);
      swap16(q[2], q[3]);
      if (r < rows) MIAIE_ST(reinterpret_cast<v4u*>(row + 16 * fg), (v4u{q[0], q[1], q[2], q[3]}));
    } else {
      static_assert(HJ == 2 || HJ == 4, "columns of a wave");
      swap16(q[0], q[1]);
      if (r < rows) MIAIE_ST(reinterpret_cast<v2u*>(row + 16 * (fg & 1) + 8 * (fg >> 1)), (v2u{q[0], q[1]}));
    }
    if (wn == 0 && fg == 0 && r < rows) MIAIE_ST(p.Hs + (size_t)(f0 / 128) * p.M + slot0 + r, scale_f32(e));
  }
}

// Inclusive sums over the lanes of a wave.
__device__ __forceinline__ int scan_wave(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // lane - 1 of sixteen
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // ... - 2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // ... - 4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // ... - 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // the last of the sixteen before
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // the last of the first half
  return v;
}

// A tile of up to ROWS slots of one expert: its tiles are ceil(count / ROWS) of rows
// times tiles_n, walked rows first, so that those which share columns of B run beside
// each other, and the workgroups of one XCD have a contiguous run of all tiles, this
// the i-th of it: few experts' operands in one L2.  Every wave finds its tile from the
// experts' counts: loads beside each other, where a walk through the order's parts would be
// three that wait for one another, and no workgroup without a tile among the others
// (such a one waits for a whole CU's LDS like the rest: 16384 slots of 64 experts at
// 256 rows a tile 235 us with as many empty ones, 168 without).  False: no tile.
struct SlotTile {
  int e, slot, rows, tn;  // rows: of the expert from this slot on
};
template <int ROWS>
__device__ __forceinline__ bool slot_tile(const Slots& s, int xcd, int i, int tiles_n, SlotTile& to) {
  const int lane = threadIdx.x & 63;
  auto count_of = [&](int e0) { return e0 + lane < s.experts ? MIAIE_LD(s.count + e0 + lane) : 0; };
  int count = count_of(0), rows = scan_wave((count + ROWS - 1) / ROWS), total = __builtin_amdgcn_readlane(rows, 63);
  for (int e0 = 64; e0 < s.experts; e0 += 64)
    total += __builtin_amdgcn_readlane(scan_wave((count_of(e0) + ROWS - 1) / ROWS), 63);
  const int tiles = total * tiles_n, each = (tiles + 7) / 8, logical = xcd * each + i;
  if (i >= each || logical >= tiles) return false;
  const int at = logical / tiles_n;
  int before = 0, blocks_before = 0, e0 = 0;  // tiles of rows, and blocks of 128 slots, before expert e0
  int blocks_to = scan_wave((count + 127) / 128);
  while (before + __builtin_amdgcn_readlane(rows, 63) <= at) {
    before += __builtin_amdgcn_readlane(rows, 63);
    blocks_before += __builtin_amdgcn_readlane(blocks_to, 63);
    e0 += 64;
    count = count_of(e0);
    rows = scan_wave((count + ROWS - 1) / ROWS);
    blocks_to = scan_wave((count + 127) / 128);
  }
  const int l = __builtin_ctzll(__ballot(before + rows > at));
  const int c = __builtin_amdgcn_readlane(count, l), n = (c + ROWS - 1) / ROWS;
  const int local = logical - (before + __builtin_amdgcn_readlane(rows, l) - n) * tiles_n, row = local % n * ROWS;
  to.e = e0 + l;
  to.slot = 128 * (blocks_before + __builtin_amdgcn_readlane(blocks_to, l) - (c + 127) / 128) + row;
  to.rows = c - row;
  to.tn = local / n;
  return true;
}

// The tile at row m0 and column n0 of expert e's product (DENSE: e = 0); `rows` of A
// and C exist from m0 on.
template <class G, Mode MODE, Out OUT, int BBLOCK>
__device__ __forceinline__ void run_tile_at(const Args& p, int8_t* lds, int e, int m0, int n0, int rows) {
  constexpr bool GLU = OUT == OUT_GLU;
  constexpr int COLS = GLU ? G::BN / 2 : G::BN;  // columns of the result
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t pch = (uint32_t)pitch(p.K);
  const int b_rows = GLU ? 2 * p.N : p.N;
  const size_t b_s_rows = BBLOCK == 1 ? (size_t)b_rows : blocks(b_rows);
  Operands o;
  o.a = p.Aq, o.as = p.As;
  o.b = p.Bq + (size_t)n0 * pch, o.bs = p.Bs + (BBLOCK == 1 ? n0 : n0 / 128);
  o.steps = (int)blocks(p.K);
  o.as_step = p.a_rows, o.bs_step = b_s_rows;
  o.rows = min(rows, G::BM), o.cols = min(p.N - n0, COLS);
  size_t to = 0;  // first element of the product in C
  if constexpr (MODE == SLOTS) o.b += (size_t)e * b_rows * pch, o.bs += (size_t)e * b_s_rows * blocks(p.K);
  if (MODE != SLOTS || !p.gather) o.a += (size_t)m0 * pch, o.as += m0;
  if constexpr (MODE == WGRAD) {  // k: the expert's slots
    const int first = MIAIE_LD(p.s.start + e);
    o.steps = (int)blocks(MIAIE_LD(p.s.count + e));
    o.a += first, o.as += (size_t)(first / 128) * p.M;
    o.b += first, o.bs += (size_t)(first / 128) * b_s_rows;
    to = (size_t)e * p.M * p.ldc;
  }
  const dbg::Span aq_span = dbg::span_of(p.Aq), as_span = dbg::span_of(p.As), bq_span = dbg::span_of(p.Bq),
                  bs_span = dbg::span_of(p.Bs);  // (debug build only)
  v4f acc[G::NI][G::NJ];
#pragma unroll
  for (int i = 0; i < G::NI; ++i)
#pragma unroll
    for (int j = 0; j < G::NJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  // rows behind the last one are copies of it, and dropped at the end
  auto row_a = [&](int r) __attribute__((always_inline)) -> uint32_t {
    r = min(r, o.rows - 1);
    if constexpr (MODE == SLOTS) {
      if (p.gather) return (uint32_t)(MIAIE_LD(p.s.row_of + m0 + r) / p.s.top_k);
    }
    return (uint32_t)r;
  };
  // GLU: row r of a wave's part of the stage is a gate's, or the same column's up
  auto row_b = [&](int r) __attribute__((always_inline)) -> uint32_t {
    if constexpr (GLU) {
      const int h = r % G::WN, f = r / G::WN * (G::WN / 2) + h % (G::WN / 2);
      return (uint32_t)(h < G::WN / 2 ? f : p.N + f);
    }
    return (uint32_t)min(r, o.cols - 1);
  };
  auto scale_b = [&](int r) __attribute__((always_inline)) -> uint32_t {
    return BBLOCK == 1 ? row_b(r) : row_b(r) / 128;
  };
  if (o.steps > 0) {
    if constexpr (G::WAVES == 4)
      multiply_small<G, BBLOCK, GLU>(lds, o, pch, pch, row_a, row_b, scale_b, aq_span, as_span, bq_span, bs_span, acc);
    else
      multiply<G, BBLOCK, GLU>(lds, o, pch, pch, row_a, row_b, scale_b, aq_span, as_span, bq_span, bs_span, acc);
  }
  if constexpr (GLU) {
    store_glu<G>(p, lds, m0, o.rows, n0, acc);
  } else {
    using T = std::conditional_t<OUT == OUT_F32, float, __bf16>;
    store_part(static_cast<T*>(p.C) + to, p.ldc, m0 + G::wm(wave) * G::WM, n0 + G::wn(wave) * G::WN, m0 + o.rows, p.N, acc);
  }
}

template <class G, Mode MODE, Out OUT, int BBLOCK>
__global__ __launch_bounds__(G::THREADS) void gemm_tile(Args p, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[G::LDS];
  constexpr int COLS = OUT == OUT_GLU ? G::BN / 2 : G::BN;
  if constexpr (MODE == SLOTS) {
    SlotTile t;
    if (!slot_tile<G::BM>(p.s, blockIdx.x % 8, blockIdx.x / 8, tiles_n, t)) return;
    run_tile_at<G, MODE, OUT, BBLOCK>(p, lds, t.e, t.slot, t.tn * COLS, t.rows);
  } else {
    const int each = tiles_m * tiles_n, e = MODE == WGRAD ? blockIdx.x / each : 0;
    int tm, tn;
    dev::tile_coords<4>(MODE == WGRAD ? blockIdx.x % each : blockIdx.x, tiles_m, tiles_n, tm, tn);
    run_tile_at<G, MODE, OUT, BBLOCK>(p, lds, e, tm * G::BM, tn * COLS, p.M - tm * G::BM);
  }
}

// Slots in tiles of 256 rows, the last 128 or fewer of an expert in one of 128.
template <class G, class H, Out OUT>
__global__ __launch_bounds__(G::THREADS) void gemm_slots(Args p, int tiles_n) {
  static_assert(G::BM == 256 && H::BM == 128 && G::BN == H::BN && G::THREADS == H::THREADS, "tiles of one launch");
  __shared__ __attribute__((aligned(1024))) int8_t lds[G::LDS > H::LDS ? G::LDS : H::LDS];
  constexpr int COLS = OUT == OUT_GLU ? G::BN / 2 : G::BN;
  SlotTile t;
  if (!slot_tile<256>(p.s, blockIdx.x % 8, blockIdx.x / 8, tiles_n, t)) return;
  if (t.rows > 128)
    run_tile_at<G, SLOTS, OUT, 128>(p, lds, t.e, t.slot, t.tn * COLS, t.rows);
  else
    run_tile_at<H, SLOTS, OUT, 128>(p, lds, t.e, t.slot, t.tn * COLS, t.rows);
}

// ---------------------------------------------------------------- few rows
// Up to four rows of A at a time by reading B as it lies in memory, straight into
// registers: a load takes whole lines of eight rows, lane l the 16 bytes l % 8 of row
// l / 8, and multiplies them in fp32 with those of A, which the workgroup keeps in
// LDS.  Bound by reading B, every byte of it once; a wave has eight to sixteen lines of
// eight rows in flight.  (On the matrix instructions, which want 16 rows' 16 bytes
// side by side, B had to go through LDS: 1 x 11008 x 4096 12.7 us.)
//
// fp32 products are exact here, where the 8-bit matrix instructions cut them off at
// 2^-13 of the largest of eight.  That moves their sums by 1.5e-5, and one in 400
// codes of a packed H with them; with many rows such steps average out, while a
// token's own MLP was up to 5.7e-3 off with a few of them (2.4e-3 without: Y and out are
// each rounded to bf16).
constexpr int STREAM_K = 64;  // blocks of k whose A is in LDS at a time

// <16 elements of a row of B, 16 elements of a row of A>
__device__ __forceinline__ float dot16(const float (&b)[16], const float (&a)[16]) {
  float p0 = b[0] * a[0], p1 = b[1] * a[1];
#pragma unroll
  for (int i = 2; i < 16; i += 2) p0 = __builtin_fmaf(b[i], a[i], p0), p1 = __builtin_fmaf(b[i + 1], a[i + 1], p1);
  return p0 + p1;
}
__device__ __forceinline__ void widen(v4u q, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const mx::v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], true);
    x[4 * i] = lo[0], x[4 * i + 1] = lo[1], x[4 * i + 2] = hi[0], x[4 * i + 3] = hi[1];
  }
}

// acc[m][u] += row m of A (in LDS, STREAM_K blocks a row) times this lane's part of
// row l / 8 of b[u], over the blocks kb0 + first .. kb0 + last - 1.  s[m][u]: lane kb
// has the scale of block kb0 + kb.
// D blocks are loaded together, and as many behind them.
template <int MR, int D>
__device__ __forceinline__ void stream(const int8_t* lds, const uint8_t* const (&b)[2], int first, int last, const float (&s)[MR][2],
                                       float (&acc)[MR][2]) {
  const int lane = threadIdx.x & 63;
  v4u q[2][D][2];
  auto load = [&](int kb, v4u (&to)[D][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u)  // (blocks behind the last one repeat it)
        to[d][u] = MIAIE_LD(reinterpret_cast<const v4u*>(b[u] + 128 * (size_t)min(kb + d, last - 1)));
  };
  auto multiply = [&](int kb, const v4u (&from)[D][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (kb + d >= last) return;
      float x[2][16];
#pragma unroll
      for (int u = 0; u < 2; ++u) widen(from[d][u], x[u]);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        float a[16];
        widen(*reinterpret_cast<const v4u*>(lds + 128 * (m * STREAM_K + kb + d) + 16 * (lane & 7)), a);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          acc[m][u] = __builtin_fmaf(dot16(x[u], a), __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s[m][u]), kb + d)), acc[m][u]);
      }
    }
  };
  if (first >= last) return;
  load(first, q[0]);
  for (int kb = first; kb < last; kb += 2 * D) {
    load(min(kb + D, last - 1), q[1]);
    multiply(kb, q[0]);
    if (kb + D >= last) break;
    load(min(kb + 2 * D, last - 1), q[0]);
    multiply(kb + D, q[1]);
  }
}

// Where a workgroup's rows and columns are.
struct StreamTile {
  const uint8_t *a, *b;  // first row of each
  const float *as, *bs;
  size_t a_step, b_step;  // floats from one block's scales to the next's
  int rows;
};

// acc[m][u] of the MR rows (those behind the last repeat it) and this wave's b0 and b1,
// the sums over the lanes of a row in each of them.  `again`: LDS holds rows that other
// waves may still read.
template <int MR, int D, class RowA>
__device__ __forceinline__ void stream_rows(int8_t* lds, const Args& p, const StreamTile& t, const uint8_t* const (&b)[2],
                                            const float* const (&bs)[2], bool again, RowA row_a, int part, int parts, float (&acc)[MR][2]) {
  const int tid = threadIdx.x, lane = tid & 63, threads = blockDim.x;
  const int steps = (int)blocks(p.K);
  const size_t pch = pitch(p.K);
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m][0] = acc[m][1] = 0.f;
  for (int kb0 = 0; kb0 < steps; kb0 += STREAM_K) {
    const int n = min(STREAM_K, steps - kb0);
    if (kb0 > 0 || again) __syncthreads();
    for (int i = tid; i < MR * n * 8; i += threads) {
      const int m = i / (8 * n), c = i % (8 * n);
      const v4u v = MIAIE_LD(reinterpret_cast<const v4u*>(t.a + row_a(min(m, t.rows - 1)) * pch + 128 * (size_t)kb0 + 16 * c));
      *reinterpret_cast<v4u*>(lds + 128 * m * STREAM_K + 16 * c) = v;
    }
    float s[MR][2];
    const size_t kb = kb0 + min(lane, n - 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float sb = MIAIE_LD(bs[u] + kb * t.b_step);
#pragma unroll
      for (int m = 0; m < MR; ++m) s[m][u] = sb * MIAIE_LD(t.as + kb * t.a_step + row_a(min(m, t.rows - 1)));
    }
    __syncthreads();
    const uint8_t* const from[2] = {b[0] + 128 * (size_t)kb0, b[1] + 128 * (size_t)kb0};
    const int each = (n + parts - 1) / parts;
    stream<MR, D>(lds, from, part * each, min(n, (part + 1) * each), s, acc);
  }
  // the eight lanes of a row
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float v = acc[m][u];
      v += __uint_as_float(mx::quad_swap<0xB1>(__float_as_uint(v)));
      v += __uint_as_float(mx::quad_swap<0x4E>(__float_as_uint(v)));
      v += __uint_as_float(mx::quad_swap<0x141>(__float_as_uint(v)));
      acc[m][u] = v;
    }
}

// f(number of rows taken together) for the rows that are left.
template <class F>
__device__ __forceinline__ void by_rows(int left, F&& f) {
  if (left == 1)
    f(std::integral_constant<int, 1>{});
  else if (left == 2)
    f(std::integral_constant<int, 2>{});
  else
    f(std::integral_constant<int, 4>{});
}

// Four waves; 4 / parts of them have 16 columns each, and `parts` share out the blocks
// of k, whose sums are added in LDS in their order.  Over slots a workgroup takes four
// rows of one expert at a time, and the launch's workgroups share out all of these: with
// an expert's to one workgroup, a popular expert's passes follow one another (256 slots
// of one expert of 64, 1024 -> 4096 columns: 155 us, 55 shared out).
template <Mode MODE, Out OUT>
__global__ __launch_bounds__(256) void gemm_stream(Args p, int tiles_n, int parts) {
  __shared__ __attribute__((aligned(16))) int8_t lds[4 * 128 * STREAM_K];
  __shared__ float sums[4][4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = wave % parts, groups = 4 / parts;
  const size_t pch = pitch(p.K);
  auto pass = [&](const StreamTile& t, int row0, int n0, bool again, auto row_a) __attribute__((always_inline)) {
    const int col = n0 + 16 * (wave / parts);  // of this wave; behind the last one it repeats that
    const uint8_t* b[2];
    const float* bs[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      b[u] = t.b + (size_t)min(col + 8 * u + (lane >> 3), p.N - 1) * pch + 16 * (lane & 7);
      bs[u] = t.bs + min(col, p.N - 1) / 128;
    }
    by_rows(t.rows, [&](auto mr) __attribute__((always_inline)) {
      constexpr int MR = decltype(mr)::value;
      float acc[MR][2];
      stream_rows<MR, 4>(lds, p, t, b, bs, again, row_a, part, parts, acc);
      if ((lane & 7) == 0)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
          for (int u = 0; u < 2; ++u) sums[wave][m][8 * u + (lane >> 3)] = acc[m][u];
    });
    __syncthreads();
    // thread: row tid / 64, column tid % 64 of the workgroup's
    const int n = n0 + lane;
    if (wave < t.rows && lane < 16 * groups && n < p.N) {
      float sum = 0.f;
      for (int k = 0; k < parts; ++k) sum += sums[lane / 16 * parts + k][wave][lane % 16];
      using T = std::conditional_t<OUT == OUT_F32, float, __bf16>;
      MIAIE_ST(static_cast<T*>(p.C) + (size_t)(row0 + wave) * p.ldc + n, (T)sum);
    }
  };
  if constexpr (MODE == SLOTS) {
    const int first = blockIdx.x / 8;
    SlotTile at;
    for (int i = first; slot_tile<4>(p.s, blockIdx.x % 8, i, tiles_n, at); i += gridDim.x / 8) {
      StreamTile t{p.Aq, p.Bq + (size_t)at.e * p.N * pch, p.As, p.Bs + (size_t)at.e * blocks(p.N) * blocks(p.K), (size_t)p.a_rows,
                   blocks(p.N), min(4, at.rows)};
      if (!p.gather) t.a += (size_t)at.slot * pch, t.as += at.slot;
      pass(t, at.slot, 16 * groups * at.tn, i > first, [&](int r) __attribute__((always_inline)) -> size_t {
        return p.gather ? (size_t)(MIAIE_LD(p.s.row_of + at.slot + r) / p.s.top_k) : (size_t)r;
      });
    }
  } else {  // (up to four rows)
    pass(StreamTile{p.Aq, p.Bq, p.As, p.Bs, (size_t)p.a_rows, blocks(p.N), p.M}, 0, 16 * groups * blockIdx.x, false,
         [&](int r) __attribute__((always_inline)) -> size_t { return (size_t)r; });
  }
}

// The block product in bf16, which holds every element: 16 conversions and four
// instructions a fragment, sums as fp32 has them.
struct Wide {
  v8bf v[4];
  __device__ __forceinline__ explicit Wide(v8i x) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
      const v2bf c0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * q], 1.f, false), c1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * q], 1.f, true),
                 c2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * q + 1], 1.f, false), c3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * q + 1], 1.f, true);
      v[q] = v8bf{c0[0], c0[1], c1[0], c1[1], c2[0], c2[1], c3[0], c3[1]};
    }
  }
};
__device__ __forceinline__ v4f mfma_wide(const Wide& b, const Wide& a) {
  v4f p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[q], a.v[q], p, 0, 0, 0);
  return p;
}

// silu(gate) up of 128 columns of H and four rows of an expert, shared out over the
// launch's workgroups as in gemm_stream (256 slots of one expert, 4096 x 1024: 470 us by
// one workgroup a column block, 40 shared out): eight waves, each with 16 gate and 16 up
// columns over all of k.  A wave copies 256 bytes (two blocks of k, a group) of its 32
// rows of B and of A's rows into a part of LDS of its own, waits for its own copies (no
// barriers) and multiplies; the next group is on its way once this one's fragments are
// in registers.  Chunk c (16 bytes) of row r lies at c ^ (r % 16).  Two workgroups fit a CU, so that one starts while another reads
// (as loads of whole lines into registers, like gemm_stream, one fits: 101 us for 86
// at 64 experts of 2048 x 4096, eight tokens of eight).
constexpr int kGluRows = 4, kGluRegion = 2 * 4096 + 256 * kGluRows;
__global__ __launch_bounds__(512, 4) void glu_rows(Args p, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[8 * kGluRegion];
  __shared__ uint32_t lmax[8][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const uint32_t row_pitch = (uint32_t)pitch(p.K);
  const size_t b_s_rows = blocks(2 * (long)p.N);
  const int steps = (int)blocks(p.K), groups = (steps + 1) / 2;
  const dbg::Span aq_span = dbg::span_of(p.Aq), bq_span = dbg::span_of(p.Bq);  // (debug build only)
  const size_t h_pitch = pitch(p.N);
  int8_t* const mine = lds + wave * kGluRegion;
  const uint32_t mine0 = dev::lds_addr(mine);
  SlotTile t;
  for (int i = blockIdx.x / 8; slot_tile<kGluRows>(p.s, blockIdx.x % 8, i, tiles_n, t); i += gridDim.x / 8) {
    const int e = t.e, tn = t.tn, slot0 = t.slot, f0 = 128 * tn, n = min(kGluRows, t.rows);
    const uint8_t* const a = p.gather ? p.Aq : p.Aq + (size_t)slot0 * row_pitch;
    const float* const as = p.gather ? p.As : p.As + slot0;
    const uint8_t* const gate = p.Bq + ((size_t)e * 2 * p.N + f0 + 16 * wave) * row_pitch;
    const uint8_t* const b[2] = {gate, gate + (size_t)p.N * row_pitch};
    const float* const gate_s = p.Bs + (size_t)e * b_s_rows * steps + f0 / 128;
    const float* const bs[2] = {gate_s, gate_s + p.N / 128};
    auto row_a = [&](int r) __attribute__((always_inline)) -> uint32_t {
      r = slot0 + min(r, n - 1);  // (rows behind the last repeat it)
      return p.gather ? (uint32_t)(MIAIE_LD(p.s.row_of + r) / p.s.top_k) : (uint32_t)(r - slot0);
    };
    const uint32_t a_row = row_a(fg), s_row = row_a(fr);
    v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
    float sa[2], sb[2][2];
    auto copy = [&](int g) __attribute__((always_inline)) {
      const uint32_t mask = 2 * g + 1 < steps ? 15 : 7;  // (half a group: its first block again)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const size_t kb = min(2 * g + k, steps - 1);
        sa[k] = MIAIE_LD(as + kb * p.a_rows + s_row);
#pragma unroll
        for (int j = 0; j < 2; ++j) sb[k][j] = MIAIE_LD(bs[j] + kb * b_s_rows);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          dev::gload_lds16(b[j] + 256 * (size_t)g, (uint32_t)(4 * x + fg) * row_pitch + 16 * ((fr ^ (4 * x + fg)) & mask),
                           mine0 + 4096 * j + 1024 * x, bq_span);
      dev::gload_lds16(a + 256 * (size_t)g, a_row * row_pitch + 16 * ((fr ^ fg) & mask), mine0 + 8192, aq_span);
    };
    auto half = [&](int k) __attribute__((always_inline)) {
      const int c0 = 8 * k + fg, c1 = c0 + 4, r = min(fr, kGluRows - 1);
      auto fragment = [&](int at, int row) __attribute__((always_inline)) {
        return Wide(join(*reinterpret_cast<const v4i*>(mine + at + 256 * row + 16 * (c0 ^ row)),
                         *reinterpret_cast<const v4i*>(mine + at + 256 * row + 16 * (c1 ^ row))));
      };
      const Wide fa = fragment(8192, r);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const v4f q = mfma_wide(fragment(4096 * j, fr), fa);
        const float f = sa[k] * sb[k][j];
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[j][x] = __builtin_fmaf(q[x], f, acc[j][x]);
      }
    };
    copy(0);
    for (int g = 0; g < groups; ++g) {
      dev::wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      half(0);
      if (2 * g + 1 < steps) half(1);
      if (g + 1 < groups) {
        dev::waitcnt<63, 0>();
        asm volatile("" ::: "memory");
        copy(g + 1);
      }
    }
    float h[4];
    uint32_t m = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      h[x] = swiglu(acc[0][x], acc[1][x]);
      m = max(m, abs_bits(h[x]));
    }
    m = max_over_16s(m);
    if (fg == 0) lmax[wave][fr] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, lmax[w][fr]);
    const uint32_t ex = scale_of(m);
    if (fr < n) {
      const size_t slot = slot0 + fr;
      MIAIE_ST(reinterpret_cast<uint32_t*>(p.Hq + slot * h_pitch + f0 + 16 * wave + 4 * fg), pack4(h[0], h[1], h[2], h[3], inverse_f32(ex)));
      if (wave == 0 && fg == 0) MIAIE_ST(p.Hs + (size_t)tn * p.M + slot, scale_f32(ex));
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- launches
// Measured (bf16 results): 8192^3 440 us (2.5 PFLOP/s) on Large; 2048 x 4096 x 4096 42
// us on Block (16 workgroups a row of tiles: one round); 4096 x 4096 over 2048 35 us on
// Large with a scale a row; 333 x 777 x 1000 5.6 us on Small; 1 x 11008 x 4096 10 us
// by gemm_stream (4.5 TB/s).  64 experts of 256 slots, 4096 x 1024: gate and up 200 us,
// down 123 us on Large and Block together; of one slot 86 us by glu_rows, 27 us on
// Small.
using Large = Tile<256, 256, 4, 2>;
using Block = Tile<128, 256, 2, 3>;
using Square = SmallTile<128, 128, 2>;
using Flat = SmallTile<64, 128, 3>;
using Small = SmallTile<64, 64, 3>;
using Glu = SmallTile<64, 256, 2>;  // (128 columns of H)

constexpr long kThreads = (1l << 32) - 8 * 512;  // HIP takes fewer than 2^32 in a launch; slots round up to eight workgroups

// Most tiles of `rows` slots that a routing can make: one more for each expert than
// its rows fill.
long most_slot_tiles(const Slots& s, int rows) {
  const long n = (long)s.tokens * s.top_k, used = std::min<long>(s.experts, n);
  return used + (n - used) / rows;
}

template <class G, Mode MODE, Out OUT, int BBLOCK>
int run_tile(miaie_ctx* ctx, const Args& p) {
  const long tiles_m = (p.M + G::BM - 1l) / G::BM, cols = OUT == OUT_GLU ? G::BN / 2 : G::BN, tiles_n = (p.N + cols - 1) / cols;
  long grid = tiles_m * tiles_n;
  if (MODE == WGRAD) grid *= p.s.experts;
  if (MODE == SLOTS) grid = (most_slot_tiles(p.s, G::BM) * tiles_n + 7) / 8 * 8;
  const hipError_t e = launch<gemm_tile<G, MODE, OUT, BBLOCK>>(ctx->device, dim3((unsigned)grid), dim3(G::THREADS), 0, ctx->stream, p,
                                                               (int)tiles_m, (int)tiles_n);
  return check_launch(ctx, e, "gemm_fp8_tile");
}

template <Out OUT>
int run_slots_large(miaie_ctx* ctx, const Args& p) {
  const long cols = OUT == OUT_GLU ? Large::BN / 2 : Large::BN, tiles_n = (p.N + cols - 1) / cols;
  const long grid = (most_slot_tiles(p.s, 256) * tiles_n + 7) / 8 * 8;
  const hipError_t e = launch<gemm_slots<Large, Block, OUT>>(ctx->device, dim3((unsigned)grid), dim3(Large::THREADS), 0, ctx->stream, p,
                                                             (int)tiles_n);
  return check_launch(ctx, e, "gemm_fp8_slots");
}

// Waves that share out k: at least eight blocks each.
int stream_parts(int K) { return blocks(K) >= 32 ? 4 : blocks(K) >= 16 ? 2 : 1; }

template <Mode MODE, Out OUT>
int run_stream(miaie_ctx* ctx, const Args& p) {
  const int parts = stream_parts(p.K);
  const long cols = 16 * (4 / parts), tiles_n = (p.N + cols - 1) / cols;
  const long grid = MODE == SLOTS ? (most_slot_tiles(p.s, 128) * tiles_n + 7) / 8 * 8 : tiles_n;
  const hipError_t e = launch<gemm_stream<MODE, OUT>>(ctx->device, dim3((unsigned)grid), dim3(256), 0, ctx->stream, p, (int)tiles_n, parts);
  return check_launch(ctx, e, "gemm_fp8_stream");
}

int run_glu_rows(miaie_ctx* ctx, const Args& p) {
  const long grid = (most_slot_tiles(p.s, 128) * (p.N / 128) + 7) / 8 * 8;
  const hipError_t e = launch<glu_rows>(ctx->device, dim3((unsigned)grid), dim3(512), 0, ctx->stream, p, p.N / 128);
  return check_launch(ctx, e, "glu_rows");
}

// ---- choice of tile: the lowest estimated time.  A CU has `at_once` workgroups of a
// tile; a workgroup's start and end, and a step's time with one, two, ... of them on
// the CU while most CUs are at work (the clock falls under that load; with few at
// work, a step alone takes idle).  Measured at 4096 columns and K = 4096, random
// elements.  The estimates are for the choice, not for the time.
struct TileTime {
  int bm, bn, at_once;
  double ends, idle, step[3];
};
constexpr TileTime kLarge{256, 256, 1, 9.0, 1.05, {1.50}}, kBlock{128, 256, 1, 6.5, 0.72, {0.95}},
    kSquare{128, 128, 2, 3.3, 0.57, {0.65, 1.09}}, kFlat{64, 128, 2, 2.3, 0.44, {0.47, 0.70}},
    kSmall{64, 64, 3, 2.0, 0.29, {0.31, 0.44, 0.54}}, kGlu{64, 256, 1, 3.0, 0.60, {0.95}};

// (none: a launch of so many tiles would be too large)
double tile_us(const TileTime& t, double tiles, int threads, long steps, int cus) {
  if (tiles * threads >= (double)kThreads) return 1e300;
  if (2 * tiles <= cus) return 1.0 + t.ends + t.idle * steps;
  const long each = (long)((tiles + cus - 1) / cus), full = each / t.at_once, rest = each % t.at_once;
  return 1.0 + full * (t.ends + t.step[t.at_once - 1] * steps) + (rest ? t.ends + t.step[rest - 1] * steps : 0.0);
}

// A kernel of the choice.  T: a tile; Stream, GluRows: few rows.
template <class T>
struct On {
  using type = T;
};
struct Stream {};
struct GluRows {};

// f(the kernel of a dense product).  Up to four rows of weights: one reading of B by
// gemm_stream (four rows, 4096 -> 11008, 4096 -> 4096 and 12288 -> 1024 columns: 16.6, 8.5
// and 16.0 us, where the tile of 64 rows takes 15.3, 11.4 and 29.8 for five to 64; two
// readings, for five to eight, 32, 16.0 and 31.9).
template <class F>
int with_dense(int M, int N, int K, int b_block, int cus, F&& f) {
  if (b_block == 128 && M <= 4) return f(Stream{});
  auto us = [&](const TileTime& t, int threads) {
    return tile_us(t, (double)((M + t.bm - 1l) / t.bm) * (double)((N + t.bn - 1l) / t.bn), threads, (long)blocks(K), cus);
  };
  const double times[] = {us(kLarge, 512), us(kBlock, 512), us(kSquare, 256), us(kFlat, 256), us(kSmall, 256)};
  switch (std::min_element(times, times + 5) - times) {
    case 0: return f(On<Large>{});
    case 1: return f(On<Block>{});
    case 2: return f(On<Square>{});
    case 3: return f(On<Flat>{});
    default: return f(On<Small>{});
  }
}

// gemm_stream over slots: a wave takes half a microsecond for a block of k, and 256 CUs
// read 4.8 TB/s of B, once for four rows of an expert.
double stream_us(double passes, int N, int K, int cus) {
  const double parts = stream_parts(K), bytes = passes * N * (double)pitch(K);
  return 2.5 + std::max(0.5 * std::ceil(blocks(K) / parts), bytes / (4.8e6 * cus / 256));
}

// f(the kernel of a product over slots of N columns, or of H with N = F).  On<Large>
// stands for tiles of both 256 and 128 rows.  An expert's last tile is half full on
// average, and tiles of up to 128 rows and columns take a tenth longer than among dense
// ones, B coming from memory.
//
// Few slots have kernels that read B once for four rows, and add exact products.
// glu_rows up to four slots an expert: one code of H that the tiles' cut-off moves weighs
// most where few rows are added up, and its time is theirs or less but for few experts (H
// of 64 experts, 4096 x 1024, random choices: 95 us for 115 of the tile of 64 rows at one
// slot an expert on average, 111 for 130 at two, 133 for 148 at four; 8 experts, 2048 x
// 1024: 18 for 20 at two, 28 for 20 at four).  gemm_stream where few matrices are read
// along a long k (8 experts, 4096 -> 4096: 5.4 us for 11.7 of one slot, 12.2 for 12.7 of
// four, 24 for 16 of eight; 64 experts, 1024 -> 4096: 7 for 6.4 of eight, 35 for 27 of
// 64), so that its time is estimated too.
template <bool GLU, class F>
int with_slots(const Slots& s, int N, int K, int cus, F&& f) {
  const double n = (double)s.tokens * s.top_k, used = std::min<double>(s.experts, n);
  const long few = GLU ? N / 128 * 512l : (N + 15l) / 16 * 256l;  // threads of a block of slots
  const bool can = n <= 4.0 * s.experts && most_slot_tiles(s, 128) * few < kThreads;
  if constexpr (GLU) {
    if (can) return f(GluRows{});
  }
  auto us = [&](const TileTime& t, int cols, int threads) {
    const double tiles_n = (double)((N + cols - 1l) / cols);
    const double us = tile_us(t, std::max(used, n / t.bm + used / 2) * tiles_n, threads, (long)blocks(K), cus);
    return most_slot_tiles(s, t.bm) * tiles_n * threads >= (double)kThreads ? 1e300 : t.bn <= 128 ? 1.1 * us : us;
  };
  if constexpr (GLU) {
    const double times[] = {us(kLarge, 128, 512), us(kBlock, 128, 512), us(kGlu, 128, 256)};
    switch (std::min_element(times, times + 3) - times) {
      case 1: return f(On<Block>{});
      case 2: return f(On<Glu>{});
      default: return f(On<Large>{});
    }
  } else {
    const double times[] = {us(kLarge, 256, 512), us(kSquare, 128, 256), us(kSmall, 64, 256),
                            can ? stream_us(used + (n - used) / 4, N, K, cus) : 1e300};
    switch (std::min_element(times, times + 4) - times) {
      case 1: return f(On<Square>{});
      case 2: return f(On<Small>{});
      case 3: return f(Stream{});
      default: return f(On<Large>{});
    }
  }
}

template <Out OUT, int BBLOCK>
struct RunDense {
  miaie_ctx* ctx;
  const Args& p;
  int operator()(Stream) const {
    if constexpr (BBLOCK == 128) return run_stream<DENSE, OUT>(ctx, p);
    return MIAIE_EUNSUPPORTED;  // (not chosen)
  }
  template <class T>
  int operator()(On<T>) const { return run_tile<T, DENSE, OUT, BBLOCK>(ctx, p); }
};

template <Out OUT>
struct RunSlots {
  miaie_ctx* ctx;
  const Args& p;
  int operator()(Stream) const { return run_stream<SLOTS, OUT>(ctx, p); }
  int operator()(GluRows) const { return run_glu_rows(ctx, p); }
  int operator()(On<Large>) const { return run_slots_large<OUT>(ctx, p); }
  template <class T>
  int operator()(On<T>) const { return run_tile<T, SLOTS, OUT, 128>(ctx, p); }
};

// What a plan says of a kernel; `rows` and `cols` tell the workgroups of a tile.
template <class Rows>
struct Plan {
  Rows rows;  // tiles of so many rows
  int N, K;
  bool glu;
  miaie_gemm_plan* to;
  int fill(int kernel, int tile_m, int tile_n, int threads) const {
    *to = {kernel, tile_m, tile_n, (int)(rows(tile_m) * ((N + (long)tile_n - 1) / tile_n)), threads};
    return MIAIE_OK;
  }
  int operator()(Stream) const {
    *to = {MIAIE_KERNEL_ROWS, 4, 16 * (4 / stream_parts(K)), 0, 256};
    to->workgroups = (int)(rows(128) * ((N + to->tile_n - 1l) / to->tile_n));
    return MIAIE_OK;
  }
  int operator()(GluRows) const {
    *to = {MIAIE_KERNEL_ROWS, kGluRows, 128, (int)(rows(128) * (N / 128)), 512};
    return MIAIE_OK;
  }
  template <class T>
  int operator()(On<T>) const { return fill(MIAIE_KERNEL_PIPE, T::BM, glu ? T::BN / 2 : T::BN, T::THREADS); }
};

template <Out OUT, int BBLOCK>
int run_dense(miaie_ctx* ctx, const Args& p) {
  return with_dense(p.M, p.N, p.K, BBLOCK, ctx->cus, RunDense<OUT, BBLOCK>{ctx, p});
}

template <Out OUT>
int run_slots(miaie_ctx* ctx, const Args& p) {
  return with_slots<OUT == OUT_GLU>(p.s, p.N, p.K, ctx->cus, RunSlots<OUT>{ctx, p});
}

template <Out OUT>
int run_wgrad(miaie_ctx* ctx, const Args& p) { return run_tile<Large, WGRAD, OUT, 1>(ctx, p); }

}  // namespace

int launch_gemm_fp8(miaie_ctx* ctx, const uint8_t* Aq, const float* As, const uint8_t* Bq, const float* Bs, int b_block,
                    void* C, int dtype, int M, int N, int K, int ldc) {
  const Args p{Aq, As, Bq, Bs, C, nullptr, nullptr, M, N, K, ldc, M, 0, Slots{}};
  if (b_block == 1) return dtype == MIAIE_BF16 ? run_dense<OUT_BF16, 1>(ctx, p) : run_dense<OUT_F32, 1>(ctx, p);
  return dtype == MIAIE_BF16 ? run_dense<OUT_BF16, 128>(ctx, p) : run_dense<OUT_F32, 128>(ctx, p);
}

int launch_experts_gemm_fp8(miaie_ctx* ctx, const fp8::Slots& s, const uint8_t* Aq, const float* As, int gather,
                            const uint8_t* Bq, const float* Bs, void* C, int dtype, int N, int K, int ldc) {
  const Args p{Aq, As, Bq, Bs, C, nullptr, nullptr, s.rows, N, K, ldc, gather ? s.tokens : s.rows, gather, s};
  return dtype == MIAIE_BF16 ? run_slots<OUT_BF16>(ctx, p) : run_slots<OUT_F32>(ctx, p);
}

int launch_experts_glu_fp8(miaie_ctx* ctx, const fp8::Slots& s, const uint8_t* Xq, const float* Xs, const uint8_t* W1q,
                           const float* W1s, uint8_t* Hq, float* Hs, int D, int F) {
  const Args p{Xq, Xs, W1q, W1s, nullptr, Hq, Hs, s.rows, F, D, 0, s.tokens, 1, s};
  return run_slots<OUT_GLU>(ctx, p);
}

int launch_experts_wgrad_fp8(miaie_ctx* ctx, const fp8::Slots& s, const uint8_t* Atq, const float* Ats, const uint8_t* Btq,
                             const float* Bts, void* C, int dtype, int M, int N, int ldc) {
  const Args p{Atq, Ats, Btq, Bts, C, nullptr, nullptr, M, N, s.rows, ldc, M, 0, s};
  return dtype == MIAIE_BF16 ? run_wgrad<OUT_BF16>(ctx, p) : run_wgrad<OUT_F32>(ctx, p);
}

int plan_gemm_fp8(int M, int N, int K, int b_block, int cus, miaie_gemm_plan* to) {
  auto rows = [=](int tile) { return tile == 128 && M <= 4 && b_block == 128 ? 1l : (M + tile - 1l) / tile; };
  return with_dense(M, N, K, b_block, cus, Plan<decltype(rows)>{rows, N, K, false, to});
}

int plan_experts_fp8(const fp8::Slots& s, int N, int K, int swiglu, int cus, miaie_gemm_plan* to) {
  auto rows = [=](int tile) { return most_slot_tiles(s, tile); };
  if (swiglu) return with_slots<true>(s, N, K, cus, Plan<decltype(rows)>{rows, N, K, true, to});
  return with_slots<false>(s, N, K, cus, Plan<decltype(rows)>{rows, N, K, false, to});
}

}  // namespace miaie
