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
#include <algorithm>
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

// Exchanges between the four lanes fg = 0..3 that hold a row (16 lanes apart).
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {  // a of lanes 32.. with b of lanes 0..31
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {  // a of odd sixteens with b of even ones
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  uint32_t w = v;
  swap32(v, w);
  w = v = max(v, w);
  swap16(v, w);
  return max(v, w);
}

// Packs NB blocks (columns 32 nb ..) of row m, of which this lane holds in
// acc[2 k] and acc[2 k + 1] columns 4 fg + e and 16 + 4 fg + e of block k.  Columns
// from N on become zeros (WHOLE: there are none).  Lane fg writes block fg whole:
// the lanes' four codes of each half are exchanged as a 4 x 4 transpose.
// Maxima that keep NaN: a block with one becomes NaN, through a ReLU too.
template <int NB, bool RELU, bool WHOLE>
__device__ __forceinline__ void store_blocks(const Args& p, int m, int nb, int fg, const v4f* acc) {
  uint32_t q[4] = {0, 0, 0, 0}, s[4] = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    float x[8], amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = acc[2 * k + (e >> 2)][e & 3];
      if (RELU) x[e] = __builtin_elementwise_maximum(x[e], 0.f);
      if (!WHOLE) x[e] = 32 * (nb + k) + (e >> 2) * 16 + 4 * fg + (e & 3) < p.N ? x[e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      amax = __builtin_elementwise_maximum(__builtin_elementwise_maximum(amax, fabsf(x[e])), fabsf(x[e + 1]));
    s[k] = scale_of(row_max(__float_as_uint(amax)));
    q[k] = pack8(x, scale_f32(s[k]));
  }
  swap32(q[0], q[2]);
  swap32(q[1], q[3]);
  swap16(q[0], q[1]);
  swap16(q[2], q[3]);
  nb += fg;
  const size_t pitch = q_pitch(p.N);
  if (m >= p.M || fg >= NB) return;
  if (16 * (size_t)nb < pitch) {
    const uint4 v = make_uint4(__builtin_amdgcn_perm(q[1], q[0], 0x05040100u), __builtin_amdgcn_perm(q[3], q[2], 0x05040100u),
                               __builtin_amdgcn_perm(q[1], q[0], 0x07060302u), __builtin_amdgcn_perm(q[3], q[2], 0x07060302u));
    MIAIE_ST(reinterpret_cast<uint4*>(p.Yq + m * pitch + 16 * (size_t)nb), v);
  }
  const uint32_t sc = fg == 0 ? s[0] : fg == 1 ? s[1] : fg == 2 ? s[2] : s[3];
  MIAIE_ST(p.Ys + ((size_t)(nb >> 4) * p.M + m) * 16 + s_byte(nb), (uint8_t)sc);
}

// ---------------------------------------------------------------- few rows
// A workgroup of up to 16 waves owns 16 MI rows and 16 NJ columns; its waves
// share out the groups of 512 columns of k and add their sums in LDS, so a
// product of few rows has thousands of groups in flight at once.  Bound by
// reading B, every byte of it once (1 x 11008 x 4096: 6.1 us, 3.9 TB/s, of which
// about 1.5 are the launch and the first bytes).
//
// A wave copies its group's 256 bytes of 16 NJ rows of B and of A's rows into a
// part of LDS of its own (no barriers: it waits for its own copies) and reads
// the fragments from there.  Loaded straight into registers a fragment load
// takes 64 bytes of each of 16 rows, half of a line, and a wave's 4 KB of B took
// 2.7 us with everything in the L2 (1 x 11008 x 4096); a copy takes whole rows.
// In LDS chunk c (16 bytes) of row r lies at c ^ (r % 16), so the 16 rows of a
// fragment read cover all banks.  A has 4 AI rows there; fragment rows behind
// them repeat the last.
template <int MI, int NJ, int AI>
struct RowsGeom {
  static constexpr int B = 0, A = 4096 * NJ, SB = A + 1024 * AI, SA = SB + 256 * NJ;
  static constexpr int GROUP = SA + 256 * MI;              // bytes of a group
  static constexpr int OPS = 4 * NJ + AI + NJ + MI;        // copies of a group
  static constexpr int SUM = MI * NJ * 1024;               // bytes of a wave's sums
  static constexpr int REGION = std::max(GROUP, SUM);
  static constexpr int WAVES = std::min(16, 163840 / REGION);  // at most
  static_assert(AI <= 4 * MI, "rows of A");
};

template <int MI, int NJ, int AI, Out OUT>
__global__ __launch_bounds__((64 * RowsGeom<MI, NJ, AI>::WAVES)) void gemm_mx_rows(Args p, int tiles_n, int waves) {
  using G = RowsGeom<MI, NJ, AI>;
  constexpr int REGION = G::REGION;
  extern __shared__ __attribute__((aligned(1024))) int8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int m0 = 16 * MI * (blockIdx.x / tiles_n), n0 = 16 * NJ * (blockIdx.x % tiles_n);
  const uint32_t pitch = (uint32_t)q_pitch(p.K);
  const int groups = s_groups(p.K);
  const bool half = (pitch / 128) % 2;  // the last group has 256 columns
  v4f acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  int8_t* const mine = lds + wave * REGION;
  const uint32_t mine0 = dev::lds_addr(mine);
  const dbg::Span aq_span = dbg::span_of(p.Aq), bq_span = dbg::span_of(p.Bq), as_span = dbg::span_of(p.As),
                  bs_span = dbg::span_of(p.Bs);  // (debug build only)
  const uint8_t* const a_base = p.Aq + (size_t)m0 * pitch;
  const uint8_t* const b_base = p.Bq + (size_t)n0 * pitch;
  // copy x of an operand: rows 4 x .. 4 x + 3, 16 lanes each; rows behind the last
  // one repeat it.  A last group of 256 columns repeats its first half.
  const int a_last = p.M - 1 - m0, b_last = p.N - 1 - n0;
  auto copy = [&](int g) __attribute__((always_inline)) {
    const uint32_t mask = half && g == groups - 1 ? 7 : 15;
    auto rows = [&](const uint8_t* base, int x, int last, uint32_t st, const dbg::Span& span) __attribute__((always_inline)) {
      const int r = 4 * x + fg;
      const uint32_t off = (uint32_t)min(r, last) * pitch + 16 * ((fr ^ (r & 15)) & mask);
      dev::gload_lds16(base + 256 * (size_t)g, off, mine0 + st + 1024 * x, span);
    };
#pragma unroll
    for (int x = 0; x < 4 * NJ; ++x) rows(b_base, x, b_last, G::B, bq_span);
#pragma unroll
    for (int x = 0; x < AI; ++x) rows(a_base, x, a_last, G::A, aq_span);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      dev::gload_lds4(p.Bs + ((size_t)g * p.N + n0) * 16, 16 * (uint32_t)min(16 * j + fr, b_last) + 4 * fg,
                      mine0 + G::SB + 256 * j, bs_span);
#pragma unroll
    for (int i = 0; i < MI; ++i)
      dev::gload_lds4(p.As + ((size_t)g * p.M + m0) * 16, 16 * (uint32_t)min(16 * i + fr, a_last) + 4 * fg,
                      mine0 + G::SA + 256 * i, as_span);
  };
  auto multiply = [&](int g) __attribute__((always_inline)) {
    int sa[MI], sb[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) sb[j] = *reinterpret_cast<const int*>(mine + G::SB + 256 * j + 4 * lane);
#pragma unroll
    for (int i = 0; i < MI; ++i) sa[i] = *reinterpret_cast<const int*>(mine + G::SA + 256 * i + 4 * lane);
    auto step = [&](auto t_c) __attribute__((always_inline)) {
      constexpr int t = decltype(t_c)::value;
      v4i a[MI], b[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        b[j] = *reinterpret_cast<const v4i*>(mine + G::B + 4096 * j + 256 * fr + 16 * ((4 * t + fg) ^ fr));
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = min(16 * i + fr, 4 * AI - 1);
        a[i] = *reinterpret_cast<const v4i*>(mine + G::A + 256 * r + 16 * ((4 * t + fg) ^ (r & 15)));
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mfma<t>(b[j], a[i], acc[i][j], sb[j], sa[i]);
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    if (half && g == groups - 1) return;
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  };
  if (n0 < p.N) {
    // the next group is on its way once this one's fragments are in registers
    if (wave < groups) copy(wave);
    for (int g = wave; g < groups; g += waves) {
      dev::wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      multiply(g);
      if (g + waves < groups) {
        dev::waitcnt<63, 0>();
        asm volatile("" ::: "memory");
        copy(g + waves);
      }
    }
  }
  // each wave's sums; those of a unit of one or two column blocks are added up
  // by one wave, eight loads in flight
  if (waves > 1) {
#pragma unroll
    for (int f = 0; f < MI * NJ; ++f) *reinterpret_cast<v4f*>(mine + 1024 * f + 16 * lane) = acc[f / NJ][f % NJ];
    __syncthreads();
  }
  constexpr int UN = NJ == 1 ? 1 : 2, UNITS = MI * NJ / UN;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    if (u % waves != wave) continue;
    v4f sum[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j) sum[j] = acc[u * UN / NJ][u * UN % NJ + j];
    for (int w0 = 1; w0 < waves; w0 += 8) {
      v4f part[8][UN];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const int k = min(w0 + w, waves - 1), from = wave + k < waves ? wave + k : wave + k - waves;
#pragma unroll
        for (int j = 0; j < UN; ++j)
          part[w][j] = *reinterpret_cast<const v4f*>(lds + from * REGION + 1024 * (u * UN + j) + 16 * lane);
      }
#pragma unroll
      for (int w = 0; w < 8; ++w)
        if (w0 + w < waves)
#pragma unroll
          for (int j = 0; j < UN; ++j) sum[j] += part[w][j];
    }
    const int i = u * UN / NJ, j0 = u * UN % NJ, m = m0 + 16 * i + fr;
    if constexpr (OUT == OUT_F32 || OUT == OUT_BF16) {
      using T = std::conditional_t<OUT == OUT_F32, float, __bf16>;
#pragma unroll
      for (int j = 0; j < UN; ++j)
        store4(static_cast<T*>(p.C), p.ldc, m, n0 + 16 * (j0 + j) + 4 * fg, p.M, p.N, sum[j]);
    } else {
      store_blocks<1, OUT == OUT_MX_RELU, false>(p, m, (n0 + 16 * j0) / 32, fg, sum);
    }
  }
}

// ------------------------------------------------------------ large products
// A workgroup of 4 waves owns a BM x BN tile, each wave a quarter of
// NI x NJ blocks of 16 x 16; a k-tile is 128 columns, 64 bytes of a row of Q
// and one instruction per block.  Operands go global -> LDS
// (global_load_lds_dwordx4, no registers in between), four k-tiles ahead:
//   A in three stages of two k-tiles (a pair: whole 128-byte lines of a row, so
//     a copy moves 8 of them; per k-tile it would touch 16 lines by half);
//   B per k-tile, in a ring of seven half stages of BN / 2 columns: k-tile k's
//     half h in slot (2 k + h) % 7;
//   the scales of 512 columns (four k-tiles, a group) of all BM + BN rows in
//     one stage, from which each wave takes its 16 + 16 bytes a lane once a
//     group.
// Seven half stages rather than eight leave the 8 KB for the scales at 256 x
// 256 (160 KB in all).
//
// A k-tile t is multiplied in two phases: phase 1 (phi = 2 t) the blocks of
// the upper half of the wave's rows while the lower half's A fragments are read,
// a barrier, phase 2 (phi = 2 t + 1) the lower half while the next k-tile's
// fragments are read.  One set of fragment registers (64 at 256 x 256) then
// suffices beside the 256 accumulators.  Copies go out between the matrix
// instructions:
//   A pair p: halves at phi = 4 p - 8 and 4 p - 6 (after the barrier of k-tile
//     2 p - 5, the last of pair p - 3 in its stage);
//   B k-tile k: half 0 at phi = 2 k - 7 (after the barrier of k-tile k - 4,
//     whose half 1 had the slot), half 1 at phi = 2 k - 5 (after that of k - 3,
//     whose half 0 had it);
//   scales of group q + 1: phase 2 of k-tile 4 q (every wave has read those of
//     group q by its barrier), read from phase 2 of k-tile 4 q + 3 on.
// What the barrier of k-tile t has to make visible (k-tile t + 1) was sent by
// phi = 2 t - 3, so the copies of the three phases since may be in flight: at
// most VM of them (copies of scales in between only make the wait stricter).
// Phases before 0 are the prologue.
//
// Bound by the board's power: 8192^3 to fp32 in 271 us, 4.06 PFLOP/s (5.2 to 5.3 in
// the k-loop alone, the rest the four rounds' first loads and last stores), where
// the instruction alone reaches 7.1 on random operands.
template <int BM, int BN>
struct PipeGeom {
  static constexpr int WM = BM / 2, WN = BN / 2;        // rows and columns of a wave
  static constexpr int NI = WM / 16, NJ = WN / 16, HI = NI / 2;
  static constexpr int PH = HI * NJ;                    // instructions per phase
  static constexpr int A_PAIR = BM * 128, B_HALF = BN / 2 * 64;
  static constexpr int A_REGION = 3 * A_PAIR, B_REGION = 7 * B_HALF;
  static constexpr int S_REGION = (BM + BN) * 16;
  static constexpr int LDS = A_REGION + B_REGION + S_REGION;
  static constexpr int A_CP = A_PAIR / 4096 / 2;        // copies per thread of half a pair
  static constexpr int B_CP = B_HALF / 4096;            // ... of half a k-tile of B
  static constexpr int S_CP = (S_REGION + 4095) / 4096;
  static_assert(A_CP >= 1 && B_CP >= 1 && HI >= 1 && NI % 2 == 0, "tile too small for 4 waves");
  static_assert(LDS <= 163840, "LDS of a CU");
  // copies of A in phase 1 and of B in phase 2 of the k-tile d before the last
  static constexpr int a_copies(int d) { return d >= 4 ? A_CP : 0; }
  static constexpr int b_copies(int d) { return (d >= 4 ? B_CP : 0) + (d >= 3 ? B_CP : 0); }
  static constexpr int vm(int d) { return a_copies(d + 1) + b_copies(d + 1) + a_copies(d); }
};

// 16-byte chunk c of row r of a k-tile of B lies at c ^ b_swz(r), and of a
// pair of A at c ^ a_swz(r).  A ds_read_b128 serves 16 lanes at a time, which by
// the conflicts counted are not 16 rows at one chunk but eight rows each at two
// (0-3 and 12-15 at the one, 4-11 at the next, and the other way round); both
// forms cover all 64 banks (8192^3: conflicts in 10% of the LDS's cycles, 36%
// with B at c ^ (r >> 2), the time under the power limit the same).
__device__ __forceinline__ int a_swz(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int b_swz(int r) { return -(r >> 2) & 3; }

// acc += B fragment x A fragment, scales in byte T, in place.  (The compiler's
// form of the instruction writes other registers than it adds to and moves
// accumulators around: 30 cycles an instruction in a loop of 16 of them,
// against 17.)  No instruction but a load writes an operand within two
// instructions before its use (tests/test_mx_asm.py, tests/test_block_asm.py).
template <int T>
__device__ __forceinline__ void mfma_in_place(v4f& acc, v4i b, v4i a, int sb, int sa) {
#if MIAIE_DEVICE_CHECKS
  acc = mfma<T>(b, a, acc, sb, sa);
#else
  if constexpr (T == 0)
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else if constexpr (T == 1)
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else if constexpr (T == 2)
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0] cbsz:4 blgp:4" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa));
  else
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0] cbsz:4 blgp:4" : "+a"(acc) : "v"(b), "v"(a), "v"(sb), "v"(sa));
#endif
}

// The values are computed before this point (the compiler does not know that
// they have to be some instructions before an MFMA written in assembly, and
// would move a shift or select next to it).
template <int N>
__device__ __forceinline__ void pin(int (&v)[N]) {
  static_assert(N == 4 || N == 8, "registers of a wave's scales");
  if constexpr (N == 4)
    asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
  else
    asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]));
}

// The accumulators stay where they are up to this point (the compiler would
// read all 256 of them at once, and spill).
template <int NJ>
__device__ __forceinline__ void hold(v4f (&acc)[NJ]) {
  static_assert(NJ % 4 == 0, "four at a time");
#pragma unroll
  for (int j = 0; j < NJ; j += 4)
    asm volatile("" : "+a"(acc[j]), "+a"(acc[j + 1]), "+a"(acc[j + 2]), "+a"(acc[j + 3]));
}

// A wave's quarter at row m0 and column n0 of C.  In bf16 two blocks beside each other are exchanged between lanes fg and fg + 1 of
// a row, so that each holds eight columns of one block: 16 bytes a lane in either
// type, at any alignment.  EDGE: some columns of the product's last tiles are
// behind N.  A kernel of its own, for the branches between the stores: with them
// the lines of an fp32 C of 256 MB go to memory in parts, 30000 cycles a tile
// where 17000 do, and with both forms in one kernel the compiler spills
// accumulators.  Ordinary stores: 64 MB of fp32 tiles leave in 8.8 us, 14 us as
// non-temporal ones.
template <bool EDGE, class T, int NI, int NJ>
__device__ __forceinline__ void store_quarter(T* C, size_t ldc, int m0, int n0, int fr, int fg, int M, int N,
                                              v4f (&acc)[NI][NJ]) {
  constexpr int W = 16 / sizeof(T), NB = W / 4;  // columns of a lane, blocks exchanged
  typedef T V __attribute__((ext_vector_type(W)));
  using P = At<V, T>;
  const dbg::Span span = dbg::span_of(C);  // (debug build only)
  int m = m0 + fr;
  const int n = n0 + (NB == 1 ? 4 * fg : 16 * (fg & 1) + 8 * (fg >> 1));
  T* row = C + (size_t)m * ldc + n;
#pragma unroll
  for (int i = 0; i < NI; ++i, m += 16, row += 16 * ldc) {
    if (m < M) {
#pragma unroll
      for (int j = 0; j < NJ; j += NB) {
        V v;
        if constexpr (NB == 1) {
          v = acc[i][j];
        } else {
          typedef uint32_t v2u __attribute__((ext_vector_type(2)));
          typedef uint32_t v4u __attribute__((ext_vector_type(4)));
          const v2u a = __builtin_bit_cast(v2u, __builtin_convertvector(acc[i][j], v4bf));
          const v2u b = __builtin_bit_cast(v2u, __builtin_convertvector(acc[i][j + 1], v4bf));
          uint32_t a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];
          swap16(a0, b0);  // (the four lanes of a row are all here)
          swap16(a1, b1);
          v = __builtin_bit_cast(V, v4u{a0, a1, b0, b1});
        }
        if (!EDGE || n + 16 * j + W <= N) {
          MIAIE_ST_IN(span, reinterpret_cast<P*>(row + 16 * j), P{v});
        } else {
#pragma unroll
          for (int e = 0; e < W - 1; ++e)
            if (n + 16 * j + e < N) MIAIE_ST_IN(span, row + 16 * j + e, v[e]);
        }
      }
    }
    dev::sched_fence();  // (more rows at once spill)
  }
}

// The tile at row m0 and column n0; last: no tile of its rows is behind it.
template <int BM, int BN, Out OUT, bool EDGE>
__device__ __forceinline__ void pipe_tile(const Args& p, int8_t* lds, int m0, int n0, bool last) {
  using G = PipeGeom<BM, BN>;
  constexpr int NI = G::NI, NJ = G::NJ, HI = G::HI, PH = G::PH;
  constexpr int B0 = G::A_REGION, S0 = G::A_REGION + G::B_REGION;
  const uint32_t lds0 = dev::lds_addr(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, fr = lane & 15, fg = lane >> 4;
  const uint32_t pitch = (uint32_t)q_pitch(p.K);
  const int KT = (int)(pitch / 64);  // even

  // ---- copies: wave-uniform source plus a per-lane offset; rows behind the
  // last one are copies of it, and dropped at the end
  uint32_t a_off[2 * G::A_CP], b_off[2 * G::B_CP], s_off[G::S_CP];
#pragma unroll
  for (int x = 0; x < 2 * G::A_CP; ++x) {
    const int r = 8 * (4 * x + wave) + (lane >> 3);
    a_off[x] = (uint32_t)min(r, p.M - 1 - m0) * pitch + 16 * ((lane & 7) ^ a_swz(r));
  }
#pragma unroll
  for (int x = 0; x < 2 * G::B_CP; ++x) {
    const int r = 16 * (4 * x + wave) + (lane >> 2);
    b_off[x] = (uint32_t)min(r, p.N - 1 - n0) * pitch + 16 * ((lane & 3) ^ b_swz(r));
  }
#pragma unroll
  for (int x = 0; x < G::S_CP; ++x) {
    const int r = 64 * (4 * x + wave);  // of A's rows, then B's
    s_off[x] = 16 * (uint32_t)(r < BM ? min(r + lane, p.M - 1 - m0) : min(r - BM + lane, p.N - 1 - n0));
  }
  const uint8_t* const a_base = p.Aq + (size_t)m0 * pitch;
  const uint8_t* const b_base = p.Bq + (size_t)n0 * pitch;
  const dbg::Span aq_span = dbg::span_of(p.Aq), bq_span = dbg::span_of(p.Bq), as_span = dbg::span_of(p.As),
                  bs_span = dbg::span_of(p.Bs);  // (debug build only)
  const uint32_t ldsw = lds0 + 1024 * wave;
  auto copy_a = [&](const uint8_t* src, uint32_t st, int x) __attribute__((always_inline)) {
    dev::gload_lds16(src, a_off[x], ldsw + st + 4096 * x, aq_span);
  };
  // (copy x of half h of a k-tile of B, into the slot at byte st)
  auto copy_b = [&](const uint8_t* src, uint32_t st, int h, int x) __attribute__((always_inline)) {
    dev::gload_lds16(src, b_off[h * G::B_CP + x], ldsw + B0 + st + 4096 * x, bq_span);
  };
  auto copy_s = [&](int q) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < G::S_CP; ++x) {
      const int r = 64 * (4 * x + wave);
      if (r < BM)
        dev::gload_lds16(p.As + ((size_t)q * p.M + m0) * 16, s_off[x], ldsw + S0 + 4096 * x, as_span);
      else if (r < BM + BN)
        dev::gload_lds16(p.Bs + ((size_t)q * p.N + n0) * 16, s_off[x], ldsw + S0 + 4096 * x, bs_span);
    }
  };

  // ---- fragments
  int a_fo[2];
#pragma unroll
  for (int par = 0; par < 2; ++par) a_fo[par] = (wm * G::WM + fr) * 128 + (((4 * par + fg) ^ a_swz(fr)) << 4);
  const int b_fo = B0 + fr * 64 + ((fg ^ b_swz(fr)) << 4);  // (a wave's columns are one half)
  const int sa_fo = S0 + (wm * G::WM + fr) * 16 + 4 * fg, sb_fo = S0 + (BM + wn * G::WN + fr) * 16 + 4 * fg;
  v4i alo[HI], ahi[HI], bs[NJ];
  int sa[NI], sb[NJ];
  auto read_a = [&](uint32_t st, int par, int i) __attribute__((always_inline)) -> v4i {
    // (readfirstlane keeps the stage's address in the base register, so that
    // 2048 i is the instruction's offset)
    return *reinterpret_cast<const v4i*>(lds + __builtin_amdgcn_readfirstlane(st) + a_fo[par] + 2048 * i);
  };
  auto read_b = [&](uint32_t st, int j) __attribute__((always_inline)) {
    bs[j] = *reinterpret_cast<const v4i*>(lds + __builtin_amdgcn_readfirstlane(st) + b_fo + 1024 * j);
  };
  auto read_sa = [&](int i) __attribute__((always_inline)) { sa[i] = *reinterpret_cast<const int*>(lds + sa_fo + 256 * i); };
  auto read_sb = [&](int j) __attribute__((always_inline)) { sb[j] = *reinterpret_cast<const int*>(lds + sb_fo + 256 * j); };

  v4f acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

  // ---- prologue: group 0's scales, then the copies of phases -8 .. -1
  copy_s(0);
#pragma unroll
  for (int phi = -8; phi < 0; ++phi) {
    if ((phi & 1) == 0) {
      const int pr = (phi + 8) / 4, h = ((phi + 8) / 2) & 1;  // pair, half of it
      if (2 * pr < KT)
#pragma unroll
        for (int x = 0; x < G::A_CP; ++x) copy_a(a_base + 128 * pr, G::A_PAIR * pr, G::A_CP * h + x);
    } else {
      const int k0 = (phi + 7) / 2, k1 = (phi + 5) / 2;
      if (k1 >= 0 && k1 < KT)
#pragma unroll
        for (int x = 0; x < G::B_CP; ++x) copy_b(b_base + 64 * k1, (2 * k1 + 1) % 7 * G::B_HALF, 1, x);
      if (k0 < KT)
#pragma unroll
        for (int x = 0; x < G::B_CP; ++x) copy_b(b_base + 64 * k0, 2 * k0 % 7 * G::B_HALF, 0, x);
    }
  }
  if (KT >= 4)
    dev::wait_vmcnt<2 * G::A_CP + 4 * G::B_CP>();  // phases -4 .. -1
  else
    dev::wait_vmcnt<0>();
  dev::barrier();
#pragma unroll
  for (int i = 0; i < NI; ++i) read_sa(i);
#pragma unroll
  for (int j = 0; j < NJ; ++j) read_sb(j);
#pragma unroll
  for (int j = 0; j < NJ; ++j) read_b(wn * G::B_HALF, j);
#pragma unroll
  for (int i = 0; i < HI; ++i) alo[i] = read_a(0, 0, i);

  // ---- state of k-tile t of pair P (wave-uniform)
  uint32_t st0 = 0, st1 = G::A_PAIR, st2 = 2 * G::A_PAIR;  // stages of pairs P, P + 1, P + 2
  const uint8_t* a_src = a_base + 2 * 128;                  // pair P + 2
  const uint8_t* b_src = b_base + 3 * 64;                   // k-tile t + 3
  uint32_t slot = 0;                                        // of k-tile t's half 0, in half stages
  auto slot_at = [&](uint32_t add) __attribute__((always_inline)) {
    const uint32_t s = slot + add;
    return (s >= 7 ? s - 7 : s) * (uint32_t)G::B_HALF;
  };
  int t = 0;

  constexpr int A_STEP = PH * 3 / (4 * HI);  // phase 1's reads of A, evenly over three quarters of it
  // k-tile t: D k-tiles before the last; PAR = t % 2 and, where it is known at
  // compile time, T4 = t % 4.  Each matrix instruction first, then, in its
  // shadow, what goes with it.
  auto tile = [&](auto par_c, auto t4_c, auto d_c) __attribute__((always_inline)) {
    constexpr int PAR = decltype(par_c)::value, T4 = decltype(t4_c)::value, D = decltype(d_c)::value;
    constexpr int BYTE = T4 >= 0 ? T4 : PAR;
    constexpr int NA = G::a_copies(D), NB = G::b_copies(D);
    constexpr bool NEXT = D >= 1;
    uint32_t b_next = 0, cp0 = 0, cp1 = 0;
#pragma unroll
    for (int x = 0; x < PH; ++x) {
      const int j = x / HI, i = dev::snake_j<HI>(x);
      mfma_in_place<BYTE>(acc[i][j], bs[j], alo[i], sb[j], sa[i]);
      dev::sched_fence();
      if (x % A_STEP == 1 && x / A_STEP < HI) ahi[x / A_STEP] = read_a(st0, PAR, HI + x / A_STEP);
#pragma unroll
      for (int c = 0; c < NA; ++c)
        if (2 + c * PH / (NA > 0 ? NA : 1) == x) copy_a(a_src, st2, G::A_CP * PAR + c);
      if (x == PH / 2 + 1) {
        // phase 2's slots: of k-tile t + 1, of (t + 4, half 0) and of (t + 3, half 1)
        b_next = slot_at(2 + wn), cp0 = slot_at(1), cp1 = slot_at(0);
        asm volatile("" : "+s"(b_next), "+s"(cp0), "+s"(cp1));
      }
      dev::sched_fence();
    }
    dev::waitcnt<G::vm(D), 0>();
    dev::barrier();
    const uint32_t st_next = PAR == 0 ? st0 : st1;
#pragma unroll
    for (int x = 0; x < PH; ++x) {
      const int j = x / HI, i = dev::snake_j<HI>(x);
      mfma_in_place<BYTE>(acc[HI + i][j], bs[j], ahi[i], sb[j], sa[HI + i]);
      dev::sched_fence();
#pragma unroll
      for (int c = 0; c < NB; ++c)
        if (2 + c * PH / (NB > 0 ? NB : 1) == x) {
          if (c < G::B_CP)
            copy_b(b_src, cp1, 1, c);
          else
            copy_b(b_src + 64, cp0, 0, c - G::B_CP);
        }
      if constexpr (T4 == 0 || (T4 < 0 && PAR == 0)) {
        if (x == PH - 1 && (t & 3) == 0 && t + 4 < KT) copy_s(t / 4 + 1);
      }
      if constexpr (NEXT) {
        if (x % HI == HI / 2 - 1 && x / HI < HI) alo[x / HI] = read_a(st_next, 1 - PAR, x / HI);
        // registers of k-tile t are read again after their last use
        if (x % HI == HI - 1) read_b(b_next, j);
        if constexpr (T4 == 3) {
          if (x < HI) read_sa(x);
          if (x % HI == HI - 1) read_sb(j);
          if (x >= PH - HI) read_sa(HI + i);
        }
      }
      dev::sched_fence();
    }
    ++t;
    b_src += 64;
    slot = slot + 2 >= 7 ? slot - 5 : slot + 2;
    if constexpr (PAR == 1) {
      const uint32_t s = st0;
      st0 = st1;
      st1 = st2;
      st2 = s;
      a_src += 128;
    }
  };
  // The scales of a pair whose place in its group is not known at compile time:
  // the group's, or the next two bytes of those.  Three wait states between
  // these instructions and the first that takes the registers.
  auto take_scales = [&]() __attribute__((always_inline)) {
    if (t & 2) {
#pragma unroll
      for (int i = 0; i < NI; ++i) sa[i] = (int)((uint32_t)sa[i] >> 16);
#pragma unroll
      for (int j = 0; j < NJ; ++j) sb[j] = (int)((uint32_t)sb[j] >> 16);
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) read_sa(i);
#pragma unroll
      for (int j = 0; j < NJ; ++j) read_sb(j);
    }
    pin(sa);
    pin(sb);
    asm volatile("s_nop 2" ::: "memory");
    dev::sched_fence();
  };
  using P0 = std::integral_constant<int, 0>;
  using P1 = std::integral_constant<int, 1>;
  using DS = std::integral_constant<int, 64>;  // steady state
  using TR = std::integral_constant<int, -1>;
  // steady k-tiles, then the last six.  (With branches of whole tails for 2, 4
  // and 6 left the register allocator moves the accumulators through memory.)
  while (t + 10 <= KT) {
    tile(P0{}, std::integral_constant<int, 0>{}, DS{});
    tile(P1{}, std::integral_constant<int, 1>{}, DS{});
    tile(P0{}, std::integral_constant<int, 2>{}, DS{});
    tile(P1{}, std::integral_constant<int, 3>{}, DS{});
  }
  while (t + 6 < KT) {
    take_scales();
    tile(P0{}, TR{}, DS{});
    tile(P1{}, TR{}, DS{});
  }
  if (KT >= 6) {
    take_scales();
    tile(P0{}, TR{}, std::integral_constant<int, 5>{});
    tile(P1{}, TR{}, std::integral_constant<int, 4>{});
  }
  if (KT >= 4) {
    take_scales();
    tile(P0{}, TR{}, std::integral_constant<int, 3>{});
    tile(P1{}, TR{}, std::integral_constant<int, 2>{});
  }
  take_scales();
  tile(P0{}, TR{}, std::integral_constant<int, 1>{});
  tile(P1{}, TR{}, std::integral_constant<int, 0>{});
  // the last results are readable after 18 wait states at most
  dev::sched_fence();
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
  for (int i = 0; i < NI; ++i) hold(acc[i]);  // (read behind the wait)
  dev::sched_fence();

  // ---- acc[i][j]: row 16 i + fr and columns 16 j + 4 fg + 0..3 of the wave's quarter
  const int mw = m0 + wm * G::WM, nw = n0 + wn * G::WN;
  if constexpr (OUT == OUT_F32 || OUT == OUT_BF16) {
    using T = std::conditional_t<OUT == OUT_F32, float, __bf16>;
    store_quarter<EDGE>(static_cast<T*>(p.C), p.ldc, mw, nw, fr, fg, p.M, p.N, acc);
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (n0 + BN <= p.N)
        store_blocks<NJ / 2, OUT == OUT_MX_RELU, true>(p, mw + 16 * i + fr, nw / 32, fg, acc[i]);
      else
        store_blocks<NJ / 2, OUT == OUT_MX_RELU, false>(p, mw + 16 * i + fr, nw / 32, fg, acc[i]);
      dev::sched_fence();  // (more rows at once spill)
    }
    if (last) {  // zeros up to the end of the last 512 columns
      const int first = (n0 + BN) / 32, blocks = 16 * s_groups(p.N) - first;
      const size_t y_pitch = q_pitch(p.N);
      const v4i zero = {0, 0, 0, 0};
      for (int x = tid; x < BM * blocks; x += 256) {
        const int m = m0 + x / blocks, nb = first + x % blocks;
        if (m >= p.M) continue;
        if (16 * (size_t)nb < y_pitch)
          MIAIE_ST(reinterpret_cast<v4i*>(p.Yq + m * y_pitch + 16 * (size_t)nb), zero);
        MIAIE_ST(p.Ys + ((size_t)(nb >> 4) * p.M + m) * 16 + s_byte(nb), (uint8_t)0);
      }
    }
  }
}

template <int BM, int BN, Out OUT, bool EDGE>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2) void gemm_mx_pipe(Args p, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[PipeGeom<BM, BN>::LDS];
  int tm, tn;
  dev::tile_coords<4>(blockIdx.x, tiles_m, tiles_n, tm, tn);
  pipe_tile<BM, BN, OUT, EDGE>(p, lds, tm * BM, tn * BN, tn == tiles_n - 1);
}

// 256 x 256 tiles over the first `wide` tile columns, then 256 x 128 tiles: the
// narrow ones fill the CUs that the last round of wide ones would leave idle
// (2048 x 11008 x 4096 packed: 344 wide tiles on 256 CUs, 60 us; 53 us as 256 wide
// and 176 narrow).
template <Out OUT, bool EDGE>
__global__ __launch_bounds__(256, 1) void gemm_mx_mixed(Args p, int tiles_m, int wide, int narrow) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[PipeGeom<256, 256>::LDS];
  int tm, tn;
  if ((int)blockIdx.x < tiles_m * wide) {
    dev::tile_coords<4>(blockIdx.x, tiles_m, wide, tm, tn);
    pipe_tile<256, 256, OUT, false>(p, lds, tm * 256, tn * 256, false);
  } else {
    dev::tile_coords<4>(blockIdx.x - tiles_m * wide, tiles_m, narrow, tm, tn);
    pipe_tile<256, 128, OUT, EDGE>(p, lds, tm * 256, wide * 256 + tn * 128, tn == narrow - 1);
  }
}

template <Out OUT>
int run_mixed(miaie_ctx* ctx, const Args& p, int wide) {
  const int tiles_m = (p.M + 255) / 256, narrow = (p.N - 256 * wide + 127) / 128;
  hipError_t e = hipSuccess;
  auto go = [&](auto k) {
    e = launch<decltype(k)::value>(ctx->device, dim3((unsigned)tiles_m * (wide + narrow)), dim3(256), 0, ctx->stream, p,
                                   tiles_m, wide, narrow);
  };
  if ((OUT == OUT_F32 || OUT == OUT_BF16) && p.N % 128)
    go(kernel_t<gemm_mx_mixed<OUT, OUT == OUT_F32 || OUT == OUT_BF16>>{});
  else
    go(kernel_t<gemm_mx_mixed<OUT, false>>{});
  return check_launch(ctx, e, "gemm_mx_mixed");
}

template <int BM, int BN, Out OUT>
int run_pipe(miaie_ctx* ctx, const Args& p) {
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  hipError_t e = hipSuccess;
  auto go = [&](auto k) {
    e = launch<decltype(k)::value>(ctx->device, dim3((unsigned)tiles_m * tiles_n), dim3(256), 0, ctx->stream, p, tiles_m,
                                   tiles_n);
  };
  if ((OUT == OUT_F32 || OUT == OUT_BF16) && p.N % BN)
    go(kernel_t<gemm_mx_pipe<BM, BN, OUT, OUT == OUT_F32 || OUT == OUT_BF16>>{});
  else
    go(kernel_t<gemm_mx_pipe<BM, BN, OUT, false>>{});
  return check_launch(ctx, e, "gemm_mx_pipe");
}

// Columns of a result that are written (a packed one has zeros up to the end of its last 512 columns).
constexpr long written_cols(Out out, int N) {
  return out == OUT_MX || out == OUT_MX_RELU ? 512l * s_groups(N) : N;
}

// Tiles and waves of a product on gemm_mx_rows: as many waves as share the groups
// of 512 columns evenly, up to 16 and to what fits the LDS.
struct RowsGrid {
  long tiles_n, tiles;
  int waves;
};
template <int MI, int NJ, int AI>
RowsGrid rows_grid(long M, long cols, int groups) {
  using G = RowsGeom<MI, NJ, AI>;
  const long tiles_n = (cols + 16 * NJ - 1) / (16 * NJ);
  const int each = (groups + G::WAVES - 1) / G::WAVES;
  return {tiles_n, (M + 16 * MI - 1) / (16 * MI) * tiles_n, (groups + each - 1) / each};
}

template <int MI, int NJ, int AI, Out OUT>
int run_rows(miaie_ctx* ctx, const Args& p) {
  const RowsGrid g = rows_grid<MI, NJ, AI>(p.M, written_cols(OUT, p.N), s_groups(p.K));
  const hipError_t e = launch<gemm_mx_rows<MI, NJ, AI, OUT>>(ctx->device, dim3((unsigned)g.tiles), dim3(64 * g.waves),
                                                                    (size_t)g.waves * RowsGeom<MI, NJ, AI>::REGION, ctx->stream,
                                                                    p, (int)g.tiles_n, g.waves);
  return check_launch(ctx, e, "gemm_mx_rows");
}

// ------------------------------------------------------------ choice of kernel
// The kernel with the lowest estimated time.  Few rows: a CU copies about 42
// bytes a ns into LDS with its waves' groups in flight, so the workgroups of one
// CU take that time for all their groups.  Large products: cycles of a workgroup's
// start, of a k-tile and of its end as measured on the tiles (a k-tile of 256 x 256
// has 64 instructions of 16 cycles on each wave), the clock 2.3 GHz with a part of
// the CUs at work and about 1.9 under the power limit.  128 x 128 tiles fit a CU
// twice, and then take 960 cycles for both where one takes 540.  (A packed result
// takes no single column block, whose two neighbours a lane needs, and no 64 x 32
// tiles, which its 512 columns at least never make the quickest.)
// The estimates are for the choice, not for the time: against the chosen kernels at
// 1 to 2048 rows of 4096 x 4096, 11008 x 4096 and 4096 x 11008 (bf16 out) they are
// 31% low to 10% high below 48 rows, 19% low to 55% high at 48 to 256 (row kernels at
// K = 11008 are the ones estimated high) and 18% low to 14% high above.  Of those
// three sizes at 48, 64, 96, 128, 192, 256, 384 and 512 rows, with the row kernels of 16 x 32
// to 64 x 64 results and the 128 x 128 and 256 x 128 tiles each timed, the chosen
// one is the quickest in 23 and 4% behind in one.
struct Choice {
  double us = 1e30;
  int kernel = -1;  // none: no kernel takes a product of that size in one launch
  int wide = 0;     // tile columns of 256 (mixed tiles)
};
void consider(Choice& best, int kernel, double us) {
  if (us < best.us) best = Choice{us, kernel, 0};
}
constexpr double kNever = 1e300;

template <int MI, int NJ, int AI>
double rows_us(long M, long cols, int groups, int cus) {
  using G = RowsGeom<MI, NJ, AI>;
  const RowsGrid g = rows_grid<MI, NJ, AI>(M, cols, groups);
  if (g.tiles * g.waves >= 1l << 26) return kNever;  // (HIP takes fewer than 2^32 threads)
  return 1.2 + 0.02 * G::OPS + (double)((g.tiles + cus - 1) / cus) * groups * G::GROUP / 42e3;
}

// Cycles of a workgroup on a tile: its start, a k-tile, its end (fp32, bf16, packed).
struct TileCycles {
  int bm;
  double start, k_tile, end[3];
};
constexpr TileCycles kTiles[] = {{256, 4500, 1320, {16500, 7800, 9900}}, {256, 3400, 840, {8200, 3800, 5800}},
                                 {128, 2400, 540, {3500, 1850, 3400}}};

double pipe_us(long tiles, int k_tiles, const TileCycles& t, double end, int cus) {
  const long rounds = (tiles + cus - 1) / cus;
  const double ghz = 2 * tiles < cus ? 2.35e3 : 1.9e3;
  if (t.bm == 128 && rounds > 1) return 1.0 + (double)((rounds + 1) / 2) * (1600 + t.start + end + 960.0 * k_tiles) / ghz;
  return 1.0 + (double)rounds * (t.start + end + t.k_tile * k_tiles) / ghz;
}

template <Out OUT>
Choice choose(int M, int N, int K, int cus) {
  constexpr bool packed = OUT == OUT_MX || OUT == OUT_MX_RELU;
  const int groups = s_groups(K), k_tiles = (int)(q_pitch(K) / 64);
  const long cols = written_cols(OUT, N);
  Choice c;
  if (M <= 4) {
    consider(c, 0, rows_us<1, 1 + packed, 1>(M, cols, groups, cus));
  } else if (M <= 8) {
    if (!packed) consider(c, 1, rows_us<1, 1, 2>(M, cols, groups, cus));
    consider(c, 2, rows_us<1, 2, 2>(M, cols, groups, cus));
    consider(c, 3, rows_us<1, 4, 2>(M, cols, groups, cus));
  } else {
    if (!packed) consider(c, 4, rows_us<1, 1, 4>(M, cols, groups, cus));
    consider(c, 5, rows_us<1, 2, 4>(M, cols, groups, cus));
    consider(c, 6, rows_us<1, 4, 4>(M, cols, groups, cus));
  }
  if (M > 16) {
    if (!packed) consider(c, 7, rows_us<2, 1, 8>(M, cols, groups, cus));
    consider(c, 8, rows_us<2, 2, 8>(M, cols, groups, cus));
    consider(c, 9, rows_us<2, 4, 8>(M, cols, groups, cus));
  }
  if (M > 32) {
    if (!packed) consider(c, 10, rows_us<4, 2, 16>(M, cols, groups, cus));
    consider(c, 11, rows_us<4, 4, 16>(M, cols, groups, cus));
  }
  // (a row's offset within a tile in 32 bits, and HIP takes fewer than 2^32 threads)
  if (q_pitch(K) < (1u << 24)) {
    constexpr int o = packed ? 2 : OUT == OUT_BF16;
    constexpr long most = 1l << 24;  // workgroups
    const long tiles_m = (M + 255l) / 256, wide = (N + 255l) / 256;
    const long square = ((M + 127l) / 128) * ((N + 127l) / 128), tall = tiles_m * ((N + 127l) / 128);
    if (square < most) consider(c, 12, pipe_us(square, k_tiles, kTiles[2], kTiles[2].end[o], cus));
    if (tall < most) consider(c, 13, pipe_us(tall, k_tiles, kTiles[1], kTiles[1].end[o], cus));
    if (tiles_m * wide < most) consider(c, 14, pipe_us(tiles_m * wide, k_tiles, kTiles[0], kTiles[0].end[o], cus));
    // whole rounds of wide tiles, then narrow ones
    if (tall < most && tiles_m * wide > cus && tiles_m <= cus && tiles_m * wide < 8l * cus) {
      const long first = tiles_m * wide / cus * cus / tiles_m;  // wide tile columns
      const long narrow = tiles_m * ((N - 256 * first + 127) / 128);
      if (first > 0 && narrow > 0) {
        const double us = pipe_us(tiles_m * first, k_tiles, kTiles[0], kTiles[0].end[o], cus) - 1.0 +
                          pipe_us(narrow, k_tiles, kTiles[1], kTiles[1].end[o], cus);
        if (us < c.us) c = Choice{us, 15, (int)first};
      }
    }
  }
  return c;
}

// A kernel of the choice as a type.
template <int MI, int NJ, int AI>
struct Rows {};
template <int BM, int BN>
struct Pipe {};
struct Mixed {
  int wide;
};

template <Out OUT, class F>
int with_kernel(const Choice& c, F&& go) {
  constexpr bool packed = OUT == OUT_MX || OUT == OUT_MX_RELU;
  switch (c.kernel) {
    case 0: return go(Rows<1, 1 + packed, 1>{});
    case 1: return go(Rows<1, 1 + packed, 2>{});
    case 2: return go(Rows<1, 2, 2>{});
    case 3: return go(Rows<1, 4, 2>{});
    case 4: return go(Rows<1, 1 + packed, 4>{});
    case 5: return go(Rows<1, 2, 4>{});
    case 6: return go(Rows<1, 4, 4>{});
    case 7: return go(Rows<2, 1 + packed, 8>{});
    case 8: return go(Rows<2, 2, 8>{});
    case 9: return go(Rows<2, 4, 8>{});
    case 10: return go(Rows<4, packed ? 4 : 2, 16>{});
    case 11: return go(Rows<4, 4, 16>{});
    case 12: return go(Pipe<128, 128>{});
    case 13: return go(Pipe<256, 128>{});
    case 14: return go(Pipe<256, 256>{});
    default: return go(Mixed{c.wide});
  }
}

template <Out OUT>
struct Runner {
  miaie_ctx* ctx;
  const Args& p;
  template <int MI, int NJ, int AI>
  int operator()(Rows<MI, NJ, AI>) const { return run_rows<MI, NJ, AI, OUT>(ctx, p); }
  template <int BM, int BN>
  int operator()(Pipe<BM, BN>) const { return run_pipe<BM, BN, OUT>(ctx, p); }
  int operator()(Mixed m) const { return run_mixed<OUT>(ctx, p, m.wide); }
};

template <Out OUT>
struct Planner {
  int M, N, K;
  miaie_gemm_plan* plan;
  template <int MI, int NJ, int AI>
  int operator()(Rows<MI, NJ, AI>) const {
    const RowsGrid g = rows_grid<MI, NJ, AI>(M, written_cols(OUT, N), s_groups(K));
    *plan = {MIAIE_KERNEL_ROWS, 16 * MI, 16 * NJ, (int)g.tiles, 64 * g.waves};
    return MIAIE_OK;
  }
  template <int BM, int BN>
  int operator()(Pipe<BM, BN>) const {
    *plan = {MIAIE_KERNEL_PIPE, BM, BN, (M + BM - 1) / BM * ((N + BN - 1) / BN), 256};
    return MIAIE_OK;
  }
  int operator()(Mixed m) const {
    *plan = {MIAIE_KERNEL_PIPE_MIXED, 256, 256, (M + 255) / 256 * (m.wide + (N - 256 * m.wide + 127) / 128), 256};
    return MIAIE_OK;
  }
};

int too_large(miaie_ctx* ctx, int M, int N, int K) {
  return fail(ctx, MIAIE_EINVAL, "gemm_mxfp4: a product of M=%d N=%d K=%d is too large for one launch", M, N, K);
}

template <Out OUT>
int run(miaie_ctx* ctx, const Args& p) {
  const Choice c = choose<OUT>(p.M, p.N, p.K, ctx->cus);
  return c.kernel < 0 ? too_large(ctx, p.M, p.N, p.K) : with_kernel<OUT>(c, Runner<OUT>{ctx, p});
}

// Up and down projection, both chosen before either is queued.
template <Out OUT>
int run_mlp(miaie_ctx* ctx, const Args& up, const Args& down) {
  const Choice u = choose<OUT_MX_RELU>(up.M, up.N, up.K, ctx->cus), d = choose<OUT>(down.M, down.N, down.K, ctx->cus);
  if (u.kernel < 0) return too_large(ctx, up.M, up.N, up.K);
  if (d.kernel < 0) return too_large(ctx, down.M, down.N, down.K);
  const int rc = with_kernel<OUT_MX_RELU>(u, Runner<OUT_MX_RELU>{ctx, up});
  return rc ? rc : with_kernel<OUT>(d, Runner<OUT>{ctx, down});
}

template <Out OUT>
int plan(int M, int N, int K, int cus, miaie_gemm_plan* to) {
  const Choice c = choose<OUT>(M, N, K, cus);
  return c.kernel < 0 ? too_large(nullptr, M, N, K) : with_kernel<OUT>(c, Planner<OUT>{M, N, K, to});
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

int launch_mlp_mxfp4(miaie_ctx* ctx, const uint8_t* Xq, const uint8_t* Xs, const uint8_t* W1q, const uint8_t* W1s,
                     const uint8_t* W2q, const uint8_t* W2s, uint8_t* Hq, uint8_t* Hs, void* Y, int dtype, int M, int K,
                     int F, int Nout, int ldy) {
  const Args up{Xq, Xs, W1q, W1s, nullptr, Hq, Hs, M, F, K, 0}, down{Hq, Hs, W2q, W2s, Y, nullptr, nullptr, M, Nout, F, ldy};
  return dtype == MIAIE_BF16 ? run_mlp<OUT_BF16>(ctx, up, down) : run_mlp<OUT_F32>(ctx, up, down);
}

int plan_gemm_mxfp4(int M, int N, int K, int out, int cus, miaie_gemm_plan* to) {
  // (with and without a ReLU a packed product takes the same kernels)
  return out == MIAIE_MXFP4 ? plan<OUT_MX>(M, N, K, cus, to) : out == MIAIE_BF16 ? plan<OUT_BF16>(M, N, K, cus, to) : plan<OUT_F32>(M, N, K, cus, to);
}

}  // namespace miaie
