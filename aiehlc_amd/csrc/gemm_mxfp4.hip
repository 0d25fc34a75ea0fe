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
// from N on become zeros.  Lane fg writes block fg whole: the lanes' four codes
// of each half are exchanged as a 4 x 4 transpose.
template <int NB, bool RELU>
__device__ __forceinline__ void store_blocks(const Args& p, int m, int nb, int fg, const v4f* acc) {
  uint32_t q[4] = {0, 0, 0, 0}, s[4] = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    float x[8];
    uint32_t amax = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int n = 32 * (nb + k) + (e >> 2) * 16 + 4 * fg + (e & 3);
      float v = acc[2 * k + (e >> 2)][e & 3];
      if (RELU) v = v < 0.f ? 0.f : v;  // (keeps NaN)
      x[e] = n < p.N ? v : 0.f;
      amax = max(amax, abs_bits(x[e]));
    }
    s[k] = scale_of(row_max(amax));
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
      store_blocks<1, OUT == OUT_MX_RELU>(p, m, n0 / 32, fg, acc[i]);
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
//   scales of group q + 1: phase 2 of k-tile 4 q (every wave took those of group
//     q into registers in phase 2 of k-tile 4 q - 1), taken in phase 2 of k-tile
//     4 q + 3.
// What the barrier of k-tile t has to make visible (k-tile t + 1) was sent by
// phi = 2 t - 3, so the copies of the three phases since may be in flight: at
// most VM of them (copies of scales in between only make the wait stricter).
// Phases before 0 are the prologue.
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
// pair of A at c ^ a_swz(r): the 16 lanes that one ds_read_b128 serves at a
// time, 16 consecutive rows at one chunk, then cover all 64 banks.
__device__ __forceinline__ int a_swz(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int b_swz(int r) { return (r >> 2) & 3; }

// acc += B fragment x A fragment, scales in byte T, in place.  (The compiler's
// form of the instruction writes other registers than it adds to and moves
// accumulators around: 30 cycles an instruction in a loop of 16 of them,
// against 17.)  No instruction but a load writes an operand within two
// instructions before its use (tests/test_mx_asm.py).
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

template <int BM, int BN, Out OUT>
__global__ __launch_bounds__(256, BM == 256 ? 1 : 2) void gemm_mx_pipe(Args p, int tiles_m, int tiles_n) {
  using G = PipeGeom<BM, BN>;
  constexpr int NI = G::NI, NJ = G::NJ, HI = G::HI, PH = G::PH;
  __shared__ __attribute__((aligned(1024))) int8_t lds[G::LDS];
  constexpr int B0 = G::A_REGION, S0 = G::A_REGION + G::B_REGION;
  const uint32_t lds0 = dev::lds_addr(lds);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, fr = lane & 15, fg = lane >> 4;
  int tm, tn;
  dev::tile_coords<4>(blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
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
  int sa[NI], sb[NJ], sa_next[NI], sb_next[NJ];
  auto read_a = [&](uint32_t st, int par, int i) __attribute__((always_inline)) -> v4i {
    // (readfirstlane keeps the stage's address in the base register, so that
    // 2048 i is the instruction's offset)
    return *reinterpret_cast<const v4i*>(lds + __builtin_amdgcn_readfirstlane(st) + a_fo[par] + 2048 * i);
  };
  auto read_b = [&](uint32_t st, int j) __attribute__((always_inline)) {
    bs[j] = *reinterpret_cast<const v4i*>(lds + __builtin_amdgcn_readfirstlane(st) + b_fo + 1024 * j);
  };
  auto read_s = [&](int x) __attribute__((always_inline)) {
    if (x < NI)
      sa_next[x] = *reinterpret_cast<const int*>(lds + sa_fo + 256 * x);
    else
      sb_next[x - NI] = *reinterpret_cast<const int*>(lds + sb_fo + 256 * (x - NI));
  };

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
  for (int x = 0; x < NI + NJ; ++x) read_s(x);
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

  // k-tile t: D k-tiles before the last; PAR = t % 2 and, where it is known at
  // compile time, T4 = t % 4 (else -1: the registers of scales are then shifted
  // by a pair's two bytes for the second pair of a group)
  auto tile = [&](auto par_c, auto t4_c, auto d_c) __attribute__((always_inline)) {
    constexpr int PAR = decltype(par_c)::value, T4 = decltype(t4_c)::value, D = decltype(d_c)::value;
    constexpr int BYTE = T4 >= 0 ? T4 : PAR;
    constexpr int NA = G::a_copies(D), NB = G::b_copies(D);
    constexpr bool NEXT = D >= 1;
#pragma unroll
    for (int x = 0; x < PH; ++x) {
      const int j = x / HI, i = dev::snake_j<HI>(x);
      mfma_in_place<BYTE>(acc[i][j], bs[j], alo[i], sb[j], sa[i]);
      if (x < HI) ahi[x] = read_a(st0, PAR, HI + x);
#pragma unroll
      for (int c = 0; c < NA; ++c)
        if (c * PH / (NA > 0 ? NA : 1) == x) copy_a(a_src, st2, G::A_CP * PAR + c);
      dev::sched_fence();
    }
    dev::waitcnt<G::vm(D), 0>();
    dev::barrier();
    const uint32_t st_next = PAR == 0 ? st0 : st1;
    const uint32_t b_next = slot_at(2 + wn);
    const uint32_t cp0 = slot_at(1), cp1 = slot_at(0);  // (2 (t + 4)) % 7, (2 (t + 3) + 1) % 7
#pragma unroll
    for (int x = 0; x < PH; ++x) {
      const int j = x / HI, i = dev::snake_j<HI>(x);
      mfma_in_place<BYTE>(acc[HI + i][j], bs[j], ahi[i], sb[j], sa[HI + i]);
#pragma unroll
      for (int c = 0; c < NB; ++c)
        if (c * PH / (NB > 0 ? NB : 1) == x) {
          if (c < G::B_CP)
            copy_b(b_src, cp1, 1, c);
          else
            copy_b(b_src + 64, cp0, 0, c - G::B_CP);
        }
      if constexpr (T4 == 0 || (T4 < 0 && PAR == 0)) {
        if (x == 0 && (t & 3) == 0 && t + 4 < KT) copy_s(t / 4 + 1);
      }
      if constexpr (NEXT) {
        if (x < HI) alo[x] = read_a(st_next, 1 - PAR, x);
        if (x % HI == HI - 1) read_b(b_next, j);  // last use of k-tile t's fragment j
        // (where t % 4 may be 1 these are not taken, and read again at 3)
        if constexpr (T4 == 3 || (T4 < 0 && PAR == 1)) {
#pragma unroll
          for (int r = x * (NI + NJ) / PH; r < (x + 1) * (NI + NJ) / PH; ++r) read_s(r);
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
  // The scales of the pair that starts: the group's (phase 2 of the k-tile
  // before read them), or the next two bytes of those.  Three wait states between
  // these instructions and the first that takes the registers.
  auto take_scales = [&](bool shift) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i) sa[i] = shift ? (int)((uint32_t)sa[i] >> 16) : sa_next[i];
#pragma unroll
    for (int j = 0; j < NJ; ++j) sb[j] = shift ? (int)((uint32_t)sb[j] >> 16) : sb_next[j];
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
    take_scales(false);
    tile(P0{}, std::integral_constant<int, 0>{}, DS{});
    tile(P1{}, std::integral_constant<int, 1>{}, DS{});
    tile(P0{}, std::integral_constant<int, 2>{}, DS{});
    tile(P1{}, std::integral_constant<int, 3>{}, DS{});
  }
  while (t + 6 < KT) {
    take_scales(t & 2);
    tile(P0{}, TR{}, DS{});
    tile(P1{}, TR{}, DS{});
  }
  if (KT >= 6) {
    take_scales(t & 2);
    tile(P0{}, TR{}, std::integral_constant<int, 5>{});
    tile(P1{}, TR{}, std::integral_constant<int, 4>{});
  }
  if (KT >= 4) {
    take_scales(t & 2);
    tile(P0{}, TR{}, std::integral_constant<int, 3>{});
    tile(P1{}, TR{}, std::integral_constant<int, 2>{});
  }
  take_scales(t & 2);
  tile(P0{}, TR{}, std::integral_constant<int, 1>{});
  tile(P1{}, TR{}, std::integral_constant<int, 0>{});
  // the last results are readable after 18 wait states at most
  dev::sched_fence();
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
  dev::sched_fence();

  // ---- acc[i][j]: row 16 i + fr and columns 16 j + 4 fg + 0..3 of the wave's quarter
  const int mw = m0 + wm * G::WM, nw = n0 + wn * G::WN;
  if constexpr (OUT == OUT_F32 || OUT == OUT_BF16) {
    using T = std::conditional_t<OUT == OUT_F32, float, __bf16>;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        store4(static_cast<T*>(p.C), p.ldc, mw + 16 * i + fr, nw + 16 * j + 4 * fg, p.M, p.N, acc[i][j]);
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      store_blocks<NJ / 2, OUT == OUT_MX_RELU>(p, mw + 16 * i + fr, nw / 32, fg, acc[i]);
      dev::sched_fence();  // (more rows at once spill)
    }
    if (tn == tiles_n - 1) {  // zeros up to the end of the last 512 columns
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

// Tiles and workgroups of a launch; HIP takes fewer than 2^32 threads.
template <int BM, int BN, Out OUT>
int run_pipe(miaie_ctx* ctx, const Args& p) {
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  const hipError_t e = launch<gemm_mx_pipe<BM, BN, OUT>>(ctx->device, dim3((unsigned)tiles_m * tiles_n), dim3(256), 0,
                                                         ctx->stream, p, tiles_m, tiles_n);
  return check_launch(ctx, e, "gemm_mx_pipe");
}

template <Out OUT>
int run(miaie_ctx* ctx, const Args& p) {
  if (p.M > 64 && q_pitch(p.K) < (1u << 24)) {
    const long tiles = ((p.M + 255l) / 256) * ((p.N + 255l) / 256);
    if (tiles < 1l << 22) return 3 * tiles >= 2 * ctx->cus ? run_pipe<256, 256, OUT>(ctx, p) : run_pipe<128, 128, OUT>(ctx, p);
  }
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
