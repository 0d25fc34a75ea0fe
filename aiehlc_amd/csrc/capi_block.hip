// C-ABI entries of the MXFP4 operators and the norms around a block: argument
// validation, then dispatch.  As in capi.hip, everything is checked on the
// host before anything is queued.
#include "mxfp4.hpp"

using namespace miaie;

namespace {

constexpr int kMost = 1 << 30;
constexpr int kMostK = 1 << 26;  // contracted by a product (32-bit offsets of the rows of a tile)

int check_size(miaie_ctx* ctx, const char* fn, const char* name, int v) {
  if (v < 1 || v > kMost) return fail(ctx, MIAIE_EINVAL, "%s: %s=%d outside [1, 2^30]", fn, name, v);
  return MIAIE_OK;
}

int check_dtype(miaie_ctx* ctx, const char* fn, const char* name, int dtype) {
  if (dtype != MIAIE_F32 && dtype != MIAIE_BF16)
    return fail(ctx, MIAIE_EINVAL, "%s: %s=%d is neither MIAIE_F32 nor MIAIE_BF16", fn, name, dtype);
  return MIAIE_OK;
}

int check_pitch(miaie_ctx* ctx, const char* fn, const char* name, int ld, int cols) {
  if (ld < cols) return fail(ctx, MIAIE_EINVAL, "%s: row pitch %s=%d below %d columns", fn, name, ld, cols);
  return MIAIE_OK;
}

int check_elements(miaie_ctx* ctx, const char* fn, const char* name, const void* p, int dtype) {
  if (!aligned(p, dtype == MIAIE_BF16 ? 2 : 4)) return fail(ctx, MIAIE_EINVAL, "%s: %s is misaligned", fn, name);
  return MIAIE_OK;
}

int check_rows(miaie_ctx* ctx, const char* fn, const char* name, int R, int K) {
  if ((long)R * mx::s_groups(K) >= kMost)
    return fail(ctx, MIAIE_EINVAL, "%s: %s (%d rows of %d columns) is too large", fn, name, R, K);
  return MIAIE_OK;
}

// The two arrays of a packed R x K matrix.
int check_packed(miaie_ctx* ctx, const char* fn, const char* name, const uint8_t* q, const uint8_t* s, int R, int K) {
  if (!q || !s) return fail(ctx, MIAIE_EINVAL, "%s: %s%s is NULL", fn, name, !q ? "q" : "s");
  if (!aligned(q, 16) || !aligned(s, 16))
    return fail(ctx, MIAIE_EINVAL, "%s: %sq and %ss must be 16-byte aligned", fn, name, name);
  return check_rows(ctx, fn, name, R, K);
}

// 512 threads pack 64 rows of 512 columns of a packed transpose, the workgroups'
// number rounded up to 64 (quant_mxfp4.hip); HIP takes fewer than 2^32 threads.
int check_transpose(miaie_ctx* ctx, const char* fn, int R, int C) {
  if ((long)mx::s_groups(R) * 8 * mx::s_groups(C) > (1l << 23) - 64)
    return fail(ctx, MIAIE_EINVAL, "%s: R=%d C=%d too large to pack along the columns", fn, R, C);
  return MIAIE_OK;
}

}  // namespace

#define MIAIE_TRY(call)          \
  do {                           \
    if (int rc_ = (call)) return rc_; \
  } while (0)

extern "C" size_t miaie_mxfp4_q_pitch(int K) { return K < 1 || K > kMost ? 0 : mx::q_pitch(K); }

extern "C" size_t miaie_mxfp4_q_bytes(int R, int K) {
  return R < 1 || R > kMost ? 0 : (size_t)R * miaie_mxfp4_q_pitch(K);
}

extern "C" size_t miaie_mxfp4_s_bytes(int R, int K) {
  return R < 1 || R > kMost || K < 1 || K > kMost ? 0 : (size_t)R * mx::s_groups(K) * 16;
}

extern "C" int miaie_quant_mxfp4(miaie_ctx* ctx, const void* X, int dtype, int R, int C, int ldx, uint8_t* Q,
                                 uint8_t* S, uint8_t* Qt, uint8_t* St) {
  MIAIE_TRY(enter(ctx));
  MIAIE_CHECK_NOT_NULL(ctx, X);
  MIAIE_TRY(check_dtype(ctx, __func__, "dtype", dtype));
  MIAIE_TRY(check_size(ctx, __func__, "R", R));
  MIAIE_TRY(check_size(ctx, __func__, "C", C));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldx", ldx, C));
  MIAIE_TRY(check_elements(ctx, __func__, "X", X, dtype));
  if (!Q && !S && !Qt && !St) return fail(ctx, MIAIE_EINVAL, "%s: Q, S, Qt and St are all NULL", __func__);
  if (Q || S) MIAIE_TRY(check_packed(ctx, __func__, "X", Q, S, R, C));
  if (Qt || St) {
    MIAIE_TRY(check_packed(ctx, __func__, "Xt", Qt, St, C, R));
    MIAIE_TRY(check_transpose(ctx, __func__, R, C));
  }
  return launch_quant_mxfp4(ctx, X, dtype, R, C, ldx, Q, S, Qt, St);
}

extern "C" int miaie_dequant_mxfp4(miaie_ctx* ctx, const uint8_t* Q, const uint8_t* S, void* Y, int dtype, int R,
                                   int C, int ldy) {
  MIAIE_TRY(enter(ctx));
  MIAIE_CHECK_NOT_NULL(ctx, Y);
  MIAIE_TRY(check_dtype(ctx, __func__, "dtype", dtype));
  MIAIE_TRY(check_size(ctx, __func__, "R", R));
  MIAIE_TRY(check_size(ctx, __func__, "C", C));
  MIAIE_TRY(check_packed(ctx, __func__, "X", Q, S, R, C));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldy", ldy, C));
  MIAIE_TRY(check_elements(ctx, __func__, "Y", Y, dtype));
  return launch_dequant_mxfp4(ctx, Q, S, Y, dtype, R, C, ldy);
}

namespace {

int check_gemm_sizes(miaie_ctx* ctx, const char* fn, int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1 || M > kMost || N > kMost || K > kMostK)
    return fail(ctx, MIAIE_EINVAL, "%s: M=%d N=%d K=%d must be in [1, 2^30], K in [1, 2^26]", fn, M, N, K);
  return MIAIE_OK;
}

int check_gemm(miaie_ctx* ctx, const char* fn, const uint8_t* Aq, const uint8_t* As, const uint8_t* Bq,
               const uint8_t* Bs, int M, int N, int K) {
  MIAIE_TRY(check_gemm_sizes(ctx, fn, M, N, K));
  MIAIE_TRY(check_packed(ctx, fn, "A", Aq, As, M, K));
  return check_packed(ctx, fn, "B", Bq, Bs, N, K);
}

}  // namespace

extern "C" int miaie_plan_gemm_mxfp4(int M, int N, int K, int out, int cus, miaie_gemm_plan* plan) {
  if (!plan) return fail(nullptr, MIAIE_EINVAL, "%s: plan is NULL", __func__);
  MIAIE_TRY(check_gemm_sizes(nullptr, __func__, M, N, K));
  MIAIE_TRY(check_rows(nullptr, __func__, "A", M, K));
  MIAIE_TRY(check_rows(nullptr, __func__, "B", N, K));
  if (out != MIAIE_F32 && out != MIAIE_BF16 && out != MIAIE_MXFP4)
    return fail(nullptr, MIAIE_EINVAL, "%s: out=%d is none of MIAIE_F32, MIAIE_BF16 and MIAIE_MXFP4", __func__, out);
  if (out == MIAIE_MXFP4) MIAIE_TRY(check_rows(nullptr, __func__, "Y", M, N));
  if (cus < 1) return fail(nullptr, MIAIE_EINVAL, "%s: cus=%d must be >= 1", __func__, cus);
  return plan_gemm_mxfp4(M, N, K, out, cus, plan);
}

extern "C" int miaie_gemm_mxfp4(miaie_ctx* ctx, const uint8_t* Aq, const uint8_t* As, const uint8_t* Bq,
                                const uint8_t* Bs, void* C, int dtype, int M, int N, int K, int ldc) {
  MIAIE_TRY(enter(ctx));
  MIAIE_CHECK_NOT_NULL(ctx, C);
  MIAIE_TRY(check_dtype(ctx, __func__, "dtype", dtype));
  MIAIE_TRY(check_gemm(ctx, __func__, Aq, As, Bq, Bs, M, N, K));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldc", ldc, N));
  MIAIE_TRY(check_elements(ctx, __func__, "C", C, dtype));
  return launch_gemm_mxfp4(ctx, Aq, As, Bq, Bs, C, dtype, M, N, K, ldc);
}

extern "C" int miaie_gemm_mxfp4_rq(miaie_ctx* ctx, const uint8_t* Aq, const uint8_t* As, const uint8_t* Bq,
                                   const uint8_t* Bs, uint8_t* Yq, uint8_t* Ys, int M, int N, int K, int relu) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_gemm(ctx, __func__, Aq, As, Bq, Bs, M, N, K));
  MIAIE_TRY(check_packed(ctx, __func__, "Y", Yq, Ys, M, N));
  if (relu != 0 && relu != 1) return fail(ctx, MIAIE_EINVAL, "%s: relu=%d must be 0 or 1", __func__, relu);
  return launch_gemm_mxfp4_rq(ctx, Aq, As, Bq, Bs, Yq, Ys, M, N, K, relu);
}

extern "C" int miaie_mlp_mxfp4(miaie_ctx* ctx, const uint8_t* Xq, const uint8_t* Xs, const uint8_t* W1q,
                               const uint8_t* W1s, const uint8_t* W2q, const uint8_t* W2s, uint8_t* Hq, uint8_t* Hs,
                               void* Y, int dtype, int M, int K, int F, int Nout, int ldy) {
  MIAIE_TRY(enter(ctx));
  MIAIE_CHECK_NOT_NULL(ctx, Y);
  MIAIE_TRY(check_dtype(ctx, __func__, "dtype", dtype));
  if (M < 1 || K < 1 || F < 1 || Nout < 1 || M > kMost || Nout > kMost || K > kMostK || F > kMostK)
    return fail(ctx, MIAIE_EINVAL, "%s: M=%d K=%d F=%d Nout=%d must be in [1, 2^30], K and F in [1, 2^26]", __func__, M, K,
                F, Nout);
  MIAIE_TRY(check_packed(ctx, __func__, "X", Xq, Xs, M, K));
  MIAIE_TRY(check_packed(ctx, __func__, "W1", W1q, W1s, F, K));
  MIAIE_TRY(check_packed(ctx, __func__, "W2", W2q, W2s, Nout, F));
  MIAIE_TRY(check_packed(ctx, __func__, "H", Hq, Hs, M, F));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldy", ldy, Nout));
  MIAIE_TRY(check_elements(ctx, __func__, "Y", Y, dtype));
  return launch_mlp_mxfp4(ctx, Xq, Xs, W1q, W1s, W2q, W2s, Hq, Hs, Y, dtype, M, K, F, Nout, ldy);
}

namespace {

// What the forward and the gradient share: sizes, pitches and types.
int check_norm(miaie_ctx* ctx, const char* fn, int rows, int cols, int ldx, int ldb, int gate_rows, int stream_dtype,
               int branch_dtype) {
  MIAIE_TRY(check_size(ctx, fn, "rows", rows));
  if (cols < 1 || cols > MIAIE_NORM_MAX_COLS)
    return fail(ctx, MIAIE_EINVAL, "%s: cols=%d outside [1, %d]", fn, cols, MIAIE_NORM_MAX_COLS);
  MIAIE_TRY(check_pitch(ctx, fn, "ldx", ldx, cols));
  MIAIE_TRY(check_pitch(ctx, fn, "ldb", ldb, cols));
  if (gate_rows < 1) return fail(ctx, MIAIE_EINVAL, "%s: gate_rows=%d must be >= 1", fn, gate_rows);
  MIAIE_TRY(check_dtype(ctx, fn, "stream_dtype", stream_dtype));
  return check_dtype(ctx, fn, "branch_dtype", branch_dtype);
}

}  // namespace

extern "C" int miaie_norm_block(miaie_ctx* ctx, const void* x, const void* b, const void* gate, const float* w_after,
                                const float* w_before, void* out, void* y, float* rstd, int rows, int cols, int ldx,
                                int ldb, int gate_rows, int stream_dtype, int branch_dtype, float alpha, float eps) {
  MIAIE_TRY(enter(ctx));
  MIAIE_CHECK_NOT_NULL(ctx, x);
  MIAIE_TRY(check_norm(ctx, __func__, rows, cols, ldx, ldb, gate_rows, stream_dtype, branch_dtype));
  if (!(eps >= 0.f)) return fail(ctx, MIAIE_EINVAL, "%s: eps=%g must be >= 0", __func__, eps);
  if (!b && !y) return fail(ctx, MIAIE_EINVAL, "%s: neither b nor y: nothing to do", __func__);
  if (b ? !w_after || !out : w_after || out || gate)
    return fail(ctx, MIAIE_EINVAL, "%s: b takes w_after and out (and may take gate); without b they are NULL", __func__);
  if ((y == nullptr) != (w_before == nullptr))
    return fail(ctx, MIAIE_EINVAL, "%s: y and w_before come together", __func__);
  const struct {
    const char* name;
    const void* p;
    int dtype;
  } elements[] = {{"x", x, stream_dtype},        {"out", out, stream_dtype},      {"b", b, branch_dtype},
                  {"y", y, branch_dtype},        {"gate", gate, branch_dtype},    {"w_after", w_after, MIAIE_F32},
                  {"w_before", w_before, MIAIE_F32}, {"rstd", rstd, MIAIE_F32}};
  for (const auto& e : elements) MIAIE_TRY(check_elements(ctx, __func__, e.name, e.p, e.dtype));
  return launch_norm_block(ctx, x, b, gate, w_after, w_before, out, y, rstd, rows, cols, ldx, ldb,
                           gate ? gate_rows : rows, stream_dtype, branch_dtype, alpha, eps);
}

extern "C" int miaie_norm_block_grad(miaie_ctx* ctx, const void* r, const void* b, const void* gate,
                                     const float* w_after, const float* w_before, const float* rstd, const void* dout,
                                     const void* dy, void* dx, void* db, float* dgate, float* dw_after,
                                     float* dw_before, void* work, size_t work_bytes, int rows, int cols, int ldx,
                                     int ldb, int gate_rows, int stream_dtype, int branch_dtype, float alpha) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_norm(ctx, __func__, rows, cols, ldx, ldb, gate_rows, stream_dtype, branch_dtype));
  if (!dout && !dy) return fail(ctx, MIAIE_EINVAL, "%s: neither dout nor dy", __func__);
  if (!dx && !db && !dgate && !dw_after && !dw_before)
    return fail(ctx, MIAIE_EINVAL, "%s: no gradient wanted", __func__);
  if (!b && !dy) return fail(ctx, MIAIE_EINVAL, "%s: neither b nor dy: no norm ran", __func__);
  if (dy ? !r || !w_before : w_before || dw_before)
    return fail(ctx, MIAIE_EINVAL, "%s: dy takes r and w_before; without it w_before and dw_before are NULL", __func__);
  if (b ? !w_after : w_after || gate || db || dgate || dw_after)
    return fail(ctx, MIAIE_EINVAL, "%s: b takes w_after; without it gate, w_after, db, dgate and dw_after are NULL",
                __func__);
  if (dgate && !gate) return fail(ctx, MIAIE_EINVAL, "%s: dgate without gate", __func__);
  MIAIE_CHECK_NOT_NULL(ctx, rstd);
  if (dgate || dw_after || dw_before) {
    MIAIE_CHECK_NOT_NULL(ctx, work);
    if (work_bytes < MIAIE_NORM_WORK_BYTES(cols))
      return fail(ctx, MIAIE_EINVAL, "%s: work_bytes=%zu below MIAIE_NORM_WORK_BYTES(%d) = %zu", __func__, work_bytes,
                  cols, MIAIE_NORM_WORK_BYTES(cols));
  }
  const struct {
    const char* name;
    const void* p;
    int dtype;
  } elements[] = {{"r", r, stream_dtype},       {"dout", dout, stream_dtype},      {"dx", dx, stream_dtype},
                  {"b", b, branch_dtype},       {"gate", gate, branch_dtype},      {"dy", dy, branch_dtype},
                  {"db", db, branch_dtype},     {"w_after", w_after, MIAIE_F32},   {"w_before", w_before, MIAIE_F32},
                  {"rstd", rstd, MIAIE_F32},    {"dgate", dgate, MIAIE_F32},       {"dw_after", dw_after, MIAIE_F32},
                  {"dw_before", dw_before, MIAIE_F32}, {"work", work, MIAIE_F32}};
  for (const auto& e : elements) MIAIE_TRY(check_elements(ctx, __func__, e.name, e.p, e.dtype));
  return launch_norm_block_grad(ctx, r, b, gate, w_after, w_before, rstd, dout, dy, dx, db, dgate, dw_after, dw_before,
                                static_cast<float*>(work), rows, cols, ldx, ldb, gate ? gate_rows : rows, stream_dtype,
                                branch_dtype, b ? alpha : 1.f);
}
