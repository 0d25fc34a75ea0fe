// C-ABI entries of the 8-bit floating point operators, the routing of tokens and
// the experts' products: argument validation, then dispatch.  As in capi.hip,
// everything is checked on the host before anything is queued.
#include "fp8.hpp"

using namespace miaie;

#define MIAIE_TRY(call)               \
  do {                                \
    if (int rc_ = (call)) return rc_; \
  } while (0)

namespace {

constexpr int kMost = 1 << 30;       // rows and columns of a matrix
constexpr int kMostMN = 1 << 25;     // of a product
constexpr int kMostK = 1 << 23;      // contracted by one (32-bit offsets of the 256 rows of a tile)
constexpr int kMostPairs = 1 << 23;  // token and choice (slots are contracted too)
constexpr int kMostWidth = 1 << 20;  // of a row of the experts' matrices

int check_range(miaie_ctx* ctx, const char* fn, const char* name, int v, int most) {
  if (v < 1 || v > most) return fail(ctx, MIAIE_EINVAL, "%s: %s=%d outside [1, %d]", fn, name, v, most);
  return MIAIE_OK;
}

int check_dtype(miaie_ctx* ctx, const char* fn, int dtype) {
  if (dtype != MIAIE_F32 && dtype != MIAIE_BF16)
    return fail(ctx, MIAIE_EINVAL, "%s: dtype=%d is neither MIAIE_F32 nor MIAIE_BF16", fn, dtype);
  return MIAIE_OK;
}

// dtype of a result over tokens, and that of the slots' rows behind it.
int check_slot_dtypes(miaie_ctx* ctx, const char* fn, int* dtype, int* y_dtype) {
  const bool wide = *dtype == (MIAIE_BF16 | MIAIE_F32_SLOTS);
  if (wide) *dtype = MIAIE_BF16;
  *y_dtype = wide ? MIAIE_F32 : *dtype;
  return check_dtype(ctx, fn, *dtype);
}

int check_block(miaie_ctx* ctx, const char* fn, const char* name, int block) {
  if (block != 1 && block != 128) return fail(ctx, MIAIE_EINVAL, "%s: %s=%d is neither 1 nor 128", fn, name, block);
  return MIAIE_OK;
}

int check_pitch(miaie_ctx* ctx, const char* fn, const char* name, int ld, int cols) {
  if (ld < cols) return fail(ctx, MIAIE_EINVAL, "%s: row pitch %s=%d below %d columns", fn, name, ld, cols);
  return MIAIE_OK;
}

// An array of `bytes`-sized elements; `may_be_null` for one that may be left out.
int check_array(miaie_ctx* ctx, const char* fn, const char* name, const void* p, int bytes, bool may_be_null = false) {
  if (!p && !may_be_null) return fail(ctx, MIAIE_EINVAL, "%s: %s is NULL", fn, name);
  if (!aligned(p, bytes)) return fail(ctx, MIAIE_EINVAL, "%s: %s is misaligned", fn, name);
  return MIAIE_OK;
}
int check_elements(miaie_ctx* ctx, const char* fn, const char* name, const void* p, int dtype) {
  return check_array(ctx, fn, name, p, dtype == MIAIE_BF16 ? 2 : 4);
}

int check_packed(miaie_ctx* ctx, const char* fn, const char* name, const uint8_t* q, const float* s) {
  if (!q || !s) return fail(ctx, MIAIE_EINVAL, "%s: %s%s is NULL", fn, name, !q ? "q" : "s");
  if (!aligned(q, 16) || !aligned(s, 4))  // (an expert's scales follow the one's before)
    return fail(ctx, MIAIE_EINVAL, "%s: %sq must be 16-byte and %ss 4-byte aligned", fn, name, name);
  return MIAIE_OK;
}

// One or both forms of a conversion's result.
int check_forms(miaie_ctx* ctx, const char* fn, const uint8_t* Q, const float* S, const uint8_t* Qt, const float* St) {
  if (!Q && !S && !Qt && !St) return fail(ctx, MIAIE_EINVAL, "%s: Q, S, Qt and St are all NULL", fn);
  if (Q || S) MIAIE_TRY(check_packed(ctx, fn, "X", Q, S));
  if (Qt || St) MIAIE_TRY(check_packed(ctx, fn, "Xt", Qt, St));
  return MIAIE_OK;
}

// 512 threads pack 128 x 128; HIP takes fewer than 2^32 threads.
bool tiles_fit(long R, long C) { return fp8::blocks(R) * fp8::blocks(C) < 1u << 23; }

int check_tiles(miaie_ctx* ctx, const char* fn, long R, long C) {
  if (!tiles_fit(R, C))
    return fail(ctx, MIAIE_EINVAL, "%s: %ld rows of %ld columns are too large", fn, R, C);
  return MIAIE_OK;
}

int check_slots(miaie_ctx* ctx, const char* fn, int tokens, int top_k, int experts) {
  MIAIE_TRY(check_range(ctx, fn, "experts", experts, MIAIE_MAX_EXPERTS));
  MIAIE_TRY(check_range(ctx, fn, "top_k", top_k, MIAIE_MAX_TOP_K));
  if (tokens < 1 || (long)tokens * top_k > kMostPairs)
    return fail(ctx, MIAIE_EINVAL, "%s: tokens=%d times top_k=%d outside [1, 2^23]", fn, tokens, top_k);
  return MIAIE_OK;
}

// What every call on an order starts with.
int check_order(miaie_ctx* ctx, const char* fn, const int* order, int tokens, int top_k, int experts) {
  MIAIE_TRY(check_array(ctx, fn, "order", order, 4));
  return check_slots(ctx, fn, tokens, top_k, experts);
}

int check_width(miaie_ctx* ctx, const char* fn, const char* name, int v) { return check_range(ctx, fn, name, v, kMostWidth); }

int check_hidden(miaie_ctx* ctx, const char* fn, int F) {
  MIAIE_TRY(check_width(ctx, fn, "F", F));
  if (F % 128) return fail(ctx, MIAIE_EINVAL, "%s: F=%d is not a multiple of 128", fn, F);
  return MIAIE_OK;
}

// A product over slots: workgroups of a launch, and 32-bit offsets of gathered rows.
int check_slot_product(miaie_ctx* ctx, const char* fn, int tokens, int top_k, int experts, long N, int K, bool gather) {
  if (fp8::slot_rows(tokens, top_k, experts) / 128 * (long)fp8::blocks(N) > 1l << 22)
    return fail(ctx, MIAIE_EINVAL, "%s: the slots of %d tokens x %d choices by %ld columns are too large", fn, tokens, top_k, N);
  if (gather && (size_t)tokens * fp8::pitch(K) >= 1ull << 32)
    return fail(ctx, MIAIE_EINVAL, "%s: %d tokens of %d columns are 2^32 bytes or more", fn, tokens, K);
  return MIAIE_OK;
}

}  // namespace

extern "C" size_t miaie_fp8_q_pitch(int K) { return K < 1 || K > kMost ? 0 : fp8::pitch(K); }

extern "C" size_t miaie_fp8_q_bytes(int R, int K) {
  return R < 1 || R > kMost || K < 1 || K > kMost || !tiles_fit(R, K) ? 0 : (size_t)R * fp8::pitch(K);
}

extern "C" size_t miaie_fp8_s_bytes(int R, int K, int block) {
  if (!miaie_fp8_q_bytes(R, K) || (block != 1 && block != 128)) return 0;
  return 4 * fp8::blocks(K) * (block == 1 ? (size_t)R : fp8::blocks(R));
}

extern "C" int miaie_quant_fp8(miaie_ctx* ctx, const void* X, int dtype, int R, int C, int ldx, int block, uint8_t* Q,
                               float* S, uint8_t* Qt, float* St) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_range(ctx, __func__, "R", R, kMost));
  MIAIE_TRY(check_range(ctx, __func__, "C", C, kMost));
  MIAIE_TRY(check_tiles(ctx, __func__, R, C));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldx", ldx, C));
  MIAIE_TRY(check_block(ctx, __func__, "block", block));
  MIAIE_TRY(check_elements(ctx, __func__, "X", X, dtype));
  MIAIE_TRY(check_forms(ctx, __func__, Q, S, Qt, St));
  return launch_quant_fp8(ctx, X, dtype, R, C, ldx, block, Q, S, Qt, St);
}

extern "C" int miaie_dequant_fp8(miaie_ctx* ctx, const uint8_t* Q, const float* S, int block, void* Y, int dtype, int R,
                                 int C, int ldy) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_range(ctx, __func__, "R", R, kMost));
  MIAIE_TRY(check_range(ctx, __func__, "C", C, kMost));
  MIAIE_TRY(check_tiles(ctx, __func__, R, C));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldy", ldy, C));
  MIAIE_TRY(check_block(ctx, __func__, "block", block));
  MIAIE_TRY(check_packed(ctx, __func__, "X", Q, S));
  MIAIE_TRY(check_elements(ctx, __func__, "Y", Y, dtype));
  return launch_dequant_fp8(ctx, Q, S, block, Y, dtype, R, C, ldy);
}

namespace {

int check_gemm_sizes(miaie_ctx* ctx, const char* fn, int M, int N, int K) {
  MIAIE_TRY(check_range(ctx, fn, "M", M, kMostMN));
  MIAIE_TRY(check_range(ctx, fn, "N", N, kMostMN));
  MIAIE_TRY(check_range(ctx, fn, "K", K, kMostK));
  if ((long)((M + 255l) / 256) * ((N + 255l) / 256) >= 1l << 23)
    return fail(ctx, MIAIE_EINVAL, "%s: a product of M=%d N=%d is too large for one launch", fn, M, N);
  return MIAIE_OK;
}

}  // namespace

extern "C" int miaie_plan_gemm_fp8(int M, int N, int K, int b_block, int cus, miaie_gemm_plan* plan) {
  if (!plan) return fail(nullptr, MIAIE_EINVAL, "%s: plan is NULL", __func__);
  MIAIE_TRY(check_gemm_sizes(nullptr, __func__, M, N, K));
  MIAIE_TRY(check_block(nullptr, __func__, "b_block", b_block));
  if (cus < 1) return fail(nullptr, MIAIE_EINVAL, "%s: cus=%d must be >= 1", __func__, cus);
  return plan_gemm_fp8(M, N, K, b_block, cus, plan);
}

extern "C" int miaie_gemm_fp8(miaie_ctx* ctx, const uint8_t* Aq, const float* As, const uint8_t* Bq, const float* Bs,
                              int b_block, void* C, int dtype, int M, int N, int K, int ldc) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_gemm_sizes(ctx, __func__, M, N, K));
  MIAIE_TRY(check_block(ctx, __func__, "b_block", b_block));
  MIAIE_TRY(check_packed(ctx, __func__, "A", Aq, As));
  MIAIE_TRY(check_packed(ctx, __func__, "B", Bq, Bs));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldc", ldc, N));
  MIAIE_TRY(check_elements(ctx, __func__, "C", C, dtype));
  return launch_gemm_fp8(ctx, Aq, As, Bq, Bs, b_block, C, dtype, M, N, K, ldc);
}

namespace {

// What routing and its gradient share.
int check_routing(miaie_ctx* ctx, const char* fn, const void* logits, int dtype, int tokens, int top_k, int experts, int ld,
                  int scoring, int renormalize, float scale) {
  MIAIE_TRY(check_dtype(ctx, fn, dtype));
  MIAIE_TRY(check_elements(ctx, fn, "logits", logits, dtype));
  MIAIE_TRY(check_range(ctx, fn, "tokens", tokens, 1 << 25));
  MIAIE_TRY(check_range(ctx, fn, "experts", experts, MIAIE_MAX_EXPERTS));
  MIAIE_TRY(check_range(ctx, fn, "top_k", top_k, MIAIE_MAX_TOP_K));
  MIAIE_TRY(check_pitch(ctx, fn, "ld", ld, experts));
  if (scoring != MIAIE_SOFTMAX && scoring != MIAIE_SIGMOID)
    return fail(ctx, MIAIE_EINVAL, "%s: scoring=%d is neither MIAIE_SOFTMAX nor MIAIE_SIGMOID", fn, scoring);
  if (renormalize != 0 && renormalize != 1)
    return fail(ctx, MIAIE_EINVAL, "%s: renormalize=%d must be 0 or 1", fn, renormalize);
  if (!(scale - scale == 0.f)) return fail(ctx, MIAIE_EINVAL, "%s: scale=%g is not finite", fn, scale);
  return MIAIE_OK;
}

}  // namespace

extern "C" int miaie_route_experts(miaie_ctx* ctx, const void* logits, int dtype, const float* bias, int* idx, float* w,
                                   int tokens, int top_k, int experts, int ld, int scoring, int groups, int groups_kept,
                                   int group_top, int renormalize, float scale) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_routing(ctx, __func__, logits, dtype, tokens, top_k, experts, ld, scoring, renormalize, scale));
  MIAIE_TRY(check_array(ctx, __func__, "bias", bias, 4, true));
  MIAIE_TRY(check_array(ctx, __func__, "idx", idx, 4));
  MIAIE_TRY(check_array(ctx, __func__, "w", w, 4));
  MIAIE_TRY(check_range(ctx, __func__, "groups", groups, 64));
  if (experts % groups)
    return fail(ctx, MIAIE_EINVAL, "%s: groups=%d does not divide experts=%d", __func__, groups, experts);
  MIAIE_TRY(check_range(ctx, __func__, "groups_kept", groups_kept, groups));
  MIAIE_TRY(check_range(ctx, __func__, "group_top", group_top, 2));
  if (top_k > experts / groups * groups_kept)
    return fail(ctx, MIAIE_EINVAL, "%s: top_k=%d of %d experts in the groups that stay", __func__, top_k,
                experts / groups * groups_kept);
  return launch_route_experts(ctx, logits, dtype, bias, idx, w, tokens, experts, top_k, ld, scoring, groups, groups_kept,
                              group_top, renormalize, scale);
}

extern "C" int miaie_route_experts_grad(miaie_ctx* ctx, const void* logits, int dtype, const int* idx, const float* dw,
                                        float* dlogits, int tokens, int top_k, int experts, int ld, int ldd, int scoring,
                                        int renormalize, float scale) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_routing(ctx, __func__, logits, dtype, tokens, top_k, experts, ld, scoring, renormalize, scale));
  MIAIE_TRY(check_array(ctx, __func__, "idx", idx, 4));
  MIAIE_TRY(check_array(ctx, __func__, "dw", dw, 4));
  MIAIE_TRY(check_array(ctx, __func__, "dlogits", dlogits, 4));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldd", ldd, experts));
  return launch_route_experts_grad(ctx, logits, dtype, idx, dw, dlogits, tokens, experts, top_k, ld, ldd, scoring,
                                   renormalize, scale);
}

namespace {
bool slots_in_range(int tokens, int top_k, int experts) {
  return tokens >= 1 && top_k >= 1 && top_k <= MIAIE_MAX_TOP_K && (long)tokens * top_k <= kMostPairs && experts >= 1 &&
         experts <= MIAIE_MAX_EXPERTS;
}
}  // namespace

extern "C" size_t miaie_experts_rows(int tokens, int top_k, int experts) {
  return slots_in_range(tokens, top_k, experts) ? (size_t)fp8::slot_rows(tokens, top_k, experts) : 0;
}

extern "C" size_t miaie_experts_order_bytes(int tokens, int top_k, int experts) {
  return slots_in_range(tokens, top_k, experts) ? 4 * fp8::slot_ints(tokens, top_k, experts) : 0;
}

extern "C" int miaie_experts_order(miaie_ctx* ctx, const int* idx, int* order, int tokens, int top_k, int experts) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_array(ctx, __func__, "idx", idx, 4));
  return launch_experts_order(ctx, fp8::slots_of(order, tokens, top_k, experts), idx);
}

extern "C" int miaie_experts_mlp_fp8(miaie_ctx* ctx, const int* order, const float* w, const uint8_t* Xq, const float* Xs,
                                     const uint8_t* W1q, const float* W1s, const uint8_t* W2q, const float* W2s, uint8_t* Hq,
                                     float* Hs, void* Y, void* out, int dtype, int tokens, int top_k, int experts, int D,
                                     int F, int Nout, int ldo) {
  int y_dtype;
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_slot_dtypes(ctx, __func__, &dtype, &y_dtype));
  MIAIE_TRY(check_width(ctx, __func__, "D", D));
  MIAIE_TRY(check_hidden(ctx, __func__, F));
  MIAIE_TRY(check_width(ctx, __func__, "Nout", Nout));
  MIAIE_TRY(check_array(ctx, __func__, "w", w, 4));
  MIAIE_TRY(check_packed(ctx, __func__, "X", Xq, Xs));
  MIAIE_TRY(check_packed(ctx, __func__, "W1", W1q, W1s));
  MIAIE_TRY(check_packed(ctx, __func__, "W2", W2q, W2s));
  MIAIE_TRY(check_packed(ctx, __func__, "H", Hq, Hs));
  MIAIE_TRY(check_elements(ctx, __func__, "Y", Y, y_dtype));
  MIAIE_TRY(check_elements(ctx, __func__, "out", out, dtype));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldo", ldo, Nout));
  MIAIE_TRY(check_slot_product(ctx, __func__, tokens, top_k, experts, 2l * F, D, true));
  MIAIE_TRY(check_slot_product(ctx, __func__, tokens, top_k, experts, Nout, F, false));
  if (2 * (size_t)F * fp8::pitch(D) >= 1ull << 32)
    return fail(ctx, MIAIE_EINVAL, "%s: 2 F = %d rows of D = %d columns are 2^32 bytes or more", __func__, 2 * F, D);
  const fp8::Slots s = fp8::slots_of(order, tokens, top_k, experts);
  MIAIE_TRY(launch_experts_glu_fp8(ctx, s, Xq, Xs, W1q, W1s, Hq, Hs, D, F));
  MIAIE_TRY(launch_experts_gemm_fp8(ctx, s, Hq, Hs, 0, W2q, W2s, Y, y_dtype, Nout, F, Nout));
  return launch_experts_combine(ctx, s, Y, y_dtype, w, out, dtype, Nout, Nout, ldo);
}

extern "C" int miaie_experts_gemm_fp8(miaie_ctx* ctx, const int* order, const uint8_t* Aq, const float* As,
                                      const uint8_t* Bq, const float* Bs, void* C, int dtype, int tokens, int top_k,
                                      int experts, int N, int K, int ldc, int gather) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_width(ctx, __func__, "N", N));
  MIAIE_TRY(check_width(ctx, __func__, "K", K));
  MIAIE_TRY(check_packed(ctx, __func__, "A", Aq, As));
  MIAIE_TRY(check_packed(ctx, __func__, "B", Bq, Bs));
  MIAIE_TRY(check_elements(ctx, __func__, "C", C, dtype));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldc", ldc, N));
  if (gather != 0 && gather != 1) return fail(ctx, MIAIE_EINVAL, "%s: gather=%d must be 0 or 1", __func__, gather);
  MIAIE_TRY(check_slot_product(ctx, __func__, tokens, top_k, experts, N, K, gather));
  return launch_experts_gemm_fp8(ctx, fp8::slots_of(order, tokens, top_k, experts), Aq, As, gather, Bq, Bs, C, dtype, N, K,
                                 ldc);
}

extern "C" int miaie_plan_experts_fp8(int tokens, int top_k, int experts, int N, int K, int swiglu, int cus,
                                      miaie_gemm_plan* plan) {
  if (!plan) return fail(nullptr, MIAIE_EINVAL, "%s: plan is NULL", __func__);
  MIAIE_TRY(check_slots(nullptr, __func__, tokens, top_k, experts));
  if (swiglu != 0 && swiglu != 1) return fail(nullptr, MIAIE_EINVAL, "%s: swiglu=%d must be 0 or 1", __func__, swiglu);
  MIAIE_TRY(swiglu ? check_hidden(nullptr, __func__, N) : check_width(nullptr, __func__, "N", N));
  MIAIE_TRY(check_width(nullptr, __func__, "K", K));
  MIAIE_TRY(check_slot_product(nullptr, __func__, tokens, top_k, experts, swiglu ? 2l * N : N, K, false));
  if (cus < 1) return fail(nullptr, MIAIE_EINVAL, "%s: cus=%d must be >= 1", __func__, cus);
  fp8::Slots s{};  // (its sizes alone)
  s.tokens = tokens, s.top_k = top_k, s.experts = experts;
  return plan_experts_fp8(s, N, K, swiglu, cus, plan);
}

extern "C" int miaie_experts_quant_fp8(miaie_ctx* ctx, const int* order, const void* X, int dtype, const float* w,
                                       uint8_t* Q, float* S, uint8_t* Qt, float* St, int tokens, int top_k, int experts,
                                       int C, int ldx) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_width(ctx, __func__, "C", C));
  MIAIE_TRY(check_tiles(ctx, __func__, fp8::slot_rows(tokens, top_k, experts), C));
  MIAIE_TRY(check_elements(ctx, __func__, "X", X, dtype));
  MIAIE_TRY(check_array(ctx, __func__, "w", w, 4, true));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldx", ldx, C));
  MIAIE_TRY(check_forms(ctx, __func__, Q, S, Qt, St));
  return launch_experts_quant_fp8(ctx, fp8::slots_of(order, tokens, top_k, experts), X, dtype, w, C, ldx, Q, S, Qt, St);
}

extern "C" int miaie_experts_swiglu_fp8(miaie_ctx* ctx, const int* order, const void* GU, int dtype, uint8_t* Q, float* S,
                                        uint8_t* Qt, float* St, int tokens, int top_k, int experts, int F, int ldgu) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_hidden(ctx, __func__, F));
  MIAIE_TRY(check_tiles(ctx, __func__, fp8::slot_rows(tokens, top_k, experts), F));
  MIAIE_TRY(check_elements(ctx, __func__, "GU", GU, dtype));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldgu", ldgu, 2 * F));
  MIAIE_TRY(check_forms(ctx, __func__, Q, S, Qt, St));
  return launch_experts_swiglu_fp8(ctx, fp8::slots_of(order, tokens, top_k, experts), GU, dtype, F, ldgu, Q, S, Qt, St);
}

extern "C" int miaie_experts_swiglu_grad_fp8(miaie_ctx* ctx, const int* order, const void* GU, int dtype, const float* dH,
                                             uint8_t* Q, float* S, uint8_t* Qt, float* St, int tokens, int top_k,
                                             int experts, int F, int ldgu, int ldh) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_hidden(ctx, __func__, F));
  MIAIE_TRY(check_tiles(ctx, __func__, fp8::slot_rows(tokens, top_k, experts), 2l * F));
  MIAIE_TRY(check_elements(ctx, __func__, "GU", GU, dtype));
  MIAIE_TRY(check_array(ctx, __func__, "dH", dH, 4));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldgu", ldgu, 2 * F));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldh", ldh, F));
  MIAIE_TRY(check_forms(ctx, __func__, Q, S, Qt, St));
  return launch_experts_swiglu_grad_fp8(ctx, fp8::slots_of(order, tokens, top_k, experts), GU, dtype, dH, F, ldgu, ldh, Q, S,
                                        Qt, St);
}

extern "C" int miaie_experts_wgrad_fp8(miaie_ctx* ctx, const int* order, const uint8_t* Atq, const float* Ats,
                                       const uint8_t* Btq, const float* Bts, void* C, int dtype, int tokens, int top_k,
                                       int experts, int M, int N, int ldc) {
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_dtype(ctx, __func__, dtype));
  MIAIE_TRY(check_width(ctx, __func__, "M", M));
  MIAIE_TRY(check_width(ctx, __func__, "N", N));
  if ((long)experts * ((M + 255) / 256) * ((N + 255) / 256) >= 1l << 23)
    return fail(ctx, MIAIE_EINVAL, "%s: %d products of M=%d N=%d are too large for one launch", __func__, experts, M, N);
  MIAIE_TRY(check_packed(ctx, __func__, "At", Atq, Ats));
  MIAIE_TRY(check_packed(ctx, __func__, "Bt", Btq, Bts));
  MIAIE_TRY(check_elements(ctx, __func__, "C", C, dtype));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldc", ldc, N));
  return launch_experts_wgrad_fp8(ctx, fp8::slots_of(order, tokens, top_k, experts), Atq, Ats, Btq, Bts, C, dtype, M, N, ldc);
}

extern "C" int miaie_experts_combine(miaie_ctx* ctx, const int* order, const void* Y, const float* w, void* out, int dtype,
                                     int tokens, int top_k, int experts, int C, int ldy, int ldo) {
  int y_dtype;
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_slot_dtypes(ctx, __func__, &dtype, &y_dtype));
  MIAIE_TRY(check_width(ctx, __func__, "C", C));
  MIAIE_TRY(check_elements(ctx, __func__, "Y", Y, y_dtype));
  MIAIE_TRY(check_array(ctx, __func__, "w", w, 4, true));
  MIAIE_TRY(check_elements(ctx, __func__, "out", out, dtype));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldy", ldy, C));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldo", ldo, C));
  return launch_experts_combine(ctx, fp8::slots_of(order, tokens, top_k, experts), Y, y_dtype, w, out, dtype, C, ldy, ldo);
}

extern "C" int miaie_experts_combine_grad(miaie_ctx* ctx, const int* order, const void* Y, const void* dout, float* dw,
                                          int dtype, int tokens, int top_k, int experts, int C, int ldy, int ldo) {
  int y_dtype;
  MIAIE_TRY(enter(ctx));
  MIAIE_TRY(check_order(ctx, __func__, order, tokens, top_k, experts));
  MIAIE_TRY(check_slot_dtypes(ctx, __func__, &dtype, &y_dtype));
  MIAIE_TRY(check_width(ctx, __func__, "C", C));
  MIAIE_TRY(check_elements(ctx, __func__, "Y", Y, y_dtype));
  MIAIE_TRY(check_elements(ctx, __func__, "dout", dout, dtype));
  MIAIE_TRY(check_array(ctx, __func__, "dw", dw, 4));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldy", ldy, C));
  MIAIE_TRY(check_pitch(ctx, __func__, "ldo", ldo, C));
  return launch_experts_combine_grad(ctx, fp8::slots_of(order, tokens, top_k, experts), Y, y_dtype, dout, dw, dtype, C, ldy,
                                     ldo);
}
