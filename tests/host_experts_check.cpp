// Run by tests/test_host_experts.py, without a GPU: the 8-bit, routing and experts'
// wrappers of miaie.hpp over entry points that record their arguments.  Operands that
// do not fit together, or buffers too short, have to be refused before an entry point
// is called; those that fit have to reach it with the sizes and arrays they stand for.
#include <cstdio>
#include <string>
#include <vector>

#include "miaie.hpp"

static std::string last;  // the last compute call: name and sizes
static int calls = 0;
static std::vector<const void*> pointers;  // its arrays

template <class... I>
static int called(const char* name, std::vector<const void*> arrays, I... sizes) {
  ++calls;
  last = name;
  pointers = std::move(arrays);
  ((last += " " + std::to_string(sizes)), ...);
  return MIAIE_OK;
}

extern "C" {
int miaie_init(miaie_ctx** ctx, int) { return *ctx = reinterpret_cast<miaie_ctx*>(8), MIAIE_OK; }
int miaie_finish(miaie_ctx*) { return MIAIE_OK; }
const char* miaie_last_error_string(const miaie_ctx*) { return "recorded"; }
int miaie_alloc(miaie_ctx*, size_t, void** p) {  // addresses of their own, never read
  static uintptr_t next = 0;
  return *p = reinterpret_cast<void*>(next += 4096), MIAIE_OK;
}
int miaie_free(miaie_ctx*, void*) { return MIAIE_OK; }
size_t miaie_fp8_q_bytes(int R, int K) { return (size_t)R * ((K + 127) / 128 * 128); }
size_t miaie_fp8_s_bytes(int R, int K, int block) { return (size_t)4 * ((K + 127) / 128) * ((R + block - 1) / block); }
size_t miaie_experts_rows(int T, int k, int E) {
  const int n = T * k, used = E < n ? E : n;
  return 128 * (used + (n - used) / 128);
}
size_t miaie_experts_order_bytes(int T, int k, int E) { return 4 * (2 * E + T * k + miaie_experts_rows(T, k, E)); }
using u8 = uint8_t;
int miaie_quant_fp8(miaie_ctx*, const void* X, int dt, int R, int C, int ldx, int block, u8* Q, float* S, u8* Qt, float* St) {
  return called("quant", {X, Q, S, Qt, St}, dt, R, C, ldx, block);
}
int miaie_dequant_fp8(miaie_ctx*, const u8* Q, const float* S, int block, void* Y, int dt, int R, int C, int ldy) {
  return called("dequant", {Q, S, Y}, block, dt, R, C, ldy);
}
int miaie_gemm_fp8(miaie_ctx*, const u8* Aq, const float* As, const u8* Bq, const float* Bs, int block, void* C, int dt, int M,
                   int N, int K, int ldc) {
  return called("gemm", {Aq, As, Bq, Bs, C}, block, dt, M, N, K, ldc);
}
int miaie_route_experts(miaie_ctx*, const void* l, int dt, const float* bias, int* idx, float* w, int T, int k, int E, int ld,
                        int scoring, int groups, int kept, int top, int renorm, float scale) {
  return called("route", {l, bias, idx, w}, dt, T, k, E, ld, scoring, groups, kept, top, renorm, (int)(8 * scale));
}
int miaie_route_experts_grad(miaie_ctx*, const void* l, int dt, const int* idx, const float* dw, float* dl, int T, int k, int E,
                             int ld, int ldd, int scoring, int renorm, float scale) {
  return called("route_grad", {l, idx, dw, dl}, dt, T, k, E, ld, ldd, scoring, renorm, (int)(8 * scale));
}
int miaie_experts_order(miaie_ctx*, const int* idx, int* order, int T, int k, int E) { return called("order", {idx, order}, T, k, E); }
int miaie_experts_mlp_fp8(miaie_ctx*, const int* o, const float* w, const u8* Xq, const float* Xs, const u8* W1q, const float* W1s,
                          const u8* W2q, const float* W2s, u8* Hq, float* Hs, void* Y, void* out, int dt, int T, int k, int E, int D,
                          int F, int N, int ldo) {
  return called("mlp", {o, w, Xq, Xs, W1q, W1s, W2q, W2s, Hq, Hs, Y, out}, dt, T, k, E, D, F, N, ldo);
}
int miaie_experts_gemm_fp8(miaie_ctx*, const int* o, const u8* Aq, const float* As, const u8* Bq, const float* Bs, void* C, int dt,
                           int T, int k, int E, int N, int K, int ldc, int gather) {
  return called("slots", {o, Aq, As, Bq, Bs, C}, dt, T, k, E, N, K, ldc, gather);
}
int miaie_experts_quant_fp8(miaie_ctx*, const int* o, const void* X, int dt, const float* w, u8* Q, float* S, u8* Qt, float* St,
                            int T, int k, int E, int C, int ldx) {
  return called("quant_slots", {o, X, w, Q, S, Qt, St}, dt, T, k, E, C, ldx);
}
int miaie_experts_swiglu_fp8(miaie_ctx*, const int* o, const void* GU, int dt, u8* Q, float* S, u8* Qt, float* St, int T, int k,
                             int E, int F, int ld) {
  return called("swiglu", {o, GU, Q, S, Qt, St}, dt, T, k, E, F, ld);
}
int miaie_experts_swiglu_grad_fp8(miaie_ctx*, const int* o, const void* GU, int dt, const float* dH, u8* Q, float* S, u8* Qt,
                                  float* St, int T, int k, int E, int F, int ld, int ldh) {
  return called("swiglu_grad", {o, GU, dH, Q, S, Qt, St}, dt, T, k, E, F, ld, ldh);
}
int miaie_experts_wgrad_fp8(miaie_ctx*, const int* o, const u8* Aq, const float* As, const u8* Bq, const float* Bs, void* C, int dt,
                            int T, int k, int E, int M, int N, int ldc) {
  return called("wgrad", {o, Aq, As, Bq, Bs, C}, dt, T, k, E, M, N, ldc);
}
int miaie_experts_combine(miaie_ctx*, const int* o, const void* Y, const float* w, void* out, int dt, int T, int k, int E, int C,
                          int ldy, int ldo) {
  return called("combine", {o, Y, w, out}, dt, T, k, E, C, ldy, ldo);
}
int miaie_experts_combine_grad(miaie_ctx*, const int* o, const void* Y, const void* dout, float* dw, int dt, int T, int k, int E,
                               int C, int ldy, int ldo) {
  return called("combine_grad", {o, Y, dout, dw}, dt, T, k, E, C, ldy, ldo);
}
}

static int failures = 0;

static void report(bool ok, int line, const char* what) {
  if (ok) return;
  ++failures;
  std::printf("line %d: %s; last call: %s\n", line, what, last.c_str());
}

template <class F>
static void refused(int line, const char* text, F&& f) {
  const int before = calls;
  try {
    f();
    report(false, line, "not refused");
  } catch (const miaie::Error& e) {
    report(e.code() == MIAIE_EINVAL && std::string(e.what()).find(text) != std::string::npos, line, e.what());
  }
  report(calls == before, line, "an entry point was called");
}

template <class F>
static void reaches(int line, const char* want, std::vector<const void*> arrays, F&& f) {
  try {
    f();
    report(last == want, line, want);
    report(pointers == arrays, line, "the arrays are not where they belong");
  } catch (const miaie::Error& e) {
    report(false, line, e.what());
  }
}

#define REFUSED(text, call) refused(__LINE__, text, [&] { call; })
#define REACHES(want, arrays, call) reaches(__LINE__, want, arrays, [&] { call; })
#define P(...) (std::vector<const void*>{__VA_ARGS__})
#define M(m) m.q.data(), m.s.data()

int main() {
  using namespace miaie;
  Context ctx;
  Fp8Matrix A(ctx, 5, 300), B(ctx, 7, 300, 128), Bt(ctx, 300, 7, 128), longer(ctx, 7, 301), A2(ctx, 5, 300, 1, 2), At(ctx, 300, 5);
  Buffer<float> x(ctx, 1500), x1(ctx, 1499), c(ctx, 35), c1(ctx, 34);
  Buffer<uint16_t> h(ctx, 2100), h1(ctx, 2099);

  REACHES("quant 0 5 300 300 1", P(x.data(), M(A), nullptr, nullptr), quant_fp8(x, A));
  REACHES("quant 1 7 300 300 128", P(h.data(), M(B), nullptr, nullptr), quant_fp8(h, B));
  REFUSED("X is smaller", quant_fp8(x1, A));
  REFUSED("several", quant_fp8(x, A2));
  REACHES("quant 0 300 5 5 1", P(x.data(), nullptr, nullptr, M(A)), quant_fp8_t(x, A));
  REFUSED("X is smaller", quant_fp8_t(x1, A));
  REACHES("quant 1 7 300 300 128", P(h.data(), M(B), M(Bt)), quant_fp8_both(h, B, Bt));
  REFUSED("transpose", quant_fp8_both(h, B, At));
  REFUSED("X is smaller", quant_fp8_both(h1, B, Bt));
  Fp8Matrix B3(ctx, 7, 300, 128, 3), B3t(ctx, 300, 7, 128, 3);
  REACHES("quant 1 7 300 300 128", P(h.data(), B3.q.data() + 2 * 7 * 384, B3.s.data() + 2 * 3, nullptr, nullptr), quant_fp8_at(h, B3, 2));
  REACHES("quant 1 7 300 300 128", P(h.data(), B3.q.data() + 7 * 384, B3.s.data() + 3, B3t.q.data() + 300 * 128, B3t.s.data() + 3),
          quant_fp8_at(h, B3, 1, &B3t));
  REFUSED("no such", quant_fp8_at(h, B3, 3));
  REFUSED("no such", quant_fp8_at(h, B3, -1));
  REFUSED("X is smaller", quant_fp8_at(h1, B3, 0));
  REFUSED("transposes", quant_fp8_at(h, B3, 0, &Bt));
  REACHES("dequant 1 1 5 300 300", P(M(A), h.data()), dequant_fp8(A, h));
  REFUSED("Y is smaller", dequant_fp8(A, x1));
  REACHES("gemm 128 0 5 7 300 7", P(M(A), M(B), c.data()), gemm_fp8(A, B, c));
  REACHES("gemm 1 0 5 5 300 5", P(M(A), M(A), c.data()), gemm_fp8(A, A, c));
  REFUSED("blocks of 128", gemm_fp8(B, A, c));
  REFUSED("several", gemm_fp8(A, A2, c));
  REFUSED("different lengths", gemm_fp8(A, longer, c));
  REFUSED("C is smaller", gemm_fp8(A, B, c1));

  const Routing r{10, 2, 8, MIAIE_SIGMOID, 4, 2, 2, false, 2.5f};
  Buffer<float> l(ctx, 80), l1(ctx, 79), bias(ctx, 8), bias1(ctx, 7), w(ctx, 20), w1(ctx, 19), dl(ctx, 80);
  Buffer<int32_t> idx(ctx, 20), idx1(ctx, 19);
  REACHES("route 0 10 2 8 8 1 4 2 2 0 20", P(l.data(), bias.data(), idx.data(), w.data()), route_experts(l, &bias, idx, w, r));
  REACHES("route 1 10 2 8 8 0 1 1 1 1 8", P(h.data(), nullptr, idx.data(), w.data()),
          route_experts(h, nullptr, idx, w, Routing{10, 2, 8}));
  REFUSED("logits", route_experts(l1, &bias, idx, w, r));
  REFUSED("bias", route_experts(l, &bias1, idx, w, r));
  REFUSED("idx or w", route_experts(l, &bias, idx1, w, r));
  REFUSED("idx or w", route_experts(l, &bias, idx, w1, r));
  REACHES("route_grad 0 10 2 8 8 8 1 0 20", P(l.data(), idx.data(), w.data(), dl.data()), route_experts_grad(l, idx, w, dl, r));
  REFUSED("dlogits", route_experts_grad(l, idx, w, l1, r));
  REFUSED("idx or dw", route_experts_grad(l, idx, w1, dl, r));

  ExpertsOrder o(ctx, 10, 2, 8);
  const int R = o.rows();  // 8 * 128
  REACHES("order 10 2 8", P(idx.data(), o.order.data()), experts_order(idx, o));
  REFUSED("idx", experts_order(idx1, o));

  const int D = 40, F = 128, N = 30;
  Fp8Matrix X(ctx, 10, D), W1(ctx, 2 * F, D, 128, 8), W2(ctx, N, F, 128, 8), H(ctx, R, F), Xr(ctx, R, D);
  Fp8Matrix W1of7(ctx, 2 * F, D, 128, 7), W1half(ctx, F, D, 128, 8), W2rows(ctx, N, F, 1, 8), Ht(ctx, F, R), Xt(ctx, D, R);
  Buffer<uint16_t> Y(ctx, R * N), Y1(ctx, R * N - 1), out(ctx, 10 * N), out1(ctx, 10 * N - 1), GU(ctx, R * 2 * F), GU1(ctx, R * 2 * F - 1);
  auto mlp = P(o.order.data(), w.data(), M(X), M(W1), M(W2), M(H), Y.data(), out.data());
  REACHES("mlp 1 10 2 8 40 128 30 30", mlp, experts_mlp_fp8(o, w, X, W1, W2, H, Y, out));
  REFUSED("tokens' rows", experts_mlp_fp8(o, w, Xr, W1, W2, H, Y, out));
  REFUSED("each expert", experts_mlp_fp8(o, w, X, W1of7, W2, H, Y, out));
  REFUSED("each expert", experts_mlp_fp8(o, w, X, W1half, W2, H, Y, out));
  REFUSED("each expert", experts_mlp_fp8(o, w, X, W1, W2rows, H, Y, out));
  REFUSED("H does", experts_mlp_fp8(o, w, X, W1, W2, Ht, Y, out));
  REFUSED("too small", experts_mlp_fp8(o, w1, X, W1, W2, H, Y, out));
  REFUSED("too small", experts_mlp_fp8(o, w, X, W1, W2, H, Y1, out));
  REFUSED("too small", experts_mlp_fp8(o, w, X, W1, W2, H, Y, out1));

  REACHES("slots 1 10 2 8 256 40 256 1", P(o.order.data(), M(X), M(W1), GU.data()), experts_gemm_fp8(o, X, W1, GU, true));
  REACHES("slots 1 10 2 8 30 128 30 0", P(o.order.data(), M(H), M(W2), Y.data()), experts_gemm_fp8(o, H, W2, Y));
  REFUSED("tokens' rows", experts_gemm_fp8(o, H, W2, Y, true));
  REFUSED("slots' rows", experts_gemm_fp8(o, X, W1, GU));
  REFUSED("each expert", experts_gemm_fp8(o, H, W1, GU));
  REFUSED("C is smaller", experts_gemm_fp8(o, H, W2, Y1));

  Buffer<float> xt(ctx, 10 * D), xt1(ctx, 10 * D - 1), dH(ctx, R * F), dH1(ctx, R * F - 1);
  REACHES("quant_slots 0 10 2 8 40 40", P(o.order.data(), xt.data(), w.data(), M(Xr), M(Xt)),
          experts_quant_fp8(o, xt, &w, &Xr, &Xt, D));
  REACHES("quant_slots 0 10 2 8 40 40", P(o.order.data(), xt.data(), nullptr, nullptr, nullptr, M(Xt)),
          experts_quant_fp8(o, xt, nullptr, nullptr, &Xt, D));
  REFUSED("X or w", experts_quant_fp8(o, xt1, &w, &Xr, &Xt, D));
  REFUSED("X or w", experts_quant_fp8(o, xt, &w1, &Xr, &Xt, D));
  REFUSED("shape", experts_quant_fp8(o, xt, &w, &X, &Xt, D));
  REFUSED("shape", experts_quant_fp8(o, xt, &w, &Xr, &Xr, D));
  REACHES("swiglu 1 10 2 8 128 256", P(o.order.data(), GU.data(), M(H), M(Ht)), experts_swiglu_fp8(o, GU, &H, &Ht, F));
  REFUSED("GU", experts_swiglu_fp8(o, GU1, &H, &Ht, F));
  REFUSED("shape", experts_swiglu_fp8(o, GU, &Ht, &Ht, F));
  Fp8Matrix G(ctx, R, 2 * F), Gt(ctx, 2 * F, R);
  REACHES("swiglu_grad 1 10 2 8 128 256 128", P(o.order.data(), GU.data(), dH.data(), M(G), M(Gt)),
          experts_swiglu_grad_fp8(o, GU, dH, &G, &Gt, F));
  REFUSED("GU or dH", experts_swiglu_grad_fp8(o, GU, dH1, &G, &Gt, F));
  REFUSED("shape", experts_swiglu_grad_fp8(o, GU, dH, &H, &Gt, F));

  Buffer<float> dW(ctx, 8 * 2 * F * D), dW1(ctx, 8 * 2 * F * D - 1);
  REACHES("wgrad 0 10 2 8 256 40 40", P(o.order.data(), M(Gt), M(Xt), dW.data()), experts_wgrad_fp8(o, Gt, Xt, dW));
  REFUSED("along the slots", experts_wgrad_fp8(o, G, Xt, dW));
  REFUSED("C is smaller", experts_wgrad_fp8(o, Gt, Xt, dW1));
  REACHES("combine 1 10 2 8 30 30 30", P(o.order.data(), Y.data(), w.data(), out.data()), experts_combine(o, Y, &w, out, N));
  REACHES("combine 1 10 2 8 30 30 30", P(o.order.data(), Y.data(), nullptr, out.data()), experts_combine(o, Y, nullptr, out, N));
  REFUSED("too small", experts_combine(o, Y1, &w, out, N));
  REFUSED("too small", experts_combine(o, Y, &w1, out, N));
  REFUSED("too small", experts_combine(o, Y, &w, out1, N));
  REACHES("combine_grad 1 10 2 8 30 30 30", P(o.order.data(), Y.data(), out.data(), w.data()),
          experts_combine_grad(o, Y, out, w, N));
  REFUSED("too small", experts_combine_grad(o, Y, out1, w, N));
  REFUSED("too small", experts_combine_grad(o, Y, out, w1, N));
  if (!failures) std::printf("ok\n");
  return failures ? 1 : 0;
}
